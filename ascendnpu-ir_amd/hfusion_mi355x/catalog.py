"""The HFusion groups this package compiles ahead of time.

`__graft_entry__.build()` compiles each entry, so that `smoke()` and
`bench.py` on a GPU machine load prebuilt code objects: the headline
workloads of `groups.CONFIGS` at their full sizes, the bf16 and [K, N]-layout
contractions, the block-scaled fp8 contraction, the transpose+cast group, the layer norm,
block-scaled codes and weight product of a 4096-wide layer, the same layer's
norm, cache and attention in serving, and the reduced
RMSNorm+quant group the smoke check runs.  The parity cases the tests compile (ragged sizes,
every op family of the generic lowering, dynamic dims) live beside the tests.
"""
from . import groups as g


def entries():
    """name -> IR text of every prebuilt product group."""
    e = {}
    for name, c in g.CONFIGS.items():
        e[name] = c["fn"](**c["kw"])
    e["bf16_mmad"] = g.bf16_mmad(4096, 4096, 4096)
    e["rmsnorm_quant_256"] = g.rmsnorm_quant(256, 4096)
    e["transpose_cast"] = g.transpose_cast(4096, 8192)
    # the W8A8 contraction with B in the [K, N] layout of linalg.matmul
    e["w8a8_dequant_kn"] = g.w8a8_dequant(4096, 4096, 4096, b_layout="kn").replace("@w8a8_dequant(", "@w8a8_dequant_kn(")
    # block-scaled fp8 (hfusion.matmul_mx), e4m3 x e4m3 with e8m0 scales
    e["mx_fp8"] = g.matmul_mx(4096, 4096, 4096, name="mx_fp8")
    # block-scaled fp4 (e2m1, two values per byte), 4096^3 logical
    e["mx_fp4"] = g.matmul_mx(4096, 4096, 4096, fa="e2m1", fb="e2m1", via="bitcast", name="mx_fp4")
    # layer norm of a training batch with its input kept in 8 bits, and the
    # gradient that reads it; of a decoding step (any row count)
    e["layer_norm"] = g.layer_norm(8192, 4096, ckpt="e4m3")
    e["layer_norm_grad"] = g.layer_norm_grad(8192, 4096, ckpt="e4m3")
    e["layer_norm_rt"] = _any_rows(g.layer_norm, cols=4096)
    # block-scaled codes of a batch and of a decoding step, of a weight, and back
    e["quantize_mx"] = g.quantize_mx(8192, 4096)
    e["quantize_mx_rt"] = _any_rows(g.quantize_mx, cols=4096)
    e["quantize_mx_weight"] = g.quantize_mx(4096, 4096, fmt="e2m1", axis=0)
    e["dequantize_mx_weight"] = g.dequantize_mx(4096, 4096, fmt="e2m1", axis=0)
    # the linear layer with a 4-bit weight, any row count
    e["linear_mx_rt"] = _any_rows(g.linear_mx, n=4096, k=4096, bias=True)
    # the attention half of a decoder layer in serving: the residual's norm into
    # int8 codes, rotation and append to an 8-bit cache of 64 sequences, and the
    # attention over it, any row count
    cache = dict(heads=32, kv_heads=8, dim=128, slots=64, room=8192, blocks=4096, block=64)
    e["rms_norm"] = g.rms_norm(8192, 4096)
    e["rms_norm_rt"] = _any_rows(g.rms_norm, cols=4096)
    e["append_kv_rt"] = _any_rows(g.append_kv, **cache)
    e["paged_attention_rt"] = _any_rows(g.paged_attention, **cache)
    return e


def _any_rows(build, **kw):
    """The group at a launch-time row count (104729 is no other dim of it)."""
    return g.with_dynamic_rows(build(104729, **kw), 104729)


def options(name):
    """Compiler options of an entry: names in _rt take their row count at launch."""
    return "dyn=runtime" if name.endswith("_rt") else ""


def get(name):
    return entries()[name]
