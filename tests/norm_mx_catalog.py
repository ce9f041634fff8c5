"""The layer-norm and block-scaled groups the tests prebuild: every format,
element type, schedule and ragged end of each operator."""
from hfusion_mi355x import groups as g

_ANY = 7919

# rows, cols, element type, format, axis
QUANT = [
    (37, 128, "bf16", "e4m3", 1), (5, 1, "f32", "e5m2", 1), (33, 101, "f16", "e4m3", 1), (3, 4096, "bf16", "e2m1", 1),
    (7, 98, "f32", "e2m1", 1), (1, 32, "bf16", "e5m2", 1), (64, 36, "f16", "e2m1", 1), (9, 260, "f32", "e4m3", 1),
    (32, 256, "bf16", "e4m3", 0), (70, 33, "f32", "e5m2", 0), (300, 261, "f16", "e2m1", 0), (2, 1, "bf16", "e2m1", 0),
    (1, 7, "f32", "e4m3", 0), (258, 512, "bf16", "e2m1", 0), (513, 258, "f16", "e5m2", 0),
]
# rows, cols, element type, type of weight and bias, checkpoint, affine
NORM = [
    (3, 1, "f32", "f32", None, 2), (5, 7, "bf16", "f32", None, 2), (9, 64, "f16", "f16", "e4m3", 1), (6, 33, "f32", "f32", "e5m2", 2),
    (33, 512, "bf16", "bf16", None, 2), (130, 1000, "bf16", "bf16", "e4m3", 2), (40, 1024, "f16", "f32", "e5m2", 0),
    (7, 1032, "f32", "f32", None, 1), (700, 2001, "bf16", "f32", None, 2), (5, 4096, "bf16", "bf16", "e5m2", 2),
    (3, 5003, "f32", "f32", "e4m3", 2), (2, 8200, "bf16", "f32", "e4m3", 1), (2, 16384, "f16", "f32", "e4m3", 2),
    (600, 320, "f32", "f32", None, 2), (1, 16383, "f32", "f32", None, 2), (11, 96, "bf16", "bf16", None, 0),
]
# rows, outputs, k, format, bias, result
LINEAR = [
    (1, 16, 32, "e2m1", False, "bf16"), (1, 1, 64, "e4m3", True, "f32"), (3, 33, 96, "e5m2", False, "f32"), (16, 40, 288, "e4m3", True, "bf16"),
    (17, 100, 1024, "e2m1", True, "bf16"), (33, 257, 2080, "e2m1", False, "bf16"), (64, 50, 4096, "e5m2", False, "bf16"), (48, 129, 512, "e4m3", True, "f32"),
    (65, 100, 544, "e2m1", True, "bf16"), (300, 520, 256, "e4m3", False, "bf16"), (129, 31, 160, "e5m2", True, "f32"),
]
# rows enough for the weight as bf16 in the workspace
LINEAR_MANY = [(2300, 520, 1024, "e4m3", True, "bf16"), (4500, 40, 288, "e2m1", False, "f32"), (4200, 129, 96, "e5m2", True, "bf16")]
# k to the end of what a workgroup's scales leave of LDS, and past it
LINEAR_LONG = [(3, 20, 131072, "e2m1", False, "f32"), (9, 33, 98304, "e4m3", False, "f32"), (2, 16, 262144, "e5m2", False, "f32")]
# more rows than the workgroups take at once
NORM_LONG = [(2081, 2001, "bf16", "f32", None, 2), (9000, 33, "f16", "f16", "e4m3", 2), (777, 5003, "f32", "f32", None, 1),
             (4200, 160, "f32", "f32", "e5m2", 2)]
# rows too wide for two row groups a workgroup, and more of them than one launch
# of the gradient takes: every thread stores its partial sums itself; f32 rows
# past 8192 are not loaded ahead
NORM_WIDE = [(1000, 5003, "f32", "f32", None, 2), (1100, 8200, "bf16", "f32", "e4m3", 2), (900, 16383, "f32", "f32", None, 1),
             (1030, 4104, "f16", "f16", "e5m2", 1)]
# a training step of norm and linear layer: rows, columns of the norm, outputs
STEP = (96, 512, 192)
# the same at a launch-time row count, and the row counts they are called with
RT_ROWS = [1, 5, 16, 17, 40, 64, 65, 130, 515]


def quant_name(c, kind="quant"):
    r, n, el, fmt, ax = c
    return f"{kind}mx_{fmt}_{el}_{r}x{n}_a{ax}"


def norm_name(c, kind="ln"):
    r, n, el, p, ck, aff = c
    return f"{kind}_{el}_{p}_{ck or 'x'}_{r}x{n}_w{aff}"


def linear_name(c):
    m, n, k, fmt, bias, out = c
    return f"linmx_{fmt}_{m}x{n}x{k}_{'b' if bias else 'n'}_{out}"


def _norm_kw(c):
    r, n, el, p, ck, aff = c
    return dict(rows=r, cols=n, elem=el, params=p, ckpt=ck, affine=aff)


def norm_rank3():
    """[2, 3, 64]: the leading dims are the rows."""
    return g.layer_norm(6, 64, ckpt="e4m3").replace("<6x64x", "<2x3x64x").replace("<6xf32>", "<2x3xf32>").replace("<6x2xui8>", "<2x3x2xui8>")


def norm_grad_rank3():
    return g.layer_norm_grad(6, 64).replace("<6x64x", "<2x3x64x").replace("<6xf32>", "<2x3xf32>")


def entries():
    e = {}
    for c in QUANT:
        r, n, el, fmt, ax = c
        e[quant_name(c)] = g.quantize_mx(r, n, src=el, fmt=fmt, axis=ax)
        e[quant_name(c, "dequant")] = g.dequantize_mx(r, n, dst=el, fmt=fmt, axis=ax)
    for c in NORM + NORM_LONG:
        e[norm_name(c)] = g.layer_norm(**_norm_kw(c))
        e[norm_name(c, "lngrad")] = g.layer_norm_grad(**_norm_kw(c))
    for m, n, k, fmt, bias, out in LINEAR + LINEAR_MANY + LINEAR_LONG:
        e[linear_name((m, n, k, fmt, bias, out))] = g.linear_mx(m, n, k, fmt=fmt, bias=bias, out=out)
    e["linmx_filled"] = g.linear_mx(5, 48, 64, out="f32").replace("0.000000e+00", "1.500000e+00")
    e["ln_untied"], e["lngrad_untied"] = untied(g.layer_norm(9, 96, ckpt="e4m3")), untied(g.layer_norm_grad(64, 256))
    e["quantmx_untied"] = untied(g.quantize_mx(70, 64, fmt="e5m2"))
    e["linmx_residual"], e["linmx_residual_bf16"] = linear_epilogue(70, 48, 96), linear_epilogue(70, 48, 96, out="bf16")
    e["linmx_residual_many"] = linear_epilogue(2300, 520, 1024)
    e["ln_rank3"], e["lngrad_rank3"] = norm_rank3(), norm_grad_rank3()
    rt = lambda ir: g.with_dynamic_rows(ir, _ANY)  # noqa: E731
    e["quantmx_e4m3_rt"] = rt(g.quantize_mx(_ANY, 100))
    e["quantmx_e2m1_rt"] = rt(g.quantize_mx(_ANY, 4096, fmt="e2m1"))
    e["dequantmx_e2m1_rt"] = rt(g.dequantize_mx(_ANY, 4096, fmt="e2m1"))
    e["ln_rt"] = rt(g.layer_norm(_ANY, 1000, ckpt="e4m3"))
    e["lngrad_rt"] = rt(g.layer_norm_grad(_ANY, 1000, ckpt="e4m3", params="f32"))
    e["lngrad_wide_rt"] = rt(g.layer_norm_grad(_ANY, 4096))
    for c in NORM_WIDE:
        e[norm_name(c)] = g.layer_norm(**_norm_kw(c))
        e[norm_name(c, "lngrad")] = g.layer_norm_grad(**_norm_kw(c))
    m, k, n = STEP
    e["step_norm"], e["step_norm_grad"] = g.layer_norm(m, k, ckpt="e4m3"), g.layer_norm_grad(m, k, ckpt="e4m3")
    e["step_codes"], e["step_values"] = g.quantize_mx(n, k, fmt="e2m1"), g.dequantize_mx(n, k, fmt="e2m1")
    e["step_linear"], e["step_linear_grad"] = g.linear_mx(m, n, k, bias=True), g.bf16_mmad(m, k, n, b_layout="kn")
    e["lngrad_long_rt"] = rt(g.layer_norm_grad(_ANY, 5000, params="f32"))
    e["lngrad_plain_rt"] = rt(g.layer_norm_grad(_ANY, 96, affine=0))
    e["linmx_e2m1_rt"] = rt(g.linear_mx(_ANY, 130, 544, bias=True))
    e["linmx_e4m3_rt"] = rt(g.linear_mx(_ANY, 1040, 1024, fmt="e4m3"))
    # the norm, the quantisation of its result and the block-scaled product
    e["prog_norm_matmul_mx"] = g.layer_norm_matmul_mx(100, 208, 384)
    e["prog_norm_linear_mx"] = g.layer_norm_linear_mx(20, 208, 384)
    e["prog_norm_linear_mx_many"] = g.layer_norm_linear_mx(2300, 1040, 1024)
    return e


def untied(ir):
    """The group with buffers of its own for its results: their destinations
    are tensor.empty, not arguments."""
    head, body = ir.split(") -> (", 1) if ") -> (" in ir else ir.split(") -> ", 1)
    outs = body[body.index("outs(") + 5:]
    outs = outs[:outs.index(")")]
    names, types = (v.split(", ") for v in outs.split(" : "))
    for n, t in zip(names, types):
        assert f", {n}: {t}" in head
        head = head.replace(f", {n}: {t}", "")
    empties = "".join(f"    {n} = tensor.empty() : {t}\n" for n, t in zip(names, types))
    at = body.index("{\n") + 2
    return head + (") -> (" if ") -> (" in ir else ") -> ") + body[:at] + empties + body[at:]


def linear_epilogue(m, n, k, out="f32"):
    """linear_mx with a residual [m, n] and a factor per row: (a w + residual) * factor."""
    C, O = f"tensor<{m}x{n}xf32>", f"tensor<{m}x{n}x{out}>"
    ir = g.linear_mx(m, n, k, bias=True, out=out)
    ir = ir.replace(f"%bias: tensor<{n}xf32>", f"%res: {C}, %factor: tensor<{m}xf32>")
    ir = ir.replace(f"%bb = linalg.broadcast ins(%bias : tensor<{n}xf32>) outs(%e1 : {C}) dimensions = [0]",
                    f"%bb = linalg.broadcast ins(%factor : tensor<{m}xf32>) outs(%e1 : {C}) dimensions = [1]\n"
                    f"    %e5 = tensor.empty() : {C}\n"
                    f"    %cr = linalg.elemwise_binary {{fun = #linalg.binary_fn<add>}} ins(%c, %res : {C}, {C}) outs(%e5 : {C}) -> {C}")
    return ir.replace("binary_fn<add>}} ins(%c, %bb".replace("}}", "}"), "binary_fn<mul>} ins(%cr, %bb")
