"""Layer norm with its gradient, block-scaled quantisation and the block-scaled weight product, in plain form and through the package.

The path these operators lie on is a linear layer behind a norm, with its
activations and weights in few bits: the norm saves what its backward pass
needs (its input in 8 bits), activations and weights become 8- or 4-bit
codes with one power-of-two scale per 32 elements, and a serving program
multiplies a few tokens by such weights.

operators ("op")
  ln      layer norm: y, mean and 1/std, and with "ckpt" the input as
          block-scaled 8-bit codes (the activation checkpoint)
  ln_grad its gradient: dx, dgamma, dbeta, from the input or from its checkpoint
  quant   block-scaled 8-bit codes and scales of a matrix, blocks along a row
          (axis 1) or down a column (axis 0); with "back" also read back to
          bf16, which is how 4-bit codes show the values they stand for
  linear  bf16 rows times a block-scaled weight [N, K], bias, bf16 out
"rt" takes the row count at launch (one compiled group for all).
"""
import functools
import math
import os
import sys

import torch

own = False

E2M1, E4M3, E5M2 = "e2m1", "e4m3", "e5m2"
# exponent of the largest binade, bits of the mantissa, smallest exponent, largest value
_FORMATS = {E2M1: (2, 1, 0, 6.0), E4M3: (8, 3, -6, 448.0), E5M2: (15, 2, -14, 57344.0)}
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_CODES = {E4M3: torch.float8_e4m3fn, E5M2: torch.float8_e5m2}
_EPS = 1e-5
_BLOCK = 32
# a row count that no other size of a drawn case has: the compiled group's
# rows are left open in its place
_ANY_ROWS = 104729


def listed():
    return [
        # the norm of a training step's tokens; its input is kept in 8 bits
        dict(name="ln_train", op="ln", rows=8192, cols=4096, type="bf16", params="bf16", ckpt=E4M3, rt=False),
        # the norm of one decoding step's tokens: launch and row latency
        dict(name="ln_decode", op="ln", rows=16, cols=4096, type="bf16", params="bf16", ckpt="", rt=True),
        # f32 rows of an odd length, f32 weight and bias
        dict(name="ln_odd", op="ln", rows=777, cols=5003, type="f32", params="f32", ckpt="", rt=False),
        # backward of the training step, the input read from its checkpoint
        dict(name="ln_grad_train", op="ln_grad", rows=8192, cols=4096, type="bf16", params="bf16", ckpt=E4M3, rt=False),
        # backward of a short ragged batch from the saved input, f32 weights
        dict(name="ln_grad_ragged", op="ln_grad", rows=777, cols=2001, type="bf16", params="f32", ckpt="", rt=True),
        # backward of a few short rows
        dict(name="ln_grad_small", op="ln_grad", rows=64, cols=1024, type="f32", params="f32", ckpt="", rt=False),
        # activations of a prompt batch for a block-scaled fp8 product
        dict(name="quant_fp8_rows", op="quant", rows=8192, cols=4096, type="bf16", fmt=E4M3, axis=1, back=False, rt=False),
        # a linear layer's weight to 4 bits as the product's right operand, and read back
        dict(name="quant_fp4_weight", op="quant", rows=4096, cols=4096, type="bf16", fmt=E2M1, axis=0, back=True, rt=False),
        # a few tokens' activations
        dict(name="quant_decode", op="quant", rows=16, cols=4096, type="bf16", fmt=E4M3, axis=1, back=False, rt=True),
        # a linear layer with 4-bit weights for one token
        dict(name="linear_token", op="linear", m=1, n=4096, k=4096, fmt=E2M1, rt=True),
        # the same layer for a decoding batch, 8-bit weights, an odd number of outputs
        dict(name="linear_batch", op="linear", m=48, n=5003, k=4096, fmt=E4M3, rt=False),
        # the same layer on a full prompt
        dict(name="linear_prompt", op="linear", m=4096, n=4096, k=4096, fmt=E2M1, rt=True),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ln", "ln", "ln_grad", "ln_grad", "quant", "quant", "linear", "linear"])
    rt = rng.random() < 0.5
    if op == "linear":
        m = _spread(rng, 1, 4096)
        return dict(op=op, m=m, n=_spread(rng, 256, 4096), k=32 * _spread(rng, 8, 128), fmt=rng.choice([E2M1, E2M1, E4M3, E5M2]), rt=rt)
    rows = _spread(rng, 1, 8192)
    type_ = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "quant":
        fmt, axis = rng.choice([E2M1, E4M3, E5M2]), rng.choice([1, 1, 0])
        cols = _spread(rng, 64, 4096)
        if fmt == E2M1:  # two codes a byte along the blocks' axis
            rows, cols = (rows + rows % 2, cols) if axis == 0 else (rows, cols + cols % 2)
        return dict(op=op, rows=rows, cols=cols, type=type_, fmt=fmt, axis=axis, back=fmt == E2M1, rt=rt and axis == 1)
    cols = _spread(rng, 64, 16384)
    # at most the largest listed case's elements, whatever the type's width
    rows = max(1, min(rows, (8192 * 4096 // 2 if type_ == "f32" else 8192 * 4096) // cols))
    return dict(op=op, rows=rows, cols=cols, type=type_, params=rng.choice([type_, "f32"]),
                ckpt=rng.choice(["", E4M3, E5M2]), rt=rt)


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed * 1000003 + 29)

    def normal(shape, std=1.0):
        return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32) * std

    def uniform(shape, lo, hi):
        return torch.rand(shape, generator=gen, device=dev, dtype=torch.float32) * (hi - lo) + lo

    def out(shape, dtype):
        return torch.empty(shape, dtype=dtype, device=dev)

    op, s = case["op"], dict(case=case)
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        w, sw = _quantise(normal((n, k), 1.0 / math.sqrt(k)), case["fmt"])
        s.update(a=normal((m, k)).bfloat16(), w=_pack(w) if case["fmt"] == E2M1 else w.to(_CODES[case["fmt"]]), sw=sw,
                 bias=normal((n,), 0.1), out=out((m, n), torch.bfloat16))
        return s
    r, c, t = case["rows"], case["cols"], _TYPES[case["type"]]
    # activations: a spread of row sizes, an offset per row, some columns far larger than the others
    x = normal((r, c)) * uniform((r, 1), 0.25, 4.0) + normal((r, 1), 0.5)
    x[:, :: max(1, c // 7)] *= 8.0
    s["x"] = x = x.to(t)
    if op == "quant":
        blocks = (c + _BLOCK - 1) // _BLOCK if case["axis"] == 1 else (r + _BLOCK - 1) // _BLOCK
        s["scales"] = out((r if case["axis"] == 1 else c, blocks), torch.int8)
        if case["fmt"] == E2M1:
            s["codes"] = out((r, c // 2) if case["axis"] == 1 else (r // 2, c), torch.int8)
        else:
            s["codes"] = out((r, c), _CODES[case["fmt"]])
        if case["back"]:
            s["back"] = out((r, c), torch.bfloat16)
        return s
    p = _TYPES[case["params"]]
    s["gamma"] = uniform((c,), 0.5, 1.5).to(p)
    if op == "ln":
        s.update(beta=normal((c,), 0.1).to(p), y=out((r, c), t), mean=out((r,), torch.float32), rstd=out((r,), torch.float32))
        if case["ckpt"]:
            s.update(codes=out((r, c), _CODES[case["ckpt"]]), scales=out((r, (c + _BLOCK - 1) // _BLOCK), torch.int8))
        return s
    f = x.float()
    mean = f.mean(dim=1)
    s.update(dy=normal((r, c), 0.1).to(t), mean=mean, rstd=((f - mean[:, None]).square().mean(dim=1) + _EPS).rsqrt(),
             dx=out((r, c), t), dgamma=out((c,), p), dbeta=out((c,), p))
    if case["ckpt"]:
        v, s["scales"] = _quantise(f, case["ckpt"])
        s["codes"] = v.to(_CODES[case["ckpt"]])
        del s["x"]
    return s


# ---------------------------------------------------------------- plain forms
def _pow2(e):
    """2^e in f32 for whole e in [-127, 127], made from its bits: a power
    function may be an ulp off."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _quantise(x, fmt, axis=1):
    """Values of the codes and the scale bytes of f32 x, blocks along `axis`."""
    emax, mant, emin, top = _FORMATS[fmt]
    t = x if axis == 1 else x.t()
    r, c = t.shape
    blocks = (c + _BLOCK - 1) // _BLOCK
    t = torch.nn.functional.pad(t, (0, blocks * _BLOCK - c)).reshape(r, blocks, _BLOCK)
    amax = t.abs().amax(dim=2)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 1 - emax, -127).clamp(-127, 127)
    v = t * _pow2(-e)[:, :, None]
    step = _pow2(torch.frexp(v).exponent.sub(1).clamp(min=emin) - mant)
    v = (torch.round(v / step) * step).clamp(-top, top).reshape(r, blocks * _BLOCK)[:, :c]
    return (v if axis == 1 else v.t()), (e + 127).to(torch.uint8).view(torch.int8)


def _scale_of(scales, n, axis=1):
    """The f32 scales of n elements along the blocks' axis."""
    f = _pow2(scales.view(torch.uint8).to(torch.int32) - 127)
    f = f.repeat_interleave(_BLOCK, dim=1)[:, :n]
    return f if axis == 1 else f.t()


def _pack(v):
    """e2m1 values [N, K] as bytes [N, K/2], the even k in the low half."""
    a = v.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).view(torch.int8)


def _unpack(w):
    """The e2m1 values [N, K] of bytes [N, K/2]."""
    b = w.view(torch.uint8).to(torch.int32)
    code = torch.stack([b & 15, b >> 4], dim=2).reshape(w.shape[0], -1)
    m, sign = (code & 7).float(), 1.0 - 2.0 * (code >> 3).float()
    return sign * torch.where(m < 4, m * 0.5, torch.where(m < 6, m - 2, m * 2 - 8))


def _bits(scales):
    """Scale bytes as the powers of two that they stand for."""
    return scales.view(torch.float8_e8m0fnu)


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "linear":
        w = _unpack(s["w"]) if case["fmt"] == E2M1 else s["w"].float()
        return (s["a"].float() @ (w * _scale_of(s["sw"], case["k"])).t() + s["bias"]).bfloat16()
    if op == "quant":
        v, scales = _quantise(s["x"].float(), case["fmt"], case["axis"])
        if not case["back"]:
            return v.to(_CODES[case["fmt"]]), _bits(scales)
        n = case["cols"] if case["axis"] == 1 else case["rows"]
        return (v * _scale_of(scales, n, case["axis"])).bfloat16(), _bits(scales)
    t = _TYPES[case["type"]]
    if op == "ln":
        x = s["x"].float()
        mean = x.mean(dim=1)
        d = x - mean[:, None]
        rstd = 1.0 / torch.sqrt(d.square().mean(dim=1) + _EPS)
        y = (d * rstd[:, None] * s["gamma"].float() + s["beta"].float()).to(t)
        if not case["ckpt"]:
            return y, mean, rstd
        v, scales = _quantise(x, case["ckpt"])
        return y, mean, rstd, v.to(_CODES[case["ckpt"]]), _bits(scales)
    x = s["codes"].float() * _scale_of(s["scales"], case["cols"]) if case["ckpt"] else s["x"].float()
    dy = s["dy"].float()
    xh = (x - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * s["gamma"].float()
    dx = s["rstd"][:, None] * (g - g.mean(dim=1, keepdim=True) - xh * (g * xh).mean(dim=1, keepdim=True))
    p = s["gamma"].dtype
    return dx.to(t), (dy * xh).sum(dim=0).to(p), dy.sum(dim=0).to(p)


# ---------------------------------------------------------------- the package's operators
@functools.lru_cache(maxsize=None)
def _group(name, rows, rt, **kw):
    """The compiled group of one operator and size, which a program keeps; with
    "rt" `rows` stands for any row count."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ascendnpu-ir_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import hfusion_mi355x as hf

    build = getattr(hf.groups, name)
    if rt:
        return hf.DynamicGroup(hf.groups.with_dynamic_rows(build(rows, **kw), rows), runtime=True)
    return hf.load(build(rows, **kw))


def _own(s):
    case = s["case"]
    op, rt = case["op"], case["rt"]
    rows = _ANY_ROWS if rt else case["m" if op == "linear" else "rows"]
    if op == "linear":
        g = _group("linear_mx", rows, rt, n=case["n"], k=case["k"], fmt=case["fmt"], bias=True)
        return g(s["a"], s["w"], s["sw"], s["bias"], s["out"])
    if op == "quant":
        kw = dict(cols=case["cols"], fmt=case["fmt"], axis=case["axis"])
        codes, scales = _group("quantize_mx", rows, rt, src=case["type"], **kw)(s["x"], s["codes"], s["scales"])
        if not case["back"]:
            return codes, _bits(scales)
        return _group("dequantize_mx", rows, rt, dst="bf16", **kw)(codes, scales, s["back"]), _bits(scales)
    kw = dict(cols=case["cols"], elem=case["type"], params=case["params"], ckpt=case["ckpt"] or None)
    if op == "ln":
        g = _group("layer_norm", rows, rt, eps=_EPS, **kw)
        if not case["ckpt"]:
            return g(s["x"], s["gamma"], s["beta"], s["y"], s["mean"], s["rstd"])
        y, mean, rstd, codes, scales = g(s["x"], s["gamma"], s["beta"], s["y"], s["mean"], s["rstd"], s["codes"], s["scales"])
        return y, mean, rstd, codes, _bits(scales)
    x = (s["codes"], s["scales"]) if case["ckpt"] else (s["x"],)
    return _group("layer_norm_grad", rows, rt, **kw)(s["dy"], *x, s["gamma"], s["mean"], s["rstd"],
                                                            s["dx"], s["dgamma"], s["dbeta"])


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    op = case["op"]
    width = {"bf16": 2, "f16": 2, "f32": 4}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * m * k + n * k * (0.5 if case["fmt"] == E2M1 else 1) + n * k / 32 + 4 * n + 2 * m * n, "flops": 2 * m * n * k}
    r, c = case["rows"], case["cols"]
    e = width[case["type"]]
    if op == "quant":
        code = 0.5 if case["fmt"] == E2M1 else 1
        # read back: the codes and scales are read, and bf16 is written
        return {"bytes": r * c * (e + code + 1 / 32 + ((code + 1 / 32 + 2) if case["back"] else 0)), "flops": 3 * r * c}
    kept = 1 + 1 / 32 if case["ckpt"] else 0
    p = width[case["params"]]
    if op == "ln":
        return {"bytes": r * c * (2 * e + kept) + 8 * r + 2 * c * p, "flops": 8 * r * c}
    return {"bytes": r * c * (2 * e + (kept or e)) + 8 * r + 3 * c * p, "flops": 14 * r * c}


# ---------------------------------------------------------------- 64 bits
def _power(e):
    """2^e in f64 for whole e in [-300, 300], from a table of exact ones."""
    return torch.tensor([2.0 ** i for i in range(-300, 301)], dtype=torch.float64, device=e.device)[e.long() + 300]


def _exact_codes(x, fmt):
    """Codes' values and scales of f64 x [R, C], blocks along the rows: the
    nearest point of the format's grid, ties to the even one."""
    emax, mant, emin, top = _FORMATS[fmt]
    r, c = x.shape
    codes, scales = torch.empty_like(x), torch.empty((r, (c + 31) // 32), dtype=torch.float64, device=x.device)
    for b in range(scales.shape[1]):
        part = x[:, 32 * b : 32 * b + 32]
        big = part.abs().amax(dim=1)
        lead = torch.floor(torch.log2(big))
        # the logarithm next to a power of two, put right by comparison
        lead = lead.clamp(-150, 150)
        lead = torch.where(_power(lead + 1) <= big, lead + 1, torch.where(_power(lead) > big, lead - 1, lead))
        scale = _power((lead - emax).clamp(-127, 127))
        v = part / scale[:, None]
        near = torch.round(torch.log2(v.abs().clamp(min=2.0 ** emin)))
        grid = _power(torch.where(_power(near) > v.abs().clamp(min=2.0 ** emin), near - 1, near) - mant)
        low = torch.floor(v / grid)
        rest = v / grid - low
        up = (rest > 0.5) | ((rest == 0.5) & (low % 2 != 0))
        codes[:, 32 * b : 32 * b + 32] = ((low + up) * grid).clamp(-top, top)
        scales[:, b] = scale
    return codes, scales


_E2M1_VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]

    def scaled(codes, scales):
        f = _power(scales.view(torch.uint8).long() - 127)
        at = torch.arange(codes.shape[1], device=codes.device) // 32
        return codes * f[:, at]

    if op == "linear":
        if case["fmt"] == E2M1:
            table = torch.tensor(_E2M1_VALUES, dtype=torch.float64, device=s["w"].device)
            b = s["w"].view(torch.uint8).long()
            w = torch.empty((case["n"], case["k"]), dtype=torch.float64, device=b.device)
            w[:, 0::2], w[:, 1::2] = table[b % 16], table[b // 16]
        else:
            w = s["w"].double()
        return s["a"].double() @ scaled(w, s["sw"]).t().contiguous() + s["bias"].double()
    if op == "quant":
        x = s["x"].double()
        codes, scales = _exact_codes(x if case["axis"] == 1 else x.t().contiguous(), case["fmt"])
        if case["back"]:
            codes = codes * scales.repeat_interleave(32, dim=1)[:, : codes.shape[1]]
        return (codes if case["axis"] == 1 else codes.t()), scales
    gamma = s["gamma"].double()
    if op == "ln":
        x = s["x"].double()
        mean, var = x.mean(dim=1), x.var(dim=1, unbiased=False)
        rstd = (var + _EPS) ** -0.5
        y = torch.addcmul(s["beta"].double(), (x - mean[:, None]) * rstd[:, None], gamma)
        return (y, mean, rstd, *(_exact_codes(x, case["ckpt"]) if case["ckpt"] else ()))
    x = scaled(s["codes"].double(), s["scales"]) if case["ckpt"] else s["x"].double()
    dy, mean, rstd = s["dy"].double(), s["mean"].double(), s["rstd"].double()
    n = x.shape[1]
    xh = (x - mean[:, None]) * rstd[:, None]
    a, b = (dy @ gamma) / n, torch.mv(dy * xh, gamma) / n
    dx = (dy * gamma - a[:, None] - xh * b[:, None]) * rstd[:, None]
    return dx, dy.mul(xh).sum(dim=0), dy.sum(dim=0)
