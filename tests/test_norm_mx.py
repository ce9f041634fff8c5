"""Layer norm and its gradient, block-scaled codes and the block-scaled
weight product: refusals and the CPU restatement (no GPU), then every
prebuilt group of norm_mx_catalog against the formulas in 64 bits.

Codes, scales and values read back are exact.  The tolerances of the others
count, per value, half a step of the result's type (u) and for each f32 sum of
n terms (n additions + the products' rounding) * 2^-24 * sum |terms|."""
import ctypes

import numpy as np
import pytest

import hfusion_mi355x as hf
import group_catalog as cat
import norm_mx_catalog as nc
from helpers import run_gpu, to_dev, to_host
from hfusion_mi355x import groups as g
from oracle import blockscaled as bs
from oracle import interp

E24 = 2.0 ** -24
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
# smallest subnormal of the type: half of it is the rounding next to zero
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}


def note(msg):
    print(f"[case] {msg}", flush=True)


def stored(a, elem):
    """f64 values as storage of the element type (rounded), and exactly what that holds."""
    s = interp.from_f32(np.asarray(a, np.float32), elem)
    return s, interp.to_f32(interp.T(s, elem)).astype(np.float64)


def value(a, elem):
    return interp.to_f32(interp.T(np.asarray(a), elem)).astype(np.float64)


def activations(rng, rows, cols):
    x = rng.normal(size=(rows, cols)) * rng.uniform(0.25, 4, (rows, 1)) + rng.normal(0, 0.5, (rows, 1))
    x[:, :: max(1, cols // 7)] *= 8
    return x


def edge_values(rng, rows, cols, elem):
    """Activations with blocks of zeros, powers of two and ties of every
    format, subnormals, the largest values, infinities and NaN."""
    x = activations(rng, rows, cols)
    flat = x.reshape(-1)
    n = flat.size
    ties = rng.integers(-64, 65, n) / 4.0 * 2.0 ** rng.integers(-6, 7, n)
    flat[:] = np.where(rng.random(n) < 0.5, ties, flat)
    top = {"f32": 3.0e38, "bf16": 3.0e38, "f16": 65504.0}[elem]
    low = {"f32": 1e-44, "bf16": 1e-39, "f16": 6e-8}[elem]
    for k in range(0, n, 160):
        kind = (k // 160) % 7
        seg = flat[k:k + 40]
        if kind == 0:
            seg[:] = 0.0
        elif kind == 1:
            seg[:] = low * rng.integers(-3, 4, seg.size)
        elif kind == 2:
            seg[0] = top
        elif kind == 3:
            seg[-1] = np.inf
        elif kind == 4:
            seg[seg.size // 2] = np.nan
        elif kind == 5:
            seg[0] = -np.inf
        else:
            seg[:] = -2.0 ** rng.integers(-12, 12, seg.size)
    return x


# ---------------------------------------------------------------- no GPU
def refuse(ir, why, options=""):
    with pytest.raises(hf.CompileError, match=why):
        hf.compile(ir, options=options, cache=False)


def test_refused_block_scaled_codes():
    ir = g.quantize_mx(8, 64)
    refuse(ir.replace("format = 2", "format = 7"), "format other than")
    refuse(ir.replace("format = 2 : i32, ", ""), "missing format")
    refuse(ir.replace("axis = 1", "axis = 2"), "axis other")
    refuse(ir.replace("<8x2xui8>", "<8x3xui8>"), "scales shape")
    refuse(ir.replace("<8x2xui8>", "<8x2xi32>"), "e8m0")
    refuse(ir.replace("f8E4M3FN", "f8E5M2"), "codes of another type")
    refuse(ir.replace("xbf16", "xi32"), "values of type")
    refuse(ir.replace("<8x64xf8E4M3FN>", "<8x32xf8E4M3FN>"), "codes shape")
    refuse(ir.replace("outs(%q, %s", "outs(%q, %q"), "one destination")
    refuse(g.quantize_mx(8, 66, fmt="e2m1").replace("x66x", "x65x").replace("<8x33x", "<8x32x"), "odd number of 4-bit")
    refuse(g.quantize_mx(8, 64).replace("<8x64x", "<0x64x").replace("<8x2x", "<0x2x"), "empty tensor")
    refuse(g.with_dynamic_rows(g.quantize_mx(7919, 64, axis=0), 7919), "blocks down the columns", "dyn=runtime")
    refuse(g.dequantize_mx(8, 64).replace("xbf16", "xf64"), "values of type")
    for bad in (dict(fmt="e3m2"), dict(axis=2), dict(fmt="e2m1", cols=63)):
        with pytest.raises(ValueError):
            g.quantize_mx(**{**dict(rows=8, cols=64), **bad})


def test_refused_layer_norm():
    ir = g.layer_norm(8, 64, ckpt="e4m3")
    refuse(ir.replace("eps = 1.000000000e-05 : f32, ", ""), "missing eps")
    refuse(ir.replace("1.000000000e-05", "-1.0"), "eps that is negative")
    refuse(ir.replace("format = 2", "format = 3"), "4-bit checkpoint")
    refuse(ir.replace("tensor<64xbf16>", "tensor<32xbf16>"), "one element per column")
    refuse(ir.replace("tensor<64xbf16>", "tensor<64xf16>"), "another type than f32 or the rows'")
    refuse(ir.replace("tensor<8xf32>", "tensor<8xbf16>"), "must be f32")
    refuse(g.layer_norm(8, 16385), "more than 16384")
    refuse(g.layer_norm(8, 64).replace("outs(%y,", "outs(%x,"), "also a destination")
    refuse(g.layer_norm_grad(8, 16400), "more than 16384")
    refuse(g.layer_norm_grad(8, 64).replace("%dy: tensor<8x64xbf16>", "%dy: tensor<8x64xf16>"), "beside")
    refuse(g.layer_norm_grad(8, 64, params="f32").replace("%dbeta: tensor<64xf32>", "%dbeta: tensor<64xbf16>"), "destination")
    refuse(g.layer_norm_grad(8, 64).replace("%r#2", "%r#1").replace("#1, %r#1", "#1, %r#1"), "does not return|returns")
    with pytest.raises(ValueError):
        g.layer_norm(8, 64, affine=3)


def test_refused_linear():
    ir = g.linear_mx(4, 16, 64)
    refuse(ir.replace("rhsFormat = 3", "rhsFormat = 0"), "rhsFormat other")
    refuse(ir.replace("{rhsFormat = 3 : i32} ", ""), "without rhsFormat")
    refuse(ir.replace("<16x2xui8>", "<16x1xui8>"), "scales shape")
    refuse(ir.replace("<4x64xbf16>", "<4x64xf16>"), "another type than bf16")
    refuse(g.linear_mx(4, 16, 48).replace("<16x2xui8>", "<16x1xui8>"), "multiple of 32")
    refuse(ir.replace("<16x32xi8>", "<16x64xi8>"), "codes shape")
    refuse(ir.replace("rhsFormat = 3", "rhsFormat = 2"), "codes shape")
    refuse(ir.replace("%out: tensor<4x16xbf16>", "%out: tensor<2x16xbf16>"), "destination|shape inconsistent")


def test_oracle_codes():
    """The restatement: codes are the nearest values, ties to the even one;
    scales follow the largest magnitude; packing and unpacking are inverses."""
    for fmt in ("e2m1", "e4m3", "e5m2"):
        vals = bs.code_values(fmt)
        fin = vals[np.isfinite(vals)]
        pos = np.unique(np.abs(fin))
        assert pos[-1] == bs.TOP[fmt] and np.array_equal(bs.code_values(fmt)[bs.encode(pos, fmt)], pos)
        mid = (pos[:-1] + pos[1:]) / 2
        assert (bs.encode(mid, fmt) % 2 == 0).all()
        above = np.nextafter(mid, np.inf)
        assert np.array_equal(vals[bs.encode(above, fmt)], pos[1:]) and np.array_equal(vals[bs.encode(-above, fmt)], -pos[1:])
        assert (vals[bs.encode(np.array([1e9, -1e9]), fmt)] == [bs.TOP[fmt], -bs.TOP[fmt]]).all()
        x = np.zeros((1, 96))
        x[0, 40], x[0, 70] = 2.0 ** 5, 2.0 ** -140
        _, s = bs.quantize(x, fmt, 1)
        assert s.tolist() == [[0, 127 + 5 - bs.EMAX[fmt], 0]]
        x[0, 3], x[0, 41] = np.inf, np.nan
        codes, s = bs.quantize(x, fmt, 1)
        assert s.tolist() == [[255, 255, 0]] and not codes[0, :64].any()
    c = np.arange(48, dtype=np.uint8).reshape(6, 8) % 16
    for ax in (0, 1):
        assert np.array_equal(bs.unpack(bs.pack(c, ax), ax), c)


def test_oracle_norm_gradient():
    """dx, dgamma, dbeta of the formula against differences of the forward."""
    rng = np.random.default_rng(5)
    x, gm, bt, w = rng.normal(size=(4, 9)), rng.uniform(0.5, 1.5, 9), rng.normal(size=9), rng.normal(size=(4, 9))
    loss = lambda x, gm, bt: (bs.layer_norm(x, gm, bt, 1e-3)[0] * w).sum()  # noqa: E731
    _, mean, rstd = bs.layer_norm(x, gm, bt, 1e-3)
    dx, dg, db = bs.layer_norm_grad(w, x, gm, mean, rstd)
    h = 1e-6
    for arr, grad in ((x, dx), (gm, dg), (bt, db)):
        for i in np.ndindex(arr.shape):
            keep = arr[i]
            arr[i] = keep + h
            up = loss(x, gm, bt)
            arr[i] = keep - h
            down = loss(x, gm, bt)
            arr[i] = keep
            assert abs((up - down) / (2 * h) - grad[i]) < 1e-7 * (1 + abs(grad[i])) + 1e-7


def test_oracle_runs_the_programs():
    """The un-fused programs through the interpreter equal their parts by hand."""
    rng = np.random.default_rng(8)
    m, n, k = 100, 208, 384
    (xs, x), (gs, gm), (ts, bt) = (stored(a, "bf16") for a in (activations(rng, m, k), rng.uniform(0.5, 1.5, k), rng.normal(0, 0.1, k)))
    wc, ws = bs.quantize(rng.normal(size=(k, n)) / 16, "e4m3", 0)
    got = interp.run(cat.get("prog_norm_matmul_mx"), xs, gs, ts, wc, ws)[0]
    y = value(stored(bs.layer_norm(x, gm, bt, np.float32(1e-5))[0], "bf16")[0], "bf16")
    a, sa = bs.quantize(y, "e4m3", 1)
    want = bs.dequantize(a, sa, "e4m3", 1) @ bs.dequantize(wc, ws, "e4m3", 0)
    # serial f32 sums of k products
    bound = np.abs(bs.dequantize(a, sa, "e4m3", 1)) @ np.abs(bs.dequantize(wc, ws, "e4m3", 0)) * (k + 1) * E24
    assert (np.abs(got - want) <= bound + 1e-30).all()


def test_launch_time_rows_manifest():
    """One code object for every row count, and the row counts each kernel serves."""
    art = hf.compile(cat.get("linmx_e2m1_rt"), options="dyn=runtime")
    text = open(art.manifest).read()
    alts = [ln.split() for ln in text.splitlines() if ln.startswith("alt ")]
    few = [a for a in alts if len(a) == 6]
    assert few and all(a[6:] == ["pre"] for a in alts[len(few):]) and [int(a[2]) for a in alts] == sorted(int(a[2]) for a in alts)
    art = hf.compile(cat.get("lngrad_rt"), options="dyn=runtime")
    text = open(art.manifest).read()
    # (the alternatives are the launches of few rows, none behind the rows kernel)
    assert "rows_zero 1" in text and [ln.split()[2:] for ln in text.splitlines() if ln.startswith("alt ")][-1][0] == "1200"
    assert hf.compile(cat.get(nc.norm_name(nc.NORM[8], "lngrad"))).blocks[0]["workspace"] == 0
    assert "rows_zero" not in open(hf.compile(cat.get("ln_rt"), options="dyn=runtime").manifest).read()


# ---------------------------------------------------------------- block-scaled codes
def quant_args(c, x):
    r, n, el, fmt, ax = c
    codes = np.zeros((r, n // 2) if fmt == "e2m1" and ax else (r // 2, n) if fmt == "e2m1" else (r, n), np.uint8)
    return [x, codes if fmt != "e2m1" else codes.view(np.int8), np.zeros((r, (n + 31) // 32) if ax else (n, (r + 31) // 32), np.int8)]


@pytest.mark.gpu
@pytest.mark.parametrize("c", nc.QUANT, ids=nc.quant_name)
def test_quantize_exact(gpu, c):
    r, n, el, fmt, ax = c
    note(nc.quant_name(c))
    rng = np.random.default_rng(hash(c[:2]) % 1000)
    for x64 in (activations(rng, r, n), edge_values(rng, r, n, el)):
        xs, x = stored(x64, el)
        q, s = run_gpu(nc.quant_name(c), quant_args(c, xs), gpu)
        wq, ws = bs.quantize(x, fmt, ax)
        assert np.array_equal(s.view(np.uint8), ws)
        assert np.array_equal(q.view(np.uint8), bs.pack(wq, ax) if fmt == "e2m1" else wq)


@pytest.mark.gpu
@pytest.mark.parametrize("c", nc.QUANT, ids=nc.quant_name)
def test_dequantize_exact(gpu, c):
    r, n, el, fmt, ax = c
    note(nc.quant_name(c, "dequant"))
    rng = np.random.default_rng(17)
    # every code and every scale byte, the ends among them
    codes = rng.integers(0, 16 if fmt == "e2m1" else 256, (r, n)).astype(np.uint8)
    scales = rng.integers(0, 256, (r, (n + 31) // 32) if ax else (n, (r + 31) // 32)).astype(np.uint8)
    scales.flat[:: 5], scales.flat[1:: 7] = 0, 255
    q = bs.pack(codes, ax) if fmt == "e2m1" else codes
    out, = run_gpu(nc.quant_name(c, "dequant"), [q.view(np.int8) if fmt == "e2m1" else q, scales.view(np.int8),
                                                 np.zeros((r, n), interp.NP[el])], gpu)
    with np.errstate(over="ignore", invalid="ignore"):
        want = bs.dequantize(q, scales, fmt, ax).astype(np.float32)  # (exact, or past the largest f32)
        ws = interp.from_f32(want, el)
    got, want = value(out, el), value(ws, el)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    assert np.array_equal(got[ok], want[ok]) and np.array_equal(np.signbit(got[ok]), np.signbit(want[ok]))


@pytest.mark.gpu
def test_codes_at_launch_time_rows(gpu):
    import torch
    rng = np.random.default_rng(3)
    for name, cols, fmt in (("quantmx_e4m3_rt", 100, "e4m3"), ("quantmx_e2m1_rt", 4096, "e2m1")):
        grp = hf.compile(cat.get(name), options=cat.options(name), require_cached=True).load()
        for rows in (1, 3, 64, 257):
            note(f"{name} {rows}")
            xs, x = stored(activations(rng, rows, cols), "bf16")
            args = [to_dev(a, p["elem"], gpu) for a, p in zip(quant_args((rows, cols, "bf16", fmt, 1), xs), grp.meta["params"])]
            q, s = grp(*args)
            wq, ws = bs.quantize(x, fmt, 1)
            assert np.array_equal(s.cpu().numpy().view(np.uint8), ws)
            assert np.array_equal(q.view(torch.uint8).cpu().numpy(), bs.pack(wq, 1) if fmt == "e2m1" else wq)


# ---------------------------------------------------------------- layer norm
def norm_inputs(c, seed=1, shift=0.0):
    r, n, el, p, ck, aff = c
    rng = np.random.default_rng(seed + r + n)
    xs, x = stored(activations(rng, r, n) + shift, el)
    gs, gm = stored(rng.uniform(0.5, 1.5, n), p)
    ts, bt = stored(rng.normal(0, 0.1, n), p)
    ds, dy = stored(rng.normal(0, 0.1, (r, n)), el)
    return xs, x, gs, gm, ts, bt, ds, dy


def adds(n):
    """Additions on the way of one of n terms into a row's sum, at most: 16 to
    a thread's own sum (two chunks of eight), 6 over a wave, 16 waves."""
    return min(n, 40)


def check_norm(c, outs, x, gm, bt, eps=np.float32(1e-5)):
    r, n, el, p, ck, aff = c
    gm, bt = gm if aff >= 1 else np.ones(n), bt if aff >= 2 else np.zeros(n)
    y, mean, rstd = bs.layer_norm(x, gm, bt, float(eps))
    a = (adds(n) + 2) * E24
    dmu = a * np.abs(x).mean(axis=1)
    assert (np.abs(outs[1].astype(np.float64) - mean) <= dmu + 1e-45).all()
    # variance: its own sum, and the square of the mean's error; a square root,
    # a division and an addition behind it
    rel = 0.5 * a + (dmu * rstd) ** 2 + dmu * rstd * 4 * E24 + 3 * E24
    assert (np.abs(outs[2].astype(np.float64) - rstd) <= rel * rstd).all()
    xh = np.abs((x - mean[:, None]) * rstd[:, None])
    tol = (dmu * rstd)[:, None] * np.abs(gm) + xh * np.abs(gm) * (rel[:, None] + 3 * E24) + 2 * E24 * np.abs(bt)
    assert (np.abs(value(outs[0], el) - y) <= tol * 1.01 + U[el] * (np.abs(y) + tol) + TINY[el]).all()
    if ck:
        wq, ws = bs.quantize(x, ck, 1)
        assert np.array_equal(outs[4].view(np.uint8), ws) and np.array_equal(outs[3].view(np.uint8), wq)


def norm_args(c, xs, gs, ts):
    r, n, el, p, ck, aff = c
    args = [xs] + [gs, ts][:aff] + [np.zeros_like(xs), np.zeros(r, np.float32), np.zeros(r, np.float32)]
    return args + ([np.zeros((r, n), np.uint8), np.zeros((r, (n + 31) // 32), np.int8)] if ck else [])


@pytest.mark.gpu
@pytest.mark.parametrize("c", nc.NORM, ids=nc.norm_name)
def test_layer_norm(gpu, c):
    note(nc.norm_name(c))
    for shift in (0.0, 100.0):  # (rows far from zero: the variance does not come from a difference of squares)
        xs, x, gs, gm, ts, bt, _, _ = norm_inputs(c, shift=shift)
        check_norm(c, run_gpu(nc.norm_name(c), norm_args(c, xs, gs, ts), gpu), x, gm, bt)


def check_grad(c, outs, x, gm, dy, mean, rstd, groups=512):
    r, n, el, p, ck, aff = c
    gm = gm if aff >= 1 else np.ones(n)
    dx, dg, db = bs.layer_norm_grad(dy, x, gm, mean, rstd)
    xh, gg = (x - mean[:, None]) * rstd[:, None], dy * gm
    a = (adds(n) + 5) * E24
    m0, m1 = np.abs(gg).mean(axis=1, keepdims=True), np.abs(gg * xh).mean(axis=1, keepdims=True)
    tol = rstd[:, None] * (a * (m0 + np.abs(xh) * m1) + 6 * E24 * (np.abs(gg) + m0 + np.abs(xh) * m1))
    assert (np.abs(value(outs[0], el) - dx) <= tol + U[el] * (np.abs(dx) + tol) + TINY[el]).all()
    # a column: the rows of a group one after another, then the groups in 16
    # slices (and those in order)
    n_adds = -(-r // groups) + -(-min(r, 4 * groups) // 16) + 16 + 4
    for got, want, terms in zip(outs[1:], (dg, db), (np.abs(dy * xh), np.abs(dy))):
        t = n_adds * E24 * terms.sum(axis=0)
        assert (np.abs(value(got, p) - want) <= t + U[p] * (np.abs(want) + t) + TINY[p]).all()


def grad_args(c, xs, x, gs, ds):
    """Kernel arguments and the f64 x, mean and 1/std they stand for."""
    r, n, el, p, ck, aff = c
    mean, var = x.mean(axis=1).astype(np.float32), x.var(axis=1)
    rstd = (1 / np.sqrt(var + 1e-5)).astype(np.float32)
    src = [xs]
    if ck:
        codes, scales = bs.quantize(x, ck, 1)
        src, x = [codes, scales.view(np.int8)], bs.dequantize(codes, scales, ck, 1)
    args = [ds] + src + [gs][:aff] + [mean, rstd, np.zeros_like(ds)] + [np.zeros_like(gs)] * aff
    return args, x, mean.astype(np.float64), rstd.astype(np.float64)


@pytest.mark.gpu
@pytest.mark.parametrize("c", nc.NORM, ids=lambda c: nc.norm_name(c, "lngrad"))
def test_layer_norm_grad(gpu, c):
    note(nc.norm_name(c, "lngrad"))
    xs, x, gs, gm, _, _, ds, dy = norm_inputs(c)
    args, x, mean, rstd = grad_args(c, xs, x, gs, ds)
    check_grad(c, run_gpu(nc.norm_name(c, "lngrad"), args, gpu), x, gm, dy, mean, rstd)


@pytest.mark.gpu
def test_layer_norm_gradient_against_differences(gpu):
    """The GPU's gradient against differences of the GPU's own forward: the
    change of sum(y w) along a direction, f32 throughout."""
    import torch
    c = (600, 320, "f32", "f32", None, 2)
    note("gradient against differences")
    xs, x, gs, gm, ts, bt, ds, dy = norm_inputs(c)
    args, _, _, _ = grad_args(c, xs, x, gs, ds)
    dx, dg, db = run_gpu(nc.norm_name(c, "lngrad"), args, gpu)
    rng = np.random.default_rng(2)
    h = 2.0 ** -6
    for which, grad in ((0, dx), (1, dg), (2, db)):
        base = [xs, gs, ts]
        d = rng.choice([-1.0, 1.0], base[which].shape).astype(np.float32)
        vals = []
        for s in (h, -h):
            moved = [a.copy() for a in base]
            moved[which] = (moved[which] + np.float32(s) * d).astype(np.float32)
            y = run_gpu(nc.norm_name(c), norm_args(c, *moved), gpu)[0]
            vals.append((y.astype(np.float64) * dy).sum())
        got, want = (grad.astype(np.float64) * d).sum(), (vals[0] - vals[1]) / (2 * h)
        # third-order term of the difference: h^2 / 6 times a third derivative of
        # order rstd^3 per element, added at random over the elements; and the
        # rounding of y (2^-24 |y| |dy| each, at random) over 2 h
        r3 = (1 / np.sqrt(x.var(axis=1) + 1e-5)) ** 3
        curve = h * h * 8 * np.sqrt((dy ** 2 * (np.abs(x - x.mean(axis=1, keepdims=True)) + 1) ** 2 * r3[:, None] ** 2).sum()) * np.sqrt(320)
        noise = np.sqrt(((dy * 8) ** 2).sum()) * 8 * E24 / (2 * h) + np.abs(grad * d).sum() * 64 * E24
        assert abs(got - want) <= curve + noise, (which, got, want, curve, noise)


@pytest.mark.gpu
def test_layer_norm_rank3(gpu):
    note("rank 3")
    c = (6, 64, "bf16", "bf16", "e4m3", 2)
    xs, x, gs, gm, ts, bt, ds, dy = norm_inputs(c)
    args = norm_args(c, xs, gs, ts)
    shapes = [p["shape"] for p in hf.compile(cat.get("ln_rank3"), require_cached=True).blocks[0]["params"]]
    outs = run_gpu("ln_rank3", [a.reshape(s) for a, s in zip(args, shapes)], gpu)
    assert outs[0].shape == (2, 3, 64) and outs[1].shape == (2, 3)
    check_norm(c, [o.reshape((6,) + o.shape[2:]) for o in outs], x, gm, bt)
    cg = c[:4] + (None, 2)
    args, _, mean, rstd = grad_args(cg, xs, x, gs, ds)
    shapes = [p["shape"] for p in hf.compile(cat.get("lngrad_rank3"), require_cached=True).blocks[0]["params"]]
    outs = run_gpu("lngrad_rank3", [a.reshape(s) for a, s in zip(args, shapes)], gpu)
    check_grad(cg, [outs[0].reshape(6, 64)] + outs[1:], x, gm, dy, mean, rstd)


@pytest.mark.gpu
@pytest.mark.parametrize("name,cols,ck,p", [("lngrad_rt", 1000, "e4m3", "f32"), ("lngrad_wide_rt", 4096, None, "bf16")])
def test_layer_norm_at_launch_time_rows(gpu, name, cols, ck, p):
    """Any row count through one group, zero included: no rows leave zeros in
    the weight's gradients."""
    import torch
    grp = hf.compile(cat.get(name), options=cat.options(name), require_cached=True).load()
    fwd = hf.compile(cat.get("ln_rt"), options=cat.options("ln_rt"), require_cached=True).load()
    for rows in (1, 2, 37, 600, 1500, 0):
        note(f"{name} {rows}")
        c = (rows, cols, "bf16", p, ck, 2)
        if rows == 0:
            z = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt, device=gpu)  # noqa: E731
            src = [torch.zeros((0, cols), dtype=torch.uint8, device=gpu).view(torch.float8_e4m3fn), z(0, (cols + 31) // 32, dt=torch.int8)] if ck else [z(0, cols)]
            pt = torch.float32 if p == "f32" else torch.bfloat16
            dg, db = (torch.full((cols,), 7.0, dtype=pt, device=gpu) for _ in range(2))
            grp(z(0, cols), *src, z(cols, dt=pt), z(0, dt=torch.float32), z(0, dt=torch.float32), z(0, cols), dg, db)
            assert not dg.any() and not db.any()
            continue
        xs, x, gs, gm, ts, bt, ds, dy = norm_inputs(c)
        args, xv, mean, rstd = grad_args(c, xs, x, gs, ds)
        outs = grp(*(to_dev(a, q["elem"], gpu) for a, q in zip(args, grp.meta["params"])))
        check_grad(c, [to_host(o, q["elem"]) for o, q in zip(outs, grp.meta["results"])], xv, gm, dy, mean, rstd)
        if ck:
            cf = (rows, cols, "bf16", "bf16", ck, 2)
            xs, x, gs, gm, ts, bt, _, _ = norm_inputs(cf)
            outs = fwd(*(to_dev(a, q["elem"], gpu) for a, q in zip(norm_args(cf, xs, gs, ts), fwd.meta["params"])))
            check_norm(cf, [to_host(o, q["elem"]) for o, q in zip(outs, fwd.meta["results"])], x, gm, bt)


@pytest.mark.gpu
def test_layer_norm_rows_that_are_no_numbers(gpu):
    """A row with NaN or infinity gives NaN in that row alone; its checkpoint
    block is NaN, the row's others are not."""
    note("rows that are no numbers")
    c = (130, 1000, "bf16", "bf16", "e4m3", 2)
    xs, x, gs, gm, ts, bt, ds, dy = norm_inputs(c)
    x[5, 77], x[9, 999], x[64, 0] = np.nan, np.inf, -np.inf
    xs, x = stored(x, "bf16")
    outs = run_gpu(nc.norm_name(c), norm_args(c, xs, gs, ts), gpu)
    bad = np.zeros(130, bool)
    bad[[5, 9, 64]] = True
    y = value(outs[0], "bf16")
    assert np.isnan(y[bad]).all()
    check_norm((127,) + c[1:], [o[~bad] for o in outs], x[~bad], gm, bt)
    assert (outs[4].view(np.uint8) == 255).sum() == 3
    # rows of equal values: no variance, y is the bias
    xs, x = stored(np.full((130, 1000), 3.0), "bf16")
    y = value(run_gpu(nc.norm_name(c), norm_args(c, xs, gs, ts), gpu)[0], "bf16")
    assert np.array_equal(y, np.broadcast_to(bt, y.shape))


# ---------------------------------------------------------------- weight product
def linear_inputs(m, n, k, fmt, seed=4):
    rng = np.random.default_rng(seed + m + n + k)
    as_, a = stored(rng.normal(size=(m, k)), "bf16")
    codes, scales = bs.quantize(rng.normal(size=(n, k)) / np.sqrt(k), fmt, 1)
    w = bs.pack(codes, 1).view(np.int8) if fmt == "e2m1" else codes
    return as_, a, w, scales.view(np.int8), rng.normal(0, 0.1, n).astype(np.float32), bs.dequantize(w, scales, fmt, 1)


def check_linear(got, out, a, w, bias, k):
    with np.errstate(invalid="ignore"):
        want = a @ w.T + bias
    # a matrix-core step adds 32 products to the sum, at most a whole step of
    # f32 each: 32 + k/32 steps + 8 partial sums + the bias
    t = (2 * (40 + k / 32) + 2) * E24 * (np.abs(a) @ np.abs(w).T + np.abs(bias))
    assert (np.abs(value(got, out) - want) <= t + U[out] * (np.abs(want) + t)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("c", nc.LINEAR, ids=nc.linear_name)
def test_linear(gpu, c):
    m, n, k, fmt, bias, out = c
    note(nc.linear_name(c))
    as_, a, w, s, b, wv = linear_inputs(m, n, k, fmt)
    got, = run_gpu(nc.linear_name(c), [as_, w, s] + [b] * bias + [np.zeros((m, n), interp.NP[out])], gpu)
    check_linear(got, out, a, wv, b if bias else 0 * b, k)


@pytest.mark.gpu
@pytest.mark.parametrize("name,n,k,fmt,bias", [("linmx_e2m1_rt", 130, 544, "e2m1", True), ("linmx_e4m3_rt", 1040, 1024, "e4m3", False)])
def test_linear_at_launch_time_rows(gpu, name, n, k, fmt, bias):
    import torch
    grp = hf.compile(cat.get(name), options=cat.options(name), require_cached=True).load()
    for m in nc.RT_ROWS + [1100, 2100]:
        note(f"{name} {m}")
        as_, a, w, s, b, wv = linear_inputs(m, n, k, fmt)
        # (guard rows behind the result stay as they are)
        out = torch.full((m + 3, n), 9.0, dtype=torch.bfloat16, device=gpu)
        args = [to_dev(v, p["elem"], gpu) for v, p in zip([as_, w, s] + [b] * bias, grp.meta["params"])]
        got = grp(*args, out[:m])
        check_linear(to_host(got, "bf16"), "bf16", a, wv, b if bias else 0 * b, k)
        assert (out[m:] == 9.0).all()


@pytest.mark.gpu
def test_linear_scales_at_their_ends(gpu):
    """Scale bytes 0 and 254 and NaN (255) in the weight: every code's value
    as the formula has it, a NaN block in every result of its row alone."""
    note("scale bytes at their ends")
    for c in nc.LINEAR:
        m, n, k, fmt, bias, out = c
        if out != "f32":
            continue
        as_, a, w, s, b, _ = linear_inputs(m, n, k, fmt)
        sb = s.view(np.uint8).copy()
        sb[0, 0] = 0
        if n > 5:
            sb[3, -1], sb[5, 0] = 255, 0
        # (2^127 times a large code is past f32: one code of 1 in that block)
        wb = w.view(np.uint8).copy()
        if n > 8:
            sb[7, 0] = 254
            wb[7, : 16 if fmt == "e2m1" else 32] = 0
            wb[7, 0] = {"e2m1": 2, "e4m3": 0x38, "e5m2": 0x3C}[fmt]
            as_[:, 0] = 0
            as_[0, 0] = 0x3E80  # 0.25
            a = value(as_, "bf16")
        w = wb.view(w.dtype)
        wv = bs.dequantize(w, sb, fmt, 1)
        got, = run_gpu(nc.linear_name(c), [as_, w, sb.view(np.int8)] + [b] * bias + [np.zeros((m, n), np.float32)], gpu)
        nan = np.isnan(wv).any(axis=1)
        assert np.isnan(got[:, nan]).all()
        check_linear(got[:, ~nan], out, a, wv[~nan], (b if bias else 0 * b)[~nan], k)


@pytest.mark.gpu
@pytest.mark.parametrize("c", [c for c in nc.LINEAR if c[5] == "f32"], ids=nc.linear_name)
def test_linear_smallest_scales(gpu, c):
    """Weights of 2^-127 .. 2^-124 (bf16's subnormals among them) against rows
    of about 2^110: their products count as any others."""
    m, n, k, fmt, bias, out = c
    note("smallest scales " + nc.linear_name(c))
    as_, a, w, s, b, _ = linear_inputs(m, n, k, fmt)
    as_, a = stored(np.ldexp(a, 110), "bf16")
    sb = (np.arange(s.size).reshape(s.shape) % 4).astype(np.uint8)
    wv = bs.dequantize(w, sb, fmt, 1)
    got, = run_gpu(nc.linear_name(c), [as_, w, sb.view(np.int8)] + [0 * b] * bias + [np.zeros((m, n), np.float32)], gpu)
    check_linear(got, out, a, wv, 0 * b, k)


# ---------------------------------------------------------------- together, and how they are called
@pytest.mark.gpu
def test_norm_quantize_matmul_program(gpu):
    """Layer norm -> quantisation -> block-scaled contraction as one program.
    The norm's result rounds to bf16 within its tolerance, so a code next to a
    border may be the neighbour: the product is compared with the one of the
    GPU's own norm, whose codes are exact."""
    import torch
    note("prog_norm_matmul_mx")
    rng = np.random.default_rng(21)
    m, n, k = 100, 208, 384
    (xs, x), (gs, gm), (ts, bt) = (stored(a, "bf16") for a in (activations(rng, m, k), rng.uniform(0.5, 1.5, k), rng.normal(0, 0.1, k)))
    wc, ws = bs.quantize(rng.normal(size=(k, n)) / 16, "e4m3", 0)
    prog = hf.compile(cat.get("prog_norm_matmul_mx"), require_cached=True).load()
    args = [to_dev(a, p["elem"], gpu) for a, p in zip([xs, gs, ts, wc, ws.view(np.int8)], prog.meta["params"])]
    got = prog(*args).cpu().numpy()
    fwd = hf.load(g.layer_norm(m, k))
    y = fwd(*args[:3], *(torch.empty(s, dtype=d, device=gpu) for s, d in (((m, k), torch.bfloat16), ((m,), torch.float32), ((m,), torch.float32))))[0]
    q, s = bs.quantize(value(to_host(y, "bf16"), "bf16"), "e4m3", 1)
    a, b = bs.dequantize(q, s, "e4m3", 1), bs.dequantize(wc, ws, "e4m3", 0)
    # (fp8 block products: within 2^-11 of the products' magnitude sum)
    assert (np.abs(got - a @ b) <= 2.0 ** -11 * (np.abs(a) @ np.abs(b))).all()


@pytest.mark.gpu
def test_training_step_of_norm_and_linear(gpu):
    """Forward with an 8-bit checkpoint, the weight to 4 bits, the linear
    layer, and back: dy through the weight read back to bf16, then the norm's
    gradient from the checkpoint.  Each stage is held to its own tolerance on
    the stage before's output."""
    import torch
    note("training step")
    c = (130, 1000, "bf16", "bf16", "e4m3", 2)
    xs, x, gs, gm, ts, bt, _, _ = norm_inputs(c)
    outs = run_gpu(nc.norm_name(c), norm_args(c, xs, gs, ts), gpu)
    check_norm(c, outs, x, gm, bt)
    rng = np.random.default_rng(6)
    ds, dy = stored(rng.normal(0, 0.1, (130, 1000)), "bf16")
    args = [ds, outs[3], outs[4], gs, outs[1], outs[2], np.zeros_like(ds), np.zeros_like(gs), np.zeros_like(gs)]
    got = run_gpu(nc.norm_name(c, "lngrad"), args, gpu)
    kept = bs.dequantize(outs[3], outs[4], "e4m3", 1)
    check_grad(c, got, kept, gm, dy, outs[1].astype(np.float64), outs[2].astype(np.float64))
    # the checkpoint is within half a step of its block's largest binade of x
    amax = np.abs(x).reshape(130, -1)
    for b in range(0, 1000, 32):
        top = amax[:, b:b + 32].max(axis=1, keepdims=True)
        assert (np.abs(kept[:, b:b + 32] - x[:, b:b + 32]) <= top * 2.0 ** -3).all()


@pytest.mark.gpu
def test_captured_and_replayed(gpu):
    """Forward, gradient (with its workspace) and product in one captured
    graph, replayed on new inputs with eager work between the replays."""
    import torch
    note("captured")
    load = lambda n: hf.compile(cat.get(n), options=cat.options(n), require_cached=True).load()  # noqa: E731
    fwd, bwd, lin = load("ln_rt"), load("lngrad_rt"), load("linmx_e2m1_rt")
    rows, cols = 300, 1000
    dev = dict(device=gpu)
    x = torch.randn(rows, cols, **dev).bfloat16()
    dy = torch.randn(rows, cols, **dev).bfloat16()
    gm, bt = torch.rand(cols, **dev).bfloat16() + 0.5, torch.randn(cols, **dev).bfloat16()
    w = torch.randint(-128, 128, (130, 272), dtype=torch.int8, **dev)
    sc = torch.randint(115, 125, (130, 17), dtype=torch.int8, **dev)
    bias = torch.randn(130, **dev)
    a = torch.randn(100, 544, **dev).bfloat16()

    def buffers():
        e = lambda s, d: torch.zeros(s, dtype=d, **dev)  # noqa: E731
        return ([e((rows, cols), torch.bfloat16), e((rows,), torch.float32), e((rows,), torch.float32),
                 e((rows, cols), torch.uint8).view(torch.float8_e4m3fn), e((rows, 32), torch.int8)],
                [e((rows, cols), torch.bfloat16), e((cols,), torch.float32), e((cols,), torch.float32)], e((100, 130), torch.bfloat16))

    def step(o):
        fwd(x, gm, bt, *o[0])
        bwd(dy, o[0][3], o[0][4], gmf, o[0][1], o[0][2], *o[1])
        lin(a, w, sc, bias, o[2])
    gmf = gm.float()
    eager, held = buffers(), buffers()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(held)
    for i in range(4):
        x.copy_(torch.randn(rows, cols, **dev) * (i + 1))
        dy.copy_(torch.randn(rows, cols, **dev))
        a.copy_(torch.randn(100, 544, **dev))
        graph.replay()
        torch.cuda.synchronize()
        step(eager)
        torch.cuda.synchronize()
        for p, q in zip(eager[0] + eager[1] + [eager[2]], held[0] + held[1] + [held[2]]):
            assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))


@pytest.mark.gpu
def test_two_streams_with_workspaces_of_their_own(gpu):
    """Two gradients in flight at once, each with a caller's workspace; the
    same group on one stream twice gives the same bits."""
    import torch
    note("two streams")
    grp = hf.compile(cat.get("lngrad_rt"), options=cat.options("lngrad_rt"), require_cached=True).load()
    cases = []
    for seed in (1, 2):
        c = (900, 1000, "bf16", "f32", "e4m3", 2)
        xs, x, gs, gm, _, _, ds, dy = norm_inputs(c, seed=seed)
        args, xv, mean, rstd = grad_args(c, xs, x, gs, ds)
        cases.append(([to_dev(a, p["elem"], gpu) for a, p in zip(args, grp.meta["params"])], xv, gm, dy, mean, rstd))
    streams = [torch.cuda.Stream() for _ in cases]
    spaces = [torch.zeros(grp.info.workspace_bytes, dtype=torch.uint8, device=gpu) for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        for (args, *_r), s, ws in zip(cases, streams, spaces):
            grp(*args, stream=s.cuda_stream, workspace=ws)
    torch.cuda.synchronize()
    first = []
    for args, xv, gm, dy, mean, rstd in cases:
        outs = [to_host(o, q["elem"]) for o, q in zip(args[-3:], grp.meta["results"])]
        check_grad(c, outs, xv, gm, dy, mean, rstd)
        first.append(outs)
    for (args, *_r), outs in zip(cases, first):
        grp(*args)
        torch.cuda.synchronize()
        for o, q, w in zip(args[-3:], grp.meta["results"], outs):
            assert np.array_equal(to_host(o, q["elem"]).view(np.uint8), w.view(np.uint8))


@pytest.mark.gpu
def test_strided_views_and_offsets(gpu):
    """Memref descriptors: x a row-pitched view, codes at an odd offset."""
    import torch
    from hfusion_mi355x import native
    note("memref views")
    c = (33, 101, "f16", "e4m3", 1)
    r, n = 33, 101
    xs, x = stored(activations(np.random.default_rng(9), r, n), "f16")
    grp = hf.compile(cat.get(nc.quant_name(c)), require_cached=True).load()
    wide = torch.zeros((r, 150), dtype=torch.float16, device=gpu)
    wide[:, 3:104] = to_dev(xs, "f16", gpu)
    codes = torch.full((r * n + 40,), 0xA5, dtype=torch.uint8, device=gpu)
    scales = torch.full((r * 4 + 8,), 0xA5, dtype=torch.uint8, device=gpu)
    descs = [native.memref_descriptor(wide.data_ptr(), [r, n], offset=3, strides=[150, 1]),
             native.memref_descriptor(codes.data_ptr(), [r, n], offset=13), native.memref_descriptor(scales.data_ptr(), [r, 4], offset=1)]
    ptrs = (ctypes.c_void_p * 3)(*[ctypes.addressof(d) for d in descs])
    native.check(native.hfr().hfr_group_launch_memref(grp._h, ptrs, 3, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    wq, ws = bs.quantize(x, "e4m3", 1)
    got, gs = codes.cpu().numpy(), scales.cpu().numpy()
    assert np.array_equal(got[13:13 + r * n].reshape(r, n), wq) and np.array_equal(gs[1:1 + r * 4].reshape(r, 4), ws)
    assert (got[:13] == 0xA5).all() and (got[13 + r * n:] == 0xA5).all() and gs[0] == 0xA5 and (gs[1 + r * 4:] == 0xA5).all()


@pytest.mark.gpu
def test_gradient_without_allocation(gpu):
    """hfr_group_launch_noalloc: the library's scratch in place of the workspace."""
    import torch
    note("noalloc")
    c = nc.NORM_LONG[0]
    xs, x, gs, gm, _, _, ds, dy = norm_inputs(c)
    args, xv, mean, rstd = grad_args(c, xs, x, gs, ds)
    grp = hf.compile(cat.get(nc.norm_name(c, "lngrad")), require_cached=True).load()
    assert 0 < grp.info.workspace_bytes <= hf.native.hfr().hfr_scratch_bytes()
    outs = grp(*(to_dev(a, p["elem"], gpu) for a, p in zip(args, grp.meta["params"])), noalloc=True)
    torch.cuda.synchronize()
    check_grad(c, [to_host(o, q["elem"]) for o, q in zip(outs, grp.meta["results"])], xv, gm, dy, mean, rstd, groups=256)


# ---------------------------------------------------------------- workspaces, alignment, empty rows
def test_refused_empty_rows():
    for ir in (g.layer_norm(0, 64), g.layer_norm_grad(0, 64)):
        with pytest.raises(RuntimeError, match="empty tensor"):
            hf.compile(ir)


@pytest.mark.gpu
def test_refused_operands_off_their_alignment(gpu):
    """Rows and codes of the weight product start on 16 bytes, or the launch
    is refused and writes nothing; scales may start anywhere."""
    import torch
    note("alignment")
    m, n, k, fmt, bias, out = c = (17, 100, 1024, "e2m1", True, "bf16")
    grp = hf.compile(cat.get(nc.linear_name(c)), require_cached=True).load()
    as_, a, w, s, b, wv = linear_inputs(m, n, k, fmt)
    good = [to_dev(v, p["elem"], gpu) for v, p in zip([as_, w, s, b], grp.meta["params"])]

    def moved(t, by):  # a contiguous view `by` elements into a buffer
        big = torch.zeros(t.numel() + by, dtype=t.dtype, device=gpu)
        big[by:] = t.reshape(-1)
        return big[by:].view(t.shape)
    for i, by in ((0, 1), (0, 4), (1, 1), (1, 8)):
        o = torch.full((m, n), 9.0, dtype=torch.bfloat16, device=gpu)
        with pytest.raises(RuntimeError, match="does not start on 16 bytes"):
            grp(*(moved(t, by) if j == i else t for j, t in enumerate(good)), o)
        assert (o == 9.0).all()
    o = moved(torch.full((m, n), 9.0, dtype=torch.bfloat16, device=gpu), 1)
    grp(moved(good[0], 8), moved(good[1], 16), moved(good[2], 3), moved(good[3], 1), o)
    check_linear(to_host(o, "bf16"), "bf16", a, wv, b, k)


@pytest.mark.gpu
def test_refused_workspaces(gpu):
    import torch
    note("workspaces refused")
    c = nc.NORM_LONG[0]
    grp = hf.compile(cat.get(nc.norm_name(c, "lngrad")), require_cached=True).load()
    xs, x, gs, gm, _, _, ds, dy = norm_inputs(c)
    args, xv, mean, rstd = grad_args(c, xs, x, gs, ds)
    args = [to_dev(a, p["elem"], gpu) for a, p in zip(args, grp.meta["params"])]
    need = grp.info.workspace_bytes
    for ws in (torch.zeros(need - 1, dtype=torch.uint8, device=gpu), torch.zeros(need, dtype=torch.uint8),
               torch.zeros(2 * need, dtype=torch.uint8, device=gpu)[::2]):
        with pytest.raises(ValueError, match="needs a workspace"):
            grp(*args, workspace=ws)
    with pytest.raises(RuntimeError, match="start on 16 bytes"):
        grp(*args, workspace=torch.zeros(need + 4, dtype=torch.uint8, device=gpu)[4:])
    outs = grp(*args, workspace=torch.zeros(need, dtype=torch.uint8, device=gpu))
    check_grad(c, [to_host(o, q["elem"]) for o, q in zip(outs, grp.meta["results"])], xv, gm, dy, mean, rstd, groups=256)


@pytest.mark.gpu
def test_plain_calls_on_two_streams_and_graphs_that_overlap(gpu):
    """One group, plain calls in flight on two streams, and two captured
    graphs replayed on two streams at once: each has a workspace of its own."""
    import torch
    note("overlapping plain calls")
    grp = hf.compile(cat.get("lngrad_rt"), options=cat.options("lngrad_rt"), require_cached=True).load()
    lin = hf.compile(cat.get("linmx_e4m3_rt"), options=cat.options("linmx_e4m3_rt"), require_cached=True).load()
    c = (2100, 1000, "bf16", "f32", "e4m3", 2)
    cases = []
    for seed in (3, 4):
        xs, x, gs, gm, _, _, ds, dy = norm_inputs(c, seed=seed)
        args, _, _, _ = grad_args(c, xs, x, gs, ds)
        as_, _, w, s, _, _ = linear_inputs(2100, 1040, 1024, "e4m3", seed=seed)
        cases.append(([to_dev(a, p["elem"], gpu) for a, p in zip(args, grp.meta["params"])],
                      [to_dev(a, p["elem"], gpu) for a, p in zip([as_, w, s], lin.meta["params"])]
                      + [torch.zeros((2100, 1040), dtype=torch.bfloat16, device=gpu)]))

    def run(case):
        grp(*case[0])
        lin(*case[1])

    def results(case):
        return [t.clone() for t in case[0][-3:] + case[1][-1:]]

    def wipe():
        for case in cases:
            for t in case[0][-3:] + case[1][-1:]:
                t.zero_()
        torch.cuda.synchronize()
    want = []
    for case in cases:  # one after another
        run(case)
        torch.cuda.synchronize()
        want.append(results(case))
    streams = [torch.cuda.Stream() for _ in cases]

    def check():
        torch.cuda.synchronize()
        for case, w in zip(cases, want):
            for p, q in zip(results(case), w):
                assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))
    wipe()
    for _ in range(8):
        for case, s in zip(cases, streams):
            with torch.cuda.stream(s):
                run(case)
    check()
    graphs = []
    for case in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            run(case)
    for _ in range(3):
        wipe()
        for _ in range(4):
            for gr, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    gr.replay()
        check()


@pytest.mark.gpu
def test_programs_of_two_graphs(gpu):
    """A program whose product takes the weight through a workspace, captured
    twice and replayed on two streams at once."""
    import torch
    note("programs of two graphs")
    m, n, k = 2300, 1040, 1024
    prog = hf.compile(cat.get("prog_norm_linear_mx_many"), require_cached=True).load()
    assert prog.workspace_bytes >= 2 * n * k  # (the weight as bf16)
    cases, want = [], []
    for seed in (1, 2):
        rng = np.random.default_rng(seed)
        (xs, x), (gs, gm), (ts, bt) = (stored(a, "bf16") for a in (activations(rng, m, k), rng.uniform(0.5, 1.5, k), rng.normal(0, 0.1, k)))
        _, _, w, s, _, wv = linear_inputs(8, n, k, "e2m1", seed=seed)
        cases.append([to_dev(v, p["elem"], gpu) for v, p in zip([xs, gs, ts, w, s], prog.meta["params"])])
        want.append(prog(*cases[-1]))
        torch.cuda.synchronize()
        # the norm's result is within half a step of bf16 (2^-8) and its f32 sums'
        # error (below 2^-14 of a value of order 4), the product rounds once more
        y, _, _ = bs.layer_norm(x, gm, bt, 1e-5)
        t = (2.0 ** -8 * np.abs(y) + 2.0 ** -12) @ np.abs(wv).T
        t = t * (1 + 2.0 ** -8) + (2.0 ** -8 + 100 * E24) * (np.abs(y) @ np.abs(wv).T)
        assert (np.abs(value(to_host(want[-1], "bf16"), "bf16") - y @ wv.T) <= t).all()
    graphs, held = [], []
    for args in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(prog(*args))
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        for h in held:
            h.zero_()
        torch.cuda.synchronize()
        for _ in range(4):
            for gr, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    gr.replay()
        torch.cuda.synchronize()
        for h, w in zip(held, want):
            assert torch.equal(h.view(torch.uint8), w.view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("c", nc.LINEAR_MANY, ids=nc.linear_name)
def test_linear_through_the_workspace(gpu, c):
    """More rows: the weight as bf16 in the workspace; scale bytes 0 and 255
    and the largest that bf16 holds go through it too."""
    m, n, k, fmt, bias, out = c
    note(nc.linear_name(c))
    grp = hf.compile(cat.get(nc.linear_name(c)), require_cached=True).load()
    assert grp.info.workspace_bytes >= 2 * n * k
    as_, a, w, s, b, wv = linear_inputs(m, n, k, fmt)
    got, = run_gpu(nc.linear_name(c), [as_, w, s] + [b] * bias + [np.zeros((m, n), interp.NP[out])], gpu)
    check_linear(got, out, a, wv, b if bias else 0 * b, k)
    sb = s.view(np.uint8).copy()
    sb[0, 0], sb[3, -1], sb[5, 0] = 0, 255, 0
    wv = bs.dequantize(w, sb, fmt, 1)
    got, = run_gpu(nc.linear_name(c), [as_, w, sb.view(np.int8)] + [b] * bias + [np.zeros((m, n), interp.NP[out])], gpu)
    nan = np.isnan(wv).any(axis=1)
    assert nan.sum() == 1 and np.isnan(value(got, out)[:, nan]).all()
    check_linear(got[:, ~nan], out, a, wv[~nan], (b if bias else 0 * b)[~nan], k)


@pytest.mark.gpu
@pytest.mark.parametrize("name,n,k,fmt,bias", [("linmx_e2m1_rt", 130, 544, "e2m1", True), ("linmx_e4m3_rt", 1040, 1024, "e4m3", False)])
def test_linear_of_many_rows_at_launch_time(gpu, name, n, k, fmt, bias):
    """Past every kernel that reads the codes themselves."""
    import torch
    art = hf.compile(cat.get(name), options=cat.options(name), require_cached=True)
    grp = art.load()
    with open(art.manifest) as f:
        few = max(int(ln.split()[2]) for ln in f if ln.startswith("alt ") and not ln.split()[-1] == "pre")
    for m in (few, few + 1, 4500):
        note(f"{name} {m}")
        as_, a, w, s, b, wv = linear_inputs(m, n, k, fmt)
        out = torch.full((m + 3, n), 9.0, dtype=torch.bfloat16, device=gpu)
        got = grp(*(to_dev(v, p["elem"], gpu) for v, p in zip([as_, w, s] + [b] * bias, grp.meta["params"])), out[:m])
        check_linear(to_host(got, "bf16"), "bf16", a, wv, b if bias else 0 * b, k)
        assert (out[m:] == 9.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("c", nc.NORM_LONG, ids=nc.norm_name)
def test_layer_norm_of_many_rows(gpu, c):
    """Workgroups that walk several rows, the last of them partly or not there."""
    note(nc.norm_name(c))
    xs, x, gs, gm, ts, bt, ds, dy = norm_inputs(c)
    check_norm(c, run_gpu(nc.norm_name(c), norm_args(c, xs, gs, ts), gpu), x, gm, bt)
    args, x, mean, rstd = grad_args(c, xs, x, gs, ds)
    # (fewer row groups than 512: more additions one after another)
    check_grad(c, run_gpu(nc.norm_name(c, "lngrad"), args, gpu), x, gm, dy, mean, rstd, groups=256)


@pytest.mark.gpu
def test_gradient_of_rows_that_are_no_numbers(gpu):
    """NaN or infinity in dy or x: NaN in that row of dx alone, and in the
    weight's gradients where the row's values are none."""
    note("gradient of rows that are no numbers")
    c = (700, 2001, "bf16", "f32", None, 2)
    xs, x, gs, gm, _, _, ds, dy = norm_inputs(c)
    clean, xv, mean, rstd = grad_args(c, xs, x, gs, ds)
    want = run_gpu(nc.norm_name(c, "lngrad"), clean, gpu)
    dy[5, 77], dy[9, 2000] = np.nan, np.inf
    ds, dy = stored(dy, "bf16")
    got = run_gpu(nc.norm_name(c, "lngrad"), [ds] + clean[1:], gpu)
    bad = np.zeros(700, bool)
    bad[[5, 9]] = True
    dx = value(got[0], "bf16")
    assert np.isnan(dx[5]).all() and not np.isfinite(dx[9]).any()
    assert np.array_equal(got[0][~bad].view(np.uint8), want[0][~bad].view(np.uint8))
    cols = np.zeros(2001, bool)
    cols[[77, 2000]] = True
    assert np.isnan(got[2][77]) and np.isinf(got[2][2000]) and not np.isfinite(got[1][cols]).any()
    for a, b in zip(got[1:], want[1:]):
        assert np.array_equal(a[~cols], b[~cols])


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu):
    """More than 2^31 elements (4.3 GB of bf16): the last rows come out as the
    same rows alone do."""
    import torch
    note("offsets past 32 bits")
    load = lambda n: hf.compile(cat.get(n), options=cat.options(n), require_cached=True).load()  # noqa: E731
    tail = 64
    e = lambda s, d: torch.zeros(s, dtype=d, device=gpu)  # noqa: E731

    def both(grp, cols, rows, make):
        """The group over `rows` rows, whose last `tail` are random, and over those."""
        x = e((rows, cols), torch.bfloat16)
        x[-tail:] = torch.randn(tail, cols, device=gpu)
        big, small = make(rows), make(tail)
        grp(x, *big)
        grp(x[-tail:].clone(), *small)
        return x, big, small
    rows, cols = 2 ** 31 // 4096 + 200, 4096
    x, big, small = both(load("quantmx_e2m1_rt"), cols, rows, lambda r: [e((r, cols // 2), torch.int8), e((r, cols // 32), torch.int8)])
    for p, q in zip(big, small):
        assert torch.equal(p[-tail:], q) and not p[:-tail:4099].any()
    back = e((tail, cols), torch.bfloat16)
    load("dequantmx_e2m1_rt")(*big, x)
    load("dequantmx_e2m1_rt")(*small, back)
    assert torch.equal(x[-tail:], back) and not x[:-tail:4099].any()
    del x, big, small, back
    rows, cols = 2 ** 31 // 1000 + 200, 1000
    gm, bt = e((cols,), torch.bfloat16) + 1.5, e((cols,), torch.bfloat16) + 0.25
    fwd, bwd = load("ln_rt"), load("lngrad_rt")
    outs = lambda r: [e((r, cols), torch.bfloat16), e((r,), torch.float32), e((r,), torch.float32),  # noqa: E731
                      e((r, cols), torch.uint8).view(torch.float8_e4m3fn), e((r, 32), torch.int8)]
    x, big, small = both(fwd, cols, rows, lambda r: [gm, bt] + outs(r))
    for p, q in zip(big[2:], small[2:]):
        assert torch.equal(p[-tail:].view(torch.uint8), q.view(torch.uint8))
    assert (big[2][:-tail:4099] == 0.25).all()
    del big[2]
    # the gradient: x takes dy's place; rows of zeros add nothing to the weight's
    grads = lambda r: [e((r, cols), torch.bfloat16), e((cols,), torch.float32), e((cols,), torch.float32)]  # noqa: E731
    gb, gs = grads(rows), grads(tail)
    bwd(x, big[4], big[5], gm.float(), big[2], big[3], *gb)
    bwd(x[-tail:].clone(), small[5], small[6], gm.float(), small[3], small[4], *gs)
    assert torch.equal(gb[0][-tail:], gs[0]) and not gb[0][:-tail:4099].any()
    for p, q in zip(gb[1:], gs[1:]):  # (the same terms in another order)
        assert torch.allclose(p, q, rtol=0, atol=float(tail * 64 * E24 * 64))
    del x, big, small, gb, gs
    n, k = 130, 544
    as_, a, w, s, b, wv = linear_inputs(tail, n, k, "e2m1")
    lin = load("linmx_e2m1_rt")
    rows = 2 ** 31 // k + 200
    x, out = e((rows, k), torch.bfloat16), e((rows, n), torch.bfloat16)
    x[-tail:] = to_dev(as_, "bf16", gpu)
    lin(x, *(to_dev(v, p["elem"], gpu) for v, p in zip([w, s, b], lin.meta["params"][1:])), out)
    check_linear(to_host(out[-tail:], "bf16"), "bf16", a, wv, b, k)
    assert torch.equal(out[0], out[rows // 2]) and torch.equal(out[0], torch.from_numpy(b).to(gpu).bfloat16())


@pytest.mark.gpu
def test_captured_on_a_stream_without_a_workspace_yet(gpu):
    """A launch with an explicit stream, first met there under capture."""
    import torch
    note("captured on a new stream")
    grp = hf.compile(cat.get("lngrad_rt"), options=cat.options("lngrad_rt"), require_cached=True).load()
    c = (2100, 1000, "bf16", "f32", "e4m3", 2)
    xs, x, gs, gm, _, _, ds, dy = norm_inputs(c)
    args, xv, mean, rstd = grad_args(c, xs, x, gs, ds)
    args = [to_dev(a, p["elem"], gpu) for a, p in zip(args, grp.meta["params"])]
    grp(*args)  # (the first stream's)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        grp(*args, stream=side.cuda_stream)
    for _ in range(3):
        for t in args[-3:]:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check_grad(c, [to_host(o, q["elem"]) for o, q in zip(args[-3:], grp.meta["results"])], xv, gm, dy, mean, rstd, groups=256)
        grp(*args)


@pytest.mark.gpu
@pytest.mark.parametrize("c", nc.LINEAR_LONG, ids=nc.linear_name)
def test_linear_of_long_k(gpu, c):
    m, n, k, fmt, bias, out = c
    note(nc.linear_name(c))
    grp = hf.compile(cat.get(nc.linear_name(c)), require_cached=True).load()
    assert (grp.info.workspace_bytes > 0) == (k > 200000)
    as_, a, w, s, b, wv = linear_inputs(m, n, k, fmt)
    got, = run_gpu(nc.linear_name(c), [as_, w, s, np.zeros((m, n), np.float32)], gpu)
    check_linear(got, out, a, wv, 0 * b, k)


@pytest.mark.gpu
def test_linear_onto_a_constant(gpu):
    """The accumulator's fill is added, as matmul_mx does."""
    note("linear onto a constant")
    as_, a, w, s, b, wv = linear_inputs(5, 48, 64, "e2m1")
    got, = run_gpu("linmx_filled", [as_, w, s, np.zeros((5, 48), np.float32)], gpu)
    check_linear(got, "f32", a, wv, 0 * b + 1.5, 64)


@pytest.mark.gpu
def test_refused_overlapping_operands(gpu):
    """A destination over an operand, or over another destination, is refused
    and nothing is written; buffers side by side are not."""
    import torch
    note("overlaps")
    grp = hf.compile(cat.get("lngrad_wide_rt"), options=cat.options("lngrad_wide_rt"), require_cached=True).load()
    c = (20, 4096, "bf16", "bf16", None, 2)
    xs, x, gs, gm, _, _, ds, dy = norm_inputs(c)
    args, xv, mean, rstd = grad_args(c, xs, x, gs, ds)
    args = [to_dev(a, p["elem"], gpu) for a, p in zip(args, grp.meta["params"])]
    before = [t.clone() for t in args]
    for out, other in ((5, 0), (5, 1), (6, 2), (6, 7)):
        bad = list(args)
        bad[out] = bad[other]
        with pytest.raises(RuntimeError, match="is written and overlaps"):
            grp(*bad)
    both = torch.empty(2 * 20 * 4096 - 1, dtype=torch.bfloat16, device=gpu)
    both[:20 * 4096] = args[0].reshape(-1)
    with pytest.raises(RuntimeError, match="is written and overlaps"):
        grp(both[:20 * 4096].view(20, 4096), *args[1:5], both[20 * 4096 - 1:].view(20, 4096), *args[6:])
    for t, b in zip(args, before):
        assert torch.equal(t, b)
    both = torch.empty((40, 4096), dtype=torch.bfloat16, device=gpu)
    both[:20] = args[0]
    outs = grp(both[:20], *args[1:5], both[20:], *args[6:])
    check_grad(c, [to_host(o, q["elem"]) for o, q in zip(outs, grp.meta["results"])], xv, gm, dy, mean, rstd)
    lin = hf.compile(cat.get("linmx_e2m1_rt"), options=cat.options("linmx_e2m1_rt"), require_cached=True).load()
    a = torch.zeros((130, 544), dtype=torch.bfloat16, device=gpu)
    w, s, b = (torch.zeros(p["shape"], dtype=hf.runtime.torch_dtype(p["elem"]), device=gpu) for p in lin.meta["params"][1:4])
    with pytest.raises(RuntimeError, match="is written and overlaps"):
        lin(a, w, s, b, a.reshape(-1)[:130 * 130].view(130, 130))
