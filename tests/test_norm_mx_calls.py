"""Calls of the layer norms, block-scaled codes and weight product beside the
ordinary ones: results in buffers of their own, empty batches, workspaces,
launches under capture, the ends of the value ranges.  Each is compared with
the formulas in 64 bits at the tolerances of test_norm_mx."""
import numpy as np
import pytest

import hfusion_mi355x as hf
import group_catalog as cat
import norm_mx_catalog as nc
from helpers import to_dev, to_host
from oracle import blockscaled as bs
from test_norm_mx import E24, check_grad, check_linear, check_norm, grad_args, linear_inputs, norm_args, norm_inputs, note, stored, value


def load(name):
    return hf.compile(cat.get(name), options=cat.options(name), require_cached=True).load()


def device_args(grp, arrays, gpu):
    return [to_dev(a, p["elem"], gpu) for a, p in zip(arrays, grp.meta["params"])]


def host(outs, grp):
    return [to_host(o, r["elem"]) for o, r in zip(outs, grp.meta["results"])]


@pytest.mark.gpu
def test_results_in_buffers_of_their_own(gpu):
    """Made by the call, or the caller's: over an operand or another result
    they are refused, and nothing is written."""
    import torch
    note("untied results")
    c = (64, 256, "bf16", "bf16", None, 2)
    xs, x, gs, gm, ts, bt, ds, dy = norm_inputs(c)
    arrays, xv, mean, rstd = grad_args(c, xs, x, gs, ds)
    grp = load("lngrad_untied")
    args = device_args(grp, arrays, gpu)
    check_grad(c, host(grp(*args), grp), xv, gm, dy, mean, rstd)
    own = [torch.zeros(r["shape"], dtype=torch.bfloat16, device=gpu) for r in grp.meta["results"]]
    before = [t.clone() for t in args]
    for j, t in ((0, args[0]), (0, args[1]), (1, args[2]), (1, own[2]), (2, own[0].view(-1)[512:768])):
        bad = list(own)
        bad[j] = t
        with pytest.raises(RuntimeError, match="is written and overlaps"):
            grp(*args, results=bad)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(args, before)) and not any(t.any() for t in own)
    check_grad(c, host(grp(*args, results=own), grp), xv, gm, dy, mean, rstd)
    c = (9, 96, "bf16", "bf16", "e4m3", 2)
    xs, x, gs, gm, ts, bt, _, _ = norm_inputs(c)
    grp = load("ln_untied")
    args = device_args(grp, (xs, gs, ts), gpu)
    check_norm(c, host(grp(*args), grp), x, gm, bt)
    with pytest.raises(RuntimeError, match="is written and overlaps"):
        grp(*args, results=[args[0]] + list(grp(*args))[1:])
    grp = load("quantmx_untied")
    xs, x = stored(np.random.default_rng(4).normal(size=(70, 64)), "bf16")
    q, s = host(grp(to_dev(xs, "bf16", gpu)), grp)
    wq, ws = bs.quantize(x, "e5m2", 1)
    assert np.array_equal(q, wq) and np.array_equal(s.view(np.uint8), ws)


@pytest.mark.gpu
@pytest.mark.parametrize("name,m,n,k", [("linmx_residual", 70, 48, 96), ("linmx_residual_many", 2300, 520, 1024)])
def test_product_onto_its_residual(gpu, name, m, n, k):
    """(a w + residual) * factor over the residual itself; over the factor, or
    next to its own place in the residual, it is refused."""
    import torch
    note(name)
    as_, a, w, s, _, wv = linear_inputs(m, n, k, "e2m1")
    rng = np.random.default_rng(m)
    res, factor = rng.normal(size=(m, n)).astype(np.float32), rng.uniform(0.5, 2, m).astype(np.float32)
    grp = load(name)
    args = device_args(grp, [as_, w, s, res, factor], gpu)
    out = torch.zeros((m, n), device=gpu)
    grp(*args, out)
    # test_norm_mx's bound of the sums, one more addition, one product: a step each
    mag = np.abs(a) @ np.abs(wv).T + np.abs(res)
    tol = ((2 * (40 + k / 32) + 4) * E24 * mag) * factor[:, None]
    assert (np.abs(out.cpu().numpy() - (a @ wv.T + res) * factor[:, None]) <= tol).all()
    flat = torch.zeros(m * n + 8, device=gpu)
    flat[:m * n] = args[3].view(-1)
    here = flat[:m * n].view(m, n)
    for bad in (flat[4:m * n + 4].view(m, n), flat[8:].view(m, n)):
        with pytest.raises(RuntimeError, match="is written and overlaps argument 3"):
            grp(*args[:3], here, args[4], bad)
    wide = torch.ones(m * n + m, device=gpu)
    with pytest.raises(RuntimeError, match="is written and overlaps argument 4"):
        grp(*args[:4], wide[m * n - 4:m * n - 4 + m], wide[:m * n].view(m, n))
    grp(*args[:3], here, args[4], here)
    assert torch.equal(here, out) and not flat[m * n:].any()


@pytest.mark.gpu
def test_refused_programs_write_nothing(gpu):
    """A program whose last step is refused: its first ones have not run."""
    import torch
    note("refused programs")
    rng = np.random.default_rng(12)
    for name, m, n, k in (("prog_norm_linear_mx", 20, 208, 384), ("prog_norm_linear_mx_many", 2300, 1040, 1024)):
        (xs, x), (gs, gm), (ts, bt) = (stored(a, "bf16") for a in (rng.normal(size=(m, k)), rng.uniform(0.5, 1.5, k), rng.normal(0, 0.1, k)))
        _, _, w, s, _, wv = linear_inputs(8, n, k, "e2m1")
        prog = load(name)
        args = [to_dev(v, p["elem"], gpu) for v, p in zip([xs, gs, ts, w, s], prog.meta["params"])]
        room = torch.zeros(prog.workspace_bytes + 16, dtype=torch.uint8, device=gpu)
        # the result over the scales
        both = torch.zeros(2 * m * n + s.size, dtype=torch.uint8, device=gpu)
        over = both[2 * m * n - 8:2 * m * n - 8 + s.size].view(torch.int8).view(s.shape)
        over.copy_(args[4])
        keep = both.clone()
        with pytest.raises(RuntimeError, match="is written and overlaps"):
            prog(*args[:4], over, results=[both[:2 * m * n].view(torch.bfloat16).view(m, n)], workspace=room)
        if name.endswith("many"):
            with pytest.raises(RuntimeError, match="start on 16 bytes"):
                prog(*args, workspace=room[8:])
        torch.cuda.synchronize()
        assert not room.any() and torch.equal(both, keep)
        want = prog(*args)
        got = prog(*args, results=[torch.zeros((m, n), dtype=torch.bfloat16, device=gpu)], workspace=room)
        assert torch.equal(got, want) and room.any()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["ln_rt", "lngrad_rt", "lngrad_plain_rt", "quantmx_e4m3_rt", "quantmx_e2m1_rt", "dequantmx_e2m1_rt",
                                  "linmx_e2m1_rt", "linmx_e4m3_rt"])
def test_empty_batch(gpu, name):
    """No rows: the call returns its destinations and what has no row dim is as
    it was, but for the weight's gradients, which are zeros.  Plain calls,
    packed ones, slices of a batch, memref descriptors."""
    import ctypes
    import torch
    from hfusion_mi355x import native
    note("empty batch " + name)
    grp = load(name)
    assert grp.meta["params"] and all(r["tied"] >= 0 for r in grp.meta["results"])

    def make(rows):
        return [torch.full([rows if d == -1 else d for d in p["shape"]], 3, dtype=torch.float32, device=gpu)
                .to(hf.runtime.torch_dtype(p["elem"])) for p in grp.meta["params"]]
    args, batch = make(0), make(5)
    assert any(t.data_ptr() == 0 for t in args)
    cut = [t[:0] if -1 in p["shape"] else t for t, p in zip(batch, grp.meta["params"])]
    descs = [native.memref_descriptor(t.data_ptr(), list(t.shape)) for t in args]
    ptrs = (ctypes.c_void_p * len(descs))(*[ctypes.addressof(d) for d in descs])
    grads = [i for i, p in enumerate(grp.meta["params"]) if name == "lngrad_rt" and p["role"] != "in" and -1 not in p["shape"]]
    for tensors, call in ((args, lambda: grp(*args)), (args, lambda: grp.launcher(*args)()), (cut, lambda: grp(*cut)),
                          (args, lambda: native.check(native.hfr().hfr_group_launch_memref(grp._h, ptrs, len(descs), torch.cuda.current_stream().cuda_stream)))):
        for i in grads:
            tensors[i].fill_(7)
        before = [t.clone() for t in tensors]
        ret = call()
        torch.cuda.synchronize()
        if ret is not None:
            outs = ret if isinstance(ret, tuple) else (ret,)
            assert all(o is tensors[r["tied"]] for o, r in zip(outs, grp.meta["results"]))
        for i, (t, b) in enumerate(zip(tensors, before)):
            assert not t.any() if i in grads else torch.equal(t.view(torch.uint8), b.view(torch.uint8))
    assert all((t.float() == 3).all() for i, t in enumerate(batch) if i not in grads)


@pytest.mark.gpu
def test_argmax_with_a_workspace_off_16_bytes(gpu):
    """Any buffer of 64-bit words is a workspace of argmax, as it was."""
    import torch
    note("argmax workspace")
    grp = load("argmax_16")
    p = grp.meta["params"]
    x = torch.randn(p[0]["shape"], device=gpu)
    rest = [torch.zeros(q["shape"], dtype=hf.runtime.torch_dtype(q["elem"]), device=gpu) for q in p[1:]]
    want = [t.clone() for t in grp(x, *rest)]
    room = torch.zeros(grp.info.workspace_bytes + 8, dtype=torch.uint8, device=gpu)
    for _ in range(2):
        got = grp(x, *rest, workspace=room[8:])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError, match="start on 8 bytes"):
        grp(x, *rest, workspace=room[4:-4])


@pytest.mark.gpu
def test_workspace_of_the_launches_that_use_one(gpu):
    """A weight product at launch-time rows holds the weight as bf16 only once
    a launch of many rows needs it there; nor does a stream or a captured
    graph of few rows."""
    import torch
    note("workspace when used")
    art = hf.compile(hf.catalog.get("linear_mx_rt"), options="dyn=runtime", require_cached=True)
    n = k = 4096
    torch.cuda.synchronize()
    w = torch.randint(-128, 128, (n, k // 2), dtype=torch.int8, device=gpu)
    s = torch.randint(115, 125, (n, k // 32), dtype=torch.int8, device=gpu)
    bias = torch.randn(n, device=gpu)

    def tensors(rows):
        return torch.randn(rows, k, device=gpu).bfloat16(), torch.zeros((rows, n), dtype=torch.bfloat16, device=gpu)
    few, many = tensors(3), tensors(4096)
    whole = 2 * n * k

    def free():  # (what torch caches goes back at a capture, so before every look)
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        return torch.cuda.mem_get_info()[0]
    rows_of = hf.native.hfr().hfr_group_workspace_rows
    torch.cuda.synchronize()
    start = free()
    grp = art.load()
    assert grp.info.workspace_bytes == whole and [rows_of(grp._h, r) for r in (0, 1, 3, 4096, 10 ** 6)] == [0, 0, 0, whole, whole]
    loaded = free()
    assert start - loaded < whole // 2  # (its code)
    side = torch.cuda.Stream()
    grp(few[0], w, s, bias, few[1])
    want = few[1].clone()
    with torch.cuda.stream(side):
        grp(few[0], w, s, bias, few[1])
    grp(few[0], w, s, bias, few[1], workspace=torch.zeros(16, dtype=torch.uint8, device=gpu))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    with torch.cuda.graph(graph):
        grp(few[0], w, s, bias, few[1])
    assert torch.cuda.max_memory_allocated() - held < whole // 2
    few[1].zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(few[1], want) and loaded - free() < whole // 2
    with pytest.raises(ValueError, match=f"needs a workspace of {whole} bytes"):
        grp(many[0], w, s, bias, many[1], workspace=torch.zeros(16, dtype=torch.uint8, device=gpu))
    grp(many[0], w, s, bias, many[1])
    first = many[1].clone()
    one = free()
    assert loaded - one >= whole
    with torch.cuda.stream(side):
        many[1].zero_()
        grp(many[0], w, s, bias, many[1])
    torch.cuda.synchronize()
    assert torch.equal(many[1], first) and one - free() >= whole
    given = torch.zeros(whole, dtype=torch.uint8, device=gpu)
    grp(many[0], w, s, bias, many[1].zero_(), workspace=given)
    assert torch.equal(many[1], first) and given.any()
    del grp, graph
    # a gradient of few rows is one launch without one, of none too
    grp = load("lngrad_rt")
    assert [rows_of(grp._h, r) > 0 for r in (0, 1, 1200, 1201)] == [False, False, False, True]
    grp = load("argmax_16")
    assert rows_of(grp._h, -1) == grp.info.workspace_bytes > 0
    assert rows_of(load("ln_rt")._h, 5) == 0


class Spy:
    """The runtime library, with the workspaces that launches are given."""

    def __init__(self, lib):
        self.lib, self.seen = lib, []

    def __getattr__(self, name):
        fn = getattr(self.lib, name)
        at = {"hfr_group_launch_rows": 6, "hfr_group_launch": 5, "hfr_program_launch": 5}.get(name)
        if at is None:
            return fn

        def call(*args):
            self.seen.append(args[at])
            return fn(*args)
        return call


@pytest.mark.gpu
def test_every_capture_has_a_workspace_of_its_own(gpu, monkeypatch):
    """Under capture on the stream that a launch goes to, its workspace lies in
    the graph's memory: with the stream named, through a packed launch, through
    one that was packed before the capture, or in one and used behind it."""
    import torch
    from hfusion_mi355x import native
    note("workspaces under capture")
    spy = Spy(native.hfr())
    monkeypatch.setattr(native, "hfr", lambda: spy)
    c = (2100, 1000, "bf16", "f32", "e4m3", 2)
    xs, x, gs, gm, _, _, ds, dy = norm_inputs(c)
    arrays, xv, mean, rstd = grad_args(c, xs, x, gs, ds)
    grp, prog = load("lngrad_rt"), load("prog_norm_linear_mx")
    args = device_args(grp, arrays, gpu)
    m, n, k = 20, 208, 384
    pargs = [torch.zeros(p["shape"], dtype=hf.runtime.torch_dtype(p["elem"]), device=gpu) for p in prog.meta["params"]]
    out = torch.zeros((m, n), dtype=torch.bfloat16, device=gpu)
    side = torch.cuda.Stream()
    packed = grp.launcher(*args, stream=side.cuda_stream)
    torch.cuda.synchronize()
    graphs, inside = [], []
    for make in (lambda: grp(*args, stream=side.cuda_stream), packed, packed,
                 lambda: inside.append(grp.launcher(*args)) or inside[0](),
                 lambda: prog(*pargs, results=[out], stream=side.cuda_stream)):
        graphs.append(torch.cuda.CUDAGraph())
        spy.seen.clear()
        with torch.cuda.graph(graphs[-1], stream=side):
            make()
        assert len(spy.seen) == 1 and spy.seen[0] is not None
        graphs[-1].first = spy.seen[0]
    assert len({g.first for g in graphs}) == len(graphs)
    # outside a capture: the stream's
    spy.seen.clear()
    packed(), inside[0](), grp(*args, stream=side.cuda_stream), prog(*pargs, results=[out])
    assert spy.seen == [None] * 4
    torch.cuda.synchronize()
    for graph in graphs[:4]:
        for t in args[-3:]:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check_grad(c, host(args[-3:], grp), xv, gm, dy, mean, rstd, groups=256)


@pytest.mark.gpu
@pytest.mark.parametrize("c", nc.NORM_WIDE, ids=lambda c: nc.norm_name(c, "lngrad"))
def test_gradient_of_many_wide_rows(gpu, c):
    """Two launches, a row a workgroup: each thread leaves its columns' partial
    sums, the row's ragged end among them."""
    note(nc.norm_name(c, "lngrad"))
    grp = load(nc.norm_name(c, "lngrad"))
    assert grp.info.workspace_bytes == 256 * c[5] * c[1] * 4 and len(grp.meta["pre"]) == 1
    xs, x, gs, gm, _, _, ds, dy = norm_inputs(c)
    arrays, xv, mean, rstd = grad_args(c, xs, x, gs, ds)
    check_grad(c, host(grp(*device_args(grp, arrays, gpu)), grp), xv, gm, dy, mean, rstd, groups=256)


@pytest.mark.gpu
@pytest.mark.parametrize("c", nc.NORM_WIDE, ids=nc.norm_name)
def test_norm_of_many_wide_rows(gpu, c):
    """Workgroups of one row each that walk several."""
    note(nc.norm_name(c))
    grp = load(nc.norm_name(c))
    assert grp.meta["grid"][0] < c[0]
    xs, x, gs, gm, ts, bt, _, _ = norm_inputs(c)
    check_norm(c, host(grp(*device_args(grp, norm_args(c, xs, gs, ts), gpu)), grp), x, gm, bt)


@pytest.mark.gpu
def test_gradient_of_wide_rows_at_launch_time(gpu):
    """Both sides of the row count up to which one launch makes it."""
    note("lngrad_long_rt")
    grp = load("lngrad_long_rt")
    for rows in (1, 255, 896, 897, 1300):
        note(f"rows {rows}")
        assert (hf.native.hfr().hfr_group_workspace_rows(grp._h, rows) > 0) == (rows > 896)
        c = (rows, 5000, "bf16", "f32", None, 2)
        xs, x, gs, gm, _, _, ds, dy = norm_inputs(c)
        arrays, xv, mean, rstd = grad_args(c, xs, x, gs, ds)
        check_grad(c, host(grp(*device_args(grp, arrays, gpu)), grp), xv, gm, dy, mean, rstd, groups=256)


# the largest scale byte at which every finite code of the format is finite as bf16
LAST_FINITE = {"e5m2": 239, "e4m3": 246, "e2m1": 252}
ENDS = [(3, 33, 96, "e5m2", False, "f32"), (48, 129, 512, "e4m3", True, "f32"), (17, 100, 1024, "e2m1", True, "bf16"),
        (2300, 520, 1024, "e4m3", True, "bf16"), (4200, 129, 96, "e5m2", True, "bf16"), (4500, 40, 288, "e2m1", False, "f32")]


def bf16_of(w):
    """f64 values rounded to bf16, its subnormals (steps of 2^-133) among them."""
    step = np.ldexp(1.0, np.maximum(np.frexp(w)[1] - 8, -133))
    v = np.rint(w / step) * step
    return np.where(np.abs(v) >= 2.0 ** 128, np.copysign(np.inf, v), v)


@pytest.mark.gpu
@pytest.mark.parametrize("c", ENDS, ids=nc.linear_name)
def test_product_of_the_smallest_weights(gpu, c):
    """Small codes under the smallest scale bytes lie below bf16's smallest
    subnormal or between two of them: they count as what they round to."""
    m, n, k, fmt, bias, out = c
    note("smallest weights " + nc.linear_name(c))
    rng = np.random.default_rng(m + k)
    # (8-bit codes up to 1, both signs)
    codes = rng.integers(0, 16, (n, k)) if fmt == "e2m1" else rng.integers(0, 0x3C if fmt == "e5m2" else 0x38, (n, k)) + 128 * rng.integers(0, 2, (n, k))
    codes = codes.astype(np.uint8)
    w = bs.pack(codes, 1).view(np.int8) if fmt == "e2m1" else codes
    s = rng.integers(0, 4, (n, k // 32)).astype(np.uint8)
    exact = bs.dequantize(w, s, fmt, 1)
    wv = bf16_of(exact)
    assert (wv == exact).all() if fmt == "e2m1" else ((wv != exact).mean() > 0.1 and ((wv == 0) & (exact != 0)).any())
    as_, a = stored(np.ldexp(rng.normal(size=(m, k)), 110), "bf16")
    grp = load(nc.linear_name(c))
    args = [as_, w, s.view(np.int8)] + [np.zeros(n, np.float32)] * bias + [np.zeros((m, n), np.float32 if out == "f32" else np.uint16)]
    check_linear(host([grp(*device_args(grp, args, gpu))], grp)[0], out, a, wv, np.zeros(n), k)


@pytest.mark.gpu
@pytest.mark.parametrize("c", ENDS, ids=nc.linear_name)
def test_product_of_the_largest_weights(gpu, c):
    """Up to the format's last scale byte the largest code is a finite weight,
    past it an infinite one."""
    m, n, k, fmt, bias, out = c
    note("largest weights " + nc.linear_name(c))
    top = {"e5m2": 0x7B, "e4m3": 0x7E, "e2m1": 7}[fmt]
    rng = np.random.default_rng(m + k)
    codes = np.zeros((n, k), np.uint8)
    codes[:, ::32] = top + (8 if fmt == "e2m1" else 128) * rng.integers(0, 2, (n, k // 32))
    w = bs.pack(codes, 1).view(np.int8) if fmt == "e2m1" else codes
    as_, a = stored(np.ldexp(rng.uniform(1, 2, (m, k)), -40), "bf16")
    grp = load(nc.linear_name(c))
    for byte in (LAST_FINITE[fmt], LAST_FINITE[fmt] + 1):
        s = np.full((n, k // 32), 127, np.uint8)
        s[:: 2, -1] = byte
        exact = bs.dequantize(w, s, fmt, 1)
        wv = bf16_of(exact)
        assert np.isfinite(wv).all() == (byte == LAST_FINITE[fmt]) and np.isfinite(exact).all()
        args = [as_, w, s.view(np.int8)] + [np.zeros(n, np.float32)] * bias + [np.zeros((m, n), np.float32 if out == "f32" else np.uint16)]
        got = host([grp(*device_args(grp, args, gpu))], grp)[0]
        far = np.isinf(wv).any(axis=1)
        check_linear(got[:, ~far], out, a, wv[~far], np.zeros((~far).sum()), k)
        want = np.broadcast_to(np.sign(exact[far, -32]) * np.inf, (m, far.sum()))
        assert np.array_equal(value(got[:, far], out), want)


@pytest.mark.gpu
def test_training_step_with_its_weight(gpu):
    """Norm with an 8-bit checkpoint, the weight to 4 bits, the product; back
    through the weight's values (a bf16 contraction) into the norm's gradient.
    On the device throughout; each stage is held to its own tolerance on what
    the stage before left."""
    import torch
    note("training step with its weight")
    m, k, n = nc.STEP
    c = (m, k, "bf16", "bf16", "e4m3", 2)
    xs, x, gs, gm, ts, bt, _, _ = norm_inputs(c)
    rng = np.random.default_rng(31)
    (ws, w), (dcs, dc) = stored(rng.normal(size=(n, k)) / np.sqrt(k), "bf16"), stored(rng.normal(0, 0.1, (m, n)), "bf16")
    bias = rng.normal(0, 0.1, n).astype(np.float32)
    bf = lambda a: to_dev(a, "bf16", gpu)  # noqa: E731
    new = lambda name: [torch.empty(p["shape"], dtype=hf.runtime.torch_dtype(p["elem"]), device=gpu)  # noqa: E731
                        for p in groups[name].meta["params"] if p["role"] != "in"]
    groups = {s: load("step_" + s) for s in ("norm", "codes", "linear", "values", "linear_grad", "norm_grad")}
    gamma, beta, dout = bf(gs), bf(ts), bf(dcs)
    y, mean, rstd, kept, kept_s = groups["norm"](bf(xs), gamma, beta, *new("norm"))
    codes, scales = groups["codes"](bf(ws), *new("codes"))
    out = groups["linear"](y, codes, scales, torch.from_numpy(bias).to(gpu), *new("linear"))
    wd = groups["values"](codes, scales, *new("values"))
    dy = groups["linear_grad"](dout, wd, *new("linear_grad"))
    grads = groups["norm_grad"](dy, kept, kept_s, gamma, mean, rstd, *new("norm_grad"))
    torch.cuda.synchronize()
    fwd = host((y, mean, rstd, kept, kept_s), groups["norm"])
    check_norm(c, fwd, x, gm, bt)
    wq, wsc = bs.quantize(w, "e2m1", 1)
    assert np.array_equal(scales.cpu().numpy().view(np.uint8), wsc)
    assert np.array_equal(codes.cpu().numpy().view(np.uint8), bs.pack(wq, 1))
    wv = bs.dequantize(bs.pack(wq, 1), wsc, "e2m1", 1)
    assert np.array_equal(value(to_host(wd, "bf16"), "bf16"), wv)  # (exact in bf16)
    yv, dyv = value(fwd[0], "bf16"), value(to_host(dy, "bf16"), "bf16")
    check_linear(to_host(out, "bf16"), "bf16", yv, wv, bias, k)
    check_linear(to_host(dy, "bf16"), "bf16", dc, wv.T, np.zeros(k), n)
    xv = bs.dequantize(fwd[3], fwd[4], "e4m3", 1)
    check_grad(c, host(grads, groups["norm_grad"]), xv, gm, dyv, fwd[1].astype(np.float64), fwd[2].astype(np.float64))
    # in 64 bits, the same step's loss sum(out dc) moves along dy as the product says
    step = rng.normal(size=(m, k)) * 2.0 ** -10
    moved = (((yv + step) @ wv.T) * dc).sum() - ((yv - step) @ wv.T * dc).sum()
    bound = (2.0 ** -8 * np.abs(dyv) + (2 * (40 + n / 32) + 2) * E24 * (np.abs(dc) @ np.abs(wv))) * np.abs(step)
    assert abs(moved / 2 - (dyv * step).sum()) <= bound.sum()


@pytest.mark.gpu
def test_two_threads_on_one_stream(gpu):
    """Calls of one group and of one program from two threads, both on the
    default stream: a launch's kernels follow each other."""
    import threading
    import torch
    note("two threads")
    c = (1300, 1000, "bf16", "f32", "e4m3", 2)
    grp, prog = load("lngrad_rt"), load("prog_norm_linear_mx")
    m, n, k = 20, 208, 384
    work = []
    for seed in (1, 2):
        xs, x, gs, gm, _, _, ds, dy = norm_inputs(c, seed=seed)
        arrays, _, _, _ = grad_args(c, xs, x, gs, ds)
        args = device_args(grp, arrays, gpu)
        rng = np.random.default_rng(seed)
        xs, gs, ts = (stored(a, "bf16")[0] for a in (rng.normal(size=(m, k)), rng.uniform(0.5, 1.5, k), rng.normal(0, 0.1, k)))
        _, _, w, s, _, _ = linear_inputs(8, n, k, "e2m1", seed=seed)
        pargs = [to_dev(v, p["elem"], gpu) for v, p in zip([xs, gs, ts, w, s], prog.meta["params"])]
        want = [t.clone() for t in grp(*args)] + [prog(*pargs)]
        torch.cuda.synchronize()
        work.append((args, pargs, want))
    start, bad = threading.Barrier(2), []

    def run(args, pargs, want):
        try:
            start.wait()
            for _ in range(300):
                got = [t.clone() for t in grp(*args)] + [prog(*pargs)]
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    bad.append(1)
        except Exception as e:  # (a thread's own would be lost)
            bad.append(e)
    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


class OnDevice:
    """Stands for a device tensor where nothing is launched."""

    def __init__(self, t):
        self.t, self.is_cuda = t, True

    def __getattr__(self, name):
        return getattr(self.t, name)


def test_refused_results_that_are_not_dense():
    """A result's buffer is written whole from its address on: a strided or an
    expanded view of the right shape is refused."""
    import torch
    grp = object.__new__(hf.runtime.Group)
    grp.meta = {"params": [], "results": [dict(tied=-1, elem="f32", shape=(4, 8))]}
    grp.func, grp._h = "f", None
    grp.info = hf.native.GroupInfo()
    prog = object.__new__(hf.runtime.Program)
    prog.meta, prog.name, prog._h = grp.meta, "p", None
    for t in (torch.zeros(8, 8)[::2], torch.zeros(8, 4).t(), torch.zeros(4, 1).expand(4, 8), torch.zeros(4, 16)[:, 8:]):
        assert tuple(t.shape) == (4, 8)
        with pytest.raises(ValueError, match="result 0 of @f: expected contiguous"):
            grp._bind((), [OnDevice(t)], 1, None, False)
        with pytest.raises(ValueError, match="result 0 of @p: expected contiguous"):
            prog(results=[OnDevice(t)], stream=1)


@pytest.mark.parametrize("noalloc", [False, True])
def test_a_packed_launch_keeps_its_group(noalloc):
    """hf.load(...).launcher(...): the group goes when the launch does."""
    import gc
    import weakref
    import torch
    grp = object.__new__(hf.runtime.Group)
    grp.meta = {"params": [], "results": [dict(tied=-1, elem="f32", shape=(4,))]}
    grp.func, grp._h, grp.info = "f", None, hf.native.GroupInfo()
    packed, alive = grp.launcher(results=[OnDevice(torch.zeros(4))], stream=1, noalloc=noalloc), weakref.ref(grp)
    del grp
    gc.collect()
    assert alive() is not None
    del packed
    gc.collect()
    assert alive() is None


@pytest.mark.gpu
def test_a_packed_launch_of_a_group_that_nobody_holds(gpu):
    import gc
    import torch
    note("packed launch alone")
    x = torch.randn(9, 96, device=gpu).bfloat16()
    g, b = torch.rand(96, device=gpu).bfloat16(), torch.randn(96, device=gpu).bfloat16()
    want = load("ln_untied")(x, g, b)
    packed = load("ln_untied").launcher(x, g, b)
    gc.collect()
    got = packed()
    assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(got, want))
