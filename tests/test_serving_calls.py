"""Calls of the serving ops beside the ordinary ones: programs, captured and
replayed graphs, several streams, results in buffers of their own, empty
batches, buffers off 16 bytes, strided descriptors, caches past 2 GiB, shared
blocks, other scales.  Each is compared with test_serving's definitions or bit
by bit with the plain call."""
import ctypes

import numpy as np
import pytest

import hfusion_mi355x as hf
import group_catalog as cat
import serving_catalog as sc
from helpers import to_dev, to_host
from hfusion_mi355x import native
from oracle import serving as sv
from test_norm_mx import note, stored, value
from test_serving import attend_case, batch, check_attention, check_codes, load, norm_case, store_as


def same(a, b):
    import torch
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def attend_args(c, case, gpu):
    """Device arguments of one of attend_case's batches."""
    seq, pos, table, cache, qs, qv = case
    elems = [c[7], "i8", "i8", "i8", "i8", "i32", "i32", "i32", c[7]]
    arrays = [qs, cache[0], cache[1].view(np.int8), cache[2], cache[3].view(np.int8), seq, pos, table, np.zeros_like(qs)]
    t = hf.runtime.torch_dtype("f8E4M3FN" if c[8] == "e4m3" else "f8E5M2")
    dev = [to_dev(a, e, gpu) for a, e in zip(arrays, elems)]
    return [d.view(t) if i in (1, 3) else d for i, d in enumerate(dev)]


# ---------------------------------------------------------------- no GPU
def test_manifests():
    """The kernels by row count: groups of tokens in pieces, then a prompt's
    rows in pieces, then whole; each behind its own pre kernel alone."""
    def alts(name):
        text = open(hf.compile(cat.get(name), options="dyn=runtime").manifest).read()
        return [ln.split() for ln in text.splitlines() if ln.startswith("alt ")], text
    a, text = alts("pagedattn_usual_rt")
    assert [(x[1].rsplit("_", 1)[1], x[2], x[6:]) for x in a] == [("parts", "64", ["pre", "0"]), ("pieces", "2048", ["pre", "1"]), ("attention", str(1 << 31), ["pre", "2"])]
    # (prompts in whole units leave a word a tile)
    assert text.count("pre_rows 1 8\n") == text.count("pre_rows 32 8\n") == text.count("pre_workspace 16384\n") == 1 and text.count("pre_workspace ") == 3
    a, text = alts("pagedattn_group4_rt")  # a short context: nothing in pieces
    assert [x[1].rsplit("_", 1)[1] for x in a] == ["units", "attention"] and "workspace 16384 0" in text
    a, _ = alts("pagedattn_many_rt")  # more groups of tokens than are dealt out
    assert [(x[1].rsplit("_", 1)[1], int(x[2])) for x in a][:2] == [("parts", 1024), ("units", 1200)]
    a, _ = alts("appendkv_usual_rt")
    assert [(int(x[2]), int(x[3])) for x in a] == [(256, 1), (1024, 4)]
    art = hf.compile(cat.get("prog_decoder_attention"))
    assert [b["kind"] for b in art.blocks] == ["RMS_NORM", "SINGLE_CUBE", "APPEND_KV", "PAGED_ATTENTION"]


# ---------------------------------------------------------------- programs
@pytest.mark.gpu
def test_program_equals_its_parts(gpu):
    """The un-fused layer as one program, and its operators called one by one:
    the same bits in the residual sum, the cache and the result."""
    import torch
    note("decoder attention program")
    P = sc.PROGRAM
    prog = load("prog_decoder_attention")
    parts = [load(f"part_{n}") for n in ("norm", "product", "append", "attend")]
    gen = torch.Generator(device=gpu).manual_seed(5)
    rows, cols, slots, room, block = P["rows"], P["cols"], P["slots"], P["room"], P["block"]

    def random(p):
        t = hf.runtime.torch_dtype(p["elem"])
        if p["elem"] in ("bf16", "f32"):
            return torch.randn(p["shape"], generator=gen, device=gpu).to(t)
        if p["elem"] == "i8":
            return torch.randint(118, 122, p["shape"], generator=gen, device=gpu, dtype=torch.int8)
        return torch.randint(0, 0x70, p["shape"], generator=gen, device=gpu, dtype=torch.uint8).view(t)
    params = prog.meta["params"]
    args = [random(p) if p["elem"] != "i32" else None for p in params]
    seq, pos = batch([(1, room - 3, 3), (0, 40, 9), (3, 0, 5)], 3, slots)
    assert len(seq) == rows
    table = np.arange(slots * (room // block), dtype=np.int32)[::-1].reshape(slots, -1) % P["blocks"]
    for i, a in ((6, seq), (7, pos), (8, table)):
        args[i] = torch.from_numpy(a.copy()).to(gpu)
    x, res, gamma, w, sw, rot, sq, ps, tb, total = args[:10]
    cache, out = args[10:14], args[14]
    mine = [t.clone() for t in cache]
    for _ in range(2):  # (the second one over what the first one appended)
        got = prog(*args)
        codes = torch.empty((rows, cols), dtype=torch.float8_e4m3fn, device=gpu)
        scales = torch.empty((rows, cols // 32), dtype=torch.int8, device=gpu)
        s2, codes, scales = parts[0](x, res, gamma, torch.empty_like(total), codes, scales)
        qkv = parts[1](codes, w, scales, sw)
        q = torch.zeros_like(out)
        parts[2](qkv, rot, sq, ps, tb, q, *mine)
        want = torch.zeros_like(out)
        parts[3](q, *mine, sq, ps, tb, want)
        torch.cuda.synchronize()
        assert same(got[1], s2) and all(same(a, b) for a, b in zip(cache, mine)) and same(got[2], cache[0])
        ok = torch.from_numpy(np.isin(np.arange(rows), np.arange(rows - 3))).to(gpu)
        assert same(got[0][ok], want[ok]) and want[ok].float().abs().sum() > 0
        x.copy_(torch.randn(x.shape, generator=gen, device=gpu))


# ---------------------------------------------------------------- graphs and streams
@pytest.mark.gpu
@pytest.mark.parametrize("name", ["far", "far_f16", "usual"])
def test_graphs_of_one_group(gpu, name):
    """Two graphs of one group, of rows in pieces of either kind, replayed in
    turn over new queries with eager calls between: each replay is the eager
    result of its inputs, to the bit."""
    import torch
    note("graphs " + name)
    c = sc.ATTEND[name]
    rng = np.random.default_rng(9)
    grp = load(f"pagedattn_{name}_rt")
    far = min(c[5], 5000)
    cases = [attend_args(c, attend_case(rng, c, parts, pad), gpu) for parts, pad in (([(1, far - 1, 1), (0, 700, 1), (2, 64, 2)], 2),
                                                                                    ([(0, far - 100, 100), (2, 0, 33)], 1))]
    graphs = []
    for a in cases:
        grp(*a)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            grp(*a)
        graphs.append(graph)
    for k in range(3):
        for a in cases:
            a[0].copy_(torch.randn(a[0].shape, device=gpu).to(a[0].dtype))
            a[-1].zero_()
        graphs[0].replay(), graphs[1].replay()
        got = [a[-1].clone() for a in cases]
        for a, g in zip(cases, got):
            a[-1].zero_()
            grp(*a)
            torch.cuda.synchronize()
            assert same(a[-1], g) and g.float().abs().sum() > 0


@pytest.mark.gpu
def test_two_streams(gpu):
    """Launches of one group on two streams at once, each with parts of its own."""
    import torch
    note("two streams")
    c = sc.ATTEND["far"]
    rng = np.random.default_rng(10)
    grp = load("pagedattn_far_rt")
    cases = [attend_args(c, attend_case(rng, c, parts, 0), gpu) for parts in ([(1, 4999, 1), (0, 3000, 1)], [(0, 4000, 2), (2, 4500, 1)], [(2, 4000, 90)])]
    want = []
    for a in cases:
        grp(*a)
        torch.cuda.synchronize()
        want.append(a[-1].clone())
    streams = [torch.cuda.Stream() for _ in cases]
    for a in cases:
        a[-1].zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for a, s in zip(cases, streams):
            with torch.cuda.stream(s):
                grp(*a)
    torch.cuda.synchronize()
    assert all(same(a[-1], w) for a, w in zip(cases, want))


# ---------------------------------------------------------------- buffers
@pytest.mark.gpu
@pytest.mark.parametrize("name", ["rmsnorm_i8_rt", "rmsnorm_e4m3_rt", "appendkv_usual_rt", "pagedattn_usual_rt", "pagedattn_group4_rt"])
def test_empty_batch(gpu, name):
    """No rows: the call returns its destinations, and nothing is written."""
    import torch
    note("empty " + name)
    grp = load(name)
    args = [torch.full([0 if d == -1 else d for d in p["shape"]], 3, dtype=torch.float32, device=gpu).to(hf.runtime.torch_dtype(p["elem"]))
            for p in grp.meta["params"]]
    before = [t.clone() for t in args]
    out = grp(*args)
    torch.cuda.synchronize()
    outs = out if isinstance(out, tuple) else (out,)
    assert all(o is args[r["tied"]] for o, r in zip(outs, grp.meta["results"]))
    assert all(same(a, b) for a, b in zip(args, before) if a.numel())


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["group4", "far"])
def test_buffers_off_16_bytes(gpu, name):
    """Every buffer one element behind a 16-byte boundary: the same bits."""
    import torch
    note("off 16 bytes " + name)

    def moved(t):
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype if t.element_size() > 1 else torch.uint8, device=gpu)
        v = flat[1:]
        v.copy_(t.reshape(-1) if t.element_size() > 1 else t.reshape(-1).view(torch.uint8))
        return v.view(t.dtype).view(t.shape)
    c = sc.ATTEND[name]
    rng = np.random.default_rng(11)
    grp = load(f"pagedattn_{name}_rt")
    for parts in ([(1, min(c[5], 5000) - 1, 1), (0, 63, 2)], [(2, min(c[5], 5000) - 90, 90)]):
        a = attend_args(c, attend_case(rng, c, parts, 0), gpu)
        b = [moved(t) for t in a]
        grp(*a), grp(*b)
        torch.cuda.synchronize()
        assert b[1].data_ptr() % 16 == 1 and same(a[-1], b[-1]) and a[-1].float().abs().sum() > 0
    if name != "group4":
        return
    grp = load("appendkv_group4_rt")
    hq, hk, d, block, slots, room, blocks, el, fmt = sc.APPEND["group4"]
    seq, pos = batch([(1, 5, 60), (0, 15, 2)], 0, slots)
    gen = torch.Generator(device=gpu).manual_seed(3)
    table = torch.arange(slots * (room // block), dtype=torch.int32, device=gpu).reshape(slots, -1) % blocks
    a = [torch.randn((62, (hq + 2 * hk) * d), generator=gen, device=gpu).bfloat16(), torch.randn((room, sc.TURN["group4"][0]), generator=gen, device=gpu),
         torch.from_numpy(seq).to(gpu), torch.from_numpy(pos).to(gpu), table]
    a += [torch.zeros([62 if n == -1 else n for n in p["shape"]], dtype=hf.runtime.torch_dtype(p["elem"]), device=gpu) for p in grp.meta["params"][5:]]
    b = [moved(t) for t in a]
    grp(*a), grp(*b)
    torch.cuda.synchronize()
    assert all(same(x, y) for x, y in zip(a, b)) and a[6].view(torch.uint8).any()


@pytest.mark.gpu
def test_results_of_their_own(gpu):
    """A result that the call makes, and one that lies over an operand."""
    import torch
    note("untied results")
    c = sc.ATTEND["usual"]
    rng = np.random.default_rng(12)
    case = attend_case(rng, c, [(1, 600, 70)], 0)
    grp, tied = load("pagedattn_untied"), load("pagedattn_usual_rt")
    a = attend_args(c, case, gpu)
    out = grp(*a[:-1])
    tied(*a)
    torch.cuda.synchronize()
    assert same(out, a[-1])
    with pytest.raises(RuntimeError, match="is written and overlaps"):
        grp(*a[:-1], results=[a[0]])
    grp = load("rmsnorm_untied")
    cn = (33, 512, "bf16", "bf16", "i8", True)
    args, x, rv, gm = norm_case(cn, rng)
    dev = [to_dev(v, p["elem"], gpu) for v, p in zip(args[:3], grp.meta["params"])]
    got = grp(*dev)
    check_codes(cn, [to_host(t, r["elem"]) for t, r in zip(got, grp.meta["results"])], x, rv, gm)
    codes, scale = torch.empty_like(got[1]), torch.empty_like(got[2])
    got = grp(*dev, results=[dev[1], codes, scale])  # over the residual itself
    check_codes(cn, [to_host(t, r["elem"]) for t, r in zip(got, grp.meta["results"])], x, rv, gm)
    with pytest.raises(RuntimeError, match="is written and overlaps"):
        grp(*dev, results=[dev[0], codes, scale])


@pytest.mark.gpu
def test_append_to_a_strided_cache(gpu):
    """A cache that is every second head of a larger one, through memref
    descriptors: what the rows do not name stays, in it and between its heads."""
    import torch
    note("strided cache")
    hq, hk, d, block, slots, room, blocks, el, fmt = sc.APPEND["group4"]
    grp = load("appendkv_group4_rt")
    gen = torch.Generator(device=gpu).manual_seed(6)
    seq, pos = batch([(1, 5, 20), (0, 31, 2)], 2, slots)
    table = torch.arange(slots * (room // block), dtype=torch.int32, device=gpu).reshape(slots, -1) % blocks
    a = [torch.randn((24, (hq + 2 * hk) * d), generator=gen, device=gpu).bfloat16(), torch.randn((room, sc.TURN["group4"][0]), generator=gen, device=gpu),
         torch.from_numpy(seq).to(gpu), torch.from_numpy(pos).to(gpu), table]
    params = grp.meta["params"]
    byte = lambda shape: torch.randint(0, 0x70, shape, generator=gen, device=gpu, dtype=torch.uint8)  # noqa: E731
    wide = [byte((s[0], 2 * s[1], *s[2:])) for s in (p["shape"] for p in params[6:])]
    dense = [w[:, ::2].contiguous().view(hf.runtime.torch_dtype(p["elem"])) for w, p in zip(wide, params[6:])]
    q1, q2 = (torch.full((24, hq, d), 5.0, device=gpu).bfloat16() for _ in range(2))
    between = [w[:, 1::2].clone() for w in wide]
    grp(*a, q1, *dense)
    views = [w[:, ::2] for w in wide]
    descs = [native.memref_descriptor(t.data_ptr(), list(t.shape), strides=list(t.stride())) for t in a + [q2] + views]
    ptrs = (ctypes.c_void_p * len(descs))(*[ctypes.addressof(x) for x in descs])
    native.check(native.hfr().hfr_group_launch_memref(grp._h, ptrs, len(descs), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert same(q1, q2) and (q1[-2:] == 5).all()
    assert all(same(v, x) for v, x in zip(views, dense)) and all(torch.equal(w[:, 1::2], b) for w, b in zip(wide, between))


@pytest.mark.gpu
def test_cache_past_2_gib(gpu):
    """Blocks behind byte 2^31 of the keys and of the values: the same bits as
    in a small cache."""
    import torch
    note("large cache")
    big, small, append, attend = (load(n) for n in ("appendkv_big", "appendkv_small", "pagedattn_small", "pagedattn_big"))
    B = sc.BIG
    rows, slots, room, block, few = B["rows"], B["slots"], B["room"], B["block"], B["few"]
    gen = torch.Generator(device=gpu).manual_seed(8)
    seq, pos = batch([(0, 0, rows - 3), (1, 0, 3)], 0, slots)
    n = room // block
    table = np.arange(slots * n, dtype=np.int32).reshape(slots, n)
    assert table.max() < few and (B["blocks"] - few) * B["kv_heads"] * block * B["dim"] > 1 << 31
    qkv = torch.randn((rows, (B["heads"] + 2 * B["kv_heads"]) * B["dim"]), generator=gen, device=gpu).bfloat16()
    rot = torch.randn((room, B["dim"]), generator=gen, device=gpu)
    sq, ps = torch.from_numpy(seq).to(gpu), torch.from_numpy(pos).to(gpu)
    outs = []
    for app, att, shift in ((small, append, 0), (big, attend, B["blocks"] - few)):
        tb = torch.from_numpy(table + shift).to(gpu)
        cache = [torch.zeros(p["shape"], dtype=hf.runtime.torch_dtype(p["elem"]), device=gpu) for p in app.meta["params"][6:]]
        q = torch.zeros((rows, B["heads"], B["dim"]), dtype=torch.bfloat16, device=gpu)
        out = torch.zeros_like(q)
        app(qkv, rot, sq, ps, tb, q, *cache)
        att(q, *cache, sq, ps, tb, out)
        torch.cuda.synchronize()
        outs.append([q, out] + [t.view(torch.uint8)[shift:shift + few].clone() for t in cache])
        assert not cache[1][:shift].any()
        del cache
    assert all(same(a, b) for a, b in zip(*outs)) and outs[0][1].float().abs().sum() > 0


# ---------------------------------------------------------------- values
@pytest.mark.gpu
@pytest.mark.parametrize("name,scale", [("negative", -0.2), ("zero", 0.0), ("large", 3.0)])
def test_other_scales(gpu, name, scale):
    """A negative scale, none (a mean of the values), and one that leaves a few
    positions all of the weight."""
    import torch
    c = sc.ATTEND["group4"]
    rng = np.random.default_rng(13)
    grp = load(f"pagedattn_{name}_rt")
    for parts in ([(1, 150, 1), (0, 63, 2)], [(2, 60, 90), (0, 0, 5)]):
        note(f"scale {scale} {parts}")
        case = attend_case(rng, c, parts, 1, holes=True)
        seq, pos, table, cache, qs, qv = case
        out = grp(*attend_args(c, case, gpu))
        torch.cuda.synchronize()
        check_attention(c, to_host(out, c[7]), qv, cache, seq, pos, table, np.zeros(qv.shape), float(np.float32(scale)))


@pytest.mark.gpu
def test_shared_blocks(gpu):
    """Sequences that begin with the same blocks, and one that reads a block twice."""
    import torch
    note("shared blocks")
    c = sc.ATTEND["far_window"][:9] + (1500,)
    rng = np.random.default_rng(14)
    grp = load("pagedattn_far_window_rt")
    seq, pos, table, cache, qs, qv = attend_case(rng, c, [(0, 2000, 2), (1, 1900, 1), (2, 1800, 70)], 0)
    table[1, :100] = table[0, :100]
    table[2, 60] = table[2, 61] = table[2, 62]
    out = grp(*attend_args(c, (seq, pos, table, cache, qs, qv), gpu))
    torch.cuda.synchronize()
    check_attention(c, to_host(out, c[7]), qv, cache, seq, pos, table, np.zeros(qv.shape))


@pytest.mark.gpu
def test_append_twice(gpu):
    """The same rows appended again change nothing, and a row overwritten alone
    keeps its block's scale and the rows about it."""
    import torch
    note("append twice")
    hq, hk, d, block, slots, room, blocks, el, fmt = sc.APPEND["usual"]
    grp = load("appendkv_usual_rt")
    rng = np.random.default_rng(15)
    seq, pos = batch([(3, 60, 64), (1, 5, 3)], 0, slots)
    xs, x = stored(rng.normal(size=(67, (hq + 2 * hk) * d)), el)
    turn = rng.normal(size=(room, d)).astype(np.float32)
    table = rng.permutation(blocks)[:slots * 2].reshape(slots, 2).astype(np.int32)
    table = np.concatenate([table, np.full((slots, room // block - 2), -1, np.int32)], axis=1)
    cache = [torch.zeros(p["shape"], dtype=hf.runtime.torch_dtype(p["elem"]), device=gpu) for p in grp.meta["params"][6:]]
    dev = lambda a, e: to_dev(a, e, gpu)  # noqa: E731
    q = torch.zeros((67, hq, d), dtype=torch.bfloat16, device=gpu)
    args = [dev(xs, el), dev(turn, "f32"), dev(seq, "i32"), dev(pos, "i32"), dev(table, "i32"), q]
    grp(*args, *cache)
    torch.cuda.synchronize()
    first = [t.clone() for t in cache]
    grp(*args, *cache)
    torch.cuda.synchronize()
    assert all(same(a, b) for a, b in zip(cache, first))
    host = [t.view(torch.uint8).cpu().numpy() for t in cache]
    one, at = np.array([3], np.int32), np.array([100], np.int32)
    y, yv = stored(rng.normal(size=(1, (hq + 2 * hk) * d)) * 0.25, el)
    want = sv.append_kv(yv.astype(np.float32), turn, one, at, table, np.zeros((1, hq, d), np.uint16), *host, fmt, 0, store_as(el))
    grp(dev(y, el), args[1], dev(one, "i32"), dev(at, "i32"), args[4], q[:1].contiguous(), *cache)
    torch.cuda.synchronize()
    for t, w in zip(cache, want[1:]):
        assert np.array_equal(t.view(torch.uint8).cpu().numpy(), w)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["group4", "far", "usual", "many"])
def test_batches_of_padding(gpu, name):
    """Rows that are all padding leave everything as it was, and the call behind
    them has its rows."""
    import torch
    note("padding alone " + name)
    c = sc.ATTEND[name]
    grp = load(f"pagedattn_{name}_rt")
    for rows in (1, 9, 300, 1300):
        case = attend_case(np.random.default_rng(rows), c, [(1, 7, 1)], rows)
        args = attend_args(c, case, gpu)
        pad = [t[1:].clone() if i in (0, 5, 6) else t.clone() for i, t in enumerate(args[:-1])] + [torch.full_like(args[-1][1:], 3.0)]
        grp(*pad)
        out = grp(*args)
        torch.cuda.synchronize()
        assert (pad[-1] == 3.0).all()
        check_attention(c, to_host(out, c[7]), case[5], case[3], *case[:3], np.zeros(case[5].shape))


@pytest.mark.gpu
@pytest.mark.parametrize("own", [False, True], ids=["one stream", "streams"])
def test_two_threads(gpu, own):
    """Calls of one handle from two threads, on one stream or on one each."""
    import threading

    import torch
    note(f"two threads {own}")
    c = sc.ATTEND["far"]
    grp = load("pagedattn_far_rt")
    rng = np.random.default_rng(21)
    args = [attend_args(c, attend_case(rng, c, parts, 2), gpu) for parts in ([(0, 4990, 3), (2, 3000, 1)], [(1, 4000, 150)])]
    want = []
    for a in args:
        want.append(grp(*a).clone())
        a[-1].zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    bad = []

    def calls(i):
        try:
            with torch.cuda.stream(streams[i if own else 0]):
                for _ in range(20):
                    grp(*args[i])
                streams[i if own else 0].synchronize()
        except Exception as e:  # noqa: BLE001
            bad.append(e)
    threads = [threading.Thread(target=calls, args=(i,)) for i in range(len(args))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not bad and all(same(a[-1], w) for a, w in zip(args, want))
