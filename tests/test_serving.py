"""The serving ops, a residual stream's norm into 8-bit codes, appending to the
paged 8-bit cache and the attention that reads it: refusals and the CPU
restatement (no GPU), then every prebuilt group of serving_catalog against the
definitions.

Norm and append are exact, bit by bit: their roundings are part of their
definition.  The attention's tolerance counts, per value, with N positions
seen, D channels and P = sum p |v|:
  scores: D + 8 f32 roundings of at most sum |q k| scale, in the numerator and
    the denominator                        2 (D + 8) 2^-23 sum |q k| P
  exp2 of the hardware (1 ulp) and its argument's rounding       2^-20 P
  N f32 additions in both sums             2 N 2^-23 P
  p to 16 bits (half a step)               2^-8 P, of f16 queries 2^-11 P and
                                           2^-25 |v| for each position
  the result's own rounding (half a step)"""
import numpy as np
import pytest

import hfusion_mi355x as hf
import group_catalog as cat
import serving_catalog as sc
from helpers import run_gpu, to_dev, to_host
from hfusion_mi355x import groups as g
from launch_checks import Checked
from oracle import blockscaled as bs
from oracle import interp
from oracle import serving as sv
from test_norm_mx import TINY, U, edge_values, note, refuse, stored, value


def load(name):
    return hf.compile(cat.get(name), options=cat.options(name), require_cached=True).load()


def store_as(elem):
    def store(a):
        s = interp.from_f32(np.asarray(a, np.float32), elem)
        return s, interp.to_f32(interp.T(s, elem)).astype(np.float32)
    return store


# ---------------------------------------------------------------- no GPU
def test_refused_rms_norm():
    ir = g.rms_norm(8, 64)
    refuse(ir.replace("eps = 9.99999999999999955e-07 : f64", "other = 1 : i32"), "missing eps")
    refuse(ir.replace("9.99999999999999955e-07", "-1.0"), "eps that is negative")
    refuse(ir.replace("tensor<64xbf16>", "tensor<32xbf16>"), "one element per column")
    refuse(ir.replace("tensor<64xbf16>", "tensor<64xf16>"), "another type than f32 or the rows'")
    refuse(ir.replace("tensor<8xf32>", "tensor<8xbf16>"), "scales of i8 codes")
    refuse(ir.replace("<8x64xi8>", "<8x32xi8>"), "codes")
    refuse(ir.replace("%residual: tensor<8x64xbf16>", "%residual: tensor<8x64xf16>").replace("ins(%x, %residual, %gamma : tensor<8x64xbf16>, tensor<8x64xbf16>",
                                                                                            "ins(%x, %residual, %gamma : tensor<8x64xbf16>, tensor<8x64xf16>"), "beside")
    refuse(ir.replace("xbf16", "xi32"), "values of type")
    refuse(g.rms_norm(8, 16385), "more than 16384")
    refuse(ir.replace("outs(%sum,", "outs(%residual,"), "also a destination")
    mx = g.rms_norm(8, 64, out="e4m3")
    refuse(mx.replace("format = 2", "format = 3"), "4-bit codes")
    refuse(mx.replace("format = 2", "format = 9"), "format other")
    refuse(mx.replace("<8x2xui8>", "<8x3xui8>"), "scales shape")
    refuse(mx.replace("f8E4M3FN", "f8E5M2"), "codes of another type")
    with pytest.raises(ValueError):
        g.rms_norm(8, 64, out="e2m1")


def test_refused_append():
    ir = sc.append("group4", 9)
    refuse(ir.replace("format = 2 : i32, ", ""), "missing format")
    refuse(ir.replace("format = 2", "format = 3"), "4-bit cache")
    refuse(ir.replace("format = 2", "format = 1"), "codes of another type")
    refuse(ir.replace("pairs = 0", "pairs = 2"), "pairs other")
    refuse(ir.replace("<160x64xf32>", "<160x40xf32>"), "multiple of 16")
    refuse(ir.replace("<160x64xf32>", "<160x96xf32>"), "multiple of 16 up to the head")
    refuse(ir.replace("<160x64xf32>", "<160x64xbf16>"), "not f32")
    refuse(ir.replace("<9x768xbf16>", "<9x704xbf16>"), "rows tensor")
    refuse(ir.replace("<9x768xbf16>", "<9x768xf16>"), "rows tensor")
    refuse(ir.replace("tensor<9xi32>", "tensor<8xi32>"), "one per row")
    refuse(ir.replace("tensor<9xi32>", "tensor<9xi64>"), "must be i32")
    refuse(ir.replace("<5x10xi32>", "<5x10xi64>"), "not i32")
    refuse(ir.replace("<40x2xui8>", "<40x1xui8>"), "scales shape")
    refuse(ir.replace("<40x2x64x16x", "<40x2x16x64x"), "codes shape")
    refuse(ir.replace("x16x64x", "x24x64x").replace("x64x16x", "x64x24x"), "16, 32, 64 or 128")
    refuse(ir.replace("9x8x64x", "9x7x64x"), "no multiple of the cache's heads|rows tensor")
    refuse(ir.replace("outs(%q, %k, %ks", "outs(%q, %k, %vs"), "one destination")
    # a cache of the group's own would lose the other blocks
    from norm_mx_catalog import untied
    refuse(untied(ir), "not a group argument")
    for bad in (dict(fmt="e2m1"), dict(heads=3), dict(dim=48), dict(block=24)):
        with pytest.raises(ValueError):
            g.append_kv(**{**dict(rows=4, heads=4, kv_heads=2, dim=64, slots=1, room=64, blocks=4), **bad})


def test_refused_attention():
    ir = sc.attend("window", 9)
    refuse(ir.replace("scale = 1.250000000e-01 : f32, ", ""), "missing scale")
    refuse(ir.replace("scale = 1.250000000e-01", "scale = 1.0e39"), "scale")
    refuse(ir.replace("window = 50", "window = -1"), "negative window")
    refuse(ir.replace("format = 2 : i32, ", ""), "missing format")
    refuse(ir.replace("x8x64xbf16", "x8x64xf32"), "another type than bf16 or f16")
    refuse(ir.replace("%out: tensor<9x8x64xbf16>", "%out: tensor<9x8x64xf16>"), "destination|beside")
    refuse(ir.replace("<90x2xui8>", "<90x2xi32>"), "e8m0")
    refuse(ir.replace("outs(%out :", "outs(%q :"), "also a destination")
    rt = g.with_dynamic_rows(sc.attend("usual", 7919), 7919)
    refuse(rt.replace("%pos: tensor<?xi32>", "%pos: tensor<70xi32>").replace("tensor<?xi32>, tensor<?xi32>, tensor<6x", "tensor<?xi32>, tensor<70xi32>, tensor<6x"),
           "one per row", "dyn=runtime")


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return tmp_path_factory.mktemp("checks")


def test_destinations_apart(folder):
    """The norm's sum may be the residual's buffer and nothing else; the cache
    and the queries overlap nothing."""
    c = Checked(sc.norm(130, 1000, "bf16", "bf16", "e4m3", True), folder)
    names = ["x", "residual", "gamma", "sum", "q", "s"]
    assert len(c.at) == len(names) and c.why() == ""
    assert c.why({3: c.at[1]}) == ""
    for i, j, off in ((3, 1, 16), (3, 0, 0), (3, 2, 0), (4, 0, 0), (4, 1, 0), (5, 4, 8), (4, 3, 2)):
        assert "is written and overlaps" in c.why({i: c.at[j] + off}), (names[i], names[j])
    c = Checked(sc.append("group4", 33), folder)
    assert c.why() == ""
    for i in range(5, 10):
        for j in range(10):
            if i != j:
                assert "is written and overlaps" in c.why({i: c.at[j]})
    c = Checked(g.with_dynamic_rows(sc.attend("group4", 7919), 7919), folder, options="dyn=runtime", rows=12)
    assert c.why() == ""
    for j in range(8):
        assert "is written and overlaps" in c.why({8: c.at[j]})
    art = hf.compile(sc.append("group4", 33))
    assert [p["role"] for p in art.blocks[0]["params"]] == ["in"] * 5 + ["inout"] * 5


def test_most_rows(folder):
    """More rows than a launch has workgroups for are refused, not cut short:
    16 rows (five workgroups) and 64 rows (two heads) a tile, 2^24 workgroups of
    256 threads less one."""
    refuse(g.append_kv(1 << 27, 8, 2, 64, 5, 160, 40), "more rows than a launch takes")
    refuse(g.paged_attention(1 << 29, 4, 2, 64, 5, 160, 40), "more rows than a launch takes")
    refuse(g.paged_attention(1 << 33, 4, 2, 64, 5, 160, 40), "more rows than a launch takes")
    for ir, most in ((g.append_kv(7919, 8, 2, 64, 5, 160, 40), (2 ** 24 - 1) // 5 * 16), (g.paged_attention(7919, 4, 2, 64, 5, 160, 40), (2 ** 24 - 1) // 2 * 64)):
        c = Checked(g.with_dynamic_rows(ir, 7919), folder, options="dyn=runtime", rows=12)
        assert c.why() == ""
        c.rows = most + 1
        assert f"takes at most {most} rows a launch, got {most + 1}" in c.why()


def test_oracle_append_in_parts():
    """Tokens appended one by one leave the scales of one append of all, and
    codes within what the roundings on the way cost: a code is rounded at most
    once more for each time its scale grew."""
    rng = np.random.default_rng(3)
    hq, hk, d, block, slots, room, blocks, _, fmt = sc.APPEND["group4"]
    store = store_as("bf16")
    n = 40
    qkv = store(rng.normal(size=(n, (hq + 2 * hk) * d)) * 2.0 ** np.arange(n)[:, None] ** 0.5)[1]
    rot = rng.normal(size=(room, d)).astype(np.float32)
    table = rng.permutation(blocks)[:slots * (room // block) // 2].reshape(slots, -1)
    seq, pos = np.full(n, 2), np.arange(3, 3 + n)
    state = [np.zeros((n, hq, d), np.uint16), np.zeros((blocks, hk, block, d), np.uint8), np.zeros((blocks, hk), np.uint8),
             np.zeros((blocks, hk, d, block), np.uint8), np.zeros((blocks, hk), np.uint8)]
    whole = sv.append_kv(qkv, rot, seq, pos, table, *state, fmt, 0, store)
    for t in range(n):
        q = state[0][t:t + 1]
        state = [state[0]] + list(sv.append_kv(qkv[t:t + 1], rot, seq[t:t + 1], pos[t:t + 1], table, q, *state[1:], fmt, 0, store)[1:])
    values = bs.code_values(fmt)
    for a, b in ((1, 2), (3, 4)):
        assert np.array_equal(whole[b], state[b]) and len(np.unique(whole[b])) > 3
        assert np.abs(values[whole[a]] - values[state[a]]).max() <= 2 * 2.0 ** -4 * 16  # (below 16 a step is at most 1)
    # the scale holds what it has to, and half of it would not
    for amax in (448.0, 449.0, 1.75, 1.76, 2.0 ** -130, 3e38, 0.0):
        b = sv.scale_byte(amax, "e4m3")
        assert 448.0 * 2.0 ** (b - 127) >= amax and (b == 0 or 448.0 * 2.0 ** (b - 128) < amax)


def test_oracle_attention_by_hand():
    """Two heads over one kv head, three positions of which the window leaves two."""
    k = bs.encode(np.array([1.0, -2.0, 0.5])[None, None, :, None] * np.ones((1, 1, 3, 32)), "e4m3")
    k = np.concatenate([k, np.full((1, 1, 13, 32), 0x7F, np.uint8)], axis=2)
    v = np.ascontiguousarray(np.swapaxes(np.concatenate([bs.encode(np.array([4.0, 8.0, 16.0])[:, None] * np.ones((3, 32)), "e4m3"),
                                                         np.full((13, 32), 0x7F, np.uint8)])[None, None], 2, 3))
    one = np.full((1, 1), 127, np.uint8)
    q = np.stack([np.full(32, 0.125), np.full(32, -0.25)])[None]
    for window, seen in ((0, [0, 1, 2]), (2, [1, 2])):
        out, size, _ = sv.paged_attention(q, k, one, v, one, [0], [2], np.zeros((1, 1), int), np.zeros((1, 2, 32)), "e4m3", 0.5, window)
        for h, a in enumerate((0.125, -0.25)):
            x = np.array([1.0, -2.0, 0.5])[seen] * a * 32 * 0.5
            p = np.exp(x) / np.exp(x).sum()
            assert np.allclose(out[0, h], (p * np.array([4.0, 8.0, 16.0])[seen]).sum(), rtol=1e-12) and np.allclose(size, np.abs(out))


# ---------------------------------------------------------------- norm
def norm_case(c, rng, edges=False):
    r, n, el, p, out, res = c
    make = (lambda: edge_values(rng, r, n, el)) if edges else (lambda: rng.normal(size=(r, n)) * rng.uniform(0.1, 30, (r, 1)))
    xs, x = stored(make(), el)
    rs, rv = stored(make(), el)
    gs, gm = stored(rng.uniform(0.5, 1.5, n), p)
    codes = np.zeros((r, n), np.int8 if out == "i8" else np.uint8)
    scales = np.zeros(r, np.float32) if out == "i8" else np.zeros((r, (n + 31) // 32), np.int8)
    args = [xs] + ([rs] if res else []) + [gs] + ([np.zeros_like(xs)] if res else []) + [codes, scales]
    return args, x.astype(np.float32), rv.astype(np.float32) if res else None, gm


def check_codes(c, got, x, rv, gm, eps=1e-6):
    r, n, el, p, out, res = c
    kept, codes, scales = sv.rms_norm(x, rv, gm, eps, out, store_as(el))
    if res:
        a, b = value(got[0], el), value(kept, el)
        assert np.array_equal(a, b, equal_nan=True)
    assert np.array_equal(got[-2].view(np.uint8), codes.view(np.uint8))
    if out == "i8":
        assert np.array_equal(got[-1], scales, equal_nan=True)
    else:
        assert np.array_equal(got[-1].view(np.uint8), scales)


@pytest.mark.gpu
@pytest.mark.parametrize("c", sc.NORM, ids=sc.norm_name)
def test_norm_codes_exact(gpu, c):
    note(sc.norm_name(c))
    rng = np.random.default_rng(c[0] + c[1])
    for edges in (False, True):
        args, x, rv, gm = norm_case(c, rng, edges)
        check_codes(c, run_gpu(sc.norm_name(c), args, gpu), x, rv, gm)


@pytest.mark.gpu
def test_norm_ties_and_extremes(gpu):
    """Rows of one size (every code a tie or next to one), of zeros, of the
    smallest and largest numbers; eps 0 makes NaN of a row of zeros."""
    note("norm extremes")
    for name, c, eps in (("rmsnorm_i8_f32_f32_7x1032_x", (7, 1032, "f32", "f32", "i8", False), 1e-6), ("rmsnorm_eps0", (6, 100, "bf16", "bf16", "i8", True), 0.0)):
        r, n, el = c[:3]
        x = np.zeros((r, n))
        x[0] = np.arange(n) % 255 - 127
        x[1] = (np.arange(n) % 509 - 254) / 2
        x[2, 5] = 1e-44 if el == "f32" else 1e-40
        x[3] = 3e38
        x[4] = 2.0 ** -70 * (np.arange(n) % 255 - 127)
        xs, xv = stored(x, el)
        gs, gm = stored(np.ones(n), c[3])
        zero = [np.zeros_like(xs)]
        args = [xs] + (zero if c[5] else []) + [gs] + (zero if c[5] else []) + [np.zeros((r, n), np.int8), np.zeros(r, np.float32)]
        check_codes(c, run_gpu(name, args, gpu), xv.astype(np.float32), np.zeros_like(xv, dtype=np.float32) if c[5] else None, gm, eps)


@pytest.mark.gpu
@pytest.mark.parametrize("name,cols,p,out", [("rmsnorm_i8_rt", 1000, "bf16", "i8"), ("rmsnorm_e4m3_rt", 4096, "f32", "e4m3")])
def test_norm_at_launch_time_rows(gpu, name, cols, p, out):
    """Any row count, the sum over its residual, a row's codes whatever the
    rows beside it; no rows are no launch."""
    import torch
    rng = np.random.default_rng(8)
    grp = load(name)
    last = None
    for rows in (1, 2, 37, 600, 3001):
        note(f"{name} {rows}")
        c = (rows, cols, "bf16", p, out, True)
        args, x, rv, gm = norm_case(c, rng)
        dev = [to_dev(a, q["elem"], gpu) for a, q in zip(args, grp.meta["params"])]
        dev[3] = dev[1]  # in place
        got = grp(*dev)
        check_codes(c, [to_host(t, q["elem"]) for t, q in zip(got, grp.meta["results"])], x, rv, gm)
        last = dev
    first = [t.clone() for t in last[3:]]
    dev = [t[:5].contiguous() if t.shape[0] == 3001 else t for t in to_again(last, args, grp, gpu)]
    out5 = grp(*dev)
    for a, b in zip(out5, first):
        assert torch.equal(a.view(torch.uint8), b[:5].view(torch.uint8))
    empty = [t[:0] if t.shape[0] == 5 else t for t in dev]
    grp(*empty)
    torch.cuda.synchronize()


def to_again(last, args, grp, gpu):
    """The call's arguments as they were before the sum went over the residual."""
    return [to_dev(a, q["elem"], gpu) for a, q in zip(args, grp.meta["params"])]


@pytest.mark.gpu
def test_norm_rank3(gpu):
    note("rank 3")
    c = (6, 64, "bf16", "bf16", "i8", True)
    args, x, rv, gm = norm_case(c, np.random.default_rng(2))
    shapes = [p["shape"] for p in hf.compile(cat.get("rmsnorm_rank3"), require_cached=True).blocks[0]["params"]]
    got = run_gpu("rmsnorm_rank3", [a.reshape(s) for a, s in zip(args, shapes)], gpu)
    assert got[0].shape == (2, 3, 64) and got[2].shape == (2, 3)
    check_codes(c, [got[0].reshape(6, 64), got[1].reshape(6, 64), got[2].reshape(6)], x, rv, gm)


# ---------------------------------------------------------------- batches
def batch(parts, pad=0, slots=0):
    """seq and pos of (sequence, first position, tokens) and rows that pad: no
    position, no such sequence, a position past the table."""
    seq = [s for s, _, n in parts for _ in range(n)]
    pos = [p + i for _, p, n in parts for i in range(n)]
    kinds = [(0, -1), (slots, 3), (-1, 0), (0, 1 << 30), (-(1 << 31), -(1 << 31))]
    seq += [kinds[i % 5][0] for i in range(pad)]
    pos += [kinds[i % 5][1] for i in range(pad)]
    return np.array(seq, np.int32), np.array(pos, np.int32)


def paged_table(rng, slots, room, block, blocks, used):
    """Blocks of the sequences that hold `used` positions each; the entries
    behind are blocks of others, none, or out of range."""
    per = -(-room // block)
    table = rng.choice([-1, 1 << 30, blocks, -(1 << 31)], (slots, per)).astype(np.int32)
    free = list(rng.permutation(blocks))
    for s, n in enumerate(used):
        for i in range(-(-n // block)):
            table[s, i] = free.pop()
    return table, free


def append_batches(c):
    hq, hk, d, block, slots, room, blocks, el, fmt = c
    if slots > 100:  # row counts of every tile
        yield [(s, 5 + s % 40, 1) for s in range(300)], 2
        yield [(s, s % 50, 2) for s in range(600)], 0
        return
    yield [(0, 0, 1)], 0
    yield [(1, block - 1, 2), (0, block, 1), (2, 3, 5)], 3
    yield [(slots - 1, room - block - 1, block + 1), (0, block // 2, block + 3)], 0
    yield [(s, 7 * s + 1, 1) for s in range(slots)], 5
    yield [(2, 0, 2 * block - 1)], 1


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(sc.APPEND))
def test_append_exact(gpu, name):
    """Every row, code and scale byte, those of rows and blocks that the batch
    does not name left as they were.  Each batch goes behind what is there:
    small values, larger ones (scales grow), zeros, infinities and NaN."""
    import torch
    c = sc.APPEND[name]
    hq, hk, d, block, slots, room, blocks, el, fmt = c
    rot, pairs = sc.TURN[name]
    rng = np.random.default_rng(len(name))
    grp = load(f"appendkv_{name}_rt")
    store = store_as(el)
    for i, (parts, pad) in enumerate(append_batches(c)):
        for kind in range(4):
            note(f"{name} batch {i} kind {kind}")
            seq, pos = batch(parts, pad, slots)
            t = len(seq)
            table, free = paged_table(rng, slots, room, block, blocks, [max([p + n for s2, p, n in parts if s2 == s] or [0]) for s in range(slots)])
            if kind == 3 and len(parts) > 1:
                table[parts[1][0]] = [-1, blocks, 1 << 30, -7][i % 4]  # nowhere to go
            x = rng.normal(size=(t, (hq + 2 * hk) * d)) * [1.0, 40.0, 1.0, 1.0][kind]
            if kind == 2:
                x[0, hq * d:] = 0.0
                x[-1, (hq + hk) * d + 5] = np.inf
                x[t // 2, hq * d + 3] = np.nan
            xs, xv = store(x)
            turn = rng.normal(size=(room, rot)).astype(np.float32)
            # what is there: codes of finite values, scales about those of the new tokens
            code = lambda shape: rng.integers(0, 0x78, shape).astype(np.uint8) | (rng.integers(0, 2, shape) << 7).astype(np.uint8)  # noqa: E731
            k, v = code((blocks, hk, block, d)), code((blocks, hk, d, block))
            low = 127 - bs.EMAX[fmt] + (6 if kind == 3 else 0)
            ks, vs = (rng.integers(low, low + 4, (blocks, hk)).astype(np.uint8) for _ in range(2))
            ks.flat[::11] = 255
            vs.flat[::13] = 0
            q = np.full((t, hq, d), 7, xs.dtype)
            want = sv.append_kv(xv.astype(np.float32), turn, seq, pos, table, q, k, ks, v, vs, fmt, pairs, store)
            args = [xs, turn, seq, pos, table, q, k, ks.view(np.int8), v, vs.view(np.int8)]
            dev = [to_dev(a, p["elem"], gpu) for a, p in zip(args, grp.meta["params"])]
            outs = grp(*dev)
            torch.cuda.synchronize()
            got = [to_host(o, r["elem"]) for o, r in zip(outs, grp.meta["results"])]
            a, b = value(got[0], el), value(want[0], el)
            assert np.array_equal(a, b, equal_nan=True), "queries"
            for j, what in ((2, "key scales"), (4, "value scales"), (1, "keys"), (3, "values")):
                x, y = (bs.code_values(fmt)[m] if j in (1, 3) else m.view(np.uint8) for m in (got[j], want[j]))
                where = np.argwhere(~((x == y) | ((x != x) & (y != y))))
                assert not len(where), (what, len(where), where[:4].tolist())


@pytest.mark.gpu
def test_append_at_one_row_count(gpu):
    """The group compiled for its rows equals the one that takes any."""
    import torch
    note("append static")
    name, rows = sc.STATIC["append"]
    hq, hk, d, block, slots, room, blocks, el, fmt = sc.APPEND[name]
    rng = np.random.default_rng(4)
    seq, pos = batch([(3, 60, 64), (1, 5, 3)], 3, slots)
    table, _ = paged_table(rng, slots, room, block, blocks, [0, 8, 0, 124, 0, 0])
    outs = []
    for grp in (load("appendkv_static"), load(f"appendkv_{name}_rt")):
        gen = torch.Generator(device=gpu).manual_seed(1)
        dev = [torch.randn((rows, (hq + 2 * hk) * d), generator=gen, device=gpu).bfloat16(), torch.randn((room, d), generator=gen, device=gpu)]
        dev += [torch.from_numpy(a).to(gpu) for a in (seq, pos, table)]
        dev += [torch.zeros([rows if n == -1 else n for n in p["shape"]], dtype=hf.runtime.torch_dtype(p["elem"]), device=gpu) for p in grp.meta["params"][5:]]
        outs.append(grp(*dev))
    torch.cuda.synchronize()
    for a, b in zip(*outs):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) and a.view(torch.uint8).any()


# ---------------------------------------------------------------- attention
def cache_of(rng, c, wide=False):
    hq, hk, d, block, slots, room, blocks, el, fmt = c[:9]
    top = 0x78 if fmt == "e5m2" else 0x7F
    code = lambda shape: rng.integers(0, top, shape).astype(np.uint8) | (rng.integers(0, 2, shape) << 7).astype(np.uint8)  # noqa: E731
    k, v = code((blocks, hk, block, d)), code((blocks, hk, d, block))
    low = 127 - bs.EMAX[fmt]
    ks = rng.integers(low - 3, low, (blocks, hk)).astype(np.uint8)
    vs = rng.integers(low - (40 if wide else 2), low + 1, (blocks, hk)).astype(np.uint8)
    return k, ks, v, vs


def attend_batches(c):
    hq, hk, d, block, slots, room, blocks, el, fmt, window = c
    if slots > 100:  # groups of tokens whose tiles each thread has several of
        yield [(s, (s * 37) % 190, 1 + s % 6) for s in range(slots)], 3, {}
        yield [(s, (s * 37) % 190, 7) for s in range(slots)], 0, {}
        yield [(s, 1 + s % 20, 1) for s in range(slots - 1)] + [(slots - 1, 4000, 3)], 0, {}
        yield [(s, 1 + s % 190, 1) for s in range(slots - 1)] + [(slots - 1, 900, 1200)], 0, {}
        return
    far = min(room, 5000)
    yield [(0, 0, 1)], 0, {}
    yield [(1, far - 1, 1), (0, 63, 1), (2, 64, 1)], 3, {}
    yield [(0, block - 1, 1), (2, block, 2), (1, 5, 7)], 0, dict(wide=True)
    yield [(1, far - 70, 70), (0, 0, 33)], 5, {}
    yield [(2, 3 * block - 2, 6), (0, 40, 4), (1, 20, 1)], 1, dict(holes=True)
    yield [(s, 11 * s + 2, 3) for s in range(slots)], 2, dict(nan=True)
    # rows of prompts: tiles of several sequences, ends inside a tile
    yield [(0, far - 130, 129), (1, 10, 31), (2, 1, 90)], 3, dict(wide=True)
    yield [(0, 0, 17), (2, far - 61, 60), (1, 2 * block, 40)], 0, dict(holes=True)
    yield [(1, far // 2, 75), (0, 3, 64), (2, 0, 1)], 2, dict(nan=True)
    # single tokens and short runs beside prompts, over the tiles' ends
    yield [(1, 7, 1), (0, 3, 30), (2, far // 4, 4), (1, 9, 3), (0, far - 90, 90), (2, far // 4 + 9, 1)], 2, {}
    yield [(0, 0, 1), (1, far - 1, 1), (2, 30, 16), (1, 2, 17), (0, far // 8, 5), (2, 1, 59), (1, far // 3, 2)], 0, dict(wide=True)
    for slope in (-3, 3):
        yield [(0, far - 130, 129), (1, 2 * block, 40)], 0, dict(slope=slope)
        yield [(0, far - 2, 1), (1, 2 * block, 2)], 0, dict(slope=slope)


def check_attention(c, outs, q, cache, seq, pos, table, before, scale=None):
    hq, hk, d, block, slots, room, blocks, el, fmt, window = c
    k, ks, v, vs = cache
    scale = float(np.float32(d ** -0.5)) if scale is None else scale
    want, size, reach = sv.paged_attention(q, k, ks, v, vs, seq, pos, table, before, fmt, scale, window)
    n = np.maximum(np.asarray(pos, np.float64), 0)[:, None, None] + 65
    n = np.minimum(n, window + 65 if window else n)
    step = U[el]
    p16 = 2.0 ** -8 if el == "bf16" else 2.0 ** -11
    vmax = np.nanmax(np.abs(bs.code_values(fmt)[v[:, :, :, :]]) * np.where(vs == 255, 0, bs.scale_values(vs))[:, :, None, None], initial=0,
                     where=np.isfinite(bs.code_values(fmt)[v]))
    tol = size * (p16 + 2.0 ** -20 + 2 * (d + 8) * 2.0 ** -23 * reach[:, :, None] + 2 * n * 2.0 ** -23)
    if el == "f16":
        tol = tol + 2.0 ** -25 * n * vmax
    got = value(outs, el)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    with np.errstate(invalid="ignore"):
        ok = np.abs(got - want) <= tol + step * (np.abs(want) + tol) + TINY[el]
    assert (ok | nan).all(), (np.argwhere(~(ok | nan))[:5], np.nanmax(np.abs(got - want)))


def attend_case(rng, c, parts, pad, wide=False, holes=False, nan=False, slope=0):
    hq, hk, d, block, slots, room, blocks, el, fmt, window = c
    seq, pos = batch(parts, pad, slots)
    used = [max([p + n for s2, p, n in parts if s2 == s] or [0]) for s in range(slots)]
    table, free = paged_table(rng, slots, room, block, blocks, used)
    k, ks, v, vs = cache = cache_of(rng, c, wide)
    if slope:  # values' scales that fall (or rise) from block to block
        low = 127 - bs.EMAX[fmt]
        for s, n in enumerate(used):
            for i in range(-(-n // block)):
                step = i if slope < 0 else -(-n // block) - i
                vs[table[s, i]] = max(1, low - abs(slope) * step)
    # memory that no token has come to: NaN codes behind each end, in blocks of nobody
    for s, n in enumerate(used):
        if n % block:
            k[table[s, n // block], :, n % block:], v[table[s, n // block], :, :, n % block:] = 0xFF, 0x7F
    for b in free:
        k[b], v[b], ks[b], vs[b] = 0xFF, 0x7F, 255, 255
    for s, n in enumerate(used):  # stale entries that name them
        if n and free and -(-n // block) < table.shape[1]:
            table[s, -(-n // block)] = free[0]
    if holes:
        table[parts[0][0], 1] = -1
        table[parts[-1][0], : -(-used[parts[-1][0]] // block)] = -5  # nothing to see
    if nan:
        vs[table[parts[1][0], 0], 0] = 255
        ks[table[parts[2][0], 0], -1] = 255
    qs, qv = stored(rng.normal(size=(len(seq), hq, d)), el)
    return seq, pos, table, cache, qs, qv


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(sc.ATTEND))
def test_attention(gpu, name):
    import torch
    c = sc.ATTEND[name]
    rng = np.random.default_rng(len(name) + c[2])
    grp = load(f"pagedattn_{name}_rt")
    for i, (parts, pad, more) in enumerate(attend_batches(c)):
        note(f"{name} batch {i}")
        seq, pos, table, cache, qs, qv = attend_case(rng, c, parts, pad, **more)
        before = np.full(qv.shape, 3.0)
        args = [qs, cache[0], cache[1].view(np.int8), cache[2], cache[3].view(np.int8), seq, pos, table, store_as(c[7])(before)[0]]
        dev = [to_dev(a, p["elem"], gpu) for a, p in zip(args, grp.meta["params"])]
        out = grp(*dev)
        torch.cuda.synchronize()
        check_attention(c, to_host(out, c[7]), qv, cache, seq, pos, table, before)


@pytest.mark.gpu
def test_attention_at_one_row_count(gpu):
    import torch
    name, rows = sc.STATIC["attend"]
    note("attention static")
    c = sc.ATTEND[name]
    rng = np.random.default_rng(31)
    seq, pos, table, cache, qs, qv = attend_case(rng, c, [(0, 3000, 1), (5, 100, 64), (2, 0, 2)], 3)
    assert len(seq) == rows
    grp = load("pagedattn_static")
    args = [qs, cache[0], cache[1].view(np.int8), cache[2], cache[3].view(np.int8), seq, pos, table, np.zeros_like(qs)]
    dev = [to_dev(a, p["elem"], gpu) for a, p in zip(args, grp.meta["params"])]
    check_attention(c, to_host(grp(*dev), c[7]), qv, cache, seq, pos, table, np.zeros(qv.shape))
    torch.cuda.synchronize()


# ---------------------------------------------------------------- together
@pytest.mark.gpu
def test_layer_steps(gpu):
    """A prompt and then tokens one by one through norm, int8 product, append
    and attention, as a serving loop runs them: each op against its definition
    on what the one before it left, eager and as a captured graph that is
    replayed over new tokens."""
    import torch
    note("layer steps")
    L = sc.LAYER
    cols, heads, kv, dim, slots, room, blocks, block = (L[k] for k in ("cols", "heads", "kv_heads", "dim", "slots", "room", "blocks", "block"))
    width = (heads + 2 * kv) * dim
    norm, product, append, attend = (load(f"layer_{n}_rt") for n in ("norm_i8", "qkv", "append", "attend"))
    rng = np.random.default_rng(77)
    wq = rng.integers(-127, 128, (width, cols)).astype(np.int8)
    sch = (rng.uniform(0.5, 1.5, width) / 127 / np.sqrt(cols)).astype(np.float32)
    gs, gm = stored(rng.uniform(0.5, 1.5, cols), "bf16")
    angle = np.arange(room)[:, None] * 100.0 ** (-np.arange(dim // 2) / (dim // 2))
    rot = np.concatenate([np.cos(angle), np.sin(angle)], axis=1).astype(np.float32)
    table = np.stack([rng.permutation(blocks)[: room // block] for _ in range(1)] * slots).astype(np.int32)
    order = rng.permutation(blocks)
    table[:] = -1
    table[0, :3], table[2, :4] = order[:3], order[3:7]
    dev = lambda a, e: to_dev(a, e, gpu)  # noqa: E731
    W, S, Gm, R, Tb = dev(wq, "i8"), dev(sch, "f32"), dev(gs, "bf16"), dev(rot, "f32"), dev(table, "i32")
    cache = [torch.zeros(p["shape"], dtype=hf.runtime.torch_dtype(p["elem"]), device=gpu) for p in append.meta["params"][6:]]
    host = [np.zeros(p["shape"], np.uint8) for p in append.meta["params"][6:]]

    def buffers(rows):
        new = lambda *s, dt=torch.bfloat16: torch.zeros((rows, *s), dtype=dt, device=gpu)  # noqa: E731
        return dict(x=new(cols), res=new(cols), codes=new(cols, dt=torch.int8), scale=new(dt=torch.float32), qkv=new(width), q=new(heads, dim),
                    seq=new(dt=torch.int32), pos=new(dt=torch.int32), out=new(heads, dim))

    def step(b):
        norm(b["x"], b["res"], Gm, b["res"], b["codes"], b["scale"])
        product(b["codes"], W, b["scale"], S, b["qkv"])
        append(b["qkv"], R, b["seq"], b["pos"], Tb, b["q"], *cache)
        attend(b["q"], *cache, b["seq"], b["pos"], Tb, b["out"])

    def fill(b, seq, pos):
        rows = len(seq)
        (xs, x), (rs, rv) = (stored(rng.normal(size=(rows, cols)), "bf16") for _ in range(2))
        for t, a, e in (("x", xs, "bf16"), ("res", rs, "bf16"), ("seq", seq, "i32"), ("pos", pos, "i32")):
            b[t].copy_(dev(a, e))
        b["q"].zero_(), b["out"].zero_()
        return x.astype(np.float32), rv.astype(np.float32)

    def check(b, seq, pos, x, rv):
        nonlocal host
        torch.cuda.synchronize()
        c = (len(seq), cols, "bf16", "bf16", "i8", True)
        codes, scale = to_host(b["codes"], "i8"), to_host(b["scale"], "f32")
        check_codes(c, [to_host(b["res"], "bf16"), codes, scale], x, rv, gm)
        acc = codes.astype(np.int64) @ wq.T.astype(np.int64)
        want = interp.from_f32((acc.astype(np.float32) * scale[:, None]) * sch, "bf16")
        got = to_host(b["qkv"], "bf16")
        assert np.array_equal(got, want)
        qkv = value(got, "bf16").astype(np.float32)
        host = list(sv.append_kv(qkv, rot, seq, pos, table, np.zeros((len(seq), heads, dim), np.uint16), *host, "e4m3", 0, store_as("bf16")))
        q = host.pop(0)
        assert np.array_equal(value(to_host(b["q"], "bf16"), "bf16"), value(q, "bf16"))
        values = bs.code_values("e4m3")
        for i, t in enumerate(cache):
            t = t.view(torch.uint8).cpu().numpy()
            assert np.array_equal(t, host[i]) if i % 2 else np.array_equal(values[t], values[host[i]])
        spec = (heads, kv, dim, block, slots, room, blocks, "bf16", "e4m3", 0)
        check_attention(spec, to_host(b["out"], "bf16"), value(q, "bf16"), host, seq, pos, table, np.zeros(q.shape))

    # the prompts of two sequences, with rows that pad
    seq, pos = batch([(2, 0, 45), (0, 0, 30)], 2, slots)
    b = buffers(len(seq))
    x, rv = fill(b, seq, pos)
    step(b)
    check(b, seq, pos, x, rv)
    # token by token, the graph captured once on a stream of its own
    seq = np.array([0, 2, 0], np.int32)
    b = buffers(3)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    for i in range(5):
        pos = np.array([30 + i, 45 + i, -1], np.int32)
        x, rv = fill(b, seq, pos)
        torch.cuda.synchronize()
        if i == 0:
            with torch.cuda.stream(side):
                step(b)
        elif i == 1:
            with torch.cuda.graph(graph, stream=side):
                step(b)
            graph.replay()
        else:
            graph.replay()
        check(b, seq, pos, x, rv)
