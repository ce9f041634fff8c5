"""Attention over caches whose blocks hold values of very different sizes, and
over tables that name what a window has left behind: a row's result follows the
positions that it sees, whatever the blocks beside them in its tile hold.

Tolerance of a value, with N positions seen, D channels, P = sum p |v| and the
largest |v|, all over the positions that the row sees (of its own kv head):
  scores: D + 8 f32 roundings of at most sum |q k| scale, in the numerator and
    the denominator                        2 (D + 8) 2^-23 sum |q k| P
  exp2 of the hardware (1 ulp) and its argument's rounding       2^-20 P
  N f32 additions in both sums             2 N 2^-23 P
  p to 16 bits (half a step), of a prompt also in the denominator
                                           2 2^-8 P, of f16 queries 2 2^-11 P and
                                           2^-34 |v| for each position (p times 2^9
                                           is rounded, whose smallest step is 2^-24)
  the result's own rounding (half a step)"""
import numpy as np
import pytest

import serving_catalog as sc
import serving_range_catalog as rc
from helpers import to_dev, to_host
from oracle import blockscaled as bs
from oracle import serving as sv
from test_norm_mx import TINY, U, note, stored, value
from test_serving import batch, cache_of, load

TOP16 = 65504.0


def largest(cache, seq, pos, table, window, heads, fmt):
    """The largest |v| that each row and query head sees, and how many positions."""
    _, _, v, vs = cache
    blocks, kv, _, block = v.shape
    with np.errstate(invalid="ignore"):
        size = np.abs(bs.code_values(fmt)[v]).max(axis=2) * bs.scale_values(vs)[:, :, None]  # [block, head, token]
    out, n = np.zeros((len(seq), heads)), np.zeros(len(seq))
    for t in range(len(seq)):
        if 0 <= seq[t] < table.shape[0] and 0 <= pos[t] < table.shape[1] * block:
            j = sv.visible(pos[t], seq[t], table, blocks, block, window)
            n[t] = len(j)
            if len(j):
                out[t] = np.repeat(size[table[seq[t], j // block], :, j % block].max(axis=0), heads // kv)
    return out, n


def check_rows(c, outs, q, cache, seq, pos, table, before):
    hq, hk, d, block, slots, room, blocks, el, fmt, window = c
    want, size, reach = sv.paged_attention(q, *cache, seq, pos, table, before, fmt, float(np.float32(d ** -0.5)), window)
    vmax, n = largest(cache, seq, pos, table, window, hq, fmt)
    n = n[:, None, None]
    tol = size * (2 * U[el] + 2.0 ** -20 + 2 * (d + 8) * 2.0 ** -23 * reach[:, :, None] + 2 * n * 2.0 ** -23)
    if el == "f16":
        tol = tol + 2.0 ** -34 * n * vmax[:, :, None]
    got = value(outs, el)
    assert np.array_equal(np.isnan(got), np.isnan(want)), np.argwhere(np.isnan(got) != np.isnan(want))[:5]
    # (what may round to an infinity of f16 has no value to compare)
    far = np.abs(want) + tol + U[el] * (np.abs(want) + tol) > TOP16 if el == "f16" else np.zeros(want.shape, bool)
    with np.errstate(invalid="ignore"):
        ok = np.abs(got - want) <= tol + U[el] * (np.abs(want) + tol) + TINY[el]
    assert (ok | far | np.isnan(want)).all(), [(i.tolist(), got[tuple(i)], want[tuple(i)]) for i in np.argwhere(~(ok | far | np.isnan(want)))[:5]]
    return far


def run(grp, c, gpu, seq, pos, table, cache, qs, qv):
    import torch
    before = np.full(qv.shape, 3.0)
    args = [qs, cache[0], cache[1].view(np.int8), cache[2], cache[3].view(np.int8), seq, pos, table, stored(before, c[7])[0]]
    out = grp(*[to_dev(a, p["elem"], gpu) for a, p in zip(args, grp.meta["params"])])
    torch.cuda.synchronize()
    return check_rows(c, to_host(out, c[7]), qv, cache, seq, pos, table, before)


def case_of(rng, c, parts, byte, pad=0):
    """A batch over sequences whose block i has the value scale byte(i) in
    every head; blocks in any order, none behind a sequence's last row."""
    hq, hk, d, block, slots, room, blocks, el, fmt, window = c
    seq, pos = batch(parts, pad, slots)
    cache = cache_of(rng, c)
    order = list(rng.permutation(blocks))
    table = np.full((slots, -(-room // block)), -1, np.int32)
    for s in {s for s, _, _ in parts}:
        for i in range(-(-max(p + n for s2, p, n in parts if s2 == s) // block)):
            table[s, i] = order.pop()
            cache[3][table[s, i]] = byte(i)
    qs, qv = stored(rng.normal(size=(len(seq), hq, d)), el)
    return seq, pos, table, cache, qs, qv


# ---------------------------------------------------------------- blocks far apart
@pytest.mark.gpu
@pytest.mark.parametrize("down", [9, 20, 25, 31])
@pytest.mark.parametrize("name", ["group3", "alone", "far_f16", "wide_f16", "far_wide", "window_f16_64", "group20_f16", "far_group20_f16"])
def test_f16_prompt_beside_larger_blocks(gpu, name, down):
    """Rows of f16 prompts that see small values alone, and later blocks of
    the same tile 2^down larger, that the later rows see; and the other way
    round, where the large values have small weights or large ones."""
    c = sc.ATTEND.get(name) or rc.ATTEND[name]
    fmt, block, far = c[8], c[3], min(c[5], 2000)
    grp = load(f"pagedattn_{name}_rt")
    # (the largest values are some 2^14 times 1.75)
    big = 127 + 14 - bs.EMAX[fmt]
    for k, byte in enumerate((lambda i: big if i % 2 else big - down, lambda i: big - down if i % 2 else big,
                              lambda i: big - down if i < 3 else big - down // 2 if i < 5 else big)):
        note(f"{name} down {down} order {k}")
        rng = np.random.default_rng(down + k)
        run(grp, c, gpu, *case_of(rng, c, [(0, 0, 3 * block + 5), (2, far - 70, 70)], byte, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("down", [60, 99, 101, 112, 126, 127, 133, 150])
@pytest.mark.parametrize("name", ["group4", "group20", "far_alone", "usual", "far_group20", "wide", "window_64"])
def test_bf16_prompt_beside_larger_blocks(gpu, name, down):
    """The same of bf16, whose exponents are f32's: no block's values are
    taken for larger ones, and none are lost that a row sees alone."""
    c = sc.ATTEND.get(name) or rc.ATTEND[name]
    block, far = c[3], min(c[5], 2000)
    grp = load(f"pagedattn_{name}_rt")
    big = 60 + down  # (small values are some 2^-60)
    for k, byte in enumerate((lambda i: big if i % 2 else big - down, lambda i: big - down if i % 2 else big,
                              lambda i: big - down if i < 3 else big - down // 2 if i < 5 else big)):
        note(f"{name} down {down} order {k}")
        rng = np.random.default_rng(down + k)
        run(grp, c, gpu, *case_of(rng, c, [(0, 0, 3 * block + 5), (2, far - 70, 70)], byte, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["far_f16", "group20_f16", "far_alone"])
def test_graphs_of_blocks_far_apart(gpu, name):
    """A prompt over such blocks captured and replayed, with eager calls between:
    the eager result to the bit, and the same over and over."""
    import torch
    from test_serving_calls import attend_args, same
    c = sc.ATTEND.get(name) or rc.ATTEND[name]
    far, down = min(c[5], 2000), 25 if c[7] == "f16" else 120
    note(f"graph {name}")
    grp = load(f"pagedattn_{name}_rt")
    a = attend_args(c, case_of(np.random.default_rng(6), c, [(0, 0, 3 * c[3] + 5), (1, 40, 2), (2, far - 70, 70)], lambda k: 135 if k % 2 else 135 - down, 1), gpu)
    grp(*a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grp(*a)
    for _ in range(3):
        a[0].copy_(torch.randn(a[0].shape, device=gpu).to(a[0].dtype))
        a[-1].zero_()
        graph.replay()
        got = a[-1].clone()
        for _ in range(2):
            a[-1].zero_()
            grp(*a)
            torch.cuda.synchronize()
            assert same(a[-1], got) and got.float().abs().sum() > 0


# ---------------------------------------------------------------- windows
def placeholder(rng, c, case, scale):
    """Names one block of NaN codes in the place of all that lie before the
    window of a sequence's first row."""
    seq, pos, table, (k, ks, v, vs), qs, qv = case
    block, window, fmt = c[3], c[9], c[8]
    free = [b for b in range(len(k)) if b not in table]
    k[free[0]], v[free[0]], ks[free[0]], vs[free[0]] = 0xFF, 0x7F, scale, scale
    gone = 0
    for s in set(seq[(seq >= 0) & (seq < len(table)) & (pos >= 0)].tolist()):
        first = pos[(seq == s) & (pos >= 0)].min()
        n = max(0, (first - window + 1) // block)
        table[s, :n] = free[0]
        gone += n
    return gone


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0, 127, 200, 254, 255])
@pytest.mark.parametrize("name", ["window", "window_f16", "far_window", "far_longer"] + [n for n in rc.ATTEND if "window" in n])
def test_blocks_before_the_window(gpu, name, scale):
    """What lies before the window of a sequence's first row may be anything:
    a placeholder of NaN codes, whatever its scale.  Single tokens and a few at
    a time, rows of prompts, and both in one batch."""
    c = sc.ATTEND.get(name) or rc.ATTEND[name]
    slots, room, window = c[4], c[5], c[9]
    rng = np.random.default_rng(scale + len(name))
    low = 127 - bs.EMAX[c[8]]
    grp = load(f"pagedattn_{name}_rt")
    near = min(room, window + 200)
    for i, parts in enumerate(([(0, near - 3, 1), (1, window + 20, 1), (2, window + 33, 1)], [(0, near - 7, 6), (2, window + 61, 3)],
                               [(1, near - 90, 90), (0, window + 7, 33)], [(1, window + 17, 100), (0, near - 4, 3), (2, near - 1, 1)])):
        note(f"{name} scale {scale} batch {i}")
        case = case_of(rng, c, parts, lambda i: low - i % 3)
        assert placeholder(rng, c, case, scale) > 0 or c[3] == 128  # (of which a short batch may see every block)
        run(grp, c, gpu, *case)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["group3", "alone", "far_f16", "wide_f16", "far_wide", "group4", "group20", "far_alone", "usual", "far_group20", "wide"])
def test_rows_before_far_larger_values(gpu, name):
    """Rows that see small values alone, beside rows of the same sequence
    that see values up to f32's largest, in the next block and in the next tile:
    a few at a time and as rows of a prompt."""
    c = sc.ATTEND[name]
    block, el, slots = c[3], c[7], c[4]
    grp = load(f"pagedattn_{name}_rt")
    low = 127 - bs.EMAX[c[8]] - (14 if el == "f16" else 90)
    for big in (low + 40, 190, 254 - bs.EMAX[c[8]] - 16):
        for i, (parts, edge) in enumerate((([(0, 0, 140)], block), ([(0, 0, 140)], 64), ([(2, 64 - 2, 4)], 64), ([(1, block - 3, 6), (0, 3 * block - 1, 2)], block))):
            note(f"{name} big {big} batch {i}")
            rng = np.random.default_rng(big + i)
            case = case_of(rng, c, parts, lambda k: big if k * block >= edge else low)
            far = run(grp, c, gpu, *case)
            assert not far[case[1] < edge].any()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["group3", "alone", "far_f16", "wide_f16", "far_wide", "group4", "group20", "far_alone", "usual", "far_group20", "wide"])
def test_smallest_codes_beside_larger_blocks(gpu, name):
    """Values that are the format's smallest numbers, as far below the tile's
    largest block as one product takes them, and one further: as exact as others."""
    c = sc.ATTEND[name]
    block, el, fmt = c[3], c[7], c[8]
    grp = load(f"pagedattn_{name}_rt")
    for down in (7, 8, 9) if el == "f16" else (98, 99, 100, 101):
        for parts in ([(0, 0, 140)], [(0, block - 3, 6)]):
            note(f"{name} down {down} {parts}")
            rng = np.random.default_rng(down)
            big = 141 if el == "f16" else 136
            seq, pos, table, cache, qs, qv = case_of(rng, c, parts, lambda k: big if k else big - down)
            v = cache[2][table[0, 0]]
            v[:] = rng.integers(1, 4, v.shape) | (rng.integers(0, 2, v.shape) << 7)
            far = run(grp, c, gpu, seq, pos, table, cache, qs, qv)
            assert not far[pos < block].any()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [12, 18, 23, 25, 27])
@pytest.mark.parametrize("name", ["group3", "alone", "far_f16", "wide_f16", "far_wide", "window_f16_64"])
def test_f16_small_weights_of_large_values(gpu, name, bits):
    """Positions behind the first 64 (of blocks of 128, 128) hold values near f16's
    largest at weights of some 2^-bits of the first ones', which hold small
    values: both count in the result.  Single tokens, a few, and rows of a prompt."""
    c = sc.ATTEND.get(name) or rc.ATTEND[name]
    hq, hk, d, block, slots, room, blocks, el, fmt, window = c
    grp = load(f"pagedattn_{name}_rt")
    big, edge = 127 + 14 - bs.EMAX[fmt], max(64, block)
    for parts in ([(0, edge + 40, 1)], [(1, edge + 20, 7), (0, edge + 30, 2)], [(2, edge + 3, 30), (0, 0, edge + 60)]):
        note(f"{name} bits {bits} {parts}")
        rng = np.random.default_rng(bits)
        seq, pos, table, cache, qs, qv = case_of(rng, c, parts, lambda k: big if k * block >= edge else big - 30)
        # all queries 1; the first keys' scores 0, the others' lower by bits log 2 and a bit more
        qs, qv = stored(np.ones(qv.shape), el)
        k, ks, v, _ = cache
        ks[:] = 127
        code = bs.encode(np.array([-bits * np.log(2) / np.sqrt(d)]), fmt)[0]
        for s in {s for s, _, _ in parts}:
            for i, b in enumerate(table[s]):
                if i * block < edge:
                    k[b] = 0
                elif b >= 0:  # (values of one sign, of the largest binades)
                    k[b] = np.where(rng.random(k[b].shape) < 0.5, code, code + 1)
                    v[b] = rng.integers(0x70, 0x7B, v[b].shape)
        run(grp, c, gpu, seq, pos, table, cache, qs, qv)
