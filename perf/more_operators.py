"""The attention half of a decoder layer in serving, in plain form and through the package.

The path these operators lie on is one step of a serving loop: the residual
stream gets the last layer's output added and is normalised into 8-bit codes
for the next product; the product's queries, keys and values are rotated to
their positions and the keys and values join a paged cache that holds 8 bits
a value; the queries attend to that cache.

operators ("op")
  norm    s = x + residual, root-mean-square norm of s times a weight, as 8-bit
          codes with scales: "i8" with one f32 scale a row, "e4m3" / "e5m2"
          with a power-of-two scale for each 32 columns
  append  rows of queries, keys and values, rotated to their positions: the
          queries to a tensor of their own, the keys and values to the paged
          cache (8-bit codes, one power-of-two scale for each block of tokens
          and head)
  attend  attention of those queries over the cache, causal, optionally over a
          window of the last positions only
A batch is rows of tokens: `seq` says which sequence a row belongs to, `pos`
its position there, -1 for a row that pads the batch.  A sequence's new rows
lie together, their positions following each other.  "rt" takes the row count
at launch (one compiled group for all).

The cache: keys [blocks, kv heads, block, dim], values [blocks, kv heads, dim,
block], scale bytes [blocks, kv heads] of each; `table` [slots, blocks a
sequence may have] holds each sequence's blocks in order.
"""
import functools
import math
import os
import sys

import torch

own = False

E4M3, E5M2, I8 = "e4m3", "e5m2", "i8"
# exponent of the largest binade, largest value
_FORMATS = {E4M3: (8, 448.0), E5M2: (15, 57344.0)}
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_CODES = {E4M3: torch.float8_e4m3fn, E5M2: torch.float8_e5m2}
_WIDTH = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-6
# a row count that no other size of a case has: the compiled group's rows are
# left open in its place
_ANY_ROWS = 104729


def _cache(slots, seqs, new, past, pad, heads, kv, dim, block, room, type, fmt, rt, **more):
    """A case of the paged cache: `seqs` of `slots` sequences get up to `new`
    tokens behind up to `past` earlier ones; a table row has room for `room`."""
    return dict(slots=slots, seqs=seqs, new=new, past=past, pad=pad, heads=heads, kv=kv, dim=dim, block=block, room=room, type=type, fmt=fmt,
                rt=rt, **more)


def listed():
    return [
        # a prompt's tokens ahead of an int8 product, one scale a token
        dict(name="norm_prompt", op="norm", rows=8192, cols=4096, type="bf16", params="bf16", out=I8, residual=True, rt=False),
        # one decoding step's tokens: launch and row latency
        dict(name="norm_decode", op="norm", rows=16, cols=4096, type="bf16", params="bf16", out=I8, residual=True, rt=True),
        # an odd number of wide f16 rows ahead of a block-scaled product
        dict(name="norm_blocks", op="norm", rows=2003, cols=8192, type="f16", params="f32", out=E4M3, residual=True, rt=True),
        # f32 rows of an odd length, the first norm of a model (no residual yet)
        dict(name="norm_odd", op="norm", rows=777, cols=5003, type="f32", params="f32", out=E5M2, residual=False, rt=False),
        # prompts of three sequences join the cache, two of them behind earlier parts
        dict(name="append_prompt", op="append", style="half", rot=128,
             **_cache(4, 3, 4096, 1000, 0, 32, 8, 128, 64, 8192, "bf16", E4M3, False)),
        # one decoding step of 64 sequences
        dict(name="append_decode", op="append", style="half", rot=128,
             **_cache(64, 64, 1, 4000, 0, 32, 8, 128, 64, 8192, "bf16", E4M3, True)),
        # a ragged batch of short pieces, neighbouring pairs rotated, a part of each head only
        dict(name="append_ragged", op="append", style="pairs", rot=32,
             **_cache(16, 13, 101, 333, 5, 12, 4, 96, 16, 1024, "f16", E5M2, True)),
        # one token behind a long context
        dict(name="attend_token", op="attend", window=0, **_cache(1, 1, 1, 32767, 0, 32, 8, 128, 64, 32768, "bf16", E4M3, True)),
        # one decoding step of 48 sequences of all lengths, in a batch padded to 64
        dict(name="attend_batch", op="attend", window=0, **_cache(64, 48, 1, 8100, 16, 32, 8, 128, 64, 8192, "bf16", E4M3, True)),
        # a few proposed tokens of each of eight short sequences, checked in one step
        dict(name="attend_few", op="attend", window=0, **_cache(8, 8, 4, 500, 0, 32, 8, 128, 16, 2048, "bf16", E4M3, True)),
        # whole prompts of four sequences
        dict(name="attend_prompt", op="attend", window=0, **_cache(4, 4, 4096, 0, 0, 32, 8, 128, 64, 4096, "bf16", E4M3, False)),
        # a piece of a long prompt, over a window of the last positions
        dict(name="attend_piece", op="attend", window=4096, **_cache(2, 1, 1001, 15000, 0, 16, 2, 64, 32, 16384, "f16", E5M2, True)),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "append", "append", "attend", "attend", "attend"])
    rt = rng.random() < 0.5
    if op == "norm":
        type_, cols = rng.choice(["bf16", "bf16", "f16", "f32"]), _spread(rng, 64, 16384)
        # at most the largest listed case's elements, whatever the type's width
        rows = max(1, min(_spread(rng, 1, 8192), (8192 * 4096 // 2 if type_ == "f32" else 8192 * 4096) // cols))
        return dict(op=op, rows=rows, cols=cols, type=type_, params=rng.choice([type_, "f32"]), out=rng.choice([I8, I8, E4M3, E5M2]),
                    residual=rng.random() < 0.7, rt=rt)
    kv, group, dim, block = rng.choice([1, 2, 4, 8]), rng.choice([1, 3, 4, 8]), rng.choice([64, 96, 128, 256]), rng.choice([16, 32, 64, 128])
    kind = rng.choice(["decode", "few", "prompt"])
    if kind == "decode":
        seqs, new, past = _spread(rng, 1, 64), 1, _spread(rng, 1, 16000)
    elif kind == "few":
        seqs, new, past = _spread(rng, 1, 32), rng.randint(2, 8), _spread(rng, 1, 8000)
    else:
        seqs, new, past = rng.randint(1, 4), _spread(rng, 16, 2048), rng.choice([0, _spread(rng, 1, 4000)])
    pad = rng.choice([0, 0, rng.randint(1, 9)])
    room = -(-(past + new) // block) * block + block * rng.randint(0, 3)
    case = _cache(seqs + rng.randint(0, 3), seqs, new, past, pad, kv * group, kv, dim, block, room, rng.choice(["bf16", "bf16", "f16"]),
                  rng.choice([E4M3, E4M3, E5M2]), rt)
    if op == "append":
        case.update(type=rng.choice([case["type"], case["type"], "f32"]), style=rng.choice(["half", "half", "pairs"]),
                    rot=rng.choice([dim, dim, dim // 2]))
    else:
        case["window"] = rng.choice([0, 0, _spread(rng, 16, 4096)])
    return dict(op=op, **case)


# ---------------------------------------------------------------- a batch's lengths
def _part(i):
    """Fractions in [0, 1) spread evenly, in no order."""
    return (i + 1) * 0.6180339887498949 % 1.0


def _lengths(case):
    """(new tokens, earlier tokens) of each sequence: ragged, the first the longest."""
    n, new, past = case["seqs"], case["new"], case["past"]
    return [(new if i == 0 else 1 + int((new - 1) * _part(i)), past if i == 0 else int(past * _part(2 * i + 1))) for i in range(n)]


def _rows(case):
    return sum(n for n, _ in _lengths(case)) + case["pad"]


def _visible(case):
    """Positions that the sequences' rows see, and that are read at all."""
    seen = read = 0
    w = case["window"] or 1 << 60
    for new, past in _lengths(case):
        full = max(0, min(new, w - past))  # rows that see everything before them
        seen += full * past + full * (full + 1) // 2 + (new - full) * w
        read += min(past + new, w + new - 1)
    return seen, read


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed * 1000003 + 41)

    def normal(shape, std=1.0):
        return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32) * std

    def uniform(shape, lo, hi):
        return torch.rand(shape, generator=gen, device=dev, dtype=torch.float32) * (hi - lo) + lo

    def out(shape, dtype):
        return torch.zeros(shape, dtype=dtype, device=dev)

    s = dict(case=case)
    t = _TYPES[case["type"]]
    if case["op"] == "norm":
        r, c = case["rows"], case["cols"]
        # a residual stream: a spread of row sizes, some columns far larger than the others
        x = normal((r, c)) * uniform((r, 1), 0.25, 4.0)
        x[:, :: max(1, c // 7)] *= 8.0
        s.update(x=x.to(t), gamma=uniform((c,), 0.5, 1.5).to(_TYPES[case["params"]]))
        if case["residual"]:
            s.update(residual=normal((r, c), 2.0).to(t), sum=out((r, c), t))
        if case["out"] == I8:
            s.update(codes=out((r, c), torch.int8), scales=out((r,), torch.float32))
        else:
            s.update(codes=out((r, c), _CODES[case["out"]]), scales=out((r, (c + 31) // 32), torch.int8))
        return s
    slots, kv, d, block, room = case["slots"], case["kv"], case["dim"], case["block"], case["room"]
    lengths = _lengths(case)
    # the batch's rows; the padding ones last
    which = torch.randperm(slots, generator=gen, device=dev)[: len(lengths)].tolist()
    seq = [q for q, (new, _) in zip(which, lengths) for _ in range(new)] + [0] * case["pad"]
    pos = [past + i for new, past in lengths for i in range(new)] + [-1] * case["pad"]
    s.update(seq=torch.tensor(seq, dtype=torch.int32, device=dev), pos=torch.tensor(pos, dtype=torch.int32, device=dev))
    # the blocks that each sequence needs, from anywhere in the pool
    needs = [-(-(new + past) // block) for new, past in lengths]
    blocks = sum(needs) + 3
    order = torch.randperm(blocks, generator=gen, device=dev).to(torch.int32)
    table = torch.full((slots, -(-room // block)), -1, dtype=torch.int32, device=dev)
    at = 0
    for q, n in zip(which, needs):
        table[q, :n] = order[at : at + n]
        at += n
    s["table"] = table
    # what the cache holds already: keys with some large channels, values
    # smaller; heads of different sizes
    size = uniform((1, kv, 1, 1), 0.5, 2.0)
    keys = normal((blocks, kv, block, d)) * size
    keys[:, :, :, :: max(1, d // 5)] *= 4.0
    s["k"], s["ks"] = _block_codes(keys, case["fmt"])
    s["v"], s["vs"] = _block_codes(normal((blocks, kv, d, block), 0.5) * size, case["fmt"])
    rows, heads = len(seq), case["heads"]
    s["longest"] = (max(n for n, _ in lengths), max(n + p for n, p in lengths))
    if case["op"] == "append":
        s["qkv"] = (normal((rows, (heads + 2 * kv) * d)) * uniform((rows, 1), 0.5, 2.0)).to(t)
        half = case["rot"] // 2
        far = torch.arange(room, dtype=torch.float64, device=dev)[:, None]
        angle = far * 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
        s["rot"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        s["q"] = out((rows, heads, d), t)
    else:
        s["q"] = (normal((rows, heads, d)) * uniform((1, heads, 1), 0.5, 2.0)).to(t)
        s["out"] = out((rows, heads, d), t)
    return s


# ---------------------------------------------------------------- plain forms
def _pow2(e):
    """2^e in f32 for whole e in [-127, 127], made from its bits: a power
    function may be an ulp off."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _scale_byte(amax, fmt):
    """The byte E + 127 of the smallest 2^E that keeps values up to amax in the format's range."""
    emax, top = _FORMATS[fmt]
    m, e = torch.frexp(amax)  # m in [0.5, 1)
    e = e - 1 - emax + (m * 2.0 ** (emax + 1) > top)
    byte = torch.where(amax > 0, e, -127).clamp(-127, 127) + 127
    return torch.where(torch.isfinite(amax), byte, 255)


def _to_codes(v, byte, fmt):
    """8-bit codes of f32 v over the scale of its byte; zeros where that is 255."""
    top = _FORMATS[fmt][1]
    v = torch.where(byte < 255, v * _pow2(127 - byte.clamp(max=254)), 0.0)
    return v.clamp(-top, top).to(_CODES[fmt])


def _block_codes(x, fmt):
    """Codes and scale bytes of x [blocks, heads, ...], a scale for each block and head."""
    byte = _scale_byte(x.abs().amax(dim=(2, 3)), fmt)
    return _to_codes(x, byte[:, :, None, None], fmt), byte.to(torch.uint8).view(torch.int8)


def _byte(scales):
    return scales.view(torch.uint8).to(torch.int32)


def _value(byte):
    """2^E of scale bytes; NaN for 255."""
    return torch.where(byte < 255, _pow2(byte.clamp(max=254) - 127), float("nan"))


def _bits(scales):
    """Scale bytes as the powers of two that they stand for."""
    return scales.view(torch.float8_e8m0fnu)


def _plain_norm(s):
    case = s["case"]
    x = s["x"].float()
    if case["residual"]:
        total = (x + s["residual"].float()).to(s["x"].dtype)
        x = total.float()
    # the mean of squares in 64 bits: a code is the same in any order of the sum
    rstd = (1.0 / torch.sqrt(x.double().square().mean(dim=1) + _EPS)).float()
    y = x * rstd[:, None] * s["gamma"].float()
    if case["out"] == I8:
        scales = y.abs().amax(dim=1) / 127.0
        ok = torch.isfinite(scales) & (scales > 0)
        codes = torch.where(ok[:, None], torch.round(y / scales[:, None]), 0.0).clamp(-127, 127).to(torch.int8)
    else:
        emax, top = _FORMATS[case["out"]]
        r, c = y.shape
        blocks = torch.nn.functional.pad(y, (0, -c % 32)).reshape(r, -1, 32)
        amax = blocks.abs().amax(dim=2)
        byte = torch.where(amax > 0, torch.frexp(amax).exponent - 1 - emax, -127).clamp(-127, 127) + 127
        byte = torch.where(torch.isfinite(amax), byte, 255)
        codes = _to_codes(blocks, byte[:, :, None], case["out"]).reshape(r, -1)[:, :c].contiguous()
        scales = _bits(byte.to(torch.uint8).view(torch.int8))
    return (total, codes, scales) if case["residual"] else (codes, scales)


def _rotated(x, turn, style):
    """f32 x [rows, heads, dim], its first channels rotated by turn [rows, rot]
    (cosines, then sines): channel i with i + rot/2 ("half"), or 2 i with 2 i + 1 ("pairs")."""
    rot = turn.shape[1]
    cos, sin = turn[:, None, : rot // 2], turn[:, None, rot // 2 :]
    a, b = (x[:, :, : rot // 2], x[:, :, rot // 2 : rot]) if style == "half" else (x[:, :, 0:rot:2], x[:, :, 1:rot:2])
    first, second = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([first, second], dim=2) if style == "half" else torch.stack([first, second], dim=3).flatten(2)
    return torch.cat([turned, x[:, :, rot:]], dim=2)


def _plain_append(s):
    case = s["case"]
    kv, d, block, fmt = case["kv"], case["dim"], case["block"], case["fmt"]
    rows = (s["pos"] >= 0).nonzero()[:, 0]
    seq, pos = s["seq"][rows].long(), s["pos"][rows].long()
    qkv = s["qkv"][rows].float().reshape(len(rows), -1, d)
    q, k, v = qkv.split([case["heads"], kv, kv], dim=1)
    turn = s["rot"][pos]
    s["q"][rows] = _rotated(q, turn, case["style"]).to(s["q"].dtype)
    # the blocks that get tokens, and where the first of them goes
    blocks, which = torch.unique(s["table"][seq, pos // block].long(), return_inverse=True)
    at = pos % block
    first = torch.full(blocks.shape, block, device=pos.device).scatter_reduce(0, which, at, "amin")
    earlier = torch.arange(block, device=pos.device) < first[:, None]
    for new, codes, scales, turned in ((_rotated(k, turn, case["style"]), s["k"], s["ks"], False), (v, s["v"], s["vs"], True)):
        # NaN counts as more than any number
        size = torch.where(torch.isnan(new), float("inf"), new.abs()).amax(dim=2)
        amax = torch.zeros((len(blocks), kv), device=pos.device).scatter_reduce(0, which[:, None].expand(-1, kv), size, "amax")
        old = torch.where(first[:, None] > 0, _byte(scales)[blocks], 0)
        byte = torch.maximum(old, _scale_byte(amax, fmt))
        scales.view(torch.uint8)[blocks] = byte.to(torch.uint8)
        held = codes.view(torch.uint8)[blocks]
        held = held.transpose(2, 3).contiguous() if turned else held
        # codes that stay keep their values under a larger scale
        rescaled = held.view(_CODES[fmt]).float() * _pow2((old - byte).clamp(min=-127))[:, :, None, None]
        rescaled = torch.where((byte < 255)[:, :, None, None], rescaled, 0.0).to(_CODES[fmt]).view(torch.uint8)
        held = torch.where(earlier[:, None, :, None], rescaled, held)
        held[which, :, at] = _to_codes(new, byte[which][:, :, None], fmt).view(torch.uint8)
        codes.view(torch.uint8)[blocks] = held.transpose(2, 3).contiguous() if turned else held
    return s["q"], s["k"], _bits(s["ks"]), s["v"], _bits(s["vs"])


def _plain_attend(s):
    case = s["case"]
    heads, kv, d, block = case["heads"], case["kv"], case["dim"], case["block"]
    new, far = s["longest"]
    rows = (s["pos"] >= 0).nonzero()[:, 0]
    seq, pos = s["seq"][rows].long(), s["pos"][rows].long()
    # the sequences' rows and keys side by side
    slots = case["slots"]
    first = torch.full((slots,), 1 << 30, device=pos.device).scatter_reduce(0, seq, pos, "amin")
    place = pos - first[seq]
    at = torch.full((slots, new), -1, device=pos.device)
    at[seq, place] = pos
    q = torch.zeros((slots, new, heads, d), device=pos.device)
    q[seq, place] = s["q"][rows].float()
    group = heads // kv
    q = q.reshape(slots, new, kv, group, d).permute(0, 2, 3, 1, 4).reshape(slots, kv, group * new, d)
    table = s["table"][:, : -(-far // block)].long()
    there = (table >= 0).repeat_interleave(block, dim=1)
    table = table.clamp(min=0)

    def values(codes, scales):
        return codes.view(torch.uint8)[table].view(_CODES[case["fmt"]]).float() * _value(_byte(scales)[table])[:, :, :, None, None]

    k = values(s["k"], s["ks"]).permute(0, 2, 4, 1, 3).reshape(slots, kv, d, -1)
    v = values(s["v"], s["vs"]).permute(0, 2, 1, 4, 3).reshape(slots, kv, -1, d)
    key = torch.arange(k.shape[3], device=pos.device)
    seen = (key <= at[:, :, None]) & there[:, None, :]
    if case["window"]:
        seen &= key > at[:, :, None] - case["window"]
    v = torch.where(seen.any(dim=1)[:, None, :, None], v, 0.0)
    scores = torch.matmul(q * (1.0 / math.sqrt(d)), k).reshape(slots, kv, group, new, -1)
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(scores - scores.amax(dim=4, keepdim=True).clamp(min=-3e38))
    del scores
    total = p.sum(dim=4, keepdim=True)
    o = torch.matmul(p.reshape(slots, kv, group * new, -1), v).reshape(slots, kv, group, new, d) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(slots, new, heads, d)
    s["out"][rows] = o[seq, place].to(s["out"].dtype)
    return s["out"]


def _plain(s):
    return {"norm": _plain_norm, "append": _plain_append, "attend": _plain_attend}[s["case"]["op"]](s)


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
    if op == "norm":
        g = _group("rms_norm", _ANY_ROWS if rt else case["rows"], rt, cols=case["cols"], elem=case["type"], params=case["params"],
                   out=case["out"], residual=case["residual"], eps=_EPS)
        if case["residual"]:
            total, codes, scales = g(s["x"], s["residual"], s["gamma"], s["sum"], s["codes"], s["scales"])
            return total, codes, scales if case["out"] == I8 else _bits(scales)
        codes, scales = g(s["x"], s["gamma"], s["codes"], s["scales"])
        return codes, scales if case["out"] == I8 else _bits(scales)
    rows = _ANY_ROWS if rt else s["seq"].shape[0]
    kw = dict(heads=case["heads"], kv_heads=case["kv"], dim=case["dim"], slots=case["slots"], room=case["room"], blocks=s["k"].shape[0],
              block=case["block"], elem=case["type"], fmt=case["fmt"])
    if op == "append":
        g = _group("append_kv", rows, rt, rot=case["rot"], pairs=case["style"] == "pairs", **kw)
        q, k, ks, v, vs = g(s["qkv"], s["rot"], s["seq"], s["pos"], s["table"], s["q"], s["k"], s["ks"], s["v"], s["vs"])
        return q, k, _bits(ks), v, _bits(vs)
    g = _group("paged_attention", rows, rt, window=case["window"], **kw)
    return g(s["q"], s["k"], s["ks"], s["v"], s["vs"], s["seq"], s["pos"], s["table"], s["out"])


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    e = _WIDTH[case["type"]]
    if case["op"] == "norm":
        r, c = case["rows"], case["cols"]
        kept = 4 * r if case["out"] == I8 else r * ((c + 31) // 32)
        return {"bytes": r * c * (e * (3 if case["residual"] else 1) + 1) + kept + c * _WIDTH[case["params"]], "flops": 8 * r * c}
    lengths = _lengths(case)
    rows, heads, kv, d, block = sum(n for n, _ in lengths), case["heads"], case["kv"], case["dim"], case["block"]
    table = 4 * sum(-(-(n + p) // block) for n, p in lengths)
    if case["op"] == "append":
        turns = 4 * case["rot"] * max(n for n, _ in lengths)
        touched = sum((p + n - 1) // block - p // block + 1 for n, p in lengths)
        return {"bytes": rows * d * ((2 * heads + 2 * kv) * e + 2 * kv) + 8 * rows + turns + 4 * touched + 4 * touched * kv,
                "flops": rows * d * (3 * heads + 6 * kv)}
    seen, read = _visible(case)
    return {"bytes": 2 * rows * heads * d * e + 2 * read * kv * d + 2 * kv * table // 4 + table + 8 * rows, "flops": 4 * seen * heads * d}


# ---------------------------------------------------------------- 64 bits
def _power(e):
    """2^e in f64 for whole e in [-300, 300], from a table of exact ones."""
    return torch.tensor([2.0 ** i for i in range(-300, 301)], dtype=torch.float64, device=e.device)[e.long() + 300]


def _near(v, fmt):
    """The format's value nearest to f64 v, ties to the even code, saturated."""
    emax, top = _FORMATS[fmt]
    mant, low = (3, -6) if fmt == E4M3 else (2, -14)
    size = v.abs().clamp(min=2.0 ** low)
    lead = torch.floor(torch.log2(size))
    lead = torch.where(_power(lead + 1) <= size, lead + 1, torch.where(_power(lead) > size, lead - 1, lead))
    grid = _power(lead - mant)
    down = torch.floor(v / grid)
    rest = v / grid - down
    up = (rest > 0.5) | ((rest == 0.5) & (down % 2 != 0))
    return ((down + up) * grid).clamp(-top, top)


def _lead(x):
    """floor(log2 x) of f64 x > 0."""
    lead = torch.floor(torch.log2(x)).clamp(-250, 250)
    return torch.where(_power(lead + 1) <= x, lead + 1, torch.where(_power(lead) > x, lead - 1, lead))


def _exact_norm(case, s):
    x = s["x"].double()
    outs = []
    if case["residual"]:
        # (the sum is kept in the rows' type, and the norm is of what is kept)
        outs.append(x + s["residual"].double())
        x = (s["x"].float() + s["residual"].float()).to(s["x"].dtype).double()
    y = x * (x.square().mean(dim=1, keepdim=True) + _EPS) ** -0.5 * s["gamma"].double()
    if case["out"] == I8:
        return (*outs, None, y.abs().amax(dim=1) / 127)
    emax = _FORMATS[case["out"]][0]
    codes, scales = torch.empty_like(y), torch.empty((y.shape[0], (y.shape[1] + 31) // 32), dtype=torch.float64, device=y.device)
    for b in range(scales.shape[1]):
        part = y[:, 32 * b : 32 * b + 32]
        scale = _power((_lead(part.abs().amax(dim=1)) - emax).clamp(-127, 127))
        codes[:, 32 * b : 32 * b + 32] = _near(part / scale[:, None], case["out"])
        scales[:, b] = scale
    return (*outs, codes, scales)


def _exact_append(case, s):
    heads, kv, d, block, fmt, rot = case["heads"], case["kv"], case["dim"], case["block"], case["fmt"], case["rot"]
    emax, top = _FORMATS[fmt]
    half = rot // 2
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double().transpose(2, 3).contiguous()
    ks, vs = _power(_byte(s["ks"]) - 127), _power(_byte(s["vs"]) - 127)
    lo = torch.arange(half, device=q.device)
    lo, hi = (lo, lo + half) if case["style"] == "half" else (2 * lo, 2 * lo + 1)
    start = 0
    where = s["seq"].tolist()
    for new, past in _lengths(case):
        x = s["qkv"][start : start + new].double().reshape(new, -1, d)
        c, z = s["rot"][past : past + new, None, :half].double(), s["rot"][past : past + new, None, half:].double()
        t = x.clone()
        t[:, :, lo] = x[:, :, lo] * c - x[:, :, hi] * z
        t[:, :, hi] = x[:, :, hi] * c + x[:, :, lo] * z
        q[start : start + new] = t[:, :heads]
        ids = s["table"][where[start]].tolist()
        at = past
        while at < past + new:
            n, o, blk = min(block - at % block, past + new - at), at % block, ids[at // block]
            for codes, scales, fresh in ((k, ks, t[at - past : at - past + n, heads : heads + kv]), (v, vs, x[at - past : at - past + n, heads + kv :])):
                amax = fresh.abs().amax(dim=(0, 2))
                scale = _power(_lead(amax) - emax)
                scale = torch.where(amax > top * scale, 2 * scale, scale)
                if o > 0:
                    grown = torch.maximum(scale, scales[blk])
                    codes[blk, :, :o] = _near(codes[blk, :, :o] * (scales[blk] / grown)[:, None, None], fmt)
                    scale = grown
                codes[blk, :, o : o + n] = _near(fresh.transpose(0, 1) / scale[:, None, None], fmt)
                scales[blk] = scale
            at += n
        start += new
    return q, k, ks, v.transpose(2, 3), vs


def _exact_attend(case, s):
    heads, kv, d, block = case["heads"], case["kv"], case["dim"], case["block"]
    out, start, where = s["out"].double(), 0, s["seq"].tolist()
    for new, past in _lengths(case):
        n = past + new
        ids = s["table"][where[start], : -(-n // block)].long()
        at = torch.arange(n, device=out.device)
        seen = at[None, :] <= at[past:, None]
        if case["window"]:
            seen = seen & (at[None, :] > at[past:, None] - case["window"])
        for h in range(kv):
            k = s["k"][:, h].contiguous().view(torch.uint8)[ids].view(_CODES[case["fmt"]]).double()
            v = s["v"][:, h].contiguous().view(torch.uint8)[ids].view(_CODES[case["fmt"]]).double()
            k = (k * _power(_byte(s["ks"])[ids, h] - 127)[:, None, None]).reshape(-1, d)[:n]
            v = (v * _power(_byte(s["vs"])[ids, h] - 127)[:, None, None]).transpose(1, 2).reshape(-1, d)[:n]
            for g in range(h * heads // kv, (h + 1) * heads // kv):
                x = s["q"][start : start + new, g].double() @ k.t().contiguous() * d ** -0.5
                out[start : start + new, g] = torch.softmax(x.masked_fill(~seen, float("-inf")), dim=1) @ v
        start += new
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "append": _exact_append, "attend": _exact_attend}[case["op"]](case, s)
