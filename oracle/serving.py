"""CPU restatement of the serving ops, rms_norm, append_kv and paged_attention
(TEST INFRASTRUCTURE ONLY, as interp.py): written from the meaning that their
builders in hfusion_mi355x.groups state, apart from the kernels.  The
reference's dialect has no such ops."""
import numpy as np

from . import blockscaled as bs

F = np.float32


def rms_norm(x, residual, gamma, eps, out, store):
    """(stored sum, codes, scales) of f32 x and residual (or None); `store`
    rounds f32 to the rows' type and gives (storage, its f32 values).  Every
    step is the definition's own rounding, so the result is exact."""
    kept = None
    if residual is not None:
        with np.errstate(invalid="ignore", over="ignore"):
            kept, x = store((x + residual).astype(F))
    with np.errstate(all="ignore"):
        ms = np.square(x.astype(np.float64)).sum(axis=-1) / x.shape[-1] + eps
        rstd = (1.0 / np.sqrt(ms)).astype(F)
        y = (x * rstd[..., None]).astype(F) * gamma.astype(F)
        if out != "i8":
            codes, scales = bs.quantize(y.astype(np.float64), out, y.ndim - 1)
            return kept, codes, scales
        amax = np.abs(y).max(axis=-1)  # (NaN if any is)
        scales = amax * (F(1.0) / F(127.0))
        ok = np.isfinite(scales) & (scales > 0)
        q = np.rint(y / np.where(ok, scales, F(1.0))[..., None])
        codes = np.where(ok[..., None], np.clip(q, -127, 127), 0).astype(np.int8)
    return kept, codes, scales


def scale_byte(amax, fmt):
    """Byte of the smallest power of two that keeps amax in the format's range."""
    if not np.isfinite(amax):
        return 255
    e = -127
    while e < 127 and amax > bs.TOP[fmt] * 2.0 ** e:
        e += 1
    return e + 127


def rotate(x, turn, pairs):
    """f32 x [heads, dim] with its first channels rotated by turn [rot], each product and sum rounded to f32."""
    half = turn.size // 2
    i = np.arange(half)
    lo, hi = (2 * i, 2 * i + 1) if pairs else (i, i + half)
    c, s = turn[:half], turn[half:]
    out = x.copy()
    with np.errstate(all="ignore"):
        out[:, lo] = (x[:, lo] * c).astype(F) - (x[:, hi] * s).astype(F)
        out[:, hi] = (x[:, hi] * c).astype(F) + (x[:, lo] * s).astype(F)
    return out


def append_kv(qkv, rot, seq, pos, table, q, k, ks, v, vs, fmt, pairs, store):
    """The cache's code bits and scale bytes (uint8) and q's storage after the
    rows of f32 qkv, as new arrays."""
    q, k, ks, v, vs = (a.copy() for a in (q, k, ks, v, vs))
    blocks, kv, block, dim = k.shape
    heads = q.shape[1]
    new = {}  # block -> [(offset, keys, values)]
    for t in range(len(seq)):
        s, p = int(seq[t]), int(pos[t])
        if not (0 <= s < table.shape[0] and 0 <= p < min(table.shape[1] * block, rot.shape[0])):
            continue
        x = qkv[t].reshape(-1, dim)
        q[t] = store(rotate(x[:heads], rot[p], pairs))[0]
        b = int(table[s, p // block])
        if 0 <= b < blocks:
            new.setdefault(b, []).append((p % block, rotate(x[heads:heads + kv], rot[p], pairs), x[heads + kv:]))
    values = bs.code_values(fmt)
    for b, rows in new.items():
        first = min(o for o, _, _ in rows)
        for which, codes, scales in ((1, k, ks), (2, v, vs)):
            for h in range(kv):
                cells = codes[b, h] if which == 1 else codes[b, h].T  # [token, channel], a view
                fresh = np.stack([r[which][h] for r in rows]).astype(np.float64)
                amax = np.abs(fresh).max() if np.isfinite(fresh).all() else np.inf
                old = int(scales[b, h]) if first > 0 else 0
                now = max(old, scale_byte(amax, fmt))
                if now == 255:
                    cells[:first] = 0
                elif now != old:
                    cells[:first] = bs.encode(values[cells[:first]] * 2.0 ** (old - now), fmt)
                for (o, *_), val in zip(rows, fresh):
                    cells[o] = 0 if now == 255 else bs.encode(val * 2.0 ** (127 - now), fmt)
                scales[b, h] = now
    return q, k, ks, v, vs


def visible(p, s, table, blocks, block, window):
    """Positions that a row at position p of sequence s sees."""
    j = np.arange(max(0, p - window + 1) if window else 0, p + 1)
    b = table[s, j // block]
    return j[(b >= 0) & (b < blocks)]


def paged_attention(q, k, ks, v, vs, seq, pos, table, out, fmt, scale, window):
    """f64 result of f64 q (rows that pad the batch as in `out`), and sum p |v|
    and sum |q k| scale of each row and head's largest score error."""
    out = out.copy()
    size, reach = np.zeros_like(out), np.zeros(out.shape[:2])
    blocks, kv, block, dim = k.shape
    heads = q.shape[1]
    codes = bs.code_values(fmt)
    held = {}

    def cache(s, g, n):
        """Keys and values of the first n positions of a sequence (of blocks that it has not: of some block)."""
        if (s, g) not in held or len(held[s, g][0]) < n:
            j = np.arange(max([n] + [int(p) + 1 for s2, p in zip(seq, pos) if s2 == s and p < table.shape[1] * block]))
            b = np.clip(table[s, j // block], 0, blocks - 1)
            held[s, g] = (codes[k[b, g, j % block]] * bs.scale_values(ks[b, g])[:, None], codes[v[b, g, :, j % block]] * bs.scale_values(vs[b, g])[:, None])
        return held[s, g]
    for t in range(len(seq)):
        s, p = int(seq[t]), int(pos[t])
        if not (0 <= s < table.shape[0] and 0 <= p < table.shape[1] * block):
            continue
        j = visible(p, s, table, blocks, block, window)
        if not len(j):
            out[t] = 0
            continue
        for g in range(kv):
            key, val = (a[j] for a in cache(s, g, p + 1))
            h = slice(g * heads // kv, (g + 1) * heads // kv)
            with np.errstate(invalid="ignore"):
                x = q[t, h] @ key.T * scale
                w = np.exp(x - x.max(axis=1, keepdims=True))
                w /= w.sum(axis=1, keepdims=True)
                out[t, h] = w @ val
                size[t, h] = w @ np.abs(val)
                reach[t, h] = (np.abs(q[t, h]) @ np.abs(key).T).max(axis=1) * abs(scale)
    return out, size, reach
