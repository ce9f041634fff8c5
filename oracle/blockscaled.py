"""CPU restatement of the block-scaled and layer-norm ops (TEST
INFRASTRUCTURE ONLY, as interp.py): the formulas in 64 bits, written apart
from the kernels.  The reference's dialect has no such ops; the meaning is the
one their builders in hfusion_mi355x.groups state."""
import numpy as np

EMAX = {"e2m1": 2, "e4m3": 8, "e5m2": 15}
TOP = {"e2m1": 6.0, "e4m3": 448.0, "e5m2": 57344.0}
FORMAT = {1: "e5m2", 2: "e4m3", 3: "e2m1"}


def code_values(fmt):
    """The value of every code (index: the bits), NaN and infinities included."""
    if fmt == "e2m1":
        v = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
        return np.concatenate([v, -v])
    mant = 3 if fmt == "e4m3" else 2
    bias = 7 if fmt == "e4m3" else 15
    b = np.arange(128)
    e, m = b >> mant, b & ((1 << mant) - 1)
    v = np.where(e == 0, m * 2.0 ** (1 - bias - mant), (1 + m / 2.0 ** mant) * 2.0 ** (e - bias))
    if fmt == "e4m3":
        v[127] = np.nan
    else:
        v[124:] = [np.inf, np.nan, np.nan, np.nan]
    return np.concatenate([v, -v])


def encode(v, fmt):
    """Bits of the code nearest to v (ties to the even code), saturated."""
    mags = code_values(fmt)[: 8 if fmt == "e2m1" else 127 if fmt == "e4m3" else 124]
    a = np.minimum(np.abs(v), TOP[fmt])
    hi = np.clip(np.searchsorted(mags, a), 0, len(mags) - 1)
    lo = np.maximum(hi - 1, 0)
    up, down = mags[hi] - a, a - mags[lo]
    pick = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    sign = np.signbit(v).astype(np.int64) * (8 if fmt == "e2m1" else 128)
    return (pick + sign).astype(np.uint8)


def scale_values(b):
    b = np.asarray(b).view(np.uint8).astype(np.int64)
    return np.where(b == 255, np.nan, np.ldexp(1.0, b - 127))


def quantize(x, fmt, axis):
    """f64 x -> (code bits, unpacked, one per element; scale bytes)."""
    t = x if axis == x.ndim - 1 else x.T
    k = t.shape[-1]
    nb = (k + 31) // 32
    pad = np.zeros(t.shape[:-1] + (nb * 32,))
    pad[..., :k] = t
    blk = pad.reshape(t.shape[:-1] + (nb, 32))
    with np.errstate(invalid="ignore"):
        amax = np.abs(blk).max(axis=-1)
    bad = ~np.isfinite(blk).all(axis=-1)
    amax = np.where(bad, 1.0, amax)
    e = np.where(amax > 0, np.frexp(amax)[1] - 1 - EMAX[fmt], -127)
    e = np.clip(e, -127, 127)
    with np.errstate(invalid="ignore"):
        codes = encode(np.where(bad[..., None], 0.0, blk) * np.ldexp(1.0, -e)[..., None], fmt)
    codes = codes.reshape(pad.shape)[..., :k]
    scales = np.where(bad, 255, e + 127).astype(np.uint8)
    return (codes if axis == x.ndim - 1 else np.ascontiguousarray(codes.T)), scales


def pack(codes, axis):
    """e2m1 codes, two a byte along the axis, the even one in the low half."""
    a = np.moveaxis(codes, axis, -1)
    return np.ascontiguousarray(np.moveaxis(a[..., 0::2] | (a[..., 1::2] << 4), -1, axis))


def unpack(b, axis):
    a = np.moveaxis(np.asarray(b).view(np.uint8), axis, -1)
    return np.ascontiguousarray(np.moveaxis(np.stack([a & 15, a >> 4], axis=-1).reshape(a.shape[:-1] + (-1,)), -1, axis))


def dequantize(codes, scales, fmt, axis):
    """f64 values of codes (packed for e2m1) and scale bytes."""
    bits = unpack(codes, axis) if fmt == "e2m1" else np.asarray(codes).view(np.uint8)
    v = code_values(fmt)[bits]
    s = scale_values(scales)
    if axis == v.ndim - 1:
        return v * np.repeat(s, 32, axis=-1)[..., : v.shape[-1]]
    return v * np.repeat(s, 32, axis=1)[:, : v.shape[0]].T


def layer_norm(x, gamma, beta, eps):
    mean = x.mean(axis=-1)
    var = ((x - mean[..., None]) ** 2).mean(axis=-1)
    rstd = 1.0 / np.sqrt(var + eps)
    y = (x - mean[..., None]) * rstd[..., None]
    if gamma is not None:
        y = y * gamma
    if beta is not None:
        y = y + beta
    return y, mean, rstd


def layer_norm_grad(dy, x, gamma, mean, rstd):
    xh = (x - mean[..., None]) * rstd[..., None]
    g = dy if gamma is None else dy * gamma
    m0, m1 = g.mean(axis=-1, keepdims=True), (g * xh).mean(axis=-1, keepdims=True)
    dx = rstd[..., None] * (g - m0 - xh * m1)
    axes = tuple(range(dy.ndim - 1))
    return dx, (dy * xh).sum(axis=axes), dy.sum(axis=axes)
