"""What the serving ops refuse or launch at the ends of their ranges, and what
they answer there."""
import numpy as np
import pytest

import hfusion_mi355x as hf
from helpers import run_gpu
from hfusion_mi355x import groups as g
from test_norm_mx import note, stored
from test_serving import check_codes


def manifest(ir, options="dyn=runtime"):
    return open(hf.compile(ir, options=options).manifest).read().splitlines()


@pytest.mark.parametrize("heads,kv,slots", [(32, 8, 64), (32, 32, 65536), (20, 1, 1 << 22), (64, 64, 1 << 20), (1024, 1024, 1 << 20)])
def test_every_kernel_has_a_launchable_grid(heads, kv, slots):
    """At the most rows that each of the attention's kernels is taken for, less than
    2^24 workgroups of 256 threads; in any order of the kernels, every row
    count up to max_rows has one."""
    ir = g.with_dynamic_rows(g.paged_attention(7919, heads=heads, kv_heads=kv, dim=32, slots=slots, room=64, blocks=64, block=16), 7919)
    lines = [ln.split() for ln in manifest(ir)]
    most = next(int(ln[1]) for ln in lines if ln[0] == "max_rows")
    pre = []  # (workgroups, rows and workgroups besides)
    for ln in lines:
        if ln[0] == "pre":
            pre.append([int(ln[2]), 1, 0])
        elif ln[0] == "pre_rows":
            pre[-1][1:] = int(ln[1]), int(ln[2])
    alts = [ln for ln in lines if ln[0] == "alt"]
    bounds = [int(ln[2]) for ln in alts]
    assert bounds and bounds[-1] >= most and bounds == sorted(bounds)
    for ln in alts:
        rows = min(int(ln[2]), most)
        grids = [-(-rows // int(ln[3])) * int(ln[4])]
        grids += [n + -(-rows // b) * c for n, b, c in pre[int(ln[7]):][:1]] if "pre" in ln else []
        assert max(grids) < 1 << 24, (ln, grids)


def test_a_static_batch_of_many_slots():
    """A row count past the decoding kernels' grid is a prompt's."""
    size = dict(heads=32, kv_heads=32, dim=32, slots=1 << 20, room=64, blocks=64, block=16)
    for rows, kind in ((1 << 18, "units"), (1 << 21, "prompt")):
        variant = next(ln for ln in manifest(g.paged_attention(rows, **size), "") if ln.startswith("variant "))
        assert variant.split()[1].rstrip(",") == kind, (rows, variant)


@pytest.mark.parametrize("scale", [2.4e38, -3.4e38, float("inf"), float("nan")])
def test_refused_scales(scale):
    """A scale that is no f32 number any more as one of exponents of 2."""
    with pytest.raises(hf.CompileError, match="a scale that is no number"):
        hf.compile(g.paged_attention(8, heads=4, kv_heads=2, dim=32, slots=2, room=64, blocks=8, block=16, scale=scale), cache=False)


@pytest.mark.gpu
def test_norm_whose_reciprocal_overflows(gpu):
    """Rows so small that 1 / sqrt(mean) is infinite in f32 (eps 0): infinite
    scales, NaN only where a row has a zero."""
    note("norm of the smallest rows")
    c = (6, 100, "bf16", "bf16", "i8", True)
    x = np.full((6, 100), 1e-40)
    x[1] *= np.where(np.arange(100) % 3, 1, -1)
    x[2, 50] = 0
    x[3] = 1.0
    xs, xv = stored(x, "bf16")
    gs, gm = stored(np.ones(100), "bf16")
    zero = np.zeros_like(xs)
    got = run_gpu("rmsnorm_eps0", [xs, zero, gs, zero, np.zeros((6, 100), np.int8), np.zeros(6, np.float32)], gpu)
    check_codes(c, got, xv.astype(np.float32), np.zeros((6, 100), np.float32), gm, 0.0)
    assert np.isinf(got[-1][[0, 1, 4, 5]]).all() and np.isnan(got[-1][2]) and np.isfinite(got[-1][3])
