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


@pytest.mark.gpu
def test_streams_hold_what_their_launches_need(gpu):
    """A handle's workspaces by what each stream's launches use: single tokens
    less than prompts, whose own comes with the first of them; the answers are
    those of a launch with a caller's workspace of full size."""
    import torch
    import serving_catalog as sc
    from test_serving import attend_case, load
    from test_serving_calls import attend_args, same
    note("workspaces by launch")
    c = sc.ATTEND["usual"]
    rng = np.random.default_rng(3)
    few, prompt = (attend_args(c, attend_case(rng, c, parts, 0), gpu) for parts in ([(0, 3000, 1), (1, 900, 2)], [(2, 1500, 150)]))
    grp = load("pagedattn_usual_rt")
    full = grp.info.workspace_bytes
    lib = hf.native.hfr()
    need = lib.hfr_group_workspace_rows(grp._h, 3)
    assert need < full // 4 and lib.hfr_group_workspace_rows(grp._h, 150) == full
    want = []
    space = torch.zeros(full, dtype=torch.uint8, device=gpu)
    for a in (few, prompt):
        grp(*a, workspace=space)
        torch.cuda.synchronize()
        want.append(a[-1].clone())
    streams = [torch.cuda.Stream() for _ in range(4)]
    for s in streams:  # (what a stream itself holds is there before)
        with torch.cuda.stream(s):
            grp(*few, workspace=space)
        torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    for s in streams:
        few[-1].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            grp(*few)
        torch.cuda.synchronize()
        assert same(few[-1], want[0])
    # (allocations are in whole pages of 2 MiB)
    assert before - torch.cuda.mem_get_info()[0] <= len(streams) * (need + (4 << 20)) < len(streams) * full // 2
    for _ in range(2):
        for s in streams[:2]:
            for a, w in ((prompt, want[1]), (few, want[0])):
                a[-1].zero_()
                torch.cuda.synchronize()
                with torch.cuda.stream(s):
                    grp(*a)
                torch.cuda.synchronize()
                assert same(a[-1], w)
