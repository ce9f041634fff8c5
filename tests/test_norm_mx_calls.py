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
from test_norm_mx import check_grad, check_norm, grad_args, norm_inputs, note, stored


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
