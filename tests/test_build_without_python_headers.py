"""The C part of plain Python calls is optional: the libraries build without
Python's headers, and calls are made without it."""
import ctypes
import subprocess

import pytest

import hfusion_mi355x as hf
import group_catalog as cat
from hfusion_mi355x import native


def commands(*more):
    return subprocess.run(["make", "-n", "-B", "-C", native.PKG_ROOT, "all", *more], check=True, capture_output=True, text=True).stdout


def test_built_where_the_headers_are():
    assert "pycall.c" in commands()


def test_left_out_without_them():
    out = commands("PYTHON=false")
    assert "pycall.c" not in out and "hfr.cpp" in out and "bishengir-compile" in out


@pytest.mark.parametrize("error", [native.NativeLibraryMissing("not built"), ImportError("another Python's")])
def test_calls_without_it(monkeypatch, error):
    def missing():
        raise error
    monkeypatch.setattr(native, "hfcall", missing)
    grp = object.__new__(hf.runtime.Group)
    grp.meta, grp.func, grp._h = hf.compile(cat.get("rmsnorm_quant_256")).blocks[0], "f", ctypes.c_void_p(8)
    try:
        assert grp._make_plan() and grp._make_call() is False
    finally:
        grp._h = None


@pytest.mark.gpu
def test_same_results_without_it(gpu, monkeypatch):
    import torch
    print("[case] calls without the C part", flush=True)
    load = lambda: hf.compile(cat.get("ln_rt"), options=cat.options("ln_rt"), require_cached=True).load()  # noqa: E731
    grp = load()
    x = torch.randn(9, 1000, device=gpu).bfloat16()
    g, b = torch.rand(1000, device=gpu).bfloat16(), torch.randn(1000, device=gpu).bfloat16()

    def outs():
        return [torch.zeros([9 if d == -1 else d for d in p["shape"]], dtype=hf.runtime.torch_dtype(p["elem"]), device=gpu)
                for p in grp.meta["params"][3:]]
    want = grp(x, g, b, *outs())

    def missing():
        raise native.NativeLibraryMissing("not built")
    monkeypatch.setattr(native, "hfcall", missing)
    other = load()
    got = other(x, g, b, *outs())
    assert grp._call and other._call is False
    assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(got, want))
