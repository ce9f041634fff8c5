"""The plain call of a group (csrc/runtime/pycall.c): which arguments it
takes, what it passes on and returns, with stand-ins for tensors and for the
launch; on the GPU the same call against one made through a launcher."""
import ctypes

import numpy as np
import pytest

import hfusion_mi355x as hf
import group_catalog as cat
from hfusion_mi355x import native

LAUNCH = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.POINTER(ctypes.c_uint64), ctypes.c_size_t,
                          ctypes.POINTER(ctypes.c_void_p), ctypes.c_size_t, ctypes.c_void_p, ctypes.c_void_p)
LAUNCH_ROWS = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.POINTER(ctypes.c_uint64), ctypes.c_size_t,
                               ctypes.POINTER(ctypes.c_void_p), ctypes.c_size_t, ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p)
F32, BF16 = object(), object()


class Fake:
    def __init__(self, dtype, shape, ptr, cuda=True, dense=True, device=0):
        self.dtype, self.shape, self.is_cuda = dtype, tuple(shape), cuda
        self._ptr, self._dense, self._device = ptr, dense, device

    def is_contiguous(self):
        return self._dense

    def data_ptr(self):
        return self._ptr

    def get_device(self):
        return self._device


def make(specs, tied, dyn=False, rc=0):
    seen = []

    def launch(h, slots, n, results, nr, *rest):
        rows = rest[0] if dyn else None
        seen.append(dict(h=h, slots=[slots[i] for i in range(n)], nr=nr, results=[results[i] for i in range(nr)], rows=rows,
                         ws=rest[-2], stream=rest[-1]))
        return rc
    fn = (LAUNCH_ROWS if dyn else LAUNCH)(launch)
    call = native.hfcall().plan(ctypes.cast(fn, ctypes.c_void_p).value, 0x55, dyn, Fake, lambda dev: 0x1000 + dev, specs, tied)
    call_keep.append(fn)
    return call, seen


call_keep = []


def test_passes_and_returns():
    call, seen = make(((F32, (4, 3)), (BF16, (3,)), (F32, (4, 3))), (2,))
    a, b, o = Fake(F32, (4, 3), 0x10, device=2), Fake(BF16, (3,), 2 ** 63 + 8), Fake(F32, (4, 3), 0x30)
    assert call(a, b, o) is o
    assert seen == [dict(h=0x55, slots=[0x10, 2 ** 63 + 8, 0x30], nr=1, results=[None], rows=None, ws=None, stream=0x1002)]
    two, _ = make(((F32, (4, 3)), (BF16, (3,)), (F32, (4, 3))), (2, 0))
    assert two(a, b, o) == (o, a)


@pytest.mark.parametrize("change", [dict(dtype=BF16), dict(shape=(3, 4)), dict(shape=(4, 3, 1)), dict(shape=(12,)), dict(cuda=False), dict(dense=False)])
def test_does_not_take(change):
    call, seen = make(((F32, (4, 3)), (F32, (4, 3))), (1,))
    kw = dict(dtype=F32, shape=(4, 3), ptr=0x10)
    ok = Fake(**kw)
    assert call(ok, Fake(**{**kw, **change})) is None and call(Fake(**{**kw, **change}), ok) is None
    assert call(ok) is None and call(ok, ok, ok) is None and call(ok, 3.0) is None and not seen

    class Sub(Fake):
        pass
    assert call(ok, Sub(**kw)) is None and not seen


def test_launch_time_rows():
    call, seen = make(((F32, (-1, 3)), (BF16, (3,)), (F32, (-1,))), (2,), dyn=True)
    x, g = Fake(F32, (7, 3), 1), Fake(BF16, (3,), 2)
    assert call(x, g, Fake(F32, (7,), 3)) is not None and seen[-1]["rows"] == 7
    assert call(x, g, Fake(F32, (6,), 3)) is None and call(Fake(F32, (7, 4), 1), g, Fake(F32, (7,), 3)) is None and len(seen) == 1
    assert call(Fake(F32, (0, 3), 0), g, Fake(F32, (0,), 0)) is not None and seen[-1]["rows"] == 0


def test_error_code_and_python_errors():
    call, _ = make(((F32, (1,)),), (0,), rc=-2)
    assert call(Fake(F32, (1,), 1)) == -2
    broken = Fake(F32, (1,), 1)
    del broken.is_cuda
    with pytest.raises(AttributeError):
        call(broken)
    with pytest.raises(OverflowError):
        call(Fake(F32, (2 ** 70,), 1))


def test_refused_plans():
    plan = native.hfcall().plan
    spec = ((F32, (1,)),)
    for bad in ((0, 1, False, Fake, id, spec, (0,)), (1, 0, False, Fake, id, spec, (0,)), (1, 1, False, Fake, id, (), (0,)),
                (1, 1, False, Fake, id, spec, ()), (1, 1, False, Fake, id, spec, (-1,)), (1, 1, False, Fake, id, spec, (1,)),
                (1, 1, False, Fake, id, ((F32, (1,) * 9),), (0,)), (1, 1, False, Fake, id, spec * 25, (0,))):
        with pytest.raises(ValueError):
            plan(*bad)


def test_under_capture():
    """A group with a workspace leaves a captured call to the Python path."""
    seen, state = [], [False]

    def launch(*a):
        seen.append(a[0])
        return 0
    fn = LAUNCH(launch)
    call_keep.append(fn)
    call = native.hfcall().plan(ctypes.cast(fn, ctypes.c_void_p).value, 0x55, False, Fake, lambda dev: 0, ((F32, (4,)),), (0,),
                                lambda: state[0])
    a = Fake(F32, (4,), 0x10)
    assert call(a) is a and len(seen) == 1
    state[0] = True
    assert call(a) is None and len(seen) == 1

    def broken():
        raise OSError("capture")
    call = native.hfcall().plan(ctypes.cast(fn, ctypes.c_void_p).value, 0x55, False, Fake, lambda dev: 0, ((F32, (4,)),), (0,), broken)
    with pytest.raises(OSError, match="capture"):
        call(a)


@pytest.mark.gpu
def test_same_as_a_launcher(gpu):
    import torch
    print("[case] plain calls", flush=True)
    grp = hf.compile(cat.get("rmsnorm_quant_256"), require_cached=True).load()
    x = torch.randn(256, 4096, device=gpu).bfloat16()
    gm = torch.rand(4096, device=gpu).bfloat16()
    out = [(torch.zeros(256, 4096, dtype=torch.int8, device=gpu), torch.zeros(256, device=gpu)) for _ in range(2)]
    q, s = grp(x, gm, *out[0])
    assert q is out[0][0] and s is out[0][1] and grp._call
    grp.launcher(x, gm, *out[1])()
    torch.cuda.synchronize()
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    # what the plain call does not take is refused with the reason
    for bad, why in (((x.cpu(), gm, *out[0]), "device tensor"), ((x.float(), gm, *out[0]), "expected contiguous"),
                     ((x.t(), gm, *out[0]), "expected contiguous"), ((x, gm, out[0][0]), "takes 4 arguments")):
        with pytest.raises((TypeError, ValueError), match=why):
            grp(*bad)
    # on the stream that is current
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out[0][0].zero_()
        grp(x, gm, *out[0])
    side.synchronize()
    assert np.array_equal(out[0][0].cpu().numpy(), out[1][0].cpu().numpy())
