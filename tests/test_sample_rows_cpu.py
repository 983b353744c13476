"""Argument checks of sampling a batch: refusals come before any device work."""
import ctypes as C

import pytest

from conftest import HAS_GPU
from tensoros_b200 import _ffi

EINVAL, ENOTSUP, ENODEV = -1, -6, -7
PTR = 1 << 20
no_gpu = pytest.mark.skipif(HAS_GPU, reason="made-up pointers; checks the no-GPU behaviour")


def sample(lib, x=0, rows=3, n=100, params=0, u=PTR, token=PTR, prob=PTR, kept=PTR):
    x = _ffi.Rows(PTR, 100, 0) if x == 0 else x
    params = _ffi.SampleParams(PTR, PTR, PTR, PTR) if params == 0 else params
    return lib.tos_sample_rows_dev(None if x is None else C.byref(x), rows, n, None if params is None else C.byref(params),
                                   u, token, prob, kept, None)


@no_gpu
def test_valid_calls_find_no_device(lib):
    assert sample(lib) == sample(lib, params=None) == sample(lib, prob=None, kept=None) == ENODEV
    assert sample(lib, params=_ffi.SampleParams(None, PTR, None, PTR)) == ENODEV
    assert sample(lib, rows=0, u=None, token=None) == sample(lib, x=_ffi.Rows(PTR, 101, 1)) == ENODEV


def test_refusals(lib):
    assert sample(lib, x=None) == sample(lib, x=_ffi.Rows(None, 100, 0)) == sample(lib, x=_ffi.Rows(PTR, 99, 0)) == EINVAL
    assert sample(lib, x=_ffi.Rows(PTR + 2, 100, 0)) == sample(lib, x=_ffi.Rows(PTR + 1, 100, 1)) == EINVAL
    assert sample(lib, rows=-1) == sample(lib, n=0) == sample(lib, n=-5) == EINVAL
    assert sample(lib, u=None) == sample(lib, token=None) == EINVAL
    for o in ("u", "token", "prob", "kept"):
        assert sample(lib, **{o: PTR + 2}) == EINVAL
    for i in range(4):
        assert sample(lib, params=_ffi.SampleParams(*[PTR + (j == i) for j in range(4)])) == EINVAL
    assert sample(lib, x=_ffi.Rows(PTR, 1 << 21, 0), n=(1 << 20) + 1) == ENOTSUP
    assert sample(lib, x=_ffi.Rows(PTR, 100, 24)) == ENOTSUP
    assert sample(lib, rows=(1 << 24) + 1) == ENOTSUP
    assert lib.tos_last_status() == ENOTSUP
