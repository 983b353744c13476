"""Argument checks of the 8-bit paged cache's operators: refusals come before
any device work, so they run without a GPU; a call that passes them reports
TOS_ENODEV here."""
import ctypes as C

import pytest

from conftest import HAS_GPU
from tensoros_b200 import _ffi

OK, EINVAL, ENOTSUP, ENODEV = 0, -1, -6, -7
PTR = 1 << 20          # never read: every call here is refused first, or finds no device
no_gpu = pytest.mark.skipif(HAS_GPU, reason="made-up pointers; checks the no-GPU behaviour")


def kv(**o):
    a = dict(k=PTR, v=PTR, k_scale=PTR, v_scale=PTR, type=24, block=16, n_pages=8, page_size=32, n_kv=2, head_dim=64,
             table=PTR, n_seqs=3, table_stride=4)
    a.update(o)
    return _ffi.Paged8Kv(**a)


def rows(heads=4, hd=64, type=0, **o):
    a = dict(ptr=PTR, stride=heads * hd, type=type)
    a.update(o)
    return _ffi.Rows(**a)


def ref(x):
    return None if x is None else C.byref(x)


def append(lib, c=None, k=None, v=None, cu=PTR, kl=PTR, n=2, total=8):
    c, k, v = c or kv(), k or rows(2), v or rows(2)
    return lib.tos_kv_append_paged8_dev(ref(c), ref(k), ref(v), cu, kl, n, total, None)


def read(lib, c=None, k=0, v=0, cu=PTR, kl=PTR, n=2, total=8):
    c, k, v = c or kv(), rows(2) if k == 0 else k, rows(2) if v == 0 else v
    return lib.tos_kv_read_paged8_dev(ref(c), ref(k), ref(v), cu, kl, n, total, None)


def prompt(lib, out=None, q=None, c=None, cu=PTR, kl=PTR, n=2, total=8, mq=5, tk=60, mk=40, heads=4, scale=0.1, ws=PTR,
           wsb=1 << 40):
    out, q, c = out or rows(ptr=2 * PTR), q or rows(), c or kv()
    return lib.tos_attention_prompt_paged8_dev(ref(out), ref(q), ref(c), cu, kl, n, total, mq, tk, mk, heads, scale, ws,
                                               wsb, None)


def decode(lib, out=None, q=None, c=None, kl=PTR, n=2, mk=4000, heads=4, scale=0.1, ws=PTR, wsb=1 << 40):
    out, q, c = out or rows(ptr=2 * PTR), q or rows(), c or kv()
    return lib.tos_attention_decode_paged8_dev(ref(out), ref(q), ref(c), kl, n, mk, heads, scale, ws, wsb, None)


@no_gpu
def test_valid_calls_find_no_device(lib):
    assert append(lib) == read(lib) == prompt(lib) == decode(lib) == ENODEV
    assert read(lib, k=None) == read(lib, v=None) == ENODEV
    assert append(lib, n=0, cu=None, kl=None) == ENODEV
    assert prompt(lib, n=0, cu=None, kl=None, ws=None, wsb=0) == ENODEV
    assert decode(lib, n=0, kl=None, ws=None, wsb=0) == ENODEV
    assert append(lib, c=kv(type=64, block=1)) == ENODEV


@pytest.mark.parametrize("o", [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(table=None),
                               dict(n_pages=0), dict(page_size=0), dict(n_kv=0), dict(head_dim=0), dict(n_seqs=-1),
                               dict(table_stride=0), dict(k=PTR + 8), dict(v=PTR + 1), dict(k_scale=PTR + 2),
                               dict(v_scale=PTR + 1), dict(table=PTR + 2), dict(block=0), dict(block=-16),
                               dict(block=3, page_size=48), dict(block=64), dict(block=32, page_size=48)])
def test_cache_refusals(lib, o):
    for f in (append, read, prompt, decode):
        assert f(lib, c=kv(**o)) == EINVAL
    assert lib.tos_last_status() == EINVAL


@pytest.mark.parametrize("o", [dict(type=0), dict(type=1), dict(type=8), dict(head_dim=258), dict(block=2048, page_size=2048)])
def test_cache_unsupported(lib, o):
    for f in (append, read, prompt, decode):
        assert f(lib, c=kv(**o)) == ENOTSUP


@pytest.mark.parametrize("o", [dict(ptr=None), dict(stride=2 * 64 - 1), dict(ptr=PTR + 2), dict(stride=-256)])
def test_row_refusals(lib, o):
    assert append(lib, k=rows(2, **o)) == EINVAL and append(lib, v=rows(2, **o)) == EINVAL
    assert read(lib, k=rows(2, **o)) == EINVAL and read(lib, v=rows(2, **o)) == EINVAL
    assert prompt(lib, q=rows(**o)) == EINVAL and decode(lib, out=rows(**o)) == EINVAL


def test_call_refusals(lib):
    for f in (append, read, prompt):
        assert f(lib, cu=None) == EINVAL and f(lib, cu=PTR + 2) == EINVAL
        assert f(lib, total=-1) == EINVAL
    for f in (append, read, prompt, decode):
        assert f(lib, kl=None) == EINVAL and f(lib, kl=PTR + 1) == EINVAL
        assert f(lib, n=-1) == EINVAL and f(lib, n=4) == EINVAL      # the table has 3 rows
        assert f(lib, c=kv(n_seqs=70000), n=70000) == ENOTSUP
    assert read(lib, k=None, v=None) == EINVAL
    assert append(lib, v=rows(2, type=1)) == ENOTSUP and read(lib, v=rows(2, type=1)) == ENOTSUP
    assert append(lib, k=rows(2, type=24), v=rows(2, type=24)) == ENOTSUP
    assert append(lib, total=(1 << 30) + 1) == ENOTSUP
    for f in (prompt, decode):
        assert f(lib, heads=3) == EINVAL and f(lib, heads=0) == EINVAL
        assert f(lib, scale=float("nan")) == EINVAL and f(lib, scale=3e38) == EINVAL
        assert f(lib, out=rows(), q=rows()) == EINVAL                # the same rows
        assert f(lib, out=rows(type=1, ptr=2 * PTR)) == ENOTSUP
        assert f(lib, mk=-1) == EINVAL and f(lib, mk=(1 << 25) + 1) == ENOTSUP
        assert f(lib, ws=None) == EINVAL and f(lib, ws=PTR + 16) == EINVAL
    assert prompt(lib, mq=-1) == EINVAL and prompt(lib, tk=-1) == EINVAL
    assert prompt(lib, tk=(1 << 32) + 1) == ENOTSUP and prompt(lib, mq=1 << 30) == ENOTSUP
    odd = dict(c=kv(head_dim=40, n_seqs=200), q=rows(4, 40), out=rows(4, 40, ptr=2 * PTR))
    assert decode(lib, n=200, mk=1 << 25, **odd) == ENOTSUP          # an fp16 copy of 2^32.6 keys


def test_workspaces(lib):
    f, g = lib.tos_attention_decode_paged8_workspace_bytes, lib.tos_attention_prompt_paged8_workspace_bytes
    assert f(0, 10, 4, 2, 64) == 0 and f(2, -1, 4, 2, 64) == 0 and f(2, 10, 3, 2, 64) == 0 and f(2, 10, 4, 2, 300) == 0
    assert g(0, 4, 4, 9, 9, 4, 2, 64) == 0 and g(2, 4, 4, -1, 9, 4, 2, 64) == 0
    assert f(2, 10, 4, 2, 64) == 0                                   # one piece: none
    need = f(2, 4000, 4, 2, 64)
    assert need > 0 and decode(lib, wsb=need - 1) == EINVAL
    need = g(2, 8, 5, 60, 40, 4, 2, 64)
    assert need >= 60 * 2 * 64 * 4 and prompt(lib, wsb=need - 1) == EINVAL
    # offsets are 64-bit: a hundred million keys
    assert g(1, 8, 8, 10 ** 8, 1 << 25, 64, 8, 128) > 10 ** 8 * 8 * 128 * 4
