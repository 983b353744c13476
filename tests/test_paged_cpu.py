"""Argument checks of the paged-cache operators: refusals come before any
device work, so they run without a GPU; a call that passes them reports
TOS_ENODEV here."""
import ctypes as C

import pytest

from conftest import HAS_GPU
from tensoros_b200 import _ffi

OK, EINVAL, ENOTSUP, ENODEV = 0, -1, -6, -7
PTR = 1 << 20          # never read: every call here is refused first, or finds no device
no_gpu = pytest.mark.skipif(HAS_GPU, reason="made-up pointers; checks the no-GPU behaviour")


def kv(**o):
    a = dict(k=PTR, v=PTR, type=1, n_pages=8, page_size=16, n_kv=2, head_dim=64, table=PTR, n_seqs=3, table_stride=4)
    a.update(o)
    return _ffi.PagedKv(**a)


def rows(heads=4, hd=64, type=0, **o):
    a = dict(ptr=PTR, stride=heads * hd, type=type)
    a.update(o)
    return _ffi.Rows(**a)


def ref(x):
    return None if x is None else C.byref(x)


def prompt(lib, out=None, q=None, c=None, cu=PTR, kl=PTR, n=2, total=8, mq=5, mk=40, heads=4, scale=0.1, ws=PTR,
           wsb=1 << 30):
    out, q, c = out or rows(ptr=2 * PTR), q or rows(), c or kv()
    return lib.tos_attention_prompt_paged_dev(ref(out), ref(q), ref(c), cu, kl, n, total, mq, mk, heads, scale, ws,
                                              wsb, None)


def decode(lib, out=None, q=None, c=None, kl=PTR, n=2, mk=4000, pt=PTR, pl=50, heads=4, scale=0.1, ws=PTR,
           wsb=1 << 30):
    out, q, c = out or rows(ptr=2 * PTR), q or rows(), c or kv()
    return lib.tos_attention_decode_paged_dev(ref(out), ref(q), ref(c), kl, n, mk, pt, pl, heads, scale, ws, wsb, None)


def append(lib, c=None, k=None, v=None, q=None, qo=None, n=3, heads=0, seq=PTR, slot=PTR, pos=PTR, qn=None, kn=None,
           eps=1e-6):
    c, k, v = c or kv(), k or rows(2), v or rows(2)
    return lib.tos_kv_append_paged_dev(ref(c), ref(k), ref(v), ref(q), ref(qo), n, heads, seq, slot, pos, qn, kn, eps,
                                       None, None)


def norm(lib, q=None, qo=None, k=None, ko=None, n=3, heads=4, n_kv=0, hd=64, qn=PTR, kn=None, eps=1e-6):
    q, qo = q or rows(), qo or rows()
    return lib.tos_qk_norm_rotary_dev(ref(q), ref(qo), ref(k), ref(ko), n, heads, n_kv, hd, qn, kn, eps, None, None,
                                      None)


@no_gpu
def test_valid_calls_find_no_device(lib):
    h = C.c_void_p()
    d = _ffi.RotaryDesc(rot_dim=64, base=10000.0, factor=1.0)
    assert lib.tos_rotary_create(C.byref(h), C.byref(d)) == ENODEV
    assert prompt(lib) == decode(lib) == append(lib) == norm(lib) == ENODEV
    assert prompt(lib, n=0, cu=None, kl=None) == ENODEV
    assert decode(lib, pl=0, pt=None) == ENODEV
    assert norm(lib, k=rows(2), ko=rows(2), n_kv=2) == ENODEV
    assert append(lib, q=rows(), qo=rows(type=1, ptr=2 * PTR), heads=4) == ENODEV


@pytest.mark.parametrize("o", [dict(k=None), dict(v=None), dict(table=None), dict(n_pages=0), dict(page_size=0),
                               dict(n_kv=0), dict(head_dim=0), dict(n_seqs=-1), dict(table_stride=0),
                               dict(k=PTR + 1), dict(table=PTR + 2)])
def test_cache_refusals(lib, o):
    assert prompt(lib, c=kv(**o)) == EINVAL
    assert decode(lib, c=kv(**o)) == EINVAL
    assert append(lib, c=kv(**o)) == EINVAL
    assert lib.tos_last_status() == EINVAL


@pytest.mark.parametrize("o", [dict(type=2), dict(type=8), dict(head_dim=258)])
def test_cache_unsupported(lib, o):
    assert prompt(lib, c=kv(**o)) == ENOTSUP
    assert decode(lib, c=kv(**o)) == ENOTSUP


@pytest.mark.parametrize("o", [dict(ptr=None), dict(stride=4 * 64 - 1), dict(ptr=PTR + 2), dict(stride=-256)])
def test_row_refusals(lib, o):
    assert prompt(lib, q=rows(**o)) == EINVAL
    assert decode(lib, out=rows(**o)) == EINVAL
    assert norm(lib, q=rows(**o)) == EINVAL
    assert norm(lib, qo=rows(**o)) == EINVAL
    o = dict(o)
    if "stride" in o:
        o["stride"] = 2 * 64 - 1
    assert append(lib, k=rows(2, **o)) == EINVAL
    assert append(lib, v=rows(2, **o)) == EINVAL


def test_attention_refusals(lib):
    assert prompt(lib, heads=3) == EINVAL                       # not a multiple of n_kv
    assert prompt(lib, heads=0) == EINVAL
    assert prompt(lib, scale=float("nan")) == EINVAL
    assert prompt(lib, n=4) == EINVAL                           # the table has 3 rows
    assert prompt(lib, cu=None) == EINVAL
    assert prompt(lib, kl=None) == EINVAL
    assert prompt(lib, cu=PTR + 1) == EINVAL
    for o in ("n", "total", "mq", "mk"):
        assert prompt(lib, **{o: -1}) == EINVAL
    assert prompt(lib, out=rows(), q=rows()) == EINVAL          # the same rows
    assert prompt(lib, out=rows(type=1, ptr=2 * PTR)) == ENOTSUP
    assert decode(lib, n=4) == EINVAL
    assert decode(lib, mk=-1) == EINVAL
    assert decode(lib, pl=-1) == EINVAL
    assert decode(lib, pt=None) == EINVAL
    assert decode(lib, kl=None) == EINVAL
    need = lib.tos_attention_decode_paged_workspace_bytes(2, 4000, 50, 4, 2, 64)
    assert need > 0
    assert decode(lib, wsb=need - 1) == EINVAL
    assert decode(lib, ws=None) == EINVAL
    assert decode(lib, ws=PTR + 8) == EINVAL


def test_attention_limits(lib):
    """What 32-bit counts of rows, the joining grid and the kernels' waits do not hold."""
    assert prompt(lib, mk=(1 << 25) + 1) == ENOTSUP
    assert prompt(lib, mq=1 << 30, heads=4) == ENOTSUP
    assert prompt(lib, c=kv(n_seqs=70000), n=70000) == ENOTSUP
    assert decode(lib, mk=(1 << 25) + 1) == ENOTSUP
    assert decode(lib, pl=(1 << 25) + 1) == ENOTSUP
    assert decode(lib, c=kv(n_seqs=70000), n=70000) == ENOTSUP
    assert decode(lib, scale=3e38) == EINVAL


def test_workspace_sizes(lib):
    f = lib.tos_attention_decode_paged_workspace_bytes
    assert f(0, 10, 0, 4, 2, 64) == 0 and f(2, -1, 0, 4, 2, 64) == 0 and f(2, 10, 0, 3, 2, 64) == 0
    assert f(2, 10, 0, 4, 2, 300) == 0
    assert lib.tos_attention_prompt_paged_workspace_bytes(0, 10, 10, 10, 4, 2, 64) == 0


def test_append_refusals(lib):
    assert append(lib, seq=None) == EINVAL
    assert append(lib, slot=None) == EINVAL
    assert append(lib, n=-1) == EINVAL
    assert append(lib, heads=4) == EINVAL                       # heads without q
    assert append(lib, q=rows(), qo=rows()) == EINVAL           # q without heads
    assert append(lib, c=kv(head_dim=33), k=rows(2, 33), v=rows(2, 33)) == EINVAL
    assert append(lib, v=rows(2, type=1)) == ENOTSUP            # k and v of two types
    assert append(lib, kn=PTR, eps=-1.0) == EINVAL
    assert append(lib, kn=PTR, eps=float("inf")) == EINVAL


def test_norm_refusals(lib):
    assert norm(lib, hd=63) == EINVAL
    assert norm(lib, hd=0) == EINVAL
    assert norm(lib, n=-1) == EINVAL
    assert norm(lib, n_kv=2) == EINVAL                          # heads without k
    assert norm(lib, qo=rows(type=1)) == EINVAL                 # in place with another type
    assert norm(lib, hd=258, q=rows(hd=258), qo=rows(hd=258)) == ENOTSUP
    assert norm(lib, q=rows(type=2), qo=rows(type=2)) == ENOTSUP
    assert norm(lib, eps=float("nan")) == EINVAL


@pytest.mark.parametrize("o", [dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=258), dict(layout=2), dict(base=0.0),
                               dict(base=float("nan")), dict(scaling=3), dict(scaling=1, factor=0.5),
                               dict(scaling=2, factor=2.0, orig_ctx=0, beta_fast=32.0, beta_slow=1.0),
                               dict(scaling=2, factor=2.0, orig_ctx=4096, beta_fast=1.0, beta_slow=1.0),
                               dict(scaling=2, factor=2.0, orig_ctx=4096, beta_fast=32.0, beta_slow=1.0, base=1.0)])
def test_rotary_refusals(lib, o):
    a = dict(rot_dim=64, layout=0, base=10000.0, scaling=0, factor=1.0, attn_factor=1.0)
    a.update(o)
    d, h = _ffi.RotaryDesc(**a), C.c_void_p()
    assert lib.tos_rotary_create(C.byref(h), C.byref(d)) == EINVAL and not h.value


def test_rotary_factor_refusals(lib):
    h = C.c_void_p()
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        ff = (C.c_float * 4)(1.0, 1.0, bad, 1.0)
        d = _ffi.RotaryDesc(rot_dim=8, base=10000.0, factor=1.0, freq_factors=C.cast(ff, C.c_void_p))
        assert lib.tos_rotary_create(C.byref(h), C.byref(d)) == EINVAL
    assert lib.tos_rotary_create(None, C.byref(d)) == EINVAL
    assert lib.tos_rotary_create(C.byref(h), None) == EINVAL
    lib.tos_rotary_destroy(None)


@pytest.mark.parametrize("scaling", [2, 3])
@pytest.mark.parametrize("o", [dict(orig_ctx=0), dict(beta_fast=1.0), dict(beta_slow=0.0), dict(base=1.0),
                               dict(factor=0.5), dict(attn_factor=float("inf"))])
def test_yarn_refusals(lib, scaling, o):
    a = dict(rot_dim=64, layout=0, base=10000.0, scaling=scaling, factor=2.0, orig_ctx=4096, beta_fast=32.0,
             beta_slow=1.0, attn_factor=1.0)
    a.update(o)
    d, h = _ffi.RotaryDesc(**a), C.c_void_p()
    assert lib.tos_rotary_create(C.byref(h), C.byref(d)) == EINVAL and not h.value


def test_token_arrays_are_aligned(lib):
    """Sequences, slots and positions are read as ints."""
    for o in ("seq", "slot", "pos"):
        for off in (1, 2, 3):
            assert append(lib, **{o: PTR + off}) == EINVAL, o
    q, qo = rows(), rows(ptr=2 * PTR)
    for off in (1, 2, 3):
        assert lib.tos_qk_norm_rotary_dev(ref(q), ref(qo), None, None, 3, 4, 0, 64, None, None, 0.0, None, PTR + off,
                                          None) == EINVAL
