"""Reading back, and the prompts' copy, at sizes where a CTA takes its most rows."""
import ctypes as C

import pytest
import torch

import paged8_ref as P
import paged_ref as R
from paged8_ref import I8, Cache8

pytestmark = pytest.mark.gpu


def big_cache(n, n_kv, hd):
    """One sequence of n rows in shuffled pages of 16, random bytes, scales of 1 and 2."""
    c = Cache8([0], 16, 16, n_kv, hd, I8, room=n)
    j = torch.arange(c.ks.numel(), device="cuda").view(c.ks.shape)
    c.ks.copy_(1.0 + (j * 7 % 3 == 0))
    c.vs.copy_(1.0 + (j * 5 % 3 == 0))
    c.lens = [n]
    return c


def reader(gpu, c, n):
    """A call that reads n rows back as fp16, and where they go."""
    k, v = (torch.empty(n, c.n_kv, c.hd, dtype=torch.float16, device="cuda") for _ in range(2))
    d, rk, rv, cu, kl = c.desc(), R.rows(k), R.rows(v), P.packed([n]), P.ints([n])

    def call():
        assert gpu.tos_kv_read_paged8_dev(C.byref(d), C.byref(rk), C.byref(rv), cu.data_ptr(), kl.data_ptr(), 1, n,
                                          R.stream()) == 0
    return call, k, v


def copier(gpu, c, n):
    """A prompt call of one token, nearly all of it the copy."""
    q = torch.randn(1, c.n_kv, c.hd, dtype=torch.float16, device="cuda")
    out = torch.empty_like(q)
    size = gpu.tos_attention_prompt_paged8_workspace_bytes(1, 1, 1, n, n, c.n_kv, c.n_kv, c.hd)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    d, ro, rq, cu, kl = c.desc(), R.rows(out), R.rows(q), P.packed([1]), P.ints([n])

    def call():
        assert gpu.tos_attention_prompt_paged8_dev(C.byref(ro), C.byref(rq), C.byref(d), cu.data_ptr(), kl.data_ptr(), 1, 1,
                                                   1, n, n, c.n_kv, 0.1, ws.data_ptr(), size, R.stream()) == 0
    return call, q, out


def best_us(call, n=8):
    times = []
    for _ in range(n + 3):
        a, b = torch.cuda.Event(True), torch.cuda.Event(True)
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        times.append(1e3 * a.elapsed_time(b))
    return min(times[3:])


@pytest.mark.parametrize("n_kv,hd,n", [(32, 128, 38000), (64, 128, 19100), (5, 48, 38000), (32, 256, 19100), (40, 128, 38000)])
def test_rows_of_large_calls(gpu, n_kv, hd, n):
    c = big_cache(n, n_kv, hd)
    call, k, v = reader(gpu, c, n)
    call()
    torch.cuda.synchronize()
    for x, pool in ((k, "k"), (v, "v")):
        for at in range(0, n, 4000):
            m = min(4000, n - at)
            assert torch.equal(x[at:at + m].double(), c.rows_at(0, at, at + m, pool)), (pool, at)


@pytest.mark.parametrize("n_kv,hd,n", [(32, 128, 37888), (64, 128, 18944), (32, 256, 18944)])
@pytest.mark.parametrize("what", [reader, copier])
def test_a_few_rows_more_do_not_take_several_times_as_long(gpu, what, n_kv, hd, n):
    """Around the sizes where a CTA's rows double, 5% more rows take no more than
    twice the time (they took 8 times where rows went an element a lane from there on)."""
    few, many = (best_us(what(gpu, big_cache(m, n_kv, hd), m)[0]) for m in (n, n + n // 20))
    assert many <= 2 * few, (few, many)


def test_copy_of_a_large_call(gpu):
    """Attention over 38,000 keys of 32 heads, of which the copy takes most."""
    n = 38000
    c = big_cache(n, 32, 128)
    call, q, out = copier(gpu, c, n)
    call()
    torch.cuda.synchronize()
    lim = torch.tensor([n], device="cuda")
    for h in range(0, 32, 5):
        k, v = (c.rows(0, n, pool)[:, h:h + 1] for pool in ("k", "v"))
        ref, err = P.attend(q[:, h:h + 1], k, v, float(torch.tensor(0.1)), lim)
        R.assert_rows(out[:, h:h + 1], ref, err, h)
