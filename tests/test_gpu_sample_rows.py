"""Sampling a batch on the GPU against the definition in 64 bits, token by
token."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import paged8_ref as P
import paged_ref as R
from tensoros_b200 import _ffi
from tensoros_b200 import workloads as W

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def logits(rows, n, seed=0, spread=2.0, kind=torch.float32):
    x = spread * torch.randn(rows, n, generator=gen(seed), device="cuda")
    x[:, :: max(1, n // 20)] += 6.0
    return x.to(kind)


def ptr(t):
    return None if t is None else t.data_ptr()


def call(gpu, x, u, t=None, k=None, p=None, m=None, prob=True, kept=True):
    """(tokens, probabilities, kept) by the library."""
    n = x.shape[0]
    f = lambda v: None if v is None else torch.as_tensor(v, dtype=torch.float32, device="cuda").expand(n).contiguous()  # noqa: E731
    t, p, m = f(t), f(p), f(m)
    k = None if k is None else torch.as_tensor(k, dtype=torch.int32, device="cuda").expand(n).contiguous()
    token = torch.full((n + 1,), -77, dtype=torch.int32, device="cuda")
    pr = torch.full((n,), -7.0, device="cuda") if prob else None
    ke = torch.full((n,), -77, dtype=torch.int32, device="cuda") if kept else None
    r = _ffi.Rows(x.data_ptr(), x.stride(0), R.F32 if x.dtype == torch.float32 else R.F16)
    s = _ffi.SampleParams(ptr(t), ptr(k), ptr(p), ptr(m))
    st = gpu.tos_sample_rows_dev(C.byref(r), n, x.shape[1], C.byref(s), u.data_ptr(), token.data_ptr(), ptr(pr), ptr(ke),
                                 R.stream())
    assert st == 0
    torch.cuda.synchronize()
    assert int(token[n]) == -77
    return token[:n], pr, ke


def reference(x, u, t, k, p, m):
    """One row in 64 bits: (token, probability, kept, how near u comes to a
    border, in parts of the sum)."""
    x = x.double().cpu().numpy()
    live = np.flatnonzero(~np.isneginf(x))
    if np.isnan(x).any() or live.size == 0:
        return -1, 0.0, 0, 1.0
    order = live[np.lexsort((live, -x[live]))]
    v = x[order]
    if not t > 0:
        return int(order[0]), 1.0, 1, 1.0
    d = np.where(v == v[0], 0.0, v - v[0])
    with np.errstate(over="ignore", invalid="ignore"):
        w = np.where(np.isneginf(d), 0.0, np.exp(d / t))
    n = min(k, len(w)) if k > 0 else len(w)
    c = np.cumsum(w)
    keep = n
    if p < 1:
        keep = min(keep, int(np.searchsorted(c[:n], p * c[n - 1])) + 1)
    if m > 0:
        keep = min(keep, int((w >= min(m, 1.0)).sum()))
    u = min(max(u, 0.0), float(np.float32(0.99999994))) if u == u else 0.0
    z = c[keep - 1]
    at = int(np.searchsorted(c[:keep], u * z, side="right"))
    near = np.abs(c[:keep] / z - u).min()
    return int(order[at]), w[at] / z, keep, near


def check(gpu, x, u, t=1.0, k=0, p=1.0, m=0.0):
    """Whole numbers are equal.  (Weights are whole numbers of 2^-42 of the largest,
    so sums of n are off by n 2^-43 at most, of at least 1; u at a border by
    less than that may fall to either side, which random u do not meet.)"""
    n = x.shape[0]
    per = lambda v: [float(f) for f in np.broadcast_to(np.asarray(v, np.float32), (n,))]  # noqa: E731
    token, prob, kept = call(gpu, x, u, t, k, p, m)
    for r, (t_, k_, p_, m_) in enumerate(zip(per(t), per(k), per(p), per(m))):
        want, pw, kw, near = reference(x[r], float(u[r]), t_, int(k_), p_, m_)
        assert int(kept[r]) == kw, (r, int(kept[r]), kw)
        if near > 1e-9:
            assert int(token[r]) == want, (r, int(token[r]), want, t_, k_, p_, m_, float(u[r]))
            assert abs(float(prob[r]) - pw) <= 2.0 ** -24 * pw + 1e-9
    return token


def uniform(n, seed=1):
    return torch.rand(n, generator=gen(seed), device="cuda")


FILTERS = [dict(), dict(t=0.7, k=40, p=0.95), dict(p=0.9), dict(m=0.05), dict(k=1), dict(k=5000), dict(t=2.0, p=0.999),
           dict(t=1.3, k=700, p=0.5, m=0.01), dict(k=3000, m=0.2), dict(t=0.1), dict(k=3000, p=0.99),
           dict(t=5.0, k=20000, p=0.8, m=1e-6)]


@pytest.mark.parametrize("kind", [torch.float32, torch.float16])
@pytest.mark.parametrize("o", FILTERS)
@pytest.mark.parametrize("n", [32000, 50001])
def test_filters(gpu, kind, o, n):
    check(gpu, logits(9, n, seed=n, kind=kind), uniform(9, n), **o)


@pytest.mark.parametrize("n", [1, 2, 3, 7, 64, 1000, 1023, 1025, 2047, 2049, 8193])
@pytest.mark.parametrize("o", [dict(), dict(k=3, p=0.9), dict(p=0.7, t=3.0), dict(m=0.3)])
def test_odd_sizes(gpu, n, o):
    check(gpu, logits(5, n, seed=n), uniform(5, n), **o)


@pytest.mark.parametrize("rows", [1, 37, 38, 75, 149, 400])
def test_batches(gpu, rows):
    """Every size of a cluster; every row with filters of its own."""
    g = np.random.default_rng(rows)
    pick = lambda *v: g.choice(v, rows)  # noqa: E731
    check(gpu, logits(rows, 6000, seed=rows), uniform(rows, rows), t=pick(0.0, 0.5, 1.0, 2.0, -1.0), k=pick(0, 1, 50, 3000, -3),
          p=pick(1.0, 0.5, 0.95, 2.0), m=pick(0.0, 0.01, 0.3))


@pytest.mark.parametrize("o", [dict(), dict(p=0.6), dict(k=100000), dict(k=300000, p=0.9, m=0.3), dict(t=0.5, k=50)])
def test_largest_vocabulary(gpu, o):
    check(gpu, logits(2, 1 << 20, spread=1.0), uniform(2, 3), **o)


@pytest.mark.parametrize("o", [dict(), dict(p=0.5), dict(k=20000), dict(k=20000, p=0.3), dict(m=0.999), dict(k=30000, m=1.0)])
@pytest.mark.parametrize("what", ["equal", "two", "narrow", "steps"])
def test_bins_that_overflow(gpu, what, o):
    """Ties, and values so near one another that they share a bin."""
    n, rows = 40000, 4
    x = torch.zeros(rows, n, device="cuda")
    if what == "two":
        x[:, ::3] = 1e-4
    elif what == "narrow":
        x += 1e-6 * torch.randn(rows, n, generator=gen(1), device="cuda")
    elif what == "steps":
        x = torch.round(torch.randn(rows, n, generator=gen(2), device="cuda"))
    check(gpu, x, uniform(rows, 5), **o)


@pytest.mark.parametrize("o", [dict(p=0.0), dict(p=-1.0), dict(p=1e-30), dict(k=20000, p=0.0), dict(p=0.0, m=0.5)])
@pytest.mark.parametrize("n", [1, 50, 32000])
def test_one_token_at_least_stays(gpu, n, o):
    """No top-p is too small for the first token, of very many ties too."""
    x = torch.zeros(4, n, device="cuda")
    x[1] = logits(1, n, 7)[0]
    x[2, : n // 2] = -1.0
    x[3] = (logits(1, n, 8)[0] / 4).round()
    check(gpu, x, uniform(4), **o)


@pytest.mark.parametrize("m", [0.3, 1e-6, 1e-12, 1e-18])
def test_tokens_around_min_p(gpu, m):
    """Steps of 1e-5 around the least weight, however small that is."""
    x = math.log(m) + 1e-5 * torch.arange(-2000, 2001, device="cuda", dtype=torch.float64)
    x = torch.cat([x.new_zeros(1), x]).float()[None]
    check(gpu, x.expand(3, -1).contiguous(), torch.tensor([0.2, 0.999, 0.9999999], device="cuda"), m=m)


@pytest.mark.parametrize("t", [1e-30, 1e-4, 100.0, 1e6, 1e38, float("inf")])
@pytest.mark.parametrize("o", [dict(), dict(k=9000, p=0.7), dict(m=0.9)])
def test_extreme_temperatures(gpu, t, o):
    check(gpu, logits(3, 20000, seed=8), uniform(3, 8), t=t, **o)


@pytest.mark.parametrize("kind", [torch.float32, torch.float16])
@pytest.mark.parametrize("o", [dict(), dict(k=50, p=0.9), dict(p=0.99), dict(k=30000), dict(k=4000, m=1e-9)])
def test_masked_tokens(gpu, kind, o):
    """-infinity and the type's lowest value in most places, few or one left."""
    low = torch.finfo(kind).min
    x = logits(6, 32000, seed=4, kind=kind)
    x[0, 10:] = -math.inf
    x[1, 10:] = low
    x[2, :] = -math.inf
    x[2, 31999] = -3.0
    x[3, 5:20000] = low
    x[3, 20000:] = -math.inf
    x[4, :] = low
    x[5, ::2] = -math.inf
    token = check(gpu, x, uniform(6, 4), **o)
    assert int(token[2]) == 31999 and int(token[0]) < 10 and int(token[1]) < 10


@pytest.mark.parametrize("o", [dict(), dict(t=0.0), dict(k=5, p=0.5), dict(t=float("inf"))])
def test_rows_that_are_not_finite(gpu, o):
    x = logits(6, 5000, seed=6)
    x[0, 4999] = math.nan
    x[1] = -math.inf
    x[2, [7, 70, 700]] = math.inf
    x[3, 0] = math.inf
    x[3, 1] = math.nan
    x[4, 3:] = -math.inf
    token = check(gpu, x, uniform(6, 6), **o)
    assert token[[0, 1, 3]].tolist() == [-1, -1, -1] and int(token[2]) in (7, 70, 700)


def test_random_numbers_at_their_ends(gpu):
    """u = 0: the first token; the largest below 1: the last that has weight; others as the nearest."""
    x = logits(8, 3000, seed=1, spread=0.3)
    u = torch.tensor([0.0, 0.99999994, 1.0, -1.0, math.nan, 5.0, math.inf, 0.5], device="cuda")
    for o in (dict(), dict(k=10), dict(p=0.3)):
        token = check(gpu, x, u, **o)
        for r in (0, 3, 4):
            assert int(token[r]) == int(x[r].argmax())


def test_every_token_of_a_small_row_in_its_share(gpu):
    """4096 rows of one distribution, u over a grid: tokens come in order of
    falling weight, each in its share of the grid."""
    n = 4096
    x = torch.tensor([1.0, 3.0, -1.0, 3.0, 0.5], device="cuda").expand(n, 5).contiguous()
    u = (torch.arange(n, device="cuda") + 0.5) / n
    token, prob, kept = call(gpu, x, u, t=1.5)
    w = torch.exp((x[0].double() - 3.0) / 1.5)
    share = w / w.sum()
    for i in range(5):
        assert abs(int((token == i).sum()) / n - float(share[i])) <= 1.0 / n
    assert torch.unique_consecutive(token).tolist() == [1, 3, 0, 4, 2] and bool((kept == 5).all())


def test_greedy_is_argmax(gpu):
    x = logits(4, 32000, seed=3, kind=torch.float16).float()     # ties at the top among them
    out = torch.empty(1, dtype=torch.int32, device="cuda")
    token, prob, kept = call(gpu, x, uniform(4), t=0.0)
    for r in range(4):
        assert gpu.tos_argmax_dev(x[r].data_ptr(), 32000, out.data_ptr(), R.stream()) == 0
        assert int(out) == int(token[r])
    assert bool((prob == 1).all()) and bool((kept == 1).all())


def test_parameters_left_out(gpu):
    x, u = logits(3, 4000, seed=2), uniform(3)
    want = call(gpu, x, u, 1.0, 0, 1.0, 0.0)
    for got in (call(gpu, x, u), call(gpu, x, u, prob=False, kept=False)):
        assert torch.equal(got[0], want[0])
    token = torch.empty(3, dtype=torch.int32, device="cuda")
    r = _ffi.Rows(x.data_ptr(), 4000, 0)
    assert gpu.tos_sample_rows_dev(C.byref(r), 3, 4000, None, u.data_ptr(), token.data_ptr(), None, None, R.stream()) == 0
    assert torch.equal(token, want[0])
    assert gpu.tos_sample_rows_dev(C.byref(r), 0, 4000, None, None, None, None, None, R.stream()) == 0


@pytest.mark.parametrize("kind", [torch.float32, torch.float16])
def test_unaligned_rows(gpu, kind):
    buf = logits(1, 5 * 4097 + 9, seed=9, kind=kind)[0]
    x = torch.as_strided(buf, (5, 4001), (4097, 1), 3)
    check(gpu, x, uniform(5), p=0.8)


def test_same_bits_and_two_streams(gpu):
    """Atomics in any order, streams beside one another: the same results."""
    x, u = logits(24, 60000, seed=7, spread=1.0), uniform(24)
    want = [a.clone() for a in call(gpu, x, u, 1.0, 0, 0.97, 0.0)]
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(6):
        for s in st:
            with torch.cuda.stream(s):
                for a, b in zip(call(gpu, x, u, 1.0, 0, 0.97, 0.0), want):
                    assert torch.equal(a, b)


def test_serving_step_in_a_graph(gpu):
    """Append to an 8-bit cache, attend, project to the vocabulary, sample:
    captured once, replayed with new rows, lengths, filters and random numbers."""
    heads, n_kv, hd, vocab, n = 4, 2, 64, 1024, 3
    dim = heads * hd
    c = P.Cache8([40, 3, 17], 16, 16, n_kv, hd, P.I8, room=64)
    w = W.q8_0(vocab, dim, 5, 5)
    weight = C.c_void_p()
    assert gpu.tos_weight_create(C.byref(weight), w.ctypes.data, vocab, dim, W.TYPE_Q8_0) == 0
    try:
        x = torch.randn(n, heads + 2 * n_kv, hd, generator=gen(1), device="cuda")
        att, y = torch.empty(n, dim, device="cuda"), torch.empty(n, vocab, device="cuda")
        u, t, k, token = uniform(n), torch.ones(n, device="cuda"), P.ints([0] * n), P.ints([0] * n)
        cu, kl = P.packed([1] * n), P.ints([41, 4, 18])
        an = gpu.tos_attention_decode_paged8_workspace_bytes(n, 64, heads, n_kv, hd)
        gn = gpu.tos_gemm_workspace_bytes(n, vocab, dim)
        aw, gw = (torch.empty(max(b, 256), dtype=torch.uint8, device="cuda") for b in (an, gn))
        q = x[:, :heads]
        d, rq = c.desc(), R.rows(q)
        rk, rv = R.rows(x[:, heads:heads + n_kv]), R.rows(x[:, heads + n_kv:])
        ro, rl = _ffi.Rows(att.data_ptr(), dim, 0), _ffi.Rows(y.data_ptr(), vocab, 0)
        sp = _ffi.SampleParams(t.data_ptr(), k.data_ptr(), None, None)

        def step(s):
            assert gpu.tos_kv_append_paged8_dev(C.byref(d), C.byref(rk), C.byref(rv), cu.data_ptr(), kl.data_ptr(), n, n, s) == 0
            assert gpu.tos_attention_decode_paged8_dev(C.byref(ro), C.byref(rq), C.byref(d), kl.data_ptr(), n, 64, heads, 0.125,
                                                       aw.data_ptr(), an, s) == 0
            assert gpu.tos_gemm_dev(weight, att.data_ptr(), n, y.data_ptr(), gw.data_ptr(), gn, s) == 0
            assert gpu.tos_sample_rows_dev(C.byref(rl), n, vocab, C.byref(sp), u.data_ptr(), token.data_ptr(), None, None,
                                           s) == 0

        step(R.stream())
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(torch.cuda.current_stream().cuda_stream)
        for i in range(5):
            x.copy_(torch.randn(x.shape, generator=gen(10 + i), device="cuda"))
            kl.copy_(P.ints([41 + i, 4 + i, 18 + i]))
            u.copy_(uniform(n, 20 + i))
            t.fill_(0.5 + 0.2 * i)
            k.fill_(10 * i)
            g.replay()
            torch.cuda.synchronize()
            for r in range(n):
                m = int(kl[r])
                ref, err = P.attend(q[r:r + 1], c.rows(r, m), c.rows(r, m, "v"), 0.125, torch.tensor([m], device="cuda"))
                R.assert_rows(att[r:r + 1].view(1, heads, hd), ref, err, (i, r))
                want = reference(y[r], float(u[r]), float(t[r]), 10 * i, 1.0, 0.0)
                assert int(token[r]) == want[0]
    finally:
        torch.cuda.synchronize()
        gpu.tos_weight_destroy(weight)
