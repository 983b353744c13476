"""The 8-bit paged cache on the GPU: what is stored and read back bit for bit,
attention against plain 64-bit forms (paged8_ref.py)."""
import ctypes as C

import numpy as np
import pytest
import torch

import paged8_ref as P
import paged_ref as R
from paged8_ref import F8, I8, Cache8
from paged_ref import F16, F32

pytestmark = pytest.mark.gpu
KINDS = [I8, F8]


def randn(*shape, seed=0, kind=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(R.DT[kind])


def same(a, b):
    return torch.equal(torch.nan_to_num(a.float(), nan=1e30), torch.nan_to_num(b.float(), nan=1e30))


def check_append(gpu, c, lens, k, v):
    want = P.expect_append(c, k, v, lens)
    assert P.append(gpu, c, k, v, lens, sum(lens)) == 0
    for i, (a, b, n) in enumerate(zip(lens, c.lens, range(len(lens)))):
        if a == 0:
            continue
        for name, pool, scale in (("k", want[0], want[2]), ("v", want[1], want[3])):
            pg, r = c.where(i, 0, a + b)
            assert torch.equal(getattr(c, name)[pg, r], pool[pg, r]), (name, i)
            assert same(getattr(c, name + "s")[pg, r // c.block], scale[pg, r // c.block]), (name, i)
    # nothing else changed, rows behind the last ones included
    assert torch.equal(c.k, want[0]) and torch.equal(c.v, want[1])
    assert same(c.ks, want[2]) and same(c.vs, want[3])


# ------------------------------------------------------------ append and read

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("src", [F32, F16])
@pytest.mark.parametrize("page,block,n_kv,hd,hist,lens", [
    (16, 16, 4, 128, [0, 5, 16, 31], [33, 1, 1, 40]),       # fresh, into a block, at a page's edge, over several
    (16, 1, 2, 64, [3, 0], [1, 50]),                        # a scale a row
    (64, 64, 2, 128, [0, 63, 100], [200, 1, 0]),            # four warps a block; a sequence without rows
    (24, 8, 3, 40, [0, 23], [25, 2]),                       # pages of no power of two, dims of no 16
    (128, 128, 1, 256, [1, 0], [300, 129]),                 # more rows than stay in registers
    (5, 1, 1, 7, [0, 4], [11, 3]),                          # nothing aligned
    (1024, 1024, 2, 48, [1000, 0], [40, 1]),                # the largest block
    (16, 2, 5, 80, [0, 1, 2], [3, 2, 1]),
])
def test_append(gpu, kind, src, page, block, n_kv, hd, hist, lens):
    c = Cache8(hist, page, block, n_kv, hd, kind, seed=page + hd, room=max(a + b for a, b in zip(hist, lens)))
    x = randn(sum(lens), 2 * n_kv, hd, seed=hd, kind=src)
    x[:, 0] *= 30.0                                         # a head whose scales grow
    check_append(gpu, c, lens, x[:, :n_kv], x[:, n_kv:])    # one projection's rows: strided views


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 40, 7])
def test_append_every_magnitude(gpu, kind, hd):
    """Scales at and around their borders: a row's largest magnitude is top 2^e
    or a step beside it; below the least scale, beyond the largest; zeros;
    values half way between two that the type holds."""
    top = P.TOP[kind]
    mags = []
    for e in list(range(-30, 14)):
        x = top * 2.0 ** e
        mags += [x, torch.nextafter(torch.tensor(x), torch.tensor(0.0)).item(),
                 torch.nextafter(torch.tensor(x), torch.tensor(float("inf"))).item()]
    mags += [0.0, 1e-45, 1.2e-38, 3e38]
    k = randn(len(mags), 1, hd, seed=2).clamp(-1, 1) * torch.tensor(mags, device="cuda")[:, None, None]
    k[:, 0, hd // 2] = torch.tensor(mags, device="cuda")
    halves = torch.arange(hd, device="cuda") - hd // 2 + 0.5
    v = (halves * 2.0 ** -3).expand(len(mags), 1, hd).contiguous()
    v[:, 0, 0] = top * 2.0 ** -3
    c = Cache8([0], 16, 1, 1, hd, kind, room=len(mags))
    check_append(gpu, c, [len(mags)], k, v)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [128, 24, 9])
def test_append_token_by_token_grows_scales(gpu, kind, hd):
    """Every row is larger than the last: older rows are rounded again and again."""
    c = Cache8([0, 0], 32, 16, 2, hd, kind, room=40)
    for t in range(40):
        x = randn(2, 4, hd, seed=t) * 1.3 ** t
        check_append(gpu, c, [1, 1], x[:, :2], x[:, 2:])
        c.lens = [t + 1, t + 1]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 10])
def test_append_values_that_are_not_finite(gpu, kind, hd):
    """Their block reads as NaN, of that head and side alone, and is well again
    when it is filled from its first row."""
    for bad in (float("nan"), float("inf"), -float("inf")):
        c = Cache8([0], 16, 16, 2, hd, kind, room=48)
        x = randn(40, 4, hd, seed=5)
        x[20, 1, 3] = bad
        assert P.append(gpu, c, x[:, :2], x[:, 2:], [40], 40) == 0
        c.lens = [40]
        k, v = c.rows(0), c.rows(0, pool="v")
        assert bool(torch.isnan(k[16:32, 1]).all()) and bool(torch.isfinite(k[:, 0]).all())
        assert bool(torch.isfinite(k[:16]).all()) and bool(torch.isfinite(k[32:]).all()) and bool(torch.isfinite(v).all())
        kk, vv, st = P.read(gpu, c, [40], [40], F32)
        assert st == 0 and same(kk[:40], k.float()) and same(vv[:40], v.float())
        y = randn(1, 4, hd, seed=6)
        c.lens = [30]                                       # behind it, into the same block: still NaN
        assert P.append(gpu, c, y[:, :2], y[:, 2:], [1], 1) == 0
        assert bool(torch.isnan(c.rows(0, 31)[16:31, 1]).all())
        c.lens = [16]
        check_append(gpu, c, [1], y[:, :2], y[:, 2:])
        assert bool(torch.isfinite(c.rows(0, 17)).all())


@pytest.mark.parametrize("kind", KINDS)
def test_append_bounds(gpu, kind):
    """Rows behind n_tokens, slots outside the table row and pages outside the
    pool are not stored; a block that begins with rows never held keeps their
    scale, here NaN."""
    page, hd = 16, 64
    c = Cache8([0, 0, 0, 0], page, 8, 2, hd, kind, room=32)
    c.table[1, 1] = -1
    c.table[2, 0] = c.n_pages
    before = [t.clone() for t in (c.k, c.v, c.ks, c.vs)]
    x = randn(80, 4, hd, seed=1)
    # sequence 0: 20 rows, two of them before slot 0; 1: its second page is none;
    # 2: its first is none; 3: rows on to slot 34, the table row ends at 32
    lens, kv = [20, 20, 20, 20], [18, 20, 20, 35]
    assert P.append(gpu, c, x[:, :2], x[:, 2:], lens, 78, kv_len=kv) == 0
    d = Cache8([0, 0, 0, 0], page, 8, 2, hd, kind, room=32)
    d.table = c.table
    d.k, d.v, d.ks, d.vs = [t.clone() for t in before]
    for pool, scales, y in ((d.k, d.ks, x[:, :2]), (d.v, d.vs, x[:, 2:])):
        d.put(pool, scales, 0, 0, y[2:20].double())
        d.put(pool, scales, 1, 0, y[20:36].double())
        d.put(pool, scales, 2, 16, y[56:60].double())
        pg, r = d.where(3, 15, 16)                          # joins rows that were never written: scale NaN stays
        d.put(pool, scales, 3, 16, y[61:77].double())
    for a, b in zip((c.k, c.v), (d.k, d.v)):
        pg, r = d.where(3, 15, 16)
        a[pg, r] = b[pg, r]
        assert torch.equal(a, b)
    for a, b in zip((c.ks, c.vs), (d.ks, d.vs)):
        assert same(a, b)


def test_append_many_sequences_and_garbage_lengths(gpu):
    """A hundred sequences with none to three rows; lengths that make no sense
    store nothing outside the pool."""
    n = 100
    lens = [(7 * i) % 4 for i in range(n)]
    hist = [(13 * i) % 50 for i in range(n)]
    c = Cache8(hist, 16, 16, 1, 32, I8, room=64)
    x = randn(sum(lens), 2, 32, seed=3)
    check_append(gpu, c, lens, x[:, :1], x[:, 1:])
    for kv in ([-5] * n, [2 ** 31 - 1] * n, [1 << 20] * n):
        k0 = c.k.clone()
        assert P.append(gpu, c, x[:, :1], x[:, 1:], lens, sum(lens), kv_len=kv) == 0
        assert torch.equal(c.k, k0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dst", [F32, F16])
@pytest.mark.parametrize("page,block,n_kv,hd", [(16, 16, 4, 128), (24, 8, 2, 40), (5, 1, 3, 7), (64, 32, 1, 256)])
def test_read(gpu, kind, dst, page, block, n_kv, hd):
    lens = [70, 1, 0, 33]
    c = Cache8(lens, page, block, n_kv, hd, kind, seed=4)
    take, at = [70, 1, 0, 9], 0
    k, v, st = P.read(gpu, c, take, lens, dst, total=78)
    assert st == 0
    for i, n in enumerate(take):
        got = min(n, 78 - at)
        for x, pool in ((k, "k"), (v, "v")):
            assert torch.equal(x[at:at + got].double(), c.rows(i, pool=pool)[lens[i] - n:lens[i] - n + got]), (i, pool)
        at += n
    assert bool((k[78:] == 7.0).all()) and bool((v[78:] == 7.0).all())
    # one side alone, and pages outside the pool as zeros
    c.table[0, 0] = -3
    cu, kl = P.packed([page]), P.ints([page])
    out = torch.full((page, n_kv, hd), 7.0, dtype=R.DT[dst], device="cuda")
    d, r = c.desc(), R.rows(out)
    assert gpu.tos_kv_read_paged8_dev(C.byref(d), None, C.byref(r), cu.data_ptr(), kl.data_ptr(), 1, page,
                                      R.stream()) == 0
    assert bool((out == 0).all())


# ------------------------------------------------------------------- decode

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("q", [F32, F16])
@pytest.mark.parametrize("heads,n_kv,hd,page,block,lens", [
    (32, 32, 128, 16, 16, [300, 1, 0, 17]),
    (32, 8, 128, 64, 64, [1030, 64, 63]),
    (6, 6, 48, 32, 32, [272]),
    (8, 1, 64, 16, 1, [5, 200]),
    (16, 1, 128, 24, 8, [100, 31]),                         # 16 rows a tile; steps that cross pages
    (20, 1, 128, 48, 16, [500, 9]),                         # two row tiles, the second part full
    (40, 2, 64, 16, 4, [33]),
    (4, 2, 256, 32, 32, [700, 40]),                         # 256 dims
    (12, 1, 192, 16, 16, [90]),
    (16, 4, 96, 5, 1, [77, 4]),                             # pages of five rows
    (3, 3, 16, 16, 2, [600]),
    (10, 2, 40, 32, 16, [210, 0, 3]),                       # the way over fp16
    (6, 2, 7, 5, 1, [40]),
])
def test_decode(gpu, kind, q, heads, n_kv, hd, page, block, lens):
    c = Cache8(lens, page, block, n_kv, hd, kind, seed=hd + page)
    P.check_decode(gpu, c, randn(len(lens), heads, hd, seed=1, kind=q), heads)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("q,heads,n_kv,hd", [(F32, 8, 2, 128), (F16, 4, 4, 64), (F32, 2, 1, 256)])
def test_decode_split_keys(gpu, kind, q, heads, n_kv, hd):
    """Few sequences, long: the keys are cut and joined; one sequence ends before
    most pieces begin, one is empty."""
    c = Cache8([5000, 130, 0], 32, 32, n_kv, hd, kind, seed=hd)
    P.check_decode(gpu, c, randn(3, heads, hd, seed=1, kind=q), heads, max_kv=5555)


def ragged(n, most, seed):
    """n lengths from 0 to most, a few of them around whole blocks of 128"""
    g = torch.Generator().manual_seed(seed)
    lens = (most * torch.rand(n, generator=g) ** 2).int().tolist()
    for i, v in enumerate([0, 1, 127, 128, 129, most]):
        lens[(i * 5) % n] = v
    return lens


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("q,heads,n_kv,hd,page,block,n,most", [
    (F32, 32, 8, 128, 16, 16, 12, 5000),                    # every CTA takes an even share of the keys
    (F16, 16, 16, 64, 32, 8, 20, 3000),
    (F32, 6, 6, 48, 48, 16, 40, 2000),
    (F32, 32, 2, 128, 64, 64, 40, 4000),                    # 16 rows a tile
    (F16, 24, 8, 256, 16, 16, 11, 3000),
    (F32, 8, 4, 96, 24, 8, 30, 4000),                       # by cp.async
    (F32, 20, 4, 64, 40, 8, 15, 4500),                      # by cp.async, two row tiles of 8
])
def test_decode_even_shares(gpu, kind, q, heads, n_kv, hd, page, block, n, most):
    lens = ragged(n, most, hd + n)
    c = Cache8(lens, page, block, n_kv, hd, kind, seed=n)
    P.check_decode(gpu, c, randn(n, heads, hd, seed=1, kind=q), heads)


@pytest.mark.parametrize("n", [1024, 1025])
def test_decode_many_sequences(gpu, n):
    lens = [(i * 131) % 700 for i in range(n)]
    c = Cache8(lens, 16, 16, 1, 64, I8, seed=1)
    P.check_decode(gpu, c, randn(n, 2, 64, seed=1), 2, only=list(range(0, n, 7)) + [n - 1])


@pytest.mark.parametrize("kind", KINDS)
def test_decode_scales_far_apart(gpu, kind):
    """Blocks whose scales span their whole range, the largest I8 ones (which
    need a detour in the conversion) among small ones, in one step too."""
    lo, hi = P.LIMITS[kind]
    for block in (1, 16):
        c = Cache8([200, 64], 64, block, 2, 128, kind, seed=block, spread=0.0)
        n = 64 // block
        e = (torch.arange(c.n_pages * n * 2, device="cuda") * 7 % (hi - lo + 1) + lo).view(c.n_pages, n, 2)
        c.vs.copy_(torch.exp2(e.float()))
        c.ks.copy_(torch.exp2((e % 9 - 8).float()))
        P.check_decode(gpu, c, randn(2, 8, 128, seed=2), 8)
        c.ks.fill_(2.0 ** hi)                               # scores of thousands
        P.check_decode(gpu, c, randn(2, 8, 128, seed=2), 8)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [128, 64, 40])
def test_decode_nan_blocks(gpu, kind, hd):
    """A NaN scale makes its head's rows NaN, and only where it is seen."""
    for pool in ("ks", "vs"):
        c = Cache8([100, 48, 50], 16, 16, 2, hd, kind, seed=3)
        s = getattr(c, pool)
        s[c.table[0, 3].long(), 0, 1] = float("nan")        # sequence 0, keys 48..63, head 1
        q = randn(3, 4, hd, seed=1)
        out, st = P.decode(gpu, c, q, [100, 48, 48], 4, hd ** -0.5)
        assert st == 0
        assert bool(torch.isnan(out[0, 2:]).all()) and bool(torch.isfinite(out[0, :2]).all())
        assert bool(torch.isfinite(out[1:]).all())
        out, st = P.decode(gpu, c, q, [48, 48, 48], 4, hd ** -0.5)
        assert st == 0 and bool(torch.isfinite(out).all())


@pytest.mark.parametrize("kind", KINDS)
def test_decode_odd_rows(gpu, kind):
    """Rows at odd strides and addresses, negative scale, zero scale, queries of
    zeros, huge and not finite."""
    c = Cache8([300, 20], 16, 16, 2, 64, kind, seed=8)
    buf = randn(2 * 301 + 5, seed=4)
    q = torch.as_strided(buf, (2, 4, 64), (301, 64, 1), 3)
    ob = torch.full((2 * 299 + 5,), 7.0, device="cuda")
    out = torch.as_strided(ob, (2, 4, 64), (299, 64, 1), 1)
    P.check_decode(gpu, c, q, 4, scale=-0.2, out=out)
    P.check_decode(gpu, c, q, 4, scale=0.0)
    z = randn(2, 4, 64, seed=5)
    z[0] = 0
    z[1] *= 1e30
    P.check_decode(gpu, c, z, 4, scale=1e-30)
    z[0, 1, 5] = float("nan")
    z[0, 2, 6] = float("inf")
    out, st = P.decode(gpu, c, z, c.lens, 4, 1e-30)
    assert st == 0 and bool(torch.isnan(out[0, 1:3]).all()) and bool(torch.isfinite(out[0, [0, 3]]).all())
    assert bool(torch.isfinite(out[1]).all())


def test_decode_lengths_beyond_the_table_and_bad_pages(gpu):
    for hd in (64, 40):
        c = Cache8([64, 64], 16, 16, 1, hd, I8, seed=1)
        q = randn(2, 2, hd, seed=1)
        ref = P.check_decode(gpu, c, q, 2)
        out, st = P.decode(gpu, c, q, [2 ** 31 - 1, -7], 2, hd ** -0.5, max_kv=4000)
        assert st == 0 and bool((out[1] == 0).all())
        assert bool(((out[0] - ref[0]).abs() <= 1e-5).all())   # 64 rows of the table; another split
        # a page outside the pool: its keys score 0 and weigh as such, with values of 0
        c.table[0, 2] = c.n_pages
        out, st = P.decode(gpu, c, q, [64, 64], 2, hd ** -0.5)
        assert st == 0
        k, v = (torch.cat([c.rows(0, 32, p), torch.zeros(16, 1, hd, dtype=torch.float64, device="cuda"),
                           c.rows_at(0, 48, 64, p)]) for p in ("k", "v"))
        r, err = P.attend(q[:1], k, v, hd ** -0.5, torch.tensor([64], device="cuda"))
        R.assert_rows(out[:1], r, err, "bad page")


def test_decode_offsets_beyond_32_bits(gpu):
    """The pool is 4.6 GB; sequences lie at its end."""
    c = Cache8([40], 16, 16, 8, 128, F8, seed=1, spare=0)
    pages = (1 << 32) // (16 * 8 * 128) + 5000
    big_k = torch.empty(pages, 16, 8, 128, dtype=torch.int8, device="cuda")
    big_v = torch.empty_like(big_k)
    s = torch.full((2, pages, 1, 8), float("nan"), device="cuda")
    at = pages - c.n_pages
    big_k[at:], big_v[at:], s[0, at:], s[1, at:] = c.k, c.v, c.ks, c.vs
    c.k, c.v, c.ks, c.vs, c.n_pages = big_k, big_v, s[0], s[1], pages
    c.table += at
    x = randn(3, 16, 128, seed=2)
    q = randn(1, 32, 128, seed=1)
    P.check_decode(gpu, c, q, 32)
    k, v, st = P.read(gpu, c, [40], [40], F32)
    assert st == 0 and torch.equal(k[:40].double(), c.rows(0))
    c.lens = [32]
    first = c.rows(0).clone()
    assert P.append(gpu, c, x[:, :8], x[:, 8:], [3], 3) == 0
    c.lens = [35]
    assert torch.equal(c.rows(0)[:32], first)
    assert torch.equal(c.rows(0)[32:], P.nearest(x[:, :8].double() / (n := P.needed(
        x[:, :8].abs().amax((0, 2)), F8))[:, None], F8) * n[:, None])
    P.check_prompt(gpu, c, randn(3, 32, 128, seed=3), [3], [35], 32)


@pytest.mark.parametrize("kind", KINDS)
def test_decode_long_sums_do_not_shrink(gpu, kind):
    """32,768 keys of one sign and equal weights: no accumulator cuts off."""
    n = 32768
    c = Cache8([n], 64, 64, 1, 64, kind, seed=1, spread=0.0)
    pg, r = c.where(0, 0, n)
    one = 101 if kind == I8 else torch.tensor([104.0], device="cuda").to(torch.float8_e4m3fn).view(torch.int8).item()
    c.v[pg, r] = one
    c.vs.fill_(2.0 ** -7)
    q = torch.zeros(1, 8, 64, device="cuda")
    out, st = P.decode(gpu, c, q, [n], 8, 0.1)
    want = (101 if kind == I8 else 104) * 2.0 ** -7
    assert st == 0 and float(((out - want).abs() / want).max()) <= (64 + n / 8) * R.U


@pytest.mark.parametrize("hd", [128, 40])
def test_decode_is_deterministic_and_ignores_the_workspace(gpu, hd):
    c = Cache8([4000, 17], 16, 16, 2, hd, I8, seed=6)
    q = randn(2, 8, hd, seed=1)
    a, st = P.decode(gpu, c, q, c.lens, 8, 0.1)
    n = gpu.tos_attention_decode_paged8_workspace_bytes(2, 4000, 8, 2, hd)
    b, st2 = P.decode(gpu, c, q, c.lens, 8, 0.1, ws=torch.zeros(max(n, 16), dtype=torch.uint8, device="cuda"))
    assert st == st2 == 0 and torch.equal(a, b)


# ------------------------------------------------------------------- prompts

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("q", [F32, F16])
@pytest.mark.parametrize("heads,n_kv,hd,page,block,q_lens,hist", [
    (32, 8, 128, 64, 32, [300, 1, 0, 65], [0, 40, 0, 3]),
    (8, 4, 64, 16, 16, [130, 200], [700, 0]),
    (6, 6, 48, 24, 8, [100], [31]),
    (4, 2, 256, 16, 1, [40, 9], [0, 100]),
    (10, 2, 40, 5, 1, [33, 70], [2, 0]),
    (4, 2, 7, 16, 4, [20], [11]),
    (16, 2, 128, 16, 16, [5, 3, 1], [200, 0, 77]),          # few rows a sequence
])
def test_prompt(gpu, kind, q, heads, n_kv, hd, page, block, q_lens, hist):
    kv = [a + b for a, b in zip(q_lens, hist)]
    c = Cache8(kv, page, block, n_kv, hd, kind, seed=hd + page)
    P.check_prompt(gpu, c, randn(sum(q_lens) + 2, heads, hd, seed=2, kind=q), q_lens, kv, heads,
                   total_kv=sum(kv) + 57, max_kv=max(kv) + 200)


def test_prompt_of_many_sequences(gpu):
    """More sequences than a block's threads, empty ones among them."""
    lens = [(i * 37) % 150 for i in range(700)]
    c = Cache8(lens, 16, 16, 1, 64, F8, seed=1, spread=0.2)
    P.check_prompt(gpu, c, randn(sum(lens), 2, 64, seed=1, kind=F16), lens, lens, 2)


@pytest.mark.parametrize("kind", KINDS)
def test_prompt_rows_see_no_nan_behind_them(gpu, kind):
    """Rows before a block of NaN scale do not see it; rows in and behind it do."""
    n, hd = 300, 128
    for pool in ("ks", "vs"):
        c = Cache8([n], 16, 16, 2, hd, kind, seed=2)
        q = randn(n, 8, hd, seed=3)
        ref = P.check_prompt(gpu, c, q, [n], [n], 8).clone()
        getattr(c, pool)[c.table[0, 10].long(), 0, 0] = float("nan")      # keys 160..175 of head 0
        out, st = P.prompt(gpu, c, q, [n], [n], 8, hd ** -0.5)
        assert st == 0 and torch.equal(out[:160], ref[:160]) and torch.equal(out[:, 4:], ref[:, 4:])
        assert bool(torch.isnan(out[160:, :4]).all())


def test_prompt_rows_that_see_nothing_and_short_total(gpu):
    """More queries than keys: the first see nothing; keys beyond total_kv do no harm."""
    c = Cache8([20, 500], 16, 16, 2, 64, I8, seed=5)
    q = randn(130, 4, 64, seed=1)
    P.check_prompt(gpu, c, q, [50, 80], [20, 500], 4)
    out, st = P.prompt(gpu, c, q, [50, 80], [20, 500], 4, 0.125, total_kv=0)
    torch.cuda.synchronize()
    assert st == 0


# --------------------------------------------------------------- all together

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("src", [F32, F16])
def test_serving_run(gpu, kind, src):
    """Prompts, then decoding token by token: rotation, append, attention, over
    the library's own stream order; the cache's values equal the rows within
    half a step of their block's scale."""
    heads, n_kv, hd, page, block = 8, 2, 64, 16, 16
    lens, steps = [70, 5, 33], 20
    c = Cache8([0] * 3, page, block, n_kv, hd, kind, room=96)
    rd = R.rotary_desc(hd, "half")
    rot = C.c_void_p()
    assert gpu.tos_rotary_create(C.byref(rot), C.byref(rd)) == 0
    try:
        held = [0, 0, 0]
        stored = [[], [], []]
        for step in range(steps + 1):
            new = lens if step == 0 else [1, 1, 1]
            n = sum(new)
            x = randn(n, heads + 2 * n_kv, hd, seed=step, kind=src)
            q, k, v = x[:, :heads], x[:, heads:heads + n_kv], x[:, heads + n_kv:]
            pos = P.ints([b + j for a, b in zip(new, held) for j in range(a)])
            rq, rk = R.rows(q), R.rows(k)
            assert gpu.tos_qk_norm_rotary_dev(C.byref(rq), C.byref(rq), C.byref(rk), C.byref(rk), n, heads, n_kv, hd,
                                              None, None, 0.0, rot, pos.data_ptr(), R.stream()) == 0
            c.lens = held
            assert P.append(gpu, c, k, v, new, n) == 0
            at = 0
            for i, a in enumerate(new):
                stored[i].append(k[at:at + a].double())
                at += a
            held = [a + b for a, b in zip(new, held)]
            c.lens = held
            if step == 0:
                P.check_prompt(gpu, c, q.contiguous(), new, held, heads)
            else:
                P.check_decode(gpu, c, q.contiguous(), heads)
        for i in range(3):
            pg, r = c.where(i, 0, held[i])
            s = c.ks[pg, r // block].double()[..., None]
            x = torch.cat(stored[i])
            # every rounding is half a step at most, and a block's scale grew at
            # most a few times, doubling at least: below two half steps in all
            half = s / 2 if kind == I8 else torch.maximum(x.abs() * 2.0 ** -4, s * 2.0 ** -10)
            assert bool(((c.rows(i) - x).abs() <= 2 * half * (1 + 2.0 ** -3)).all())
    finally:
        torch.cuda.synchronize()
        gpu.tos_rotary_destroy(rot)


@pytest.mark.parametrize("hd", [64, 40])
def test_graph_replay_with_changed_lengths(gpu, hd):
    """append, read, decode and prompt captured once; lengths, tables and rows
    change between replays; two graphs with a workspace each run side by side."""
    heads, n_kv, page, block, n = 4, 2, 16, 8, 3
    graphs = []
    for w in range(2):
        c = Cache8([100, 3, 50], page, block, n_kv, hd, [I8, F8][w], seed=w, room=160)
        x = randn(n, 2 * n_kv, hd, seed=w)
        q = randn(n, heads, hd, seed=w + 5)
        out, pout = torch.empty_like(q), torch.empty_like(q)
        kb = torch.empty(n, n_kv, hd, device="cuda")
        kl, cu = P.ints([101, 4, 51]), P.packed([1, 1, 1])
        dn = gpu.tos_attention_decode_paged8_workspace_bytes(n, 160, heads, n_kv, hd)
        pn = gpu.tos_attention_prompt_paged8_workspace_bytes(n, n, 1, 480, 160, heads, n_kv, hd)
        ws = torch.full((max(dn, 16),), 255, dtype=torch.uint8, device="cuda")
        pws = torch.full((pn,), 255, dtype=torch.uint8, device="cuda")
        d, rk, rv, rq, ro, rp, rb = c.desc(), R.rows(x[:, :n_kv]), R.rows(x[:, n_kv:]), R.rows(q), R.rows(out), R.rows(pout), R.rows(kb)
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            s = torch.cuda.current_stream().cuda_stream
            assert gpu.tos_kv_append_paged8_dev(C.byref(d), C.byref(rk), C.byref(rv), cu.data_ptr(), kl.data_ptr(), n, n, s) == 0
            assert gpu.tos_kv_read_paged8_dev(C.byref(d), C.byref(rb), None, cu.data_ptr(), kl.data_ptr(), n, n, s) == 0
            assert gpu.tos_attention_decode_paged8_dev(C.byref(ro), C.byref(rq), C.byref(d), kl.data_ptr(), n, 160, heads,
                                                       0.2, ws.data_ptr(), dn, s) == 0
            assert gpu.tos_attention_prompt_paged8_dev(C.byref(rp), C.byref(rq), C.byref(d), cu.data_ptr(), kl.data_ptr(), n, n,
                                                       1, 480, 160, heads, 0.2, pws.data_ptr(), pn, s) == 0
        graphs.append((g, st, c, x, q, out, pout, kb, kl, cu, ws, pws))
    held = [100, 3, 50]
    for step in range(4):
        for w, (g, st, c, x, q, out, pout, kb, kl, *_) in enumerate(graphs):
            x.copy_(randn(*x.shape, seed=100 * step + w))
            kl.copy_(P.ints([h + 1 + step for h in held]))
        torch.cuda.synchronize()
        for g, st, *_ in graphs:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for w, (g, st, c, x, q, out, pout, kb, kl, *_) in enumerate(graphs):
            for i in range(n):
                m = held[i] + 1 + step
                k, v = c.rows(i, m), c.rows(i, m, "v")
                ref, err = P.attend(q[i:i + 1], k, v, float(np.float32(0.2)), torch.tensor([m], device="cuda"))
                R.assert_rows(out[i:i + 1], ref, err, ("decode", step, w, i))
                R.assert_rows(pout[i:i + 1], ref, err, ("prompt", step, w, i))
                assert torch.equal(kb[i].double(), k[-1])


@pytest.mark.parametrize("n", [5, 20])
def test_graph_replay_shares_the_keys_anew(gpu, n):
    """Decode whose keys are dealt by the lengths (equal pieces; even shares), captured
    once: each replay deals those that are there then, and gives an eager call's bits."""
    heads, n_kv, hd, most = 32, 8, 128, 5000
    c = Cache8([most] * n, 16, 16, n_kv, hd, I8, seed=n)
    q = randn(n, heads, hd, seed=1)
    out, kl = torch.empty_like(q), P.ints([most] * n)
    size = gpu.tos_attention_decode_paged8_workspace_bytes(n, most, heads, n_kv, hd)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    d, rq, ro = c.desc(), R.rows(q), R.rows(out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        assert gpu.tos_attention_decode_paged8_dev(C.byref(ro), C.byref(rq), C.byref(d), kl.data_ptr(), n, most, heads, 0.1,
                                                   ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream) == 0
    for step, lens in enumerate([ragged(n, most, 1), [0] * n, [most] + [0] * (n - 1), [1] * n, ragged(n, 700, 2), [most] * n]):
        kl.copy_(P.ints(lens))
        out.fill_(7.0)
        g.replay()
        want = P.check_decode(gpu, c, q, heads, scale=0.1, kv_lens=lens, max_kv=most, only=[0, n // 2, n - 1])
        torch.cuda.synchronize()
        assert torch.equal(out, want), step


def test_two_streams_at_once(gpu):
    """Calls on two streams beside one another, each with its own workspace."""
    c = Cache8([6000, 900], 16, 16, 2, 128, I8, seed=1)
    q = [randn(2, 8, 128, seed=s) for s in (1, 2)]
    want = [P.decode(gpu, c, x, c.lens, 8, 0.1)[0] for x in q]
    torch.cuda.synchronize()
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i in (0, 1):
            with torch.cuda.stream(st[i]):
                got[i].append(P.decode(gpu, c, q[i], c.lens, 8, 0.1)[0])
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(x, want[i]) for x in got[i])
