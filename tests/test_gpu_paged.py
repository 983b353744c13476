"""The paged-cache operators on the GPU against plain 64-bit forms
(paged_ref.py, which derives the tolerances): per-head norm and rotary
positions, the append, prompt and decode attention, and a run of them."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import paged_ref as R
from paged_ref import F16, F32, Cache

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, kind=F32):
    return torch.randn(*shape, generator=gen(seed), device="cuda").to(R.DT[kind])


class Rotary:
    def __init__(self, gpu, d):
        self.gpu, self.d, self.h = gpu, d, C.c_void_p()
        assert gpu.tos_rotary_create(C.byref(self.h), C.byref(d)) == 0

    def __del__(self):
        torch.cuda.synchronize()
        self.gpu.tos_rotary_destroy(self.h)


# ------------------------------------------------------- norm and rotation

@pytest.mark.parametrize("tokens,heads,n_kv,hd", [(1, 32, 32, 128), (5, 6, 6, 48), (300, 8, 2, 64), (2, 3, 1, 256),
                                                  (7, 5, 1, 6), (9, 4, 4, 2), (700, 12, 4, 80)])
@pytest.mark.parametrize("src,dst", [(F32, F32), (F16, F16), (F32, F16), (F16, F32)])
def test_norm_rotary_shapes(gpu, tokens, heads, n_kv, hd, src, dst):
    layout = "half" if (heads + tokens) % 2 else "interleaved"
    d = R.rotary_desc(hd, layout)
    rot = Rotary(gpu, d)
    x = randn(tokens, heads + n_kv, hd, seed=hd + tokens, kind=src)
    q, k = x[:, :heads], x[:, heads:]                 # one projection's rows: strided views
    qo = torch.full((tokens, heads, hd), 7.0, dtype=R.DT[dst], device="cuda")
    ko = torch.full((tokens, n_kv, hd), 7.0, dtype=R.DT[dst], device="cuda")
    qw, kw = 1 + 0.1 * randn(hd, seed=1), 1 + 0.1 * randn(hd, seed=2)
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda") * 13 + 5
    a = [R.rows(t) for t in (q, qo, k, ko)]
    st = gpu.tos_qk_norm_rotary_dev(*[C.byref(r) for r in a], tokens, heads, n_kv, hd, qw.data_ptr(), kw.data_ptr(),
                                    1e-6, rot.h, pos.data_ptr(), R.stream())
    assert st == 0
    for got, x_, w in ((qo, q, qw), (ko, k, kw)):
        R.assert_rows(got, *R.norm_rotary(x_, w, float(np.float32(1e-6)), d, pos), (tokens, heads, hd, src, dst))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rot_dim", [2, 24, 32, 64, 128])
@pytest.mark.parametrize("scaling,factor,ff", [("none", 1.0, False), ("linear", 4.0, False), ("yarn", 8.0, False),
                                               ("none", 1.0, True)])
def test_rotary_parts_and_scalings(gpu, layout, rot_dim, scaling, factor, ff):
    """Part of the head, every layout and scaling, positions to the end of
    the int range, in place, without norm."""
    hd, heads, n = 128, 3, 11
    fac = 1 + np.arange(rot_dim // 2) / 7.0 if ff else None
    d = R.rotary_desc(rot_dim, layout, base=500000.0, scaling=scaling, factor=factor, orig=8192, attn=1.1, ff=fac)
    rot = Rotary(gpu, d)
    x = randn(n, heads, hd, seed=rot_dim)
    y = x.clone()
    # the last position: turns per position are known to 2^-55, so 2^31 of
    # them stay within 2^-24 turns in the 64-bit reference too
    pos = torch.tensor([0, 1, 2, 8191, 8192, 65535, 131071, 1 << 20, 1 << 24, 12345678, 3], dtype=torch.int32,
                       device="cuda")
    r = R.rows(y)
    assert gpu.tos_qk_norm_rotary_dev(C.byref(r), C.byref(r), None, None, n, heads, 0, hd, None, None, 0.0, rot.h,
                                      pos.data_ptr(), R.stream()) == 0
    R.assert_rows(y, *R.norm_rotary(x, None, 0.0, d, pos, fac), (layout, rot_dim, scaling))
    assert torch.equal(y[0, :, rot_dim:], x[0, :, rot_dim:]), "elements behind rot_dim changed"


def test_norm_without_rotation_and_large_values(gpu):
    n, heads, hd = 4, 2, 64
    x = randn(n, heads, hd, seed=3)
    x[1] *= 1e15
    x[2] = 0
    y = torch.empty_like(x)
    w = randn(hd, seed=4)
    a, b = R.rows(x), R.rows(y)
    assert gpu.tos_qk_norm_rotary_dev(None, None, C.byref(a), C.byref(b), n, 0, heads, hd, None, w.data_ptr(), 1e-5,
                                      None, None, R.stream()) == 0
    R.assert_rows(y, *R.norm_rotary(x, w, float(np.float32(1e-5)), None, None), "norm only")
    assert bool((y[2] == 0).all())


def test_rotary_unaligned_rows(gpu):
    """Rows at an odd stride from an odd element: the element-wise form."""
    n, heads, hd = 37, 3, 32
    buf = randn(n * 101 + 8, seed=5)
    x = torch.as_strided(buf, (n, heads, hd), (101, hd, 1), 1)
    out = torch.empty(n * 99 + 8, device="cuda")
    y = torch.as_strided(out, (n, heads, hd), (99, hd, 1), 3)
    d = R.rotary_desc(hd, "half")
    rot = Rotary(gpu, d)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    a, b = R.rows(x), R.rows(y)
    assert gpu.tos_qk_norm_rotary_dev(C.byref(a), C.byref(b), None, None, n, heads, 0, hd, None, None, 0.0, rot.h,
                                      pos.data_ptr(), R.stream()) == 0
    R.assert_rows(y, *R.norm_rotary(x, None, 0.0, d, pos), "unaligned")


# ----------------------------------------------------------------- append

@pytest.mark.parametrize("src,kv,page,n_kv,hd", [(F32, F16, 16, 4, 128), (F16, F16, 64, 2, 64), (F32, F32, 5, 1, 48),
                                                 (F16, F32, 1, 3, 10)])
def test_append(gpu, src, kv, page, n_kv, hd):
    """Rows land in their pages, nothing else changes, padding is skipped."""
    heads = 2 * n_kv
    lens = [3 * page + 2, 1, 2 * page]
    c = Cache(lens, page, n_kv, hd, kv, seed=page, fill=3.0)
    k0, v0 = c.k.clone(), c.v.clone()
    # tokens: (sequence, slot); padding with a bad sequence, a bad slot, a
    # table entry that points nowhere
    tok = [(0, 0), (0, 3 * page + 1), (1, 0), (2, 0), (2, 2 * page - 1), (0, page), (-1, 0), (3, 0), (1, -1),
           (2, 10 ** 9), (1, page * (c.table.shape[1] - 1))]
    good = 6
    n = len(tok)
    x = randn(n, heads + 2 * n_kv, hd, seed=9, kind=src)
    q, k, v = x[:, :heads], x[:, heads:heads + n_kv], x[:, heads + n_kv:]
    qo = torch.empty(n, heads, hd, dtype=R.DT[src], device="cuda")
    kw = 1 + 0.1 * randn(hd, seed=1)
    d = R.rotary_desc(hd, "interleaved")
    rot = Rotary(gpu, d)
    seq = torch.tensor([t[0] for t in tok], dtype=torch.int32, device="cuda")
    slot = torch.tensor([t[1] for t in tok], dtype=torch.int32, device="cuda")
    pos = torch.arange(n, dtype=torch.int32, device="cuda") + 100
    a = [R.rows(t) for t in (k, v, q, qo)]
    desc = c.desc()
    assert gpu.tos_kv_append_paged_dev(C.byref(desc), *[C.byref(r) for r in a], n, heads, seq.data_ptr(),
                                       slot.data_ptr(), pos.data_ptr(), None, kw.data_ptr(), 1e-6, rot.h,
                                       R.stream()) == 0
    eps = float(np.float32(1e-6))
    R.assert_rows(qo, *R.norm_rotary(q, None, eps, d, pos), "q")
    ref, err = R.norm_rotary(k, kw, eps, d, pos)
    for i in range(good):
        pg, r = int(c.table[tok[i][0], tok[i][1] // page]), tok[i][1] % page
        R.assert_rows(c.k[pg, r], ref[i], err[i], ("k", i))
        assert torch.equal(c.v[pg, r], v[i].to(R.DT[kv])), i
        c.k[pg, r], c.v[pg, r] = k0[pg, r], v0[pg, r]
    assert torch.equal(c.k, k0) and torch.equal(c.v, v0), "other rows changed"


# ---------------------------------------------------------- prompt attention

KINDS = [(F32, F32), (F32, F16), (F16, F16), (F16, F32)]


@pytest.mark.parametrize("qk,kv", KINDS)
@pytest.mark.parametrize("heads,n_kv,hd,page,q_lens,hist", [
    (4, 2, 128, 16, [1], [0]),
    (4, 4, 128, 64, [128, 1, 129], [0, 300, 5]),
    (8, 2, 128, 16, [257, 3, 64], [0, 130, 1]),
    (6, 6, 48, 32, [272, 16], [0, 7]),
    (8, 4, 32, 128, [200, 33], [100, 0]),
    (16, 2, 64, 8, [65, 300], [0, 63]),
    (8, 1, 96, 256, [100, 31, 1], [0, 511, 1000]),
    (5, 1, 80, 7, [40, 90], [3, 0]),
    (3, 3, 33, 3, [20, 5], [0, 9]),
    (2, 1, 256, 16, [70, 3], [0, 80]),
    (24, 8, 128, 16, [2, 0, 500, 0], [0, 40, 0, 0]),
])
def test_prompt_attention(gpu, qk, kv, heads, n_kv, hd, page, q_lens, hist):
    kv_lens = [a + b for a, b in zip(q_lens, hist)]
    c = Cache(kv_lens, page, n_kv, hd, kv, seed=hd + page)
    q = randn(sum(q_lens) + 2, heads, hd, seed=17, kind=qk) * 1.5
    R.check_prompt(gpu, c, q, q_lens, kv_lens, heads)


@pytest.mark.parametrize("qk,kv", [(F32, F16), (F16, F16), (F32, F32)])
def test_prompt_rows_that_see_nothing(gpu, qk, kv):
    """More query rows than keys: the first rows see none and give zeros."""
    q_lens, kv_lens = [40, 5, 3, 150], [10, 0, 3, 149]
    c = Cache(kv_lens, 16, 2, 128, kv, seed=1)
    q = randn(sum(q_lens), 4, 128, seed=2, kind=qk)
    out = R.check_prompt(gpu, c, q, q_lens, kv_lens, 4)
    assert bool((out[:30] == 0).all()) and bool((out[40:45] == 0).all()) and bool((out[48] == 0).all())


@pytest.mark.parametrize("qk,kv", [(F32, F16), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_prompt_unseen_values_do_not_reach_a_row(gpu, qk, kv, bad):
    """A NaN or infinity in a key or value that a row does not see (a later
    token's) leaves the row as it is; rows that see it get it."""
    n, heads, hd = 150, 4, 128
    c = Cache([n], 16, 2, hd, kv, seed=5)
    q = randn(n, heads, hd, seed=6, kind=qk)
    clean, st = R.prompt(gpu, c, q, [n], [n], heads, hd ** -0.5)
    assert st == 0
    pg, r = c.where(c.table[0], n)
    c.v[pg[100], r[100], 0, 3] = bad          # head 0's value of token 100
    c.k[pg[140], r[140], 1, 7] = float("nan")  # head 1's key of token 140
    out, st = R.prompt(gpu, c, q, [n], [n], heads, hd ** -0.5)
    assert st == 0
    err = (2.0 ** -10 if qk == F16 else 1e-5)
    assert torch.isfinite(out[:100]).all()
    assert float((out[:100].double() - clean[:100].double()).abs().max()) < err * 8
    assert not torch.isfinite(out[100:, :2, 3]).any()
    assert torch.isnan(out[140:, 2:]).all() and torch.isfinite(out[:140, 2:]).all()


def test_prompt_scores_far_apart(gpu):
    """Scores over a wide range, rising and falling along the keys: the
    running maximum moves in every tile."""
    n, heads, hd = 700, 2, 128
    for qk, kv in ((F32, F16), (F16, F16), (F32, F32)):
        c = Cache([n], 16, 1, hd, kv, seed=8)
        q = randn(n, heads, hd, seed=9, kind=qk)
        ramp = torch.linspace(0.2, 6.0, n, device="cuda")
        pg, r = c.where(c.table[0], n)
        c.k[pg, r] = (c.k[pg, r].float() * ramp[:, None, None]).to(R.DT[kv])
        R.check_prompt(gpu, c, q, [n], [n], heads)
        c.k[pg, r] = c.k[pg, r].flip(0)
        R.check_prompt(gpu, c, q, [n], [n], heads, scale=-0.11)


def test_prompt_strided_rows_and_bounds(gpu):
    """q inside a fused projection, out with gaps; lengths beyond max_kv and
    beyond the table are cut, rows beyond max_q left alone."""
    heads, n_kv, hd = 4, 2, 128
    c = Cache([90, 64], 16, n_kv, hd, F16, seed=3)
    buf = randn(60, heads + 3, hd, seed=4, kind=F16)
    q = buf[:, :heads]
    out = torch.full((60, heads + 1, hd), 7.0, dtype=torch.float16, device="cuda")[:, :heads]
    got, st = R.prompt(gpu, c, q, [30, 30], [90, 64], heads, 0.09, out=out)
    assert st == 0
    at = 0
    for i, (a, b) in enumerate(((30, 90), (30, 64))):
        k, v = c.rows(i)
        lim = torch.arange(a, device="cuda") + b - a + 1
        R.assert_rows(got[at:at + a], *R.attend(q[at:at + a], k, v, float(np.float32(0.09)), lim), i)
        at += a
    assert bool((torch.as_strided(out, (60, hd), (out.stride(0), 1), heads * hd) == 7.0).all()), "gaps changed"
    got, st = R.prompt(gpu, c, q, [30, 30], [90, 64], heads, 0.09, max_q=20, max_kv=70)
    assert st == 0
    k, v = c.rows(0)
    lim = (torch.arange(20, device="cuda") + 61).clamp(max=70)
    R.assert_rows(got[:20], *R.attend(q[:20], k[:70], v[:70], float(np.float32(0.09)), lim), "cut")
    assert bool((got[20:30] == 7.0).all())
    got, st = R.prompt(gpu, c, q, [30, 30], [10 ** 6, 64], heads, 0.09, max_kv=2 * 10 ** 6)   # the table holds 96
    assert st == 0 and bool((got[30:].isfinite()).all())


def test_bad_pages_read_as_zeros(gpu):
    heads, n_kv, hd = 4, 2, 128
    for qk, kv in ((F32, F16), (F16, F16), (F32, F32)):
        c = Cache([80, 80], 16, n_kv, hd, kv, seed=3)
        q = randn(80, heads, hd, seed=4, kind=qk)
        c.table[0, 2] = -5
        c.table[1, 1] = c.n_pages
        ref = []
        for i, bad in ((0, 2), (1, 1)):
            t = c.table[i].clone()
            t[bad] = 0
            j = torch.arange(80, device="cuda")
            k, v = c.k[t[j // 16].long(), j % 16].double(), c.v[t[j // 16].long(), j % 16].double()
            k[bad * 16:bad * 16 + 16] = 0
            v[bad * 16:bad * 16 + 16] = 0
            ref.append((k, v))
        out, st = R.prompt(gpu, c, q, [40, 40], [80, 80], heads, 0.1)
        assert st == 0
        dec, st = R.decode(gpu, c, q[:2], [80, 80], heads, 0.1)
        assert st == 0
        for i, (k, v) in enumerate(ref):
            lim = torch.arange(40, device="cuda") + 41
            R.assert_rows(out[40 * i:40 * i + 40], *R.attend(q[40 * i:40 * i + 40], k, v, float(np.float32(0.1)), lim), i)
            R.assert_rows(dec[i:i + 1], *R.attend(q[i:i + 1], k, v, float(np.float32(0.1)),
                                                  torch.tensor([80], device="cuda")), i)


# ---------------------------------------------------------- decode attention

@pytest.mark.parametrize("qk,kv", KINDS)
@pytest.mark.parametrize("heads,n_kv,hd,page,lens,prefix", [
    (32, 32, 128, 16, [1], 0),
    (6, 6, 48, 32, [272], 0),
    (32, 8, 128, 64, [1, 500, 33, 4, 0, 129], 0),
    (32, 8, 128, 16, [5, 700, 64, 1], 1000),
    (8, 1, 128, 16, [2000], 0),
    (16, 2, 64, 8, [300, 1, 77], 63),
    (40, 2, 96, 128, [90, 300], 130),
    (5, 1, 80, 7, [40, 90], 30),
    (3, 3, 33, 3, [20, 5], 4),
    (4, 2, 256, 16, [70, 300], 80),
    (8, 4, 32, 16, [0, 0, 0], 300),
    (4, 4, 128, 16, [0, 0], 0),
    (16, 16, 128, 32, [64] * 40, 700),
])
def test_decode_attention(gpu, qk, kv, heads, n_kv, hd, page, lens, prefix):
    c = Cache(lens, page, n_kv, hd, kv, seed=hd + page, prefix=prefix)
    q = randn(len(lens), heads, hd, seed=23, kind=qk) * 1.5
    R.check_decode(gpu, c, q, heads)


@pytest.mark.parametrize("qk,kv", [(F32, F16), (F16, F16), (F32, F32)])
def test_decode_long(gpu, qk, kv):
    """A long own part beside short ones, and a long prefix."""
    c = Cache([20011, 3, 900], 16, 2, 128, kv, seed=2)
    R.check_decode(gpu, c, randn(3, 8, 128, seed=3, kind=qk), 8)
    c = Cache([3, 900], 64, 2, 128, kv, seed=2, prefix=20011)
    R.check_decode(gpu, c, randn(2, 8, 128, seed=3, kind=qk), 8)


def test_decode_offsets_beyond_32_bits(gpu):
    """Pages whose element offsets pass 2^31 (and byte offsets 2^32)."""
    page, n_kv, hd = 64, 8, 128
    n_pages = (1 << 31) // (page * n_kv * hd) + 64
    c = Cache([200, 130], page, n_kv, hd, F16, seed=4)
    k = torch.empty(n_pages, page, n_kv, hd, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    shift = n_pages - c.n_pages
    k[shift:], v[shift:] = c.k, c.v
    c.k, c.v, c.n_pages = k, v, n_pages
    c.table = torch.where(c.table < 1 << 29, c.table + shift, c.table)
    q = randn(2, 16, hd, seed=5, kind=F16)
    R.check_decode(gpu, c, q, 16)
    q = randn(150, 16, hd, seed=5, kind=F32)
    R.check_prompt(gpu, c, q, [100, 50], [200, 130], 16)


def test_decode_is_deterministic_and_ignores_the_workspace(gpu):
    c = Cache([700, 30, 1500], 16, 4, 128, F16, seed=6, prefix=900)
    q = randn(3, 16, 128, seed=7)
    n = gpu.tos_attention_decode_paged_workspace_bytes(3, 1500, 900, 16, 4, 128)
    outs = []
    for fill in (0, 255, 63):
        ws = torch.full((n,), fill, dtype=torch.uint8, device="cuda")
        outs.append(R.decode(gpu, c, q, c.lens, 16, 0.08, ws=ws)[0])
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


# ------------------------------------------------------------- used together

@pytest.mark.parametrize("kv", [F16, F32])
def test_serving_run(gpu, kv):
    """Two prompts behind a shared prefix are appended and attended, then
    three decode steps; fp32 rows of one fused projection throughout."""
    heads, n_kv, hd, page, prefix = 8, 2, 64, 16, 50
    lens = [37, 90]
    d = R.rotary_desc(hd, "half", scaling="linear", factor=2.0)
    rot = Rotary(gpu, d)
    qw, kw = 1 + 0.1 * randn(hd, seed=1), 1 + 0.1 * randn(hd, seed=2)
    eps = float(np.float32(1e-6))
    c = Cache([0, 0], page, n_kv, hd, kv, seed=1, prefix=prefix, room=128)
    desc = c.desc()

    def step(rows_, seq, slot):
        n = rows_.shape[0]
        q, k, v = rows_[:, :heads], rows_[:, heads:heads + n_kv], rows_[:, heads + n_kv:]
        qo = torch.empty(n, heads, hd, device="cuda")
        sq = torch.tensor(seq, dtype=torch.int32, device="cuda")
        sl = torch.tensor(slot, dtype=torch.int32, device="cuda")
        pos = sl + prefix
        a = [R.rows(t) for t in (k, v, q, qo)]
        assert gpu.tos_kv_append_paged_dev(C.byref(desc), *[C.byref(r) for r in a], n, heads, sq.data_ptr(),
                                           sl.data_ptr(), pos.data_ptr(), qw.data_ptr(), kw.data_ptr(), 1e-6, rot.h,
                                           R.stream()) == 0
        R.assert_rows(qo, *R.norm_rotary(q, qw, eps, d, pos), "q")
        return qo

    x = randn(sum(lens), heads + 2 * n_kv, hd, seed=11)
    q = step(x, [0] * lens[0] + [1] * lens[1], list(range(lens[0])) + list(range(lens[1])))
    R.check_prompt(gpu, c, q, lens, lens, heads)
    for i in range(3):
        x = randn(2, heads + 2 * n_kv, hd, seed=20 + i)
        q = step(x, [0, 1], lens)
        lens = [n + 1 for n in lens]
        c.lens = lens
        R.check_decode(gpu, c, q, heads)


def test_graph_replay_with_changed_lengths(gpu):
    """A captured prompt call and a captured decode call, on a side stream,
    replayed after lengths, tables and queries changed; each has a workspace."""
    heads, n_kv, hd = 8, 2, 128
    c = Cache([300, 40], 16, n_kv, hd, F16, seed=1, prefix=100)
    q = randn(2, heads, hd, seed=2)
    qp = randn(64, heads, hd, seed=3, kind=F16)
    out, outp = torch.empty_like(q), torch.full_like(qp, 7.0)
    kl = torch.tensor([300, 40], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 50, 60], dtype=torch.int32, device="cuda")
    nd = gpu.tos_attention_decode_paged_workspace_bytes(2, 300, 100, heads, n_kv, hd)
    npr = gpu.tos_attention_prompt_paged_workspace_bytes(2, 64, 64, 300, heads, n_kv, hd)
    ws, wp = (torch.empty(max(n, 16), dtype=torch.uint8, device="cuda") for n in (nd, npr))
    desc, ro, rq, rop, rqp = c.desc(), R.rows(out), R.rows(q), R.rows(outp), R.rows(qp)

    def call():
        assert gpu.tos_attention_decode_paged_dev(C.byref(ro), C.byref(rq), C.byref(desc), kl.data_ptr(), 2, 300,
                                                  c.prefix_table.data_ptr(), 100, heads, 0.1, ws.data_ptr(), nd,
                                                  R.stream()) == 0
        assert gpu.tos_attention_prompt_paged_dev(C.byref(rop), C.byref(rqp), C.byref(desc), cu.data_ptr(),
                                                  kl.data_ptr(), 2, 64, 64, 300, heads, 0.1, wp.data_ptr(), npr,
                                                  R.stream()) == 0

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for lens, ql in (([300, 40], [50, 10]), ([17, 33], [5, 33]), ([1, 0], [1, 0])):
        kl.copy_(torch.tensor(lens, dtype=torch.int32))
        cu.copy_(torch.tensor([0, ql[0], sum(ql)], dtype=torch.int32))
        q.copy_(randn(2, heads, hd, seed=sum(lens)))
        outp.fill_(7.0)
        g.replay()
        pk, pv = c.prefix_rows()
        at = 0
        for i, n in enumerate(lens):
            k, v = c.rows(i, n)
            lim = (torch.arange(ql[i], device="cuda") + n - ql[i] + 1).clamp(0, n)
            R.assert_rows(outp[at:at + ql[i]], *R.attend(qp[at:at + ql[i]], k, v, float(np.float32(0.1)), lim), i)
            at += ql[i]
            k, v = torch.cat([pk, k]), torch.cat([pv, v])
            R.assert_rows(out[i:i + 1], *R.attend(q[i:i + 1], k, v, float(np.float32(0.1)),
                                                  torch.tensor([100 + n], device="cuda")), i)
        assert bool((outp[at:] == 7.0).all())


def test_two_streams_at_once(gpu):
    """Calls on two streams with a workspace each do not disturb one another."""
    heads, n_kv, hd = 16, 4, 128
    cs = [Cache([900, 200], 16, n_kv, hd, F16, seed=i, prefix=300) for i in (1, 2)]
    qs = [randn(2, heads, hd, seed=i) for i in (3, 4)]
    alone = [R.decode(gpu, c, q, c.lens, heads, 0.1)[0] for c, q in zip(cs, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    for _ in range(5):
        outs = []
        for st, c, q in zip(streams, cs, qs):
            with torch.cuda.stream(st):
                outs.append(R.decode(gpu, c, q, c.lens, heads, 0.1)[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(alone, outs))


# ------------------------------------- large enough for the tiled kernels
# (the few-rows kernels take the small calls above: 8 query rows at a time)

@pytest.mark.parametrize("qk,kv", KINDS)
@pytest.mark.parametrize("heads,n_kv,hd,page,q_lens,hist", [
    (8, 2, 128, 16, [700, 1, 129], [0, 300, 513]),          # groups of 4: row tiles end inside a token
    (6, 2, 128, 64, [513, 0, 300], [200, 7, 0]),            # groups of 3
    (16, 4, 64, 8, [1200, 33], [0, 900]),
    (12, 12, 48, 32, [900, 517], [0, 7]),
    (24, 4, 32, 128, [1100, 700], [100, 0]),
    (16, 2, 96, 256, [600, 31, 1], [0, 511, 1000]),
    (8, 8, 80, 48, [700], [31]),                            # pages of 48: no tensor-core tiles
    (4, 2, 200, 16, [500], [0]),
    (40, 1, 128, 16, [90, 2], [700, 3000]),                 # few row tiles, many keys: the key axis is split
    (8, 8, 128, 32, [40] * 50, [3 * i for i in range(50)]),  # more sequences than lanes of the plan
])
def test_prompt_attention_tiles(gpu, qk, kv, heads, n_kv, hd, page, q_lens, hist):
    kv_lens = [a + b for a, b in zip(q_lens, hist)]
    c = Cache(kv_lens, page, n_kv, hd, kv, seed=hd + page)
    q = randn(sum(q_lens) + 2, heads, hd, seed=17, kind=qk) * 1.5
    R.check_prompt(gpu, c, q, q_lens, kv_lens, heads)


@pytest.mark.parametrize("qk,kv", [(F32, F16), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("hd", [64, 128])
def test_tiles_rows_that_see_nothing_and_negative_scale(gpu, qk, kv, hd):
    q_lens, kv_lens = [900, 300, 40, 512], [700, 0, 40, 511]
    c = Cache(kv_lens, 16, 4, hd, kv, seed=1)
    q = randn(sum(q_lens), 16, hd, seed=2, kind=qk)
    out = R.check_prompt(gpu, c, q, q_lens, kv_lens, 16, scale=-0.2)
    assert bool((out[:200] == 0).all()) and bool((out[900:1200] == 0).all()) and bool((out[1240] == 0).all())
    R.check_prompt(gpu, c, q, q_lens, kv_lens, 16, scale=0.0)


@pytest.mark.parametrize("qk,kv", [(F32, F16), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,hist", [(900, 0), (60, 3000)])
def test_tiles_unseen_values_do_not_reach_a_row(gpu, qk, kv, hd, n, hist):
    """As above, over many tiles, and with the keys split."""
    heads = 16
    c = Cache([n + hist], 16, 2, hd, kv, seed=5)
    q = randn(n, heads, hd, seed=6, kind=qk)
    clean, st = R.prompt(gpu, c, q, [n], [n + hist], heads, hd ** -0.5)
    assert st == 0
    pg, r = c.where(c.table[0], n + hist)
    at, at_k = hist + n // 2, hist + n - 7
    c.v[pg[at], r[at], 0, 3] = float("inf")
    c.k[pg[at_k], r[at_k], 1, 7] = float("nan")
    out, st = R.prompt(gpu, c, q, [n], [n + hist], heads, hd ** -0.5)
    assert st == 0
    half = heads // 2
    assert torch.isfinite(out[:n // 2]).all()
    assert float((out[:n // 2].double() - clean[:n // 2].double()).abs().max()) < 8 * (2.0 ** -10 if qk == F16 else 1e-5)
    assert not torch.isfinite(out[n // 2:, :half, 3]).any()
    assert torch.isnan(out[n - 7:, half:]).all() and torch.isfinite(out[:n - 7, half:]).all()


@pytest.mark.parametrize("qk,kv", [(F32, F16), (F16, F16), (F32, F32)])
def test_tiles_scores_far_apart(gpu, qk, kv):
    """The running maximum moves in every key tile, up and (reversed) not."""
    n, heads, hd = 1000, 8, 128
    c = Cache([n], 16, 2, hd, kv, seed=8)
    q = randn(n, heads, hd, seed=9, kind=qk)
    ramp = torch.linspace(0.2, 12.0, n, device="cuda")
    pg, r = c.where(c.table[0], n)
    c.k[pg, r] = (c.k[pg, r].float() * ramp[:, None, None]).to(R.DT[kv])
    R.check_prompt(gpu, c, q, [n], [n], heads)
    c.k[pg, r] = c.k[pg, r].flip(0)
    R.check_prompt(gpu, c, q, [n], [n], heads)
    q[::3] *= 1e-4 if qk == F32 else 1.0          # small rows keep their 22 bits
    R.check_prompt(gpu, c, q, [n], [n], heads, scale=30.0 if qk == F32 else 0.1)


@pytest.mark.parametrize("qk,kv", [(F32, F16), (F16, F16)])
def test_tiles_unaligned_rows(gpu, qk, kv):
    """q and out at odd strides from odd elements."""
    n, heads, hd = 600, 8, 128
    c = Cache([n], 16, 2, hd, kv, seed=3)
    w = heads * hd + 3
    buf, obuf = randn(n * w + 8, seed=4, kind=qk), torch.full((n * w + 8,), 7.0, dtype=R.DT[qk], device="cuda")
    q = torch.as_strided(buf, (n, heads, hd), (w, hd, 1), 1)
    out = torch.as_strided(obuf, (n, heads, hd), (w, hd, 1), 5)
    got, st = R.prompt(gpu, c, q, [n], [n], heads, 0.09, out=out)
    assert st == 0
    k, v = c.rows(0)
    R.assert_rows(got, *R.attend(q, k, v, float(np.float32(0.09)), torch.arange(n, device="cuda") + 1))
    assert bool((torch.as_strided(obuf, (n, 3), (w, 1), 5 + heads * hd)[:-1] == 7.0).all())


def test_prefix_of_many_rows(gpu):
    """More decode rows than a tile over the prefix, groups that do not
    divide it, and an empty own part beside full ones."""
    for qk, kv, hd in ((F32, F16, 128), (F16, F16, 64), (F32, F32, 96), (F16, F16, 256)):
        lens = [(i * 37) % 200 for i in range(70)]
        c = Cache(lens, 16, 2, hd, kv, seed=hd, prefix=1025)
        R.check_decode(gpu, c, randn(70, 10, hd, seed=3, kind=qk), 10)


def test_tiles_that_see_nothing_many_times(gpu):
    """Whole row tiles without a key beside ones with: their rows are written
    while other warps may still be at the tile's queries."""
    heads, hd, q_lens, kv_lens = 16, 128, [900, 700, 800], [400, 0, 300]
    c = Cache(kv_lens, 16, 4, hd, F16, seed=1)
    q = randn(sum(q_lens), heads, hd, seed=2, kind=F16)
    first = R.check_prompt(gpu, c, q, q_lens, kv_lens, heads)
    for _ in range(60):
        out, st = R.prompt(gpu, c, q, q_lens, kv_lens, heads, hd ** -0.5)
        assert st == 0 and torch.equal(out, first)


@pytest.mark.parametrize("hist", [700, 9000])
def test_tiles_long_sums_do_not_shrink(gpu, hist):
    """fp32 rows over many keys with values of one sign.  A tensor-core sum
    cuts off up to a unit, 2^-23, a step; steps of 16 keys, high and low parts,
    in chains of at most 512 keys: 64 2^-23 = 7.6e-6, and scores and weights a
    tenth of that."""
    n, heads, hd = 300, 16, 128
    c = Cache([n + hist], 64, 16, hd, F16, seed=2)
    pg, r = c.where(c.table[0], n + hist)
    c.v[pg, r] = 1 + c.v[pg, r] / 16
    q = randn(n, heads, hd, seed=3)
    out, st = R.prompt(gpu, c, q, [n], [n + hist], heads, hd ** -0.5)
    assert st == 0
    k, v = c.rows(0)
    ref, _ = R.attend(q, k, v, float(np.float32(hd ** -0.5)), torch.arange(n, device="cuda") + hist + 1)
    assert float(((out.double() - ref) / ref).abs().max()) < 8.5e-6


@pytest.mark.parametrize("qk,kv", [(F32, F16), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("hd", [128, 64])
def test_prompt_of_many_sequences(gpu, qk, kv, hd):
    """More sequences than the plan sorts, empty ones among them."""
    q_lens = [(i * 7) % 23 if i % 5 else 0 for i in range(300)]
    q_lens[150] = 700
    kv_lens = [n + (i * 13) % 90 for i, n in enumerate(q_lens)]
    c = Cache(kv_lens, 16, 2, hd, kv, seed=4)
    R.check_prompt(gpu, c, randn(sum(q_lens), 8, hd, seed=5, kind=qk), q_lens, kv_lens, 8)


@pytest.mark.parametrize("qk,kv", KINDS)
@pytest.mark.parametrize("heads,n_kv,hd,page,n", [(8, 4, 128, 16, 4), (8, 4, 128, 16, 5), (4, 4, 64, 64, 32),
                                                  (4, 4, 64, 64, 33), (12, 1, 256, 5, 2), (6, 6, 48, 32, 1)])
def test_prefix_around_the_limits_of_a_row_tile(gpu, qk, kv, heads, n_kv, hd, page, n):
    """8, 10, 32 and 33 rows a key/value head behind prefixes of a page and of many splits."""
    for prefix in (1, page, 2111):
        c = Cache([(i * 37) % 150 for i in range(n)], page, n_kv, hd, kv, seed=n + prefix, prefix=prefix)
        R.check_decode(gpu, c, randn(n, heads, hd, seed=prefix, kind=qk), heads)


@pytest.mark.parametrize("qk,kv", KINDS)
@pytest.mark.parametrize("heads,n_kv,hd,page", [(71, 1, 64, 256), (128, 1, 128, 512), (28, 4, 120, 24), (9, 1, 96, 100)])
def test_wide_and_odd_groups(gpu, qk, kv, heads, n_kv, hd, page):
    """Groups that are no power of two or fill a row tile alone, pages larger than a key tile or across its end."""
    q_lens = [3, 0, 41]
    kv_lens = [300, 5, 41]
    c = Cache(kv_lens, page, n_kv, hd, kv, seed=heads)
    R.check_prompt(gpu, c, randn(sum(q_lens), heads, hd, seed=8, kind=qk), q_lens, kv_lens, heads)
    c = Cache(kv_lens, page, n_kv, hd, kv, seed=heads, prefix=777)
    R.check_decode(gpu, c, randn(3, heads, hd, seed=9, kind=qk), heads)


# ------------------------------------------ keys and values that are not finite

@pytest.mark.parametrize("qk,kv", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,hist", [(600, 0), (40, 300)])
def test_seen_nan_key_at_every_place(gpu, qk, kv, hd, n, hist):
    """A NaN in one key of each head, at all 16 places of a step and all over
    the last 128 keys: the rows that see it are NaN, the others as without it."""
    heads = 16
    c = Cache([n + hist], 16, heads, hd, kv, seed=5)
    q = randn(n, heads, hd, seed=6, kind=qk)
    k, v = c.rows(0)
    pg, r = c.where(c.table[0], n + hist)
    at = [n + hist - 128 + (17 * h) % 128 for h in range(heads)]
    for h in range(heads):
        c.k[pg[at[h]], r[at[h]], h, (5 * h) % hd] = float("nan")
    out, st = R.prompt(gpu, c, q, [n], [n + hist], heads, hd ** -0.5)
    assert st == 0
    lim = torch.arange(n, device="cuda") + hist + 1
    ref, err = R.attend(q, k, v, float(np.float32(hd ** -0.5)), lim)
    for h in range(heads):
        sees = lim > at[h]
        assert bool(torch.isnan(out[sees, h]).all()), (h, at[h])
        R.assert_rows(out[~sees, h], ref[~sees, h], err[~sees, h], (h, at[h]))


def fastest(f, times=3):
    """us of the fastest of some calls, after one"""
    f()
    best = float("inf")
    for _ in range(times):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3)
    return best


@pytest.mark.parametrize("qk,kv", KINDS)
@pytest.mark.parametrize("hd,n,hist,heads,n_kv", [(128, 70, 3000, 16, 4), (64, 300, 1900, 16, 4), (128, 1200, 0, 32, 8),
                                                  (128, 3, 1500, 8, 4), (200, 40, 700, 4, 2)])
@pytest.mark.parametrize("what", ["seen nan key", "seen inf value", "unseen nan value"])
def test_values_that_are_not_finite_cost_no_second_pass(gpu, qk, kv, hd, n, hist, heads, n_kv, what):
    """A call with a NaN or an infinity takes as long as one without, times a
    small number: no row is computed again key by key (a microsecond a key)."""
    c = Cache([n + hist], 16, n_kv, hd, kv, seed=5)
    q = randn(n, heads, hd, seed=6, kind=qk)
    args = (gpu, c, q, [n], [n + hist], heads, hd ** -0.5)
    out, st = R.prompt(*args)
    assert st == 0
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    clean = fastest(lambda: R.prompt(*args, out=out, ws=ws))
    pg, r = c.where(c.table[0], n + hist)
    at = n + hist - 1 if what.startswith("unseen") else 5
    x = c.k if what.endswith("key") else c.v
    x[pg[at], r[at], :, 3] = float("inf" if "inf" in what else "nan")
    assert fastest(lambda: R.prompt(*args, out=out, ws=ws)) < 4 * clean + 100


@pytest.mark.parametrize("qk,kv", KINDS)
@pytest.mark.parametrize("hd,n,hist,heads,n_kv", [(128, 300, 700, 16, 4), (64, 513, 0, 16, 16), (128, 1200, 0, 32, 8),
                                                  (128, 60, 5000, 16, 2), (128, 7, 300, 8, 4), (64, 9, 120, 5, 1),
                                                  (200, 90, 100, 6, 2), (80, 150, 31, 4, 4), (33, 50, 9, 3, 3)])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(gpu, qk, kv, hd, n, hist, heads, n_kv):
    """Infinities of both signs and NaN among the values of the last tokens
    and of one that all rows see: an element is the sum of those that its row
    sees, or as if there were none.  And infinite keys, which give a weight of
    zero or, at +infinity, a NaN."""
    m = n + hist
    c = Cache([m], 16, n_kv, hd, kv, seed=5)
    q = randn(n, heads, hd, seed=6, kind=qk)
    k, v = c.rows(0)
    pg, r = c.where(c.table[0], m)
    inf, nan = float("inf"), float("nan")
    back = lambda f: m - 1 - int(f * (n - 1))       # tokens of the prompt, from its end
    plan = [(back(0), 0, 0, nan), (back(.1), 0, 1, inf), (back(.2), 0, 1, inf), (back(.3), 0, 2, -inf),
            (back(.25), 0, 2, inf), (back(.6), n_kv - 1, hd - 1, -inf), (back(.9), n_kv - 1, hd // 2, nan)]
    if hist:
        plan.append((3, n_kv - 1, 5, -inf))
    extra = torch.zeros(n, heads, hd, dtype=torch.float64, device="cuda")
    lim = torch.arange(n, device="cuda") + hist + 1
    g = heads // n_kv
    for (at, h, d), x in {e[:3]: e[3] for e in plan}.items():       # short prompts: two may name one place
        c.v[pg[at], r[at], h, d] = x
        sees = (lim > at).nonzero().flatten()
        extra[sees, h * g:(h + 1) * g, d] += x
    out, st = R.prompt(gpu, c, q, [n], [m], heads, hd ** -0.5)
    assert st == 0
    ref, err = R.attend(q, k, v, float(np.float32(hd ** -0.5)), lim)
    # the plan replaced values that rows saw: their elements are infinite or NaN, all others as they were
    ok = extra == 0
    R.assert_rows(out[ok], ref[ok], err[ok], "finite")
    assert torch.equal(torch.isnan(out[~ok]), torch.isnan(extra[~ok])), "NaN"
    z = ~ok & ~torch.isnan(extra)
    assert torch.equal(out[z].double(), extra[z]), "infinities"


@pytest.mark.parametrize("qk,kv", KINDS)
@pytest.mark.parametrize("hd,n,hist,heads,n_kv", [(128, 300, 700, 16, 4), (64, 513, 0, 16, 16), (128, 60, 5000, 16, 2),
                                                  (128, 7, 300, 8, 4), (200, 90, 100, 6, 2)])
def test_infinite_keys(gpu, qk, kv, hd, n, hist, heads, n_kv):
    """An infinite element of a key: a score of -infinity weighs nothing, one
    of +infinity makes the row NaN."""
    m = n + hist
    c = Cache([m], 16, n_kv, hd, kv, seed=5)
    q = randn(n, heads, hd, seed=6, kind=qk)
    q[:, :, 7] = q[:, :, 7].abs() + 0.01
    q[:, 0, 7] *= -1
    k, v = c.rows(0)
    pg, r = c.where(c.table[0], m)
    lim = torch.arange(n, device="cuda") + hist + 1
    ats = [m - 1 - i * max(1, n // 5) for i in range(4)]
    for at in ats:
        c.k[pg[at], r[at], :, 7] = float("-inf")
        k[at, :, 7] = -1e9                             # as good as -infinity in 64 bits
    out, st = R.prompt(gpu, c, q, [n], [m], heads, hd ** -0.5)
    assert st == 0
    ref, _ = R.attend(q, k, v, float(np.float32(hd ** -0.5)), lim)
    for at in ats:
        k[at, :, 7] = 0
    _, err = R.attend(q, k, v, float(np.float32(hd ** -0.5)), lim)
    R.assert_rows(out[:, 1:], ref[:, 1:], 2 * err[:, 1:], "-inf")
    sees = lim > min(ats)
    assert bool(torch.isnan(out[sees, 0]).all()) and bool(torch.isfinite(out[~sees, 0]).all())


@pytest.mark.parametrize("qk,heads,n_kv", [(F32, 16, 4), (F16, 16, 4), (F32, 8, 1)])
def test_nan_value_behind_a_long_history(gpu, qk, heads, n_kv):
    """200,000 keys: one value that all rows see and one that few see are NaN.
    The call ends in time, and no other element changes."""
    n, m, hd = 70, 200000, 128
    c = Cache([m], 64, n_kv, hd, F16, seed=5)
    q = randn(n, heads, hd, seed=6, kind=qk)
    clean, st = R.prompt(gpu, c, q, [n], [m], heads, hd ** -0.5)
    assert st == 0
    pg, r = c.where(c.table[0], m)
    c.v[pg[5], r[5], :, 3] = float("nan")
    c.v[pg[m - 9], r[m - 9], :, 70] = float("nan")
    out, st = R.prompt(gpu, c, q, [n], [m], heads, hd ** -0.5)
    torch.cuda.synchronize()
    assert st == 0 and gpu.tos_synchronize() == 0
    assert bool(torch.isnan(out[:, :, 3]).all()) and bool(torch.isnan(out[n - 9:, :, 70]).all())
    out[:, :, 3], out[n - 9:, :, 70] = clean[:, :, 3], clean[n - 9:, :, 70]
    assert torch.equal(out, clean)


# ----------------------------------------------- long sums of values of one sign
# A tensor-core accumulator cuts off what it has no room for, so a long chain of
# sums comes out small.  Sums rounded to nearest err both ways: N additions to
# a sum that grows evenly have a standard deviation of u / sqrt(3) sqrt(N / 3),
# 2^-24 / 3 sqrt(N) of the sum.  The bounds are six of those and, once, what
# the longest chain between two roundings to nearest may lose.

def one_sign(c, m):
    """Values of every dim about one number of its own in [1, 2]"""
    pg, r = c.where(c.table[0], m)
    x = c.v[pg, r].float() / 16 + 1 + torch.arange(c.hd, device="cuda") / c.hd
    c.v[pg, r] = x.to(c.v.dtype)


def test_decode_long_sums_do_not_shrink(gpu):
    """640 sequences times heads, so that a CTA has all of one's keys: 512 steps
    a warp.  The weights' sum and the values' have 512 additions each."""
    n, heads, hd, m = 40, 16, 128, 32768
    c = Cache([m], 64, heads, hd, F16, seed=2)
    one_sign(c, m)
    k, v = c.rows(0)
    c.table, c.lens = c.table.expand(n, -1).contiguous(), [m] * n       # all read the same pages
    q = randn(n, heads, hd, seed=3)
    out, st = R.decode(gpu, c, q, c.lens, heads, hd ** -0.5)
    assert st == 0
    ref, _ = R.attend(q, k, v, float(np.float32(hd ** -0.5)), torch.full((n,), m, device="cuda"))
    rel = (out.double() - ref) / ref
    chain = 2 * 2.0 ** -23                                    # one product of 16 keys, two parts
    assert float(rel.abs().max()) < 6 * 2.0 ** -24 / 3 * (512 + 512) ** 0.5 + chain + 2.0 ** -23


@pytest.mark.parametrize("m", [700, 9000])
def test_prompt_sums_of_one_sign(gpu, m):
    """fp32 rows: chains of 24 steps of 16 keys, which lose a unit, 2^-23, each;
    one addition of the weights a key tile, of the values three tiles."""
    n, heads, hd = 300, 16, 128
    m += n
    c = Cache([m], 64, heads, hd, F16, seed=2)
    one_sign(c, m)
    k, v = c.rows(0)
    q = randn(n, heads, hd, seed=3)
    out, st = R.prompt(gpu, c, q, [n], [m], heads, hd ** -0.5)
    assert st == 0
    ref, _ = R.attend(q, k, v, float(np.float32(hd ** -0.5)), torch.arange(n, device="cuda") + m - n + 1)
    rel = (out.double() - ref) / ref
    assert float(rel.abs().max()) < 6 * 2.0 ** -24 / 3 * (m / 128 + m / 384) ** 0.5 + 24 * 2.0 ** -23 + 2.0 ** -23


@pytest.mark.parametrize("qk", [F32, F16])
def test_prompt_long_sums_do_not_shrink(gpu, qk):
    """131,072 keys in one piece (352 row tiles leave nothing to split).  fp32
    rows as above.  fp16 rows: the mean error of 128 dims' numbers, whose
    rounding, 2^-11 / sqrt(3) each, averages out, is a twentieth of half a step
    at most for a chain's loss, and five deviations of the mean."""
    n, heads, n_kv, hd, m = 700, 128, 16, 128, 131072
    c = Cache([m], 64, n_kv, hd, F16, seed=2)
    one_sign(c, m)
    q = randn(n, heads, hd, seed=3, kind=qk)
    out, st = R.prompt(gpu, c, q, [n], [m], heads, hd ** -0.5)
    assert st == 0
    pick = torch.arange(0, n, 50, device="cuda")
    k, v = c.rows(0)
    ref, _ = R.attend(q[pick, :8], k[:, :1], v[:, :1], float(np.float32(hd ** -0.5)), pick + m - n + 1)
    rel = (out[pick, :8].double() - ref) / ref
    if qk == F32:
        assert float(rel.abs().max()) < 6 * 2.0 ** -24 / 3 * (m / 128 + m / 384) ** 0.5 + 24 * 2.0 ** -23 + 2.0 ** -23
    else:
        assert abs(float(rel.mean())) < 2.0 ** -11 / 20 + 5 * 2.0 ** -11 / 3 ** 0.5 / 128 ** 0.5


# ------------------------------------------------------------------ YaRN's ramp

@pytest.mark.parametrize("rot,base,orig,factor,low,high", [
    (128, 10000.0, 4096, 4.0, 20, 46),        # 20.94 and 45.03
    (64, 10000.0, 4096, 40.0, 10, 23),        # 10.47 and 22.51
    (128, 500000.0, 8192, 8.0, 18, 35),       # 18.08 and 34.98
    (64, 1000000.0, 32768, 4.0, 11, 20),      # 11.80 and 19.83
    (64, 10000.0, 100, 8.0, 0, 10),           # -2.43 and 9.61
    (64, 10000.0, 4, 8.0, 0, 0.001),          # -13.61 and -1.57: all slow but the first
    (4, 10000.0, 10 ** 9, 8.0, 3, 3.001),     # 3.35 and 4.10: all fast
])
def test_yarn_ramp_between_rounded_edges(gpu, rot, base, orig, factor, low, high):
    """Scaling 3 against the edges, worked out apart from this code: pairs up to
    the first keep their frequency, from the second on have it divided by the
    factor, and between them go from one to the other in equal steps."""
    d = R.rotary_desc(rot, "half", base=base, factor=factor, orig=orig, attn=1.0)
    d.scaling = 3
    r = Rotary(gpu, d)
    pos = torch.tensor([1, 7, 1000, 65535], dtype=torch.int32, device="cuda")
    x = torch.zeros(4, 1, rot, device="cuda")
    x[..., :rot // 2] = 1
    y = torch.empty_like(x)
    a, b = R.rows(x), R.rows(y)
    assert gpu.tos_qk_norm_rotary_dev(C.byref(a), C.byref(b), None, None, 4, 1, 0, rot, None, None, 0.0, r.h,
                                      pos.data_ptr(), R.stream()) == 0
    mag = 1 + 0.1 * math.log(factor)
    for i in range(rot // 2):
        part = 0.0 if i <= low else 1.0 if i >= high else (i - low) / (high - low)
        angle = pos.double().cpu() * base ** (-2.0 * i / rot) * (1 - part + part / factor)
        tol = mag * (2.0 ** -22 + 4 * R.U)
        assert float((y[:, 0, i].double().cpu() - mag * torch.cos(angle)).abs().max()) < tol, i
        assert float((y[:, 0, i + rot // 2].double().cpu() - mag * torch.sin(angle)).abs().max()) < tol, i


# ------------------------------------------------------------- counts of heads

@pytest.mark.parametrize("hd,odd", [(2, 0), (4, 1), (8, 0)])
def test_rotary_of_very_many_heads(gpu, hd, odd):
    """More heads than one warp each of the largest grid, element-wise (2 dims,
    an odd address) and in 16-byte pieces."""
    heads, n_kv, n = 270001, 263001, 2
    buf = randn(n * (heads + n_kv) * hd + 8, seed=1)
    x = torch.as_strided(buf, (n, heads + n_kv, hd), ((heads + n_kv) * hd, hd, 1), odd)
    q, k = x[:, :heads], x[:, heads:]
    qo, ko = torch.empty(n, heads, hd, device="cuda"), torch.empty(n, n_kv, hd, device="cuda")
    d = R.rotary_desc(hd, "interleaved")
    rot = Rotary(gpu, d)
    pos = torch.tensor([5, 900], dtype=torch.int32, device="cuda")
    a = [R.rows(t) for t in (q, qo, k, ko)]
    assert gpu.tos_qk_norm_rotary_dev(*[C.byref(r) for r in a], n, heads, n_kv, hd, None, None, 0.0, rot.h,
                                      pos.data_ptr(), R.stream()) == 0
    R.assert_rows(qo, *R.norm_rotary(q, None, 0.0, d, pos), "q")
    R.assert_rows(ko, *R.norm_rotary(k, None, 0.0, d, pos), "k")


def test_append_of_very_many_heads(gpu):
    n_kv, hd, page = 140001, 2, 2
    c = Cache([3], page, n_kv, hd, F32, seed=1, fill=3.0)
    k, v = randn(2, n_kv, hd, seed=2), randn(2, n_kv, hd, seed=3)
    seq, slot = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, 0], [1, 2]))
    a, desc = [R.rows(t) for t in (k, v)], c.desc()
    assert gpu.tos_kv_append_paged_dev(C.byref(desc), *[C.byref(r) for r in a], None, None, 2, 0, seq.data_ptr(),
                                       slot.data_ptr(), None, None, None, 0.0, None, R.stream()) == 0
    pg, r = c.where(c.table[0], 3)
    assert torch.equal(c.k[pg[1:], r[1:]], k) and torch.equal(c.v[pg[1:], r[1:]], v)


@pytest.mark.parametrize("heads,n_kv,hd", [(32, 8, 128), (16, 4, 96)])
@pytest.mark.parametrize("n,hist", [(90, 400), (64, 1900)])
def test_short_prompts_err_little(gpu, n, hist, heads, n_kv, hd):
    """fp32 rows that see few keys, where an fp32 program errs least.  Chains of
    two key tiles, 16 steps of high and low parts, each of which loses half a
    unit, 2^-24, of the sum so far, half of the whole on the average; a tenth of
    that for all else."""
    c = Cache([n + hist], 16, n_kv, hd, F16, seed=3)
    q = randn(n, heads, hd, seed=4)
    out, st = R.prompt(gpu, c, q, [n], [n + hist], heads, hd ** -0.5)
    assert st == 0
    k, v = c.rows(0)
    ref, _ = R.attend(q, k, v, float(np.float32(hd ** -0.5)), torch.arange(n, device="cuda") + hist + 1)
    assert float((out.double() - ref).norm() / ref.norm()) < 1.1 * 32 * 2.0 ** -24 / 2
