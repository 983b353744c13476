"""Plain 64-bit forms of the 8-bit paged cache's operators, for the tests.
Values of a cache are exact in fp32 and in 64 bits, so what it stores is
compared bit for bit, and attention with the bounds of paged_ref.py (its
products, sums and weights are formed alike, and reading the cache rounds
nothing)."""
import ctypes as C

import numpy as np
import torch

import paged_ref as R
from tensoros_b200 import _ffi

I8, F8 = 24, 64
TOP = {I8: 127.0, F8: 448.0}
LIMITS = {I8: (-24, 9), F8: (-15, 7)}
ELEM = {I8: torch.int8, F8: torch.float8_e4m3fn}


def needed(amax, kind):
    """The least power of two with which magnitudes [...] fit, in 64 bits, found
    by trying every exponent."""
    out = torch.full(amax.shape, 2.0 ** LIMITS[kind][1], dtype=torch.float64, device=amax.device)
    for e in range(LIMITS[kind][1], LIMITS[kind][0] - 1, -1):
        out = torch.where(amax.double() <= TOP[kind] * 2.0 ** e, torch.full_like(out, 2.0 ** e), out)
    return torch.where(torch.isfinite(amax.double()), out, torch.full_like(out, float("nan")))


def nearest(y, kind):
    """64-bit numbers rounded to those that an element holds, ties to even."""
    if kind == I8:
        return torch.round(y).clamp(-127, 127)
    m, e = torch.frexp(y.abs())
    step = torch.ldexp(torch.ones_like(y), e.clamp(min=-5) - 4)
    return (torch.round(y / step) * step).clamp(-448, 448)


class Cache8:
    """A pool of pages with sequences in shuffled pages, filled by hand.  What no
    sequence uses holds random bytes and NaN scales, table entries that no
    sequence uses point nowhere."""

    def __init__(self, lens, page, block, n_kv, hd, kind, seed=0, spare=3, room=0, spread=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.page, self.block, self.n_kv, self.hd, self.kind = list(lens), page, block, n_kv, hd, kind
        need = [(max(n, room) + page - 1) // page for n in self.lens]
        self.n_pages = sum(need) + spare
        shape = (self.n_pages, page, n_kv, hd)
        self.k = torch.randint(-127, 128, shape, generator=g, dtype=torch.int8, device="cuda")
        self.v = torch.randint(-127, 128, shape, generator=g, dtype=torch.int8, device="cuda")
        self.ks = torch.full((self.n_pages, page // block, n_kv), float("nan"), device="cuda")
        self.vs = self.ks.clone()
        perm = torch.randperm(self.n_pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(need), max(1, max(need, default=1))), 2 ** 30, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = perm[at:at + n]
            at += n
        for i, n in enumerate(self.lens):
            for x, s in ((self.k, self.ks), (self.v, self.vs)):
                rows = torch.randn(n, n_kv, hd, generator=g, device="cuda")
                rows *= torch.exp(spread * torch.randn(n, n_kv, 1, generator=g, device="cuda"))
                self.put(x, s, i, 0, rows.double())

    def where(self, i, a, b):
        j = torch.arange(a, b, device="cuda")
        return self.table[i][j // self.page].long(), j % self.page

    def put(self, pool, scales, i, first, rows):
        """Rows first .. of sequence i, from their block's first row on, in 64 bits."""
        if rows.shape[0] == 0:
            return
        n, lo = rows.shape[0], first % self.block
        pg, r = self.where(i, first, first + n)
        blocks = (lo + n + self.block - 1) // self.block
        x = rows.new_zeros(blocks * self.block, *rows.shape[1:])
        x[lo:lo + n] = rows
        s = needed(x.view(blocks, self.block, *rows.shape[1:]).abs().amax((1, 3)), self.kind)
        s = s.repeat_interleave(self.block, 0)[lo:lo + n]
        scales[pg, r // self.block] = s.float()
        pool[pg, r] = nearest(rows / s[..., None], self.kind).to(ELEM[self.kind]).view(torch.int8)

    def rows(self, i, n=None, pool="k"):
        """Values of the first n rows of sequence i in 64 bits, [n][n_kv][hd]"""
        return self.rows_at(i, 0, self.lens[i] if n is None else n, pool)

    def rows_at(self, i, a, b, pool="k"):
        pg, r = self.where(i, a, b)
        x = getattr(self, pool)[pg, r].view(ELEM[self.kind]).double()
        return x * getattr(self, pool + "s")[pg, r // self.block].double()[..., None]

    def desc(self):
        return _ffi.Paged8Kv(self.k.data_ptr(), self.v.data_ptr(), self.ks.data_ptr(), self.vs.data_ptr(), self.kind,
                             self.block, self.n_pages, self.page, self.n_kv, self.hd, self.table.data_ptr(),
                             self.table.shape[0], self.table.stride(0))


def ints(values):
    return torch.tensor([int(v) for v in values], dtype=torch.int32, device="cuda")


def packed(lens):
    return ints(np.concatenate([[0], np.cumsum(lens)]))


def append(gpu, c, k, v, lens, total, kv_len=None, cu=None):
    """The library's call: rows of k and v behind what the sequences hold."""
    kv_len = [a + b for a, b in zip(c.lens, lens)] if kv_len is None else kv_len
    cu, kl = packed(lens) if cu is None else cu, ints(kv_len)
    d, rk, rv = c.desc(), R.rows(k), R.rows(v)
    st = gpu.tos_kv_append_paged8_dev(C.byref(d), C.byref(rk), C.byref(rv), cu.data_ptr(), kl.data_ptr(), len(lens),
                                      total, R.stream())
    if st == 0:
        torch.cuda.synchronize()
    return st


def expect_append(c, k, v, lens):
    """What the pools and scales hold after it: (k, v, ks, vs), by blocks."""
    out = []
    for pool, scales, x in ((c.k.clone(), c.ks.clone(), k), (c.v.clone(), c.vs.clone(), v)):
        at = 0
        for i, n in enumerate(lens):
            base, new = c.lens[i], x[at:at + n].double()
            at += n
            for b in range(base // c.block, (base + n + c.block - 1) // c.block if n else 0):
                lo, hi = max(base, b * c.block), min(base + n, (b + 1) * c.block)
                pg, r = c.where(i, b * c.block, hi)
                pg0, blk = pg[0], r[0] // c.block
                had = lo - b * c.block
                need = needed(new[lo - base:hi - base].abs().amax((0, 2)), c.kind)
                old = scales[pg0, blk].double()
                now = need if had == 0 else torch.where(torch.isnan(need) | torch.isnan(old), need * old,
                                                        torch.maximum(need, old))
                keep = torch.isnan(now)
                if had:
                    y = pool[pg[:had], r[:had]].view(ELEM[c.kind]).double() * (old / now)[:, None]
                    y = nearest(y, c.kind).to(ELEM[c.kind]).view(torch.int8)
                    pool[pg[:had], r[:had]] = torch.where(keep[:, None], pool[pg[:had], r[:had]], y)
                y = new[lo - base:hi - base] / now[:, None]
                y = nearest(y, c.kind).to(ELEM[c.kind]).view(torch.int8)
                pool[pg[had:], r[had:]] = torch.where(keep[:, None], pool[pg[had:], r[had:]], y)
                scales[pg0, blk] = now.float()
        out += [pool, scales]
    return out[0], out[2], out[1], out[3]


def read(gpu, c, lens, kv_len, kind, total=None, fill=7.0):
    n = sum(lens) if total is None else total
    k = torch.full((sum(lens) + 3, c.n_kv, c.hd), fill, dtype=R.DT[kind], device="cuda")
    v = k.clone()
    cu, kl = packed(lens), ints(kv_len)
    d, rk, rv = c.desc(), R.rows(k), R.rows(v)
    st = gpu.tos_kv_read_paged8_dev(C.byref(d), C.byref(rk), C.byref(rv), cu.data_ptr(), kl.data_ptr(), len(lens), n,
                                    R.stream())
    return k, v, st


def decode(gpu, c, q, kv_lens, heads, scale, out=None, max_kv=None, ws=None):
    kl = ints(kv_lens)
    max_kv = max(list(kv_lens) + [0]) if max_kv is None else max_kv
    if out is None:
        out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    n = gpu.tos_attention_decode_paged8_workspace_bytes(len(kv_lens), max_kv, heads, c.n_kv, c.hd)
    if ws is None:
        ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")   # NaN patterns: nothing may rely on it
    d, ro, rq = c.desc(), R.rows(out), R.rows(q)
    st = gpu.tos_attention_decode_paged8_dev(C.byref(ro), C.byref(rq), C.byref(d), kl.data_ptr(), len(kv_lens), max_kv,
                                             heads, scale, ws.data_ptr(), n, R.stream())
    return out, st


def prompt(gpu, c, q, q_lens, kv_lens, heads, scale, out=None, total_kv=None, max_q=None, max_kv=None, total=None,
           ws=None):
    cu, kl = packed(q_lens), ints(kv_lens)
    total = q.shape[0] if total is None else total
    total_kv = sum(kv_lens) if total_kv is None else total_kv
    max_q = max(list(q_lens) + [0]) if max_q is None else max_q
    max_kv = max(list(kv_lens) + [0]) if max_kv is None else max_kv
    if out is None:
        out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    n = gpu.tos_attention_prompt_paged8_workspace_bytes(len(q_lens), total, max_q, total_kv, max_kv, heads, c.n_kv, c.hd)
    if ws is None:
        ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")
    d, ro, rq = c.desc(), R.rows(out), R.rows(q)
    st = gpu.tos_attention_prompt_paged8_dev(C.byref(ro), C.byref(rq), C.byref(d), cu.data_ptr(), kl.data_ptr(),
                                             len(q_lens), total, max_q, total_kv, max_kv, heads, scale, ws.data_ptr(),
                                             n, R.stream())
    return out, st


def attend(q, k, v, scale, lim):
    """paged_ref.attend's values and bound, and what that bound leaves out: the
    weights of a row whose scores lie far apart.  A weight is held as an fp16
    pair of 2^7 to 2^15 times its share of the row's largest, which has 2^7 at
    least.  Its low part is off by half a step of fp16's subnormals at most,
    2^-25, so the weight by 2^-32 of the largest, and the quotient, whose
    denominator has the largest in it, by 2^-32 of the sum of |v| it sees.  (With
    values of 0 at the key of nearly all the weight, 1.2e-7 of |v| are left to
    carry the element, and this is the larger part of its error.)"""
    ref, err = R.attend(q, k, v, scale, lim)
    sums = torch.cat([torch.zeros_like(v[:1]), v.abs().cumsum(0)]) if v.shape[0] else v.new_zeros(1, *v.shape[1:])
    return ref, err + 2.0 ** -32 * sums[lim.long()].repeat_interleave(q.shape[1] // k.shape[1], 1)


def check_decode(gpu, c, q, heads, scale=None, kv_lens=None, only=None, **o):
    kv_lens = c.lens if kv_lens is None else kv_lens
    scale = c.hd ** -0.5 if scale is None else scale
    out, st = decode(gpu, c, q, kv_lens, heads, scale, **o)
    assert st == 0
    for i in range(len(kv_lens)) if only is None else only:
        n = kv_lens[i]
        lim = torch.tensor([n], device="cuda")
        ref, err = attend(q[i:i + 1], c.rows(i, n), c.rows(i, n, "v"), float(np.float32(scale)), lim)
        R.assert_rows(out[i:i + 1], ref, err, ("decode", i, n))
    return out


def check_prompt(gpu, c, q, q_lens, kv_lens, heads, scale=None, **o):
    scale = c.hd ** -0.5 if scale is None else scale
    out, st = prompt(gpu, c, q, q_lens, kv_lens, heads, scale, **o)
    assert st == 0
    at = 0
    for i, (n, m) in enumerate(zip(q_lens, kv_lens)):
        lim = (torch.arange(n, device="cuda") + (m - n) + 1).clamp(0, m)
        ref, err = attend(q[at:at + n], c.rows(i, m), c.rows(i, m, "v"), float(np.float32(scale)), lim)
        R.assert_rows(out[at:at + n], ref, err, ("prompt", i, n, m))
        at += n
    assert bool((out[at:] == 7.0).all()), "rows behind the last sequence changed"
    return out
