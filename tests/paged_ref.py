"""Plain 64-bit forms of the paged-cache operators and the error each kernel
may have, for the tests.  u = 2^-24 is fp32's half step."""
import ctypes as C
import math

import numpy as np
import torch

from tensoros_b200 import _ffi

U = 2.0 ** -24
F32, F16 = 0, 1
DT = {F32: torch.float32, F16: torch.float16}


def rows(t, stride=None):
    return _ffi.Rows(t.data_ptr(), t.stride(0) if stride is None else stride,
                     F32 if t.dtype == torch.float32 else F16)


def stream():
    return torch.cuda.current_stream().cuda_stream or 1


def half_step(t):
    return torch.finfo(t).eps / 2


# ------------------------------------------------------------------- rotation

def rotary_desc(rot, layout="half", base=10000.0, scaling="none", factor=1.0, orig=4096, fast=32.0, slow=1.0,
                attn=1.0, ff=None):
    d = _ffi.RotaryDesc(rot_dim=rot, layout=int(layout == "half"), base=base,
                        scaling=["none", "linear", "yarn"].index(scaling), factor=factor, orig_ctx=orig,
                        beta_fast=fast, beta_slow=slow, attn_factor=attn)
    if ff is not None:
        arr = np.ascontiguousarray(ff, np.float32)
        d._keep = arr
        d.freq_factors = arr.ctypes.data
    return d


def thetas(d, ff=None):
    """(angle per position of each pair, magnitude) in 64 bits"""
    out = []
    base = float(np.float32(d.base))
    for i in range(d.rot_dim // 2):
        t = base ** (-2.0 * i / d.rot_dim)
        if ff is not None:
            t /= float(np.float32(ff[i]))
        if d.scaling == 1:
            t /= d.factor
        if d.scaling == 2:
            lo, hi = (d.rot_dim * math.log(d.orig_ctx / (b * 2 * math.pi)) / (2 * math.log(base))
                      for b in (d.beta_fast, d.beta_slow))
            g = min(1.0, max(0.0, (i - lo) / (hi - lo)))
            t = (1 - g) * t + g * t / d.factor
        out.append(t)
    mag = d.attn_factor * (1 + 0.1 * math.log(d.factor)) if d.scaling == 2 else 1.0
    return np.array(out), mag


def norm_rotary(x, w, eps, d, pos, ff=None):
    """(values, error bound before the last rounding) of rows [n][heads][dim].
    The norm: a mean of dim squares, a root, a quotient and two products, each
    within (dim/8 + 16) u of its value (lanes add chains of at most dim/4
    terms, then five pairs).  The rotation: an angle within 2^-22 and two
    products and a sum, 4 u of the pair's magnitude."""
    y = x.double()
    dim = x.shape[-1]
    rel = 0.0
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
        rel = (dim / 8 + 16) * U
    err = y.abs() * rel
    if d is None:
        return y, err
    th, mag = thetas(d, ff)
    a = pos.double().cpu()[:, None] * torch.tensor(th)[None]
    c, s = (torch.cos(a) * mag).to(x.device)[:, None], (torch.sin(a) * mag).to(x.device)[:, None]
    out = y.clone()
    n = d.rot_dim // 2
    if d.layout:
        i0, i1 = torch.arange(n), torch.arange(n) + n
    else:
        i0, i1 = 2 * torch.arange(n), 2 * torch.arange(n) + 1
    p, q = y[..., i0], y[..., i1]
    out[..., i0], out[..., i1] = p * c - q * s, q * c + p * s
    e = (p.abs() + q.abs()) * mag * (rel + 2.0 ** -22 + 4 * U)
    err[..., i0] = e
    err[..., i1] = e
    return out, err


def assert_rows(got, ref, err, what=""):
    tol = err + ref.abs() * half_step(got.dtype) * (1 + 1e-3) + 2.0 ** -25   # fp16's subnormal half step
    bad = (got.double() - ref).abs() > tol
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got.double() - ref).abs() / tol).max()))


# ------------------------------------------------------------------ the cache

class Cache:
    """A pool of pages with sequences in shuffled pages.  What no sequence
    uses is NaN: unused pages, rows behind a sequence's last, table entries
    that point nowhere."""

    def __init__(self, lens, page, n_kv, hd, kind, seed=0, prefix=0, spare=3, fill=float("nan"), room=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.page, self.n_kv, self.hd, self.kind = list(lens), page, n_kv, hd, kind
        need = [(max(n, room) + page - 1) // page for n in self.lens] + [(prefix + page - 1) // page]
        self.n_pages = sum(need) + spare
        self.k = torch.full((self.n_pages, page, n_kv, hd), fill, dtype=DT[kind], device="cuda")
        self.v = self.k.clone()
        perm = torch.randperm(self.n_pages, generator=g, device="cuda").to(torch.int32)
        width = max(1, max(need))
        both = torch.full((len(need), width), 2 ** 30, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(need):
            both[i, :n] = perm[at:at + n]
            at += n
        self.table, self.prefix_table = both[:-1].contiguous(), both[-1].contiguous()
        for i, n in enumerate(self.lens + [prefix]):
            if n:
                pg, r = self.where(both[i], n)
                self.k[pg, r] = torch.randn(n, n_kv, hd, generator=g, device="cuda").to(DT[kind])
                self.v[pg, r] = torch.randn(n, n_kv, hd, generator=g, device="cuda").to(DT[kind])
        self.prefix = prefix

    def where(self, row, n):
        j = torch.arange(n, device="cuda")
        return row[j // self.page].long(), j % self.page

    def rows(self, i, n=None):
        """(k, v) of sequence i in 64 bits, [n][n_kv][hd]"""
        n = self.lens[i] if n is None else n
        if n == 0:
            z = torch.zeros(0, self.n_kv, self.hd, dtype=torch.float64, device="cuda")
            return z, z
        pg, r = self.where(self.table[i], n)
        return self.k[pg, r].double(), self.v[pg, r].double()

    def prefix_rows(self):
        if not self.prefix:
            return self.rows(0, 0)
        pg, r = self.where(self.prefix_table, self.prefix)
        return self.k[pg, r].double(), self.v[pg, r].double()

    def desc(self):
        return _ffi.PagedKv(self.k.data_ptr(), self.v.data_ptr(), self.kind, self.n_pages, self.page, self.n_kv,
                            self.hd, self.table.data_ptr(), self.table.shape[0], self.table.stride(0))


# ------------------------------------------------------------------ attention

def attend(q, k, v, scale, lim):
    """(values, error bound) of q [rows][heads][hd] over k, v [keys][n_kv][hd],
    row r seeing keys < lim[r].  The bound, of an element's sum_j p_j |v_j|:
    a score is off by at most hd u of sum_d |q_d k_d| scale (and a product of
    22-bit parts by 4 u of it), which moves every weight by that much at most
    and the quotient by twice that; weights, sums and rescalings add (64 +
    keys / 8) u (chains of at most keys / 16 terms, then a tree; two errors
    per weight).  fp16 queries: weights rounded to fp16 once, 2^-11."""
    n, H, hd = q.shape
    G = H // k.shape[1]
    out = torch.zeros(n, H, hd, dtype=torch.float64, device=q.device)
    err = torch.zeros_like(out)
    keys = k.shape[0]
    if keys == 0 or n == 0:
        return out, err
    mask = torch.arange(keys, device=q.device)[None] < lim[:, None]
    any_ = lim > 0
    for h in range(H):
        kk, vv = k[:, h // G], v[:, h // G]
        s = (q[:, h].double() @ kk.T) * scale
        a = (q[:, h].double().abs() @ kk.abs().T) * abs(scale)
        s = torch.where(mask, s, -math.inf)
        p = torch.softmax(s, -1)
        p = torch.where(any_[:, None], p, torch.zeros_like(p))
        delta = torch.where(mask, a, torch.zeros_like(a)).amax(-1) * (hd + 4) * U
        out[:, h] = p @ vv
        rel = 2 * delta + (64 + keys / 8) * U + (2.0 ** -11 if q.dtype == torch.float16 else 0.0)
        err[:, h] = (p @ vv.abs()) * rel[:, None]
    return out, err


def prompt(gpu, cache, q, q_lens, kv_lens, heads, scale, out=None, max_q=None, max_kv=None, total=None, cu=None,
           ws=None):
    """The library's call; returns (out, status)."""
    if cu is None:
        cu = torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32, device="cuda")
    kl = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    total = q.shape[0] if total is None else total
    max_q = max(list(q_lens) + [0]) if max_q is None else max_q
    max_kv = max(list(kv_lens) + [0]) if max_kv is None else max_kv
    if out is None:
        out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    n = gpu.tos_attention_prompt_paged_workspace_bytes(len(q_lens), total, max_q, max_kv, heads, cache.n_kv, cache.hd)
    if ws is None:
        ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")   # NaN patterns: nothing may rely on it
    d, ro, rq = cache.desc(), rows(out), rows(q)
    st = gpu.tos_attention_prompt_paged_dev(C.byref(ro), C.byref(rq), C.byref(d), cu.data_ptr(), kl.data_ptr(),
                                            len(q_lens), total, max_q, max_kv, heads, scale, ws.data_ptr(), n,
                                            stream())
    return out, st


def decode(gpu, cache, q, kv_lens, heads, scale, out=None, max_kv=None, ws=None):
    kl = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    max_kv = max(kv_lens) if max_kv is None else max_kv
    if out is None:
        out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    n = gpu.tos_attention_decode_paged_workspace_bytes(len(kv_lens), max_kv, cache.prefix, heads, cache.n_kv, cache.hd)
    if ws is None:
        ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")
    d, ro, rq = cache.desc(), rows(out), rows(q)
    st = gpu.tos_attention_decode_paged_dev(C.byref(ro), C.byref(rq), C.byref(d), kl.data_ptr(), len(kv_lens), max_kv,
                                            cache.prefix_table.data_ptr(), cache.prefix, heads, scale, ws.data_ptr(),
                                            n, stream())
    return out, st


def check_prompt(gpu, cache, q, q_lens, kv_lens, heads, scale=None):
    scale = cache.hd ** -0.5 if scale is None else scale
    out, st = prompt(gpu, cache, q, q_lens, kv_lens, heads, scale)
    assert st == 0
    at = 0
    for i, (n, m) in enumerate(zip(q_lens, kv_lens)):
        k, v = cache.rows(i, m)
        lim = (torch.arange(n, device="cuda") + (m - n) + 1).clamp(0, m)
        ref, err = attend(q[at:at + n], k, v, float(np.float32(scale)), lim)
        assert_rows(out[at:at + n], ref, err, ("prompt", i, n, m))
        at += n
    assert bool((out[at:] == 7.0).all()), "rows behind the last sequence changed"
    return out


def check_decode(gpu, cache, q, heads, scale=None, kv_lens=None):
    kv_lens = cache.lens if kv_lens is None else kv_lens
    scale = cache.hd ** -0.5 if scale is None else scale
    out, st = decode(gpu, cache, q, kv_lens, heads, scale)
    assert st == 0
    pk, pv = cache.prefix_rows()
    for i, n in enumerate(kv_lens):
        k, v = cache.rows(i, n)
        k, v = torch.cat([pk, k]), torch.cat([pv, v])
        ref, err = attend(q[i:i + 1], k, v, float(np.float32(scale)), torch.tensor([k.shape[0]], device="cuda"))
        assert_rows(out[i:i + 1], ref, err, ("decode", i, n))
    return out
