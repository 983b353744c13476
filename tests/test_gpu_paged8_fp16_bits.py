"""What a block of 8-bit elements stands for are fp16 numbers, so prompts over such a
cache give the bits that they give over an fp16 cache of the same values."""
import numpy as np
import pytest
import torch

import paged8_ref as P
import paged_ref as R
from paged8_ref import F8, I8, Cache8
from paged_ref import F16, F32

pytestmark = pytest.mark.gpu


def as_fp16(c, page):
    """The same sequences in an fp16 cache with pages of `page` rows."""
    f = R.Cache(c.lens, page, c.n_kv, c.hd, F16, seed=9)
    for i, n in enumerate(c.lens):
        pg, r = f.where(f.table[i], n)
        f.k[pg, r], f.v[pg, r] = (c.rows(i, n, pool).half() for pool in ("k", "v"))
        assert torch.equal(f.k[pg, r].double(), c.rows(i, n))
    return f


@pytest.mark.parametrize("kind", [I8, F8])
@pytest.mark.parametrize("src", [F32, F16])
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("heads,n_kv,hd,q_lens,hist", [
    (32, 8, 128, [300, 1, 65], [0, 40, 3]),
    (8, 4, 64, [130, 200], [1700, 0]),
    (16, 2, 128, [5, 3, 1], [200, 0, 77]),
    (4, 2, 256, [40, 9], [0, 100]),
    (10, 2, 40, [33, 70], [2, 0]),
])
def test_prompt_bits(gpu, kind, src, page, heads, n_kv, hd, q_lens, hist):
    kv = [a + b for a, b in zip(q_lens, hist)]
    c = Cache8(kv, 16, 16, n_kv, hd, kind, seed=hd + page)
    f = as_fp16(c, page)
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(sum(q_lens), heads, hd, generator=g, device="cuda").to(R.DT[src])
    scale = float(np.float32(hd ** -0.5))
    got, st = P.prompt(gpu, c, q, q_lens, kv, heads, scale)
    want, st2 = R.prompt(gpu, f, q, q_lens, kv, heads, scale)
    assert st == st2 == 0 and torch.equal(got, want)
