"""Decode over an 8-bit cache whose keys all have scales of their own, which one
lane brings and others read."""
import pytest
import torch

import paged8_ref as P
from paged8_ref import F8, I8, Cache8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [I8, F8])
@pytest.mark.parametrize("page", [16, 24])                  # by TMA; by cp.async
@pytest.mark.parametrize("heads,n_kv,hd", [(8, 1, 64), (16, 1, 128), (4, 2, 256)])
def test_every_key_has_a_scale_of_its_own(gpu, kind, page, heads, n_kv, hd):
    n = 9000
    c = Cache8([n, 31], page, 1, n_kv, hd, kind, seed=hd, spread=0.0)
    j = torch.arange(c.ks.numel(), device="cuda").view(c.ks.shape)
    c.ks.copy_(torch.exp2(-8.0 - (j * 7 % 3)))
    c.vs.copy_(torch.exp2(-8.0 + (j * 5 % 13)))
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(2, heads, hd, generator=g, device="cuda")
    out = P.check_decode(gpu, c, q, heads)
    for _ in range(20):
        again, st = P.decode(gpu, c, q, c.lens, heads, hd ** -0.5)
        assert st == 0 and torch.equal(out, again)
