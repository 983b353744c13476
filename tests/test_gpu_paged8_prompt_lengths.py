"""Prompt attention over the 8-bit paged cache where the lengths, the table and
what the workspace was sized for do not agree."""
import numpy as np
import pytest
import torch

import paged8_ref as P
import paged_ref as R
from paged8_ref import F8, I8, Cache8
from paged_ref import F16, F32

pytestmark = pytest.mark.gpu


def randn(*shape, seed=0, kind=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(R.DT[kind])


def check(out, q, q_lens, kv_lens, keys, k, v, scale):
    """Rows of sequence i see keys[i] keys at most, those of k[i] and v[i]; row r of n
    is at position kv_lens[i] - n + r."""
    at = 0
    for i, (n, m) in enumerate(zip(q_lens, kv_lens)):
        lim = (torch.arange(n, device="cuda", dtype=torch.int64) + (m - n) + 1).clamp(0, keys[i])
        ref, err = P.attend(q[at:at + n], k[i], v[i], float(np.float32(scale)), lim)
        R.assert_rows(out[at:at + n], ref, err, ("prompt", i, n, m))
        at += n


@pytest.mark.parametrize("kind", [I8, F8])
@pytest.mark.parametrize("src", [F32, F16])
@pytest.mark.parametrize("heads,n_kv,hd", [(4, 2, 64), (32, 8, 128), (10, 2, 40), (4, 2, 256)])
@pytest.mark.parametrize("q_lens,kv_lens", [
    ([50, 8], [100, 68]),                                   # some rows before the table row's end
    ([300, 1], [310, 65]),                                  # most rows behind it
    ([70, 64], [70, 64]),                                   # begins at 0
    ([5, 3], [2 ** 31 - 1, 1 << 26]),                       # far behind
])
def test_lengths_beyond_the_table_row(gpu, kind, src, heads, n_kv, hd, q_lens, kv_lens):
    """Keys end where the table row does (64 here), positions follow kv_len."""
    c = Cache8([64, 64], 16, 16, n_kv, hd, kind, seed=hd)
    q = randn(sum(q_lens), heads, hd, seed=1, kind=src)
    most = min(max(kv_lens), 1 << 12)
    out, st = P.prompt(gpu, c, q, q_lens, kv_lens, heads, hd ** -0.5, total_kv=2 * most, max_kv=most)
    assert st == 0
    k, v = ([c.rows(i, 64, pool) for i in (0, 1)] for pool in ("k", "v"))
    check(out, q, q_lens, kv_lens, [64, 64], k, v, hd ** -0.5)


@pytest.mark.parametrize("word", [0, 1, 2])
@pytest.mark.parametrize("src", [F32, F16])
@pytest.mark.parametrize("heads,n_kv,hd", [(4, 2, 64), (8, 2, 128), (10, 2, 40)])
@pytest.mark.parametrize("lens,total_kv", [
    ([20, 500, 300], 0),
    ([300, 260, 140], 500),
    ([130] + [40] * 300, 0),                                # more sequences than a block's threads
])
def test_keys_beyond_the_total_read_as_zeros(gpu, word, src, heads, n_kv, hd, lens, total_kv):
    """The workspace has room for total_kv / 128 pages of 128 keys and one for each
    sequence, dealt in the sequences' order; keys of pages beyond that are zeros,
    whatever page numbers an earlier call has left in the workspace."""
    c = Cache8(lens, 16, 16, n_kv, hd, I8, seed=hd)
    q_lens = [min(n, 30) for n in lens]
    q = randn(sum(q_lens), heads, hd, seed=1, kind=src)
    size = gpu.tos_attention_prompt_paged8_workspace_bytes(len(lens), q.shape[0], max(q_lens), total_kv, max(lens), heads,
                                                           n_kv, hd)
    ws = torch.full((size // 4 + 64,), word, dtype=torch.int32, device="cuda")
    out, st = P.prompt(gpu, c, q, q_lens, lens, heads, hd ** -0.5, total_kv=total_kv, ws=ws)
    assert st == 0
    room = total_kv // 128 + len(lens)
    k, v = [], []
    for i, n in enumerate(lens):
        pages = (n + 127) // 128
        have = min(n, 128 * max(0, min(pages, room)))
        room -= min(pages, max(room, 0))
        for to, pool in ((k, "k"), (v, "v")):
            x = c.rows(i, n, pool)
            x[have:] = 0
            to.append(x)
    check(out, q, q_lens, lens, lens, k, v, hd ** -0.5)
