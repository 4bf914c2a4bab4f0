"""Attention over an Fp8Cache where a workgroup's share of the keys holds several sequences: what one of them has wrong or
special stays its own."""
import math

import pytest
import torch

from .test_gpu_attention import tree_mask
from .test_gpu_attention8 import check, make8

pytestmark = pytest.mark.gpu

# key heads, query heads, drafted tokens, sequences: 16 to 128 shares (512 over key heads and groups of 64 rows) for 6 tiles of
# a sequence or more
SHAPES = [(32, 32, 1, 200), (32, 64, 40, 60), (8, 32, 2, 300), (16, 64, 12, 120)]


def lengths(B, seed):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(1, 150, (B,), generator=g).tolist()
    lens[B // 2] = 0
    return lens


@pytest.mark.parametrize("page", [32, 16, 5])
@pytest.mark.parametrize("Hkv,Hq,N,B", SHAPES)
def test_bad_pages_and_lengths_of_neighbours(gpu, page, Hkv, Hq, N, B):
    """Sequences with a page or length out of range are NaN, every other is as without them, bit for bit: bad pages and
    lengths leave the partition as it is (a bad length alone counts as 0, so its sequence is empty in both calls)."""
    import llima_amd
    lens = lengths(B, page + N)
    empty = [B // 3, B // 3 + 7]
    for b in empty:
        lens[b] = 0
    s, g = make8(gpu, B, N, Hq, Hkv, 64, lens, page, seed=page + B)
    clean = llima_amd.tree_attention(**s)
    if B == 60:
        check(clean, s)
    t = dict(s, block_table=s["block_table"].clone(), cache_lens=s["cache_lens"].clone())
    bad = [b for b in range(3, B, 9) if lens[b] > 0]
    for i, b in enumerate(bad):                              # first, last and a middle page; below and past the pages
        at = (0, (lens[b] - 1) // page, (lens[b] - 1) // page // 2)[i % 3]
        t["block_table"][b, at] = (-1, s["k_cache"].shape[0], -2 ** 31, 2 ** 31 - 1)[i % 4]
    t["cache_lens"][empty[0]], t["cache_lens"][empty[1]] = -5, t["block_table"].shape[1] * page + 1
    got = llima_amd.tree_attention(**t)
    good = torch.ones(B, dtype=torch.bool, device=gpu)
    good[bad + empty] = False
    assert torch.isnan(got[~good]).all()
    wrong = (got[good] != clean[good]).flatten(1).any(1).nonzero().flatten().tolist()
    assert not wrong, (len(wrong), wrong[:8])


@pytest.mark.parametrize("page", [0, 16])
@pytest.mark.parametrize("Hkv,Hq,N,B", SHAPES[1:])
def test_infinite_drafts_of_neighbours(gpu, page, Hkv, Hq, N, B):
    """Infinities and NaN in some sequences' drafted tokens: every other sequence is as without them, bit for bit."""
    import llima_amd
    s, g = make8(gpu, B, N, Hq, Hkv, 64, lengths(B, 1), page, seed=B)
    mask = tree_mask(g, B, N).to(gpu)
    clean = llima_amd.tree_attention(tree_mask=mask, **s)
    t = dict(s, k=s["k"].clone(), v=s["v"].clone())
    odd = list(range(2, B, 7))
    for i, b in enumerate(odd):
        (t["v"], t["k"])[i % 2][b, N - 1, :, i % 64] = (math.inf, math.nan, -math.inf)[i % 3]
    got = llima_amd.tree_attention(tree_mask=mask, **t)
    good = torch.ones(B, dtype=torch.bool, device=gpu)
    good[odd] = False
    assert torch.equal(got[good], clean[good])
    assert torch.equal(got[odd][:, :N - 1][~mask[odd][:, :N - 1, N - 1]], clean[odd][:, :N - 1][~mask[odd][:, :N - 1, N - 1]])
    assert not torch.isfinite(got[odd][:, N - 1]).flatten(1).all(1).any()
