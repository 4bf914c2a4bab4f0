"""Paths into an Fp8Cache whose counts are far below their places: the workgroups behind a sequence's count do nothing."""
import pytest
import torch

from .test_gpu_attention8 import F8, quantize
from .test_gpu_cache8 import same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hkv,L", [(1024, 2097160), (1024, 4194305), (512, 8388600)])
@pytest.mark.parametrize("page", [0, 8])
def test_places_times_heads_past_31_bits(gpu, Hkv, L, page):
    """(L - count) Hkv is 2^31 and more: the written tokens are the counts', and no byte beside them, in the cache or in front
    of and behind it, changes."""
    import llima_amd
    D, room, counts = 64, 16, [1, 3, 0]
    B = 1 if L >= 1 << 22 else 3
    counts = counts[:B]
    g = torch.Generator(device=gpu).manual_seed(L)
    k, v = (torch.randn(B, 4, Hkv, D, generator=g, device=gpu).bfloat16() for _ in range(2))
    nodes = torch.full((B, L), 7, dtype=torch.int32, device=gpu)              # behind the count, out of range: not read
    nodes[:, :3] = torch.tensor([2, 0, 3], dtype=torch.int32, device=gpu)
    rows = B * room
    bits = torch.full((2, rows + 64, Hkv, D), 0x38, dtype=torch.uint8, device=gpu)
    sc = torch.full((2, rows + 64, Hkv), 5.0, device=gpu)
    shape = (B * room // page, page) if page else (B, room)
    kc, vc = (llima_amd.Fp8Cache(bits[i, 32:32 + rows].view(*shape, Hkv, D).view(F8), sc[i, 32:32 + rows].view(*shape, Hkv)) for i in range(2))
    lens = torch.tensor([5, 13, 16][:B], dtype=torch.int32, device=gpu)
    table = torch.arange(B * room // page, dtype=torch.int32, device=gpu).view(B, -1) if page else None
    want_bits, want_sc = bits.clone(), sc.clone()
    for i, x in enumerate((k, v)):
        q, s = quantize(x)
        for b in range(B):
            for j in range(counts[b]):
                at = 32 + b * room + int(lens[b]) + j
                want_bits[i, at], want_sc[i, at] = q[b, (2, 0, 3)[j]].view(torch.uint8), s[b, (2, 0, 3)[j]]
    new = llima_amd.tree_commit(k, v, nodes, torch.tensor(counts, dtype=torch.int32, device=gpu), kc, vc, lens, block_table=table)
    assert new.tolist() == [int(n) + c for n, c in zip(lens, counts)]
    assert same(bits.view(F8), want_bits.view(F8)) and torch.equal(sc, want_sc)
