"""Calls over tensors of one sequence, token or head that are sliced from wider rows: the stride of a dimension of one is never
used and may be any number."""
import pytest
import torch

from .test_gpu_attention8 import F8, cache8

pytestmark = pytest.mark.gpu


def odd(t, dims, pad):
    """t with a stride in the dimensions of one that no alignment divides."""
    wide = torch.zeros(2 * t.numel() + 3 * pad + 2, dtype=torch.uint8 if t.dtype == F8 else t.dtype, device=t.device)
    st = [pad if i in dims and n == 1 else s for i, (n, s) in enumerate(zip(t.shape, t.contiguous().stride()))]
    out = wide.as_strided(t.shape, st)
    out.copy_(t.view(torch.uint8) if t.dtype == F8 else t)
    return out.view(F8) if t.dtype == F8 else out


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("B,N,Hq,Hkv", [(1, 1, 4, 1), (1, 3, 1, 1), (1, 1, 8, 2), (2, 1, 2, 1)])
def test_dimensions_of_one(gpu, eight, B, N, Hq, Hkv):
    import llima_amd
    g = torch.Generator(device=gpu).manual_seed(B + N + Hq)

    def rnd(*shape):
        return torch.randn(shape, generator=g, device=gpu).bfloat16()
    S, D = 40, 64
    q, k, v, kc, vc = rnd(B, N, Hq, D), rnd(B, N, Hkv, D), rnd(B, N, Hkv, D), rnd(B, S, Hkv, D), rnd(B, S, Hkv, D)
    lens = torch.full((B,), 33, dtype=torch.int32, device=gpu)
    nodes, counts = torch.zeros(B, 1, dtype=torch.int32, device=gpu), torch.ones(B, dtype=torch.int32, device=gpu)

    def calls(q, k, v, kc, vc):
        out = [llima_amd.tree_attention(q, k, v, kc, vc, lens)]
        new = llima_amd.tree_commit(k, v, nodes, counts, kc, vc, lens)
        assert new.tolist() == [34] * B
        if eight:
            assert llima_amd.cache_write(k, v, kc, vc, new).tolist() == [34 + N] * B
            out += llima_amd.cache_read(kc, vc, new + N)
            return out + [kc.values.view(torch.uint8).clone(), vc.scales.clone()]
        return out + [kc.clone(), vc.clone()]

    def caches(strided):
        both = [cache8(c, head_major=False) if eight else c.clone() for c in (kc, vc)]
        if not strided:
            return both
        return [llima_amd.Fp8Cache(odd(c.values, (0, 1, 2), 1001), odd(c.scales, (0, 1, 2), 77)) if eight else odd(c, (0, 1, 2), 1001) for c in both]
    want = calls(q, k, v, *caches(False))
    for dims in ((0,), (1,), (0, 1, 2)):
        t = [odd(x, dims, 1001) for x in (q, k, v)]
        assert any(s % 8 for x in t for s in x.stride()) or not any(x.shape[d] == 1 for x in t for d in dims)
        got = calls(*t, *caches(True))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
