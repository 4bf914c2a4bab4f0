"""Attention calls of more rows than a launch holds are refused with either cache (no GPU)."""
import pytest
import torch


def cache(eight, B, Hkv):
    import llima_amd
    if not eight:
        return torch.zeros(B, 1, Hkv, 64, dtype=torch.bfloat16)
    return llima_amd.Fp8Cache(torch.zeros(B, 1, Hkv, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(B, 1, Hkv))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("B,N,Hq", [(64, 1024, 1024), (1 << 16, 1, 1024), (1 << 20, 64, 1), (131073, 2, 256)])
def test_rows_past_a_launch_are_refused(monkeypatch, eight, B, N, Hq):
    """2^26 rows and more: an error, not an output that no kernel wrote."""
    import llima_amd
    from llima_amd import attention
    monkeypatch.setattr(attention, "_on_gpu", lambda *t: None)
    one = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    q, k, c = one.expand(B, N, Hq, 64), one.expand(B, N, 1, 64), cache(eight, B, 1)
    for _ in range(2):                                       # again as a call of a known form
        with pytest.raises(ValueError, match="2\\^26"):
            llima_amd.tree_attention(q, k, k, c, c, torch.zeros(B, dtype=torch.int32))
