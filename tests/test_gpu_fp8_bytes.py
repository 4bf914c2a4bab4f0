"""The bytes that the 8-bit quantisers write, against 448 x / max by one IEEE division and its rounding to e4m3 on the CPU: every
byte, so that a negative value whose quotient rounds to zero stays a negative zero."""
import pytest
import torch

from .test_gpu_attention8 import F8, quantize
from .test_gpu_norm import plain_blocks, plain_norm
from .test_gpu_sandwich import plain

pytestmark = pytest.mark.gpu


def rows(B, H, dtype, seed):
    """Values over 2^40 in every block, both signs, zeros of both signs, a block of zeros alone and one with the type's least."""
    g = torch.Generator().manual_seed(seed)
    e = torch.randint(-30 if dtype != torch.float16 else -10, 11, (B, H), generator=g)
    x = (torch.randn(B, H, generator=g) * torch.exp2(e.float())).to(dtype)
    x[:, ::7], x[:, 3::11] = 0.0, -0.0
    x[0, :128] = -0.0
    x[1, :128:2], x[1, 1:128:2] = torch.finfo(dtype).smallest_normal, -torch.finfo(dtype).smallest_normal
    x[2, :128] = -torch.finfo(dtype).smallest_normal / 8
    return x


def equal(a, b):
    a, b = (t.cpu().view(torch.uint8) for t in (a, b))
    bad = (a != b).nonzero()
    assert bad.numel() == 0, (len(bad), bad[:4].tolist(), [(int(a[tuple(i)]), int(b[tuple(i)])) for i in bad[:4]])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,H", [(4, 128), (9, 1000), (64, 4096), (5, 17000)])
def test_rows(gpu, dtype, B, H):
    import llima_amd
    x = rows(B, H, dtype, B)
    eq, _ = plain_blocks(x.float())
    got = llima_amd.quantize_rows(x.to(gpu))
    assert (eq.view(torch.uint8) == 0x80).any() and (eq.view(torch.uint8) == 0).any()
    equal(got.values, eq)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_norms(gpu, dtype):
    import llima_amd
    x, w = rows(33, 2048, dtype, 1), torch.linspace(-1.0, 1.0, 2048).to(dtype)
    res = rows(33, 2048, dtype, 2)
    for off in (0.0, 1.0):
        y, _ = plain_norm(x, w, res, 1e-5, off)
        got, _ = llima_amd.add_rms_norm(x.to(gpu), w.to(gpu), res.to(gpu), eps=1e-5, weight_offset=off, out="fp8")
        equal(got.values, plain_blocks(y)[0])
        y, _ = plain(x, w, res, w, None, 0.5, float(torch.tensor(1e-5)), off)
        got, _ = llima_amd.sandwich_norm(x.to(gpu), w.to(gpu), res.to(gpu), w.to(gpu), residual_scale=0.5, eps=1e-5,
                                         weight_offset=off, out="fp8")
        equal(got.values, plain_blocks(y)[0])


def test_head(gpu):
    import llima_amd
    V, H = 300, 576
    x = rows(V, H, torch.bfloat16, 3)
    got = llima_amd.lm_head_quantize(x.to(gpu))
    want = torch.empty(V, H, dtype=F8)
    for v in range(0, V, 128):
        for h in range(0, H, 128):
            b = x[v:v + 128, h:h + 128].float()
            top = b.abs().max().clamp_min(2.0 ** -100)
            want.view(torch.uint8)[v:v + 128, h:h + 128] = (b * 0.875 / (top * 2.0 ** -9)).to(F8).view(torch.uint8)
    equal(got.values, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_cache(gpu, dtype, D):
    import llima_amd
    T = 2048 * 64 // D
    k, v = (rows(T, 2 * D, dtype, s).view(1, T, 2, D) for s in (4, 5))
    kc, vc = llima_amd.Fp8Cache.empty(1, T, 2, D, device=gpu), llima_amd.Fp8Cache.empty(1, T, 2, D, device=gpu)
    llima_amd.cache_write(k.to(gpu), v.to(gpu), kc, vc, torch.zeros(1, dtype=torch.int32, device=gpu))
    for c, x in ((kc, k), (vc, v)):
        equal(c.values.contiguous(), quantize(x)[0])
