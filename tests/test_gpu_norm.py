"""add_rms_norm, quantize_rows and lm_head_quantize against their formulas in torch on the CPU.

Every step of the formulas is one defined operation (a 64-bit mean, one rounding of the factor,
fp32 products, one IEEE division, one rounding of the output), so the outputs are compared bit for
bit; only the order of the 64-bit sum differs, which changes the fp32 factor with probability 1e-8.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
TINY = 2.0 ** -100


def plain_blocks(y):
    """[B, H] fp32 -> (e4m3 values, scales) per 128 of a row."""
    B, H = y.shape
    n = -(-H // 128)
    b = torch.nn.functional.pad(y, (0, n * 128 - H)).view(B, n, 128)
    top = b.abs().amax(2, keepdim=True).clamp_min(TINY)
    q = (b * 0.875 / (top * 2.0 ** -9)).to(F8).view(B, n * 128)[:, :H]
    return q, (top / 448.0)[:, :, 0]


def plain_norm(x, w, res, eps, off):
    h = x.float()
    r = None
    if res is not None:
        r = (h + res.float()).to(x.dtype)
        h = r.float()
    ms = h.double().square().sum(1, keepdim=True) / h.shape[1]
    f = (1.0 / torch.sqrt(ms + float(np.float32(eps)))).float()
    return h * f * (w.float() + off), r


def same(a, b):
    """Equal values, NaN in the same places."""
    a, b = a.cpu(), b.cpu()
    assert a.shape == b.shape and a.dtype == b.dtype, (a.shape, b.shape, a.dtype, b.dtype)
    a, b = a.double(), b.double()
    assert torch.equal(torch.isnan(a), torch.isnan(b))
    bad = (torch.nan_to_num(a, nan=0.0, posinf=1e300, neginf=-1e300)
           != torch.nan_to_num(b, nan=0.0, posinf=1e300, neginf=-1e300)).nonzero()
    assert bad.numel() == 0, (bad[:5].tolist(), a[tuple(bad[0])], b[tuple(bad[0])])


def make(B, H, dtype, seed, res):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, H, generator=g) * torch.exp(torch.randn(H, generator=g))).to(dtype)
    w = (1.0 + 0.3 * torch.randn(H, generator=g)).to(dtype)
    return x, w, (2.0 * torch.randn(B, H, generator=g)).to(dtype) if res else None


SIZES = [(1, 8), (1, 64), (3, 120), (5, 128), (2, 136), (7, 1000), (1, 2048), (4, 2056), (3, 4096),
         (2, 6144), (2, 6152), (2, 8192), (3, 8200), (1, 20000), (1, 65536), (513, 256)]


@pytest.mark.parametrize("B,H", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("out", ["same", "fp8"])
def test_norm_is_its_formula(gpu, B, H, dtype, out):
    import llima_amd
    for res, off, eps in ((True, 0.0, 1e-6), (False, 1.0, 0.0)):
        x, w, r = make(B, H, dtype, 7 * B + H, res)
        y, nr = llima_amd.add_rms_norm(x.to(gpu), w.to(gpu), None if r is None else r.to(gpu), eps=eps,
                                       weight_offset=off, out=out)
        ey, er = plain_norm(x, w, r, eps, off)
        assert (nr is None) == (er is None)
        if er is not None:
            same(nr, er)
        if out == "same":
            same(y, ey.to(dtype))
        else:
            q, s = plain_blocks(ey)
            same(y.values, q)
            same(y.scales, s)


@pytest.mark.parametrize("B,H", [(1, 8), (2, 120), (3, 576), (2, 4096), (1, 16392), (70, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_rows_is_its_formula(gpu, B, H, dtype):
    import llima_amd
    x, _, _ = make(B, H, dtype, 3 * B + H, False)
    x[0, 0] = 0.0
    got = llima_amd.quantize_rows(x.to(gpu))
    q, s = plain_blocks(x.float())
    same(got.values, q)
    same(got.scales, s)


def test_quantize_rows_special_values(gpu):
    """Zero blocks, blocks below the smallest maximum, the largest values, infinities and NaN, ties."""
    import llima_amd
    x = torch.zeros(9, 256)
    x[1, :128] = 1e-38                                       # below 2^-100: rounds to 0
    x[2, 5], x[2, 200] = 3.3e38, -3.3e38
    x[3, 7] = float("inf")
    x[3, 8] = 1.0
    x[4, 9] = float("nan")
    x[5, 130] = -float("inf")
    x[6, :128] = torch.arange(128).float()
    x[7, :128] = 448.0
    x[7, 1:9] = torch.tensor([17.0, 19.0, 21.0, 23.0, 25.0, 27.0, 29.0, 31.0])   # ties of 3 mantissa bits
    x[8, 0], x[8, 1] = 448.0, 2.0 ** -10                     # half the smallest e4m3 value: to 0
    x = x.to(torch.bfloat16)
    got = llima_amd.quantize_rows(x.to(gpu))
    q, s = plain_blocks(x.float())
    same(got.values, q)
    same(got.scales, s)
    v = got.values.float().cpu()
    assert v[0].abs().sum() == 0 and v[1].abs().sum() == 0
    assert got.scales[0, 0].item() == np.float32(TINY) / np.float32(448)
    assert v[7, 1:9].tolist() == [16.0, 20.0, 20.0, 24.0, 24.0, 28.0, 28.0, 32.0] and v[8, 1] == 0
    assert torch.isnan(v[4, :128]).all() and not torch.isnan(v[4, 128:]).any()
    assert torch.isnan(v[3, 7]) and v[3, 8] == 0 and v[2, 5] == 448 and v[2, 200] == -448


def test_norm_special_rows(gpu):
    """A zero row with eps 0 is NaN and the rows beside it are not; NaN and infinities stay in their row."""
    import llima_amd
    x, w, _ = make(5, 512, torch.bfloat16, 1, False)
    x[1] = 0
    x[2, 3] = float("nan")
    x[3, 4] = float("inf")
    for out in ("same", "fp8"):
        y, _ = llima_amd.add_rms_norm(x.to(gpu), w.to(gpu), eps=0.0, out=out)
        ey, _ = plain_norm(x, w, None, 0.0, 0.0)
        if out == "same":
            same(y, ey.to(torch.bfloat16))
        else:
            q, s = plain_blocks(ey)
            same(y.values, q)
            same(y.scales, s)


def test_norm_strides_alignment_and_shapes(gpu):
    """Rows apart, unaligned rows, transposed rows, leading dimensions, no rows at all."""
    import llima_amd
    big = torch.randn(12, 1040).to(torch.bfloat16)
    w = torch.randn(520).to(torch.bfloat16)
    for x in (big[:, :520], big[:, 520:], big[:, 3:523], big[::3, 8:528], big.t()[:520].t(), big[:1, 1:521]):
        d = x.to(gpu) if x.is_contiguous() else torch.empty(0)
        b = big.to(gpu)
        d = torch.as_strided(b, x.shape, x.stride(), x.storage_offset())
        for res in (None, d.flip(0)):
            y, r = llima_amd.add_rms_norm(d, w.to(gpu), res)
            ey, er = plain_norm(x, w, None if res is None else x.flip(0), 1e-6, 0.0)
            same(y, ey.to(torch.bfloat16))
            if er is not None:
                same(r, er)
        q, s = plain_blocks(x.float())
        got = llima_amd.quantize_rows(d)
        same(got.values, q)
        same(got.scales, s)
    x = big.view(3, 4, 1040)[:, :, :520].to(gpu)
    y, r = llima_amd.add_rms_norm(x, w.to(gpu), x)
    assert y.shape == x.shape == r.shape
    y, _ = llima_amd.add_rms_norm(x, w.to(gpu), out="fp8")
    assert y.values.shape == (12, 520) and y.scales.shape == (12, 5)
    y, r = llima_amd.add_rms_norm(x[:0], w.to(gpu), x[:0])
    assert y.shape == (0, 4, 520) and r.shape == (0, 4, 520)
    assert llima_amd.quantize_rows(x[:0]).values.shape == (0, 520)


def test_norm_in_place_at_the_c_entry(gpu):
    """out_residual may be the residual's own buffer, and x's; rows both held in registers and read twice."""
    from llima_amd._lib import lib
    for H in (512, 8200):
        x, w, r = make(3, H, torch.bfloat16, H, True)
        ey, er = plain_norm(x, w, r, 1e-6, 0.0)
        for target in (0, 1):
            t = [x.to(gpu), r.to(gpu)]
            y, wd = torch.empty_like(t[0]), w.to(gpu)
            assert lib().llima_add_rms_norm(t[0].data_ptr(), t[1].data_ptr(), wd.data_ptr(), 1, 3, H, H, H,
                                            1e-6, 0.0, y.data_ptr(), None, t[target].data_ptr(),
                                            torch.cuda.current_stream().cuda_stream) == 0
            same(y, ey.to(torch.bfloat16))
            same(t[target], er)


@pytest.mark.parametrize("V,H", [(1, 64), (128, 128), (200, 320), (1000, 192), (129, 4096)])
def test_lm_head_quantize_is_its_formula(gpu, V, H):
    import llima_amd
    g = torch.Generator().manual_seed(V + H)
    w = (torch.randn(V, H, generator=g) * torch.exp(torch.randn(V, 1, generator=g))).to(torch.bfloat16)
    w[0, 0] = 0
    got = llima_amd.lm_head_quantize(w.to(gpu))
    nv, nh = -(-V // 128), -(-H // 128)
    p = torch.nn.functional.pad(w.float(), (0, nh * 128 - H, 0, nv * 128 - V)).view(nv, 128, nh, 128)
    top = p.abs().amax((1, 3), keepdim=True).clamp_min(TINY)
    q = (p * 448.0 / top).to(F8).view(nv * 128, nh * 128)[:V, :H]
    same(got.values, q)
    same(got.scales, (top / 448.0)[:, 0, :, 0])


def test_more_rows_than_a_launch_holds(gpu):
    """2^24 + 3 rows of 8: three launches, the rows around their edges, and nothing left out."""
    import llima_amd
    B, H = (1 << 24) + 3, 8
    g = torch.Generator().manual_seed(5)
    base = torch.randn(4099, H, generator=g).to(gpu, torch.bfloat16)
    x = base.repeat(B // 4099 + 1, 1)[:B].contiguous()
    w = torch.randn(H, generator=g).to(gpu, torch.bfloat16)
    y, r = llima_amd.add_rms_norm(x, w, x)
    y0, r0 = llima_amd.add_rms_norm(base, w, base)
    for got, want in ((y, y0), (r, r0)):
        n = B // 4099 * 4099
        assert torch.equal(got[:n].view(-1, 4099, H), want[None].expand(n // 4099, 4099, H))
        assert torch.equal(got[n:], want[:B - n])
    q, q0 = llima_amd.quantize_rows(x), llima_amd.quantize_rows(base)
    at = torch.tensor([0, (1 << 23) - 1, 1 << 23, (1 << 24) - 1, 1 << 24, B - 1], device=gpu)
    assert torch.equal(q.values[at].view(torch.uint8), q0.values[at % 4099].view(torch.uint8))
    assert torch.equal(q.scales[at], q0.scales[at % 4099])
