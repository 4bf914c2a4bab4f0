"""sandwich_norm against its definition: every product and sum one fp32 operation in the stated order, the means in 64
bits.  The stream and the outputs are compared bit for bit with the same operations on the CPU where the factors agree;
a factor is the nearest fp32 to a 64-bit quotient whose sum may differ by its order, by 2^-50 of it, so that it can fall
on the other side of a tie once in 2^25 rows: none of the rows here may."""
import math

import pytest
import torch

from .test_gpu_norm import plain_blocks, same

pytestmark = pytest.mark.gpu


def plain(x, post, res, pre, gate, rs, eps, off):
    def rms(h, w):
        f = (1.0 / torch.sqrt(h.double().square().mean(-1, keepdim=True) + eps)).float()
        return h * f * (w.float() + off)
    h = x.float()
    if post is not None:
        h = rms(h, post)
    if gate is not None:
        h = h * (gate.float() if torch.is_tensor(gate) else torch.tensor(gate, dtype=torch.float32))
    r = (res.float() * torch.tensor(rs, dtype=torch.float32) + h).to(x.dtype)
    return rms(r.float(), pre), r


def inputs(B, H, dtype, seed, gate):
    g = torch.Generator().manual_seed(seed)
    wide = torch.exp(0.5 * torch.randn(H, generator=g))
    x, res = ((torch.randn(B, H, generator=g) * wide).to(dtype) for _ in range(2))
    post, pre = ((torch.randn(H, generator=g) * 0.2 + 1.0).to(dtype) for _ in range(2))
    gate = {"none": None, "number": -0.7, "channel": torch.randn(H, generator=g).to(dtype),
            "token": torch.randn(B, H, generator=g).to(dtype)}[gate]
    return x, post, res, pre, gate


def on(dev, t):
    return t.to(dev) if torch.is_tensor(t) else t


@pytest.mark.parametrize("B,H", [(1, 8), (3, 120), (5, 128), (2, 2048), (3, 2056), (7, 4096), (4, 5760), (2, 6152), (3, 8192),
                                 (2, 8200), (2, 16384), (2, 16392), (1, 65536), (300, 264)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("gate,use_post", [("none", True), ("number", False), ("channel", True), ("token", True), ("token", False)])
def test_norm_is_its_definition(gpu, B, H, dtype, gate, use_post):
    import llima_amd
    x, post, res, pre, gt = inputs(B, H, dtype, B + H, gate)
    post = post if use_post else None
    kw = dict(residual_scale=0.6, eps=1e-5, weight_offset=0.5)
    y, r = plain(x, post, res, pre, gt, 0.6, float(torch.tensor(1e-5)), 0.5)
    args = [on(gpu, t) for t in (x, post, res, pre)]
    gy, gr = llima_amd.sandwich_norm(*args, gate=on(gpu, gt), **kw)
    same(gr, r)
    same(gy, y.to(dtype))
    q, gr = llima_amd.sandwich_norm(*args, gate=on(gpu, gt), out="fp8", **kw)
    eq, es = plain_blocks(y)
    same(gr, r)
    same(q.values, eq)
    same(q.scales, es)


def test_it_is_add_rms_norm_without_the_rest(gpu):
    """Without post norm, gate and scales it is the residual's addition and norm, bit for bit."""
    import llima_amd
    for dtype in (torch.bfloat16, torch.float32):
        x, _, res, pre, _ = (on(gpu, t) for t in inputs(9, 1000, dtype, 3, "none"))
        for out in ("same", "fp8"):
            a, b = llima_amd.sandwich_norm(x, None, res, pre, out=out), llima_amd.add_rms_norm(x, pre, res, out=out)
            assert torch.equal(a[1], b[1])
            if out == "same":
                assert torch.equal(a[0], b[0])
            else:
                assert torch.equal(a[0].values.float(), b[0].values.float()) and torch.equal(a[0].scales, b[0].scales)


def test_shapes_strides_and_alignment(gpu):
    """More dimensions, rows out of wider tensors, unaligned rows and weights, a gate of one row, no rows."""
    import llima_amd
    x, post, res, pre, gate = (on(gpu, t) for t in inputs(12, 256, torch.bfloat16, 5, "token"))
    y, r = llima_amd.sandwich_norm(x, post, res, pre, gate=gate)
    y3, r3 = llima_amd.sandwich_norm(x.view(3, 4, 256), post, res.view(3, 4, 256), pre, gate=gate.view(3, 4, 256))
    assert y3.shape == (3, 4, 256) and torch.equal(y3.view(12, 256), y) and torch.equal(r3.view(12, 256), r)

    def wide(t, pad):
        w = torch.zeros(t.shape[0], t.shape[1] + pad, dtype=t.dtype, device=gpu)
        w[:, pad:] = t
        return w[:, pad:]
    for pad in (8, 3):
        y2, r2 = llima_amd.sandwich_norm(wide(x, pad), post, wide(res, pad), pre, gate=wide(gate, pad))
        assert torch.equal(y2, y) and torch.equal(r2, r)
    odd = torch.zeros(257, dtype=torch.bfloat16, device=gpu)
    odd[1:] = pre
    assert torch.equal(llima_amd.sandwich_norm(x, post, res, odd[1:], gate=gate)[0], y)
    one = llima_amd.sandwich_norm(x, post, res, pre, gate=gate[:1].expand(12, 256))
    want = llima_amd.sandwich_norm(x, post, res, pre, gate=gate[0])
    assert torch.equal(one[0], want[0]) and torch.equal(one[1], want[1])
    y1, r1 = llima_amd.sandwich_norm(x[0], post, res[0], pre, gate=gate[0])
    assert y1.shape == (256,) and torch.equal(y1, y[0]) and torch.equal(r1, r[0])
    for out in ("same", "fp8"):
        y0, r0 = llima_amd.sandwich_norm(x[:0], post, res[:0], pre, gate=gate[:0], out=out)
        assert r0.shape == (0, 256)


def test_special_values_stay_in_their_row(gpu):
    import llima_amd
    x, post, res, pre, gate = (on(gpu, t) for t in inputs(6, 512, torch.bfloat16, 6, "channel"))
    y, r = llima_amd.sandwich_norm(x, post, res, pre, gate=gate)
    x2, res2 = x.clone(), res.clone()
    x2[1, 7], res2[3, 100], x2[4] = math.nan, math.inf, 0.0
    y2, r2 = llima_amd.sandwich_norm(x2, post, res2, pre, gate=gate)
    assert torch.equal(y2[[0, 2, 5]], y[[0, 2, 5]]) and torch.equal(r2[[0, 2, 5]], r[[0, 2, 5]])
    assert y2[1].isnan().all() and torch.isinf(r2[3, 100]) and torch.equal(r2[3, :100], r[3, :100])
    assert torch.equal(r2[4], res[4])                        # a block's output of zeros adds nothing


def test_rows_past_one_launch(gpu):
    """More rows than one launch takes (2^21)."""
    import llima_amd
    B = (1 << 21) + 77
    x = torch.randn(1000, 8, device=gpu).bfloat16().repeat(B // 1000 + 1, 1)[:B].contiguous()
    w = torch.ones(8, dtype=torch.bfloat16, device=gpu)
    y, r = llima_amd.sandwich_norm(x, w, x, w, gate=x)
    ey, er = llima_amd.sandwich_norm(x[:1000], w, x[:1000], w, gate=x[:1000])
    for i in (0, 1 << 20, (1 << 21) - 1000, B - B % 1000 - 1000):
        i -= i % 1000
        assert torch.equal(y[i:i + 1000], ey) and torch.equal(r[i:i + 1000], er)
    assert torch.equal(y[B - B % 1000:], ey[:B % 1000])


def test_captured(gpu):
    import llima_amd
    x, post, res, pre, gate = (on(gpu, t) for t in inputs(16, 1024, torch.bfloat16, 8, "token"))
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        q, r = llima_amd.sandwich_norm(x, post, res, pre, gate=gate, out="fp8")
    for i in range(3):
        x.normal_()
        eq, er = llima_amd.sandwich_norm(x, post, res, pre, gate=gate, out="fp8")
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(q.values.float(), eq.values.float()) and torch.equal(q.scales, eq.scales) and torch.equal(r, er)


def test_numbers_out_of_range_are_refused(gpu):
    import llima_amd
    x, post, res, pre, _ = (on(gpu, t) for t in inputs(2, 64, torch.bfloat16, 9, "none"))
    for bad in (dict(eps=-1.0), dict(eps=math.nan), dict(weight_offset=math.inf), dict(residual_scale=1e39), dict(gate=-1e39),
                dict(gate=math.nan), dict(gate=post[:32]), dict(gate=post.float()), dict(gate=x[:1])):
        with pytest.raises(ValueError):
            llima_amd.sandwich_norm(x, post, res, pre, **bad)
    for args in ((x, post, res, None), (x, post[:32], res, pre), (x, post, res, pre.float()), (x[:, :60], post[:60], res[:, :60], pre[:60])):
        with pytest.raises(ValueError):
            llima_amd.sandwich_norm(*args)
