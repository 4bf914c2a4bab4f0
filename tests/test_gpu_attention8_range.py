"""Attention over an Fp8Cache whose values' scales are far apart, against the definition in 64 bits.

Tolerance of an output, with u, the score's error and the sums' as in test_gpu_attention8.  A cached key's weight times its
value's scale is rounded to fp16 in a unit of its row's greatest W = max p max(scale, 2^-93) of the keys that its wave has met:
that stands between 2^7 and 2^15, so the rounding is relative (2^-11 at most) down to 2^-21 W and 2^-25 2^-7 W = 2^-32 W below,
times values of at most 448.  A drafted token's weight in fp16 likewise, where W is the greatest of p too.  An output
in fp16 is subnormal below 2^-14 (2^-25).
"""
import math

import pytest
import torch

from .test_gpu_attention8 import U, cache8, make8, plain
from .test_gpu_attention import make

pytestmark = pytest.mark.gpu


def check(got, s, scale):
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    B, N, Hq, D = q.shape
    G = Hq // k.shape[2]
    u = U[s["q"].dtype]
    kc, vc = plain(s["k_cache"]), plain(s["v_cache"])
    assert torch.isfinite(got).all()
    for b, n in enumerate(s["cache_lens"].tolist()):
        kb, vb = torch.cat((kc[b, :n], k[b])), torch.cat((vc[b, :n], v[b]))
        see = torch.ones(N, n + N, dtype=torch.bool, device=q.device)
        see[:, n:] = torch.ones(N, N, device=q.device).tril().bool()
        for h in range(Hq):
            kh, vh, vs = kb[:, h // G], vb[:, h // G], s["v_cache"].scales[b, :n, h // G].double()
            p = torch.softmax((q[b, :, h] @ kh.t() * scale).masked_fill(~see, -math.inf), 1)
            o, mag = p @ vh, p @ vh.abs()
            es = (D + 6) * 2.0 ** -23 * abs(scale) * (q[b, :, h].abs() @ kh.abs().t()).amax(1, keepdim=True)
            W = torch.cat((p[:, :n] * vs.clamp_min(2.0 ** -93), p.new_zeros(N, 1)), 1).amax(1, keepdim=True)
            tol = (u + 2 * es + (n + N + 64) * 2.0 ** -23) * mag + u * o.abs() + n * 448 * 2.0 ** -32 * W
            if u < 2.0 ** -8:
                tol = tol + N * float(v.abs().max()) * 2.0 ** -32 * torch.maximum(W, p[:, n:].amax(1, keepdim=True)) + 2.0 ** -25
            err = (got[b, :, h].double() - o).abs()
            bad = err > tol
            assert not bad.any(), (b, h, float((err / tol.clamp_min(1e-300)).max()), o[bad][:3].tolist(), got[b, :, h][bad][:3].tolist())


def stage(dev, dtype, D, Hq, Hkv, N, n, seed, drafts=1.0):
    """q looks at k's first value alone; every key's is 0."""
    s, _ = make(dev, 2, N, Hq, Hkv, D, [n, n // 3], 0, dtype, seed=seed)
    s["q"][:] = 0.0
    s["q"][..., 0] = 16.0
    s["k"][..., 0] = 0.0
    s["v"] *= drafts
    k = torch.randn(2, n, Hkv, D, device=dev)
    k[..., 0] = 0.0
    v = 0.5 + torch.rand(2, n, Hkv, D, device=dev)
    return s, k, v


def run(s, k, v):
    import llima_amd
    s["k_cache"], s["v_cache"] = cache8(k), cache8(v)
    check(llima_amd.tree_attention(scale=1.0, **s), s, 1.0)


SHAPES = [(64, 64, 64, 1), (128, 8, 2, 4), (128, 48, 2, 1), (256, 4, 1, 3), (64, 64, 2, 2)]


@pytest.mark.parametrize("factor", [1e4, 1e8, 1e9, 1e10, 1e20, 1e30])
@pytest.mark.parametrize("D,Hq,Hkv,N", SHAPES)
def test_a_large_value_without_weight(gpu, D, Hq, Hkv, N, factor):
    """One key in a few hundred has values far above the others' and a weight of e^-120: it changes nothing.  For the
    last query heads it has all of the weight."""
    for at in (0, 37, 899):
        s, k, v = stage(gpu, torch.bfloat16, D, Hq, Hkv, N, 900, at)
        k[:, at, :, 0] = -7.5
        v[:, at] *= factor
        s["q"][:, :, Hq - Hq // 4:, 0] = -16.0
        run(s, k, v)


@pytest.mark.parametrize("D,Hq,Hkv,N", SHAPES)
def test_a_large_value_without_weight_in_fp16(gpu, D, Hq, Hkv, N):
    for at in (0, 555):
        s, k, v = stage(gpu, torch.float16, D, Hq, Hkv, N, 900, at, drafts=2.0 ** -10)
        k[:, at, :, 0] = -7.5
        v *= 2.0 ** -12
        v[:, at] *= 2.0 ** 26
        s["q"][:, :, Hq - Hq // 4:, 0] = -16.0
        run(s, k, v)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [10, 20, 25, 40])
def test_a_heavy_key_without_a_value(gpu, dtype, bits):
    """One key takes the maximum and its values are zero; many equal weights `bits` bits below it make the output."""
    for D, Hq, Hkv, N in SHAPES[:3]:
        s, k, v = stage(gpu, dtype, D, Hq, Hkv, N, 20000, bits)
        s["k"][..., 0] = -32.0                               # drafted tokens weigh nothing
        for at in (0, 7777):
            k[:, at, :, 0], v[:, at] = bits * math.log(2.0) / 16, 0.0
            run(s, k, v * (2.0 ** (bits - 14) if dtype == torch.float16 else 1.0))


@pytest.mark.parametrize("D,Hq,Hkv,N", SHAPES)
@pytest.mark.parametrize("first,second,drafts", [
    (0.0, 0.0, 1.0), (1e-30, 1e-30, 1e-30), (1e-30, 1e-30, 1.0), (1e30, 1e30, 1.0), (0.0, 1e30, 1.0), (1e30, 0.0, 0.0),
    (1e-30, 1.0, 1e-30), (1.0, 1e30, 1e30), (3e37, 3e37, 3e37), (0.0, 1e-30, 0.0)])
def test_caches_of_small_and_large_values(gpu, D, Hq, Hkv, N, first, second, drafts):
    """All tokens of one size, and halves of two, with equal weights."""
    s, k, v = stage(gpu, torch.bfloat16, D, Hq, Hkv, N, 4000, 3, drafts=drafts)
    v[:, :2000] *= first
    v[:, 2000:] *= second
    run(s, k, v)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N", [1, 5, 11, 16])
def test_scales_of_every_size(gpu, dtype, N):
    """Scales from token to token over 2^16 (fp16) and 2^60 (bf16), with scores of ordinary spread."""
    import llima_amd
    for page in (0, 16, 7):
        s, g = make8(gpu, 2, N, 32, 8, 128, [700, 331], 0, dtype, seed=N)
        span = 30 if dtype == torch.bfloat16 else 8
        for c in (s["v_cache"],):
            e = torch.randint(-span, span + 1, c.scales.shape, generator=g).to(gpu)
            c.scales.mul_(torch.exp2(e.float()))
        got = llima_amd.tree_attention(**s) if not page else None
        if page:
            blocks = -(-700 // page)
            t = dict(s, block_table=torch.arange(2 * blocks, dtype=torch.int32, device=gpu).view(2, blocks))
            for name in ("k_cache", "v_cache"):
                c = s[name]
                pad = blocks * page - 700
                q8 = torch.nn.functional.pad(c.values.view(torch.uint8), (0, 0, 0, 0, 0, pad)).reshape(2 * blocks, page, 8, 128)
                sc = torch.nn.functional.pad(c.scales, (0, 0, 0, pad)).reshape(2 * blocks, page, 8)
                t[name] = llima_amd.Fp8Cache(q8.contiguous().view(torch.float8_e4m3fn), sc.contiguous())
            got = llima_amd.tree_attention(**t)
        check(got, s, 128 ** -0.5)
