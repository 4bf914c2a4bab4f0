"""tree_attention over an Fp8Cache against its definition in 64 bits, over the values that the cache holds.

Tolerance of an output, u = 2^-8 (bf16) or 2^-11 (fp16): a weight times its value's scale is rounded to fp16, a drafted
token's weight to the type, for the product with v (u of sum p |v| at most), the output once (u of it); a score of D exact
products, its key's scale and the scaling is off by (D + 6) 2^-23 of scale sum |q k|, which moves its weight by as much
again in the sum it is divided by; the sums over n keys, the exponentials, the scales' products and the rescaling add
(n + 64) 2^-23.  A weight in fp16 is held in units of 2^-15 times a power of two that is at most twice the largest scale, or 1
where a drafted token in fp16 was multiplied; below 2^-14 of that its absolute error is 2^-25, which times the largest
value it multiplies is 2^-40 2 max(1, scale) max(448, |v|) a key; an output in fp16 is subnormal below 2^-14 (2^-25).
"""
import math

import pytest
import torch

from .test_gpu_attention import make, tree_mask

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F8 = torch.float8_e4m3fn


def quantize(x):
    top = x.float().abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100)
    # 448 x / top without an overflow; divisions by tensors (a division by a number multiplies by its reciprocal)
    return (x.float() * 0.875 / (top * 2.0 ** -9)).to(F8), (top / torch.full_like(top, 448.0))[..., 0]


def cache8(t, head_major=True):
    """An Fp8Cache of a 16-bit cache [..., tokens, Hkv, D], in either order of tokens and heads."""
    import llima_amd
    q, s = quantize(t)
    if head_major:
        q = q.view(torch.uint8).transpose(-3, -2).contiguous().transpose(-3, -2).view(F8)
        s = s.transpose(-2, -1).contiguous().transpose(-2, -1)
    return llima_amd.Fp8Cache(q, s)


def make8(dev, *args, head_major=True, **kw):
    s, g = make(dev, *args, **kw)
    s["k_cache"], s["v_cache"] = cache8(s["k_cache"], head_major), cache8(s["v_cache"], head_major)
    return s, g


def plain(c):
    return c.values.double() * c.scales.double()[..., None]


def definition(s, mask, scale=None):
    """(out, tolerance) in 64 bits; mask bool [B, N, N] or None."""
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    B, N, Hq, D = q.shape
    Hkv = k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    u = U[s["q"].dtype]
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    table = s.get("block_table")
    kc, vc = plain(s["k_cache"]), plain(s["v_cache"])
    for b, n in enumerate(s["cache_lens"].tolist()):
        def keys(cache, new):
            rows = cache[b] if table is None else cache[table[b, :-(-n // cache.shape[1])].long()].flatten(0, 1)
            return torch.cat((rows[:n], new[b]))
        kb, vb = keys(kc, k), keys(vc, v)
        see = torch.ones(N, n + N, dtype=torch.bool, device=q.device)
        see[:, n:] = torch.ones(N, N, device=q.device).tril().bool() if mask is None else mask[b]
        for h in range(Hq):
            kh, vh = kb[:, h // (Hq // Hkv)], vb[:, h // (Hq // Hkv)]
            t = (q[b, :, h] @ kh.t() * scale).masked_fill(~see, -math.inf)
            p = torch.softmax(t, 1).masked_fill(~see.any(1, keepdim=True), 0.0)
            seen = torch.where(see.any(0)[:, None], vh, 0.0)
            o = p @ seen
            mag = p @ seen.abs()
            es = (D + 6) * 2.0 ** -23 * abs(scale) * (q[b, :, h].abs() @ torch.where(see.any(0)[:, None], kh, 0.0).abs().t()).amax(1, keepdim=True)
            a = (u + 2 * es + (n + N + 64) * 2.0 ** -23) * mag + u * o.abs()
            top = float(seen.abs().max()) if seen.numel() else 0.0
            if u < 2.0 ** -8:
                a = a + (n + N) * 2.0 ** -39 * max(448.0, top) * max(1.0, top / 448) + 2.0 ** -25
            else:
                a = a + n * 2.0 ** -39 * top
            out[b, :, h], tol[b, :, h] = o, a
    return out, tol


def check(got, s, mask=None, scale=None):
    ref, tol = definition(s, mask, scale)
    err = (got.double() - ref).abs()
    assert got.dtype == s["q"].dtype and torch.isfinite(got).all()
    assert (err <= tol + 1e-30).all(), (float((err / (tol + 1e-30)).max()), (err > tol + 1e-30).nonzero()[:4].tolist())


CASES = [  # B, N, Hq, Hkv, D, lens, page, mask
    (1, 1, 1, 1, 64, [0], 0, None), (1, 1, 4, 1, 64, [1], 0, None), (1, 1, 8, 8, 128, [31], 0, None),
    (1, 1, 32, 8, 128, [32], 0, None), (1, 1, 8, 2, 256, [17], 0, None), (2, 1, 6, 2, 128, [0, 1000], 16, None),
    (1, 16, 8, 2, 128, [500], 0, "tree"), (1, 16, 8, 2, 128, [512], 1, "tree"), (3, 5, 4, 4, 64, [0, 17, 300], 7, "tree"),
    (1, 33, 8, 2, 128, [129], 64, "tree"), (2, 33, 16, 2, 64, [31, 32], 100, "tree"), (1, 64, 8, 1, 128, [200], 48, "tree"),
    (1, 64, 3, 1, 128, [63], 64, "tree"), (2, 8, 8, 4, 256, [300, 5], 16, None), (1, 40, 16, 4, 256, [77], 0, "tree"),
    (1, 70, 12, 3, 256, [130], 32, "tree"), (1, 200, 2, 1, 64, [90], 0, "tree"), (1, 300, 4, 1, 128, [1000], 128, None),
    (5, 3, 10, 2, 128, [2000, 0, 1, 999, 64], 33, "tree"), (1, 9, 28, 4, 128, [1500], 0, "tree"),
    (70, 2, 4, 2, 64, list(range(0, 280, 4)), 5, "tree"), (1, 1, 16, 16, 128, [9000], 256, None),
    (1, 17, 32, 8, 128, [6001], 64, "tree"), (1, 1024, 1, 1, 64, [10], 0, None), (1, 2, 1024, 1024, 64, [3], 0, None),
    (2, 128, 4, 2, 128, [700, 64], 64, "tree"), (1, 1, 8, 1, 128, [40000], 32, None),
]


@pytest.mark.parametrize("B,N,Hq,Hkv,D,lens,page,kind", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_is_its_definition(gpu, B, N, Hq, Hkv, D, lens, page, kind, dtype):
    import llima_amd
    s, g = make8(gpu, B, N, Hq, Hkv, D, lens, page, dtype, seed=B + N + Hq + D)
    mask = tree_mask(g, B, N).to(gpu) if kind else None
    check(llima_amd.tree_attention(tree_mask=mask, **s), s, mask)


@pytest.mark.parametrize("page", [0, 64, 24, 16, 8, 7])
@pytest.mark.parametrize("N,Hq,Hkv", [(3, 4, 2), (1, 32, 2), (6, 8, 2), (11, 8, 2), (12, 8, 2), (16, 8, 2), (33, 8, 2), (64, 16, 4)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_kernel(gpu, dtype, D, N, Hq, Hkv, page):
    """Every number of row tiles, and several groups of them, with every way of addressing the cache, short and longer
    sequences together, with and without a mask, in both orders of tokens and heads."""
    import llima_amd
    lens = [0, 130, 700, 63]
    s, g = make8(gpu, 4, N, Hq, Hkv, D, lens, page, dtype, seed=N + D, head_major=page % 16 == 0)
    mask = tree_mask(g, 4, N).to(gpu)
    check(llima_amd.tree_attention(tree_mask=mask, **s), s, mask)
    check(llima_amd.tree_attention(scale=-0.05, **s), s, scale=-0.05)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("factors", [(1.0, 2.0 ** 12), (2.0 ** -14, 2.0 ** 9), (2.0 ** -14, 2.0 ** -14), (2.0 ** 6, 2.0 ** -20)])
def test_scales_far_apart(gpu, dtype, factors):
    """Values of unlike size from token to token, in rising and falling order, next to drafted tokens of ordinary size."""
    import llima_amd
    s, g = make(gpu, 3, 4, 8, 2, 128, [900, 70, 0], 0, dtype, seed=21)
    lo, hi = factors
    f = torch.exp2(torch.linspace(math.log2(lo), math.log2(hi), 900, device=gpu))[:, None, None]
    kc, vc = cache8(s["k_cache"]), cache8((s["v_cache"].double() * f).float())
    s["k_cache"], s["v_cache"] = kc, vc
    check(llima_amd.tree_attention(**s), s)


def test_masks_of_every_kind(gpu):
    """bool, bytes, float32, one for all sequences, strided, and rows that see nothing of the tree."""
    import llima_amd
    s, g = make8(gpu, 3, 12, 8, 2, 128, [0, 40, 130], 16, seed=4)
    mask = tree_mask(g, 3, 12).to(gpu)
    mask[0, 5] = False                                       # no cache either: nothing at all
    mask[1, 3] = False
    a = llima_amd.tree_attention(tree_mask=mask, **s)
    check(a, s, mask)
    assert (a[0, 5] == 0).all() and (a[1, 3] != 0).any()
    wide = torch.zeros(3, 12, 30, dtype=torch.bool, device=gpu)
    wide[:, :, 9:21] = mask
    for m in (mask.to(torch.uint8) * 3, mask.float(), mask.float() * 2.0 - 1.0, wide[:, :, 9:21],
              mask.transpose(1, 2).contiguous().transpose(1, 2),
              torch.where(mask, 0.5, -math.inf), torch.where(mask, 1.0, math.nan)):
        assert torch.equal(llima_amd.tree_attention(tree_mask=m, **s), a)
    one = llima_amd.tree_attention(tree_mask=mask[2], **s)
    assert torch.equal(one, llima_amd.tree_attention(tree_mask=mask[2].expand(3, 12, 12), **s))
    causal = torch.ones(12, 12, dtype=torch.bool, device=gpu).tril()
    assert torch.equal(llima_amd.tree_attention(tree_mask=causal, **s), llima_amd.tree_attention(**s))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [0, 50, 2000])
def test_what_a_row_does_not_see_does_not_reach_it(gpu, n, dtype):
    """Infinities and NaN in drafted tokens' keys and values: rows that see them get them, others do not."""
    import llima_amd
    s, g = make8(gpu, 1, 10, 4, 2, 128, [n], 16 if n else 0, dtype=dtype, seed=9)
    mask = tree_mask(g, 1, 10).to(gpu)
    mask[0, :, 7:] = False
    mask[0, 7:, :] = False
    mask[0, [7, 8, 9], [7, 8, 9]] = True
    clean = llima_amd.tree_attention(tree_mask=mask, **s)
    check(clean, s, mask)
    s["v"][0, 7, 0, 3], s["v"][0, 7, 1, 100], s["k"][0, 8, 0, 5] = math.inf, math.nan, math.nan
    s["v"][0, 9, 0, 64], s["k"][0, 9, 1, 1] = -math.inf, math.inf
    got = llima_amd.tree_attention(tree_mask=mask, **s)
    assert torch.equal(got[0, :7], clean[0, :7])
    assert torch.isinf(got[0, 7, :2, 3]).all() and (got[0, 7, :2, 3] > 0).all() and torch.isnan(got[0, 7, 2:, 100]).all()
    assert torch.isnan(got[0, 8, :2]).all() and torch.equal(got[0, 8, 2:], clean[0, 8, 2:])
    assert torch.isinf(got[0, 9, :2, 64]).all() and (got[0, 9, :2, 64] < 0).all()
    keep = torch.ones(128, dtype=torch.bool, device=gpu)
    keep[3] = False
    assert torch.equal(got[0, 7, :2, keep], clean[0, 7, :2, keep])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_special_values_in_the_cache(gpu, dtype):
    """What is cached is every row's, of its head and column alone: values times an infinite scale are infinities (NaN where the
    value is 0), a NaN score is NaN in every column, a NaN value in its own."""
    import llima_amd
    s, g = make8(gpu, 2, 3, 4, 2, 64, [400, 400], 0, dtype=dtype, seed=31)
    a = llima_amd.tree_attention(**s)
    check(a, s)
    s["v_cache"].scales[0, 100, 0] = math.inf
    s["v_cache"].values.view(torch.uint8)[0, 100, 0, 9] = 0
    s["k_cache"].scales[1, 399, 1] = math.nan
    s["v_cache"].values.view(torch.uint8)[1, 7, 0, 5] = 0x7F
    got = llima_amd.tree_attention(**s)
    row = s["v_cache"].values[0, 100, 0].float()
    want = torch.where(row == 0, math.nan, row.sign() * math.inf).expand(3, 2, 64)
    assert torch.equal(got[0, :, :2].float().nan_to_num(7.0, 1e9, -1e9), want.nan_to_num(7.0, 1e9, -1e9))
    assert torch.equal(got[0, :, 2:], a[0, :, 2:])
    assert torch.isnan(got[1, :, 2:]).all() and torch.isnan(got[1, :, :2, 5]).all()
    keep = torch.arange(64, device=gpu) != 5
    assert torch.equal(got[1, :, :2][..., keep], a[1, :, :2][..., keep])


def test_large_scores_and_scales(gpu):
    """Scores far apart (all weight on one key), equal scores, negative and zero scales."""
    import llima_amd
    s, g = make8(gpu, 2, 4, 4, 2, 64, [300, 77], 16, seed=2, qscale=60.0)
    for scale in (None, 1.0, -0.3, 0.0, 1e-4):
        check(llima_amd.tree_attention(scale=scale, **s), s, scale=scale)


@pytest.mark.parametrize("order", [1, -1])
def test_maxima_that_rise_along_the_cache(gpu, order):
    """Scores that grow (or fall) by far more than the softmax's reference moves at a time."""
    import llima_amd
    s, g = make8(gpu, 1, 2, 4, 2, 128, [3000], 0, seed=3)
    ramp = torch.linspace(0.0, 300.0, 3000, device=gpu)[::order] if order == 1 else torch.linspace(300.0, 0.0, 3000, device=gpu)
    k = torch.zeros(1, 3000, 2, 128, device=gpu)
    k[..., 0] = ramp[None, :, None]
    s["k_cache"] = cache8(k)
    s["q"][:] = 0.0
    s["q"][..., 0] = 11.0
    check(llima_amd.tree_attention(**s), s)


def test_strides_layouts_and_shared_pages(gpu):
    import llima_amd
    s, g = make8(gpu, 2, 6, 8, 2, 128, [100, 33], 0, seed=3)
    mask = tree_mask(g, 2, 6).to(gpu)
    a = llima_amd.tree_attention(tree_mask=mask, **s)
    check(a, s, mask)
    t = dict(s)
    kc, vc = s["k_cache"], s["v_cache"]
    bits = torch.stack((vc.values.view(torch.uint8), kc.values.view(torch.uint8)), 3)       # K and V side by side
    both = torch.stack((vc.scales, kc.scales), 2)
    t["k_cache"] = llima_amd.Fp8Cache(bits[:, :, :, 1].view(F8), both[:, :, 1])
    t["v_cache"] = llima_amd.Fp8Cache(bits[:, :, :, 0].view(F8), both[:, :, 0])
    qkv = torch.randn(2, 6, 12, 128, device=gpu).to(torch.bfloat16)
    qkv[:, :, :8], qkv[:, :, 8:10], qkv[:, :, 10:] = s["q"], s["k"], s["v"]
    t["q"], t["k"], t["v"] = qkv[:, :, :8], qkv[:, :, 8:10], qkv[:, :, 10:]
    assert torch.equal(llima_amd.tree_attention(tree_mask=mask, **t), a)
    odd = torch.empty(2, 6, 8, 129, device=gpu, dtype=torch.bfloat16)[..., 1:]
    odd.copy_(s["q"])
    t["q"] = odd
    assert torch.equal(llima_amd.tree_attention(tree_mask=mask, **t), a)
    # the same cache in pages of 4, the second sequence's first pages the first one's
    p = llima_amd.Fp8Cache.empty(60, 4, 2, 128, device=gpu)
    pv = llima_amd.Fp8Cache.empty(60, 4, 2, 128, device=gpu)
    for c in (p, pv):
        c.values.view(torch.uint8).fill_(0x7F)
        c.scales.fill_(math.nan)
    table = torch.full((2, 40), 12345, dtype=torch.int32, device=gpu)     # entries past the length are not read
    ids = torch.randperm(60)[:34].tolist()
    for b, n in ((0, 100), (1, 33)):
        for j in range(0, n, 4):
            page = ids.pop()
            w = min(4, n - j)
            for new, old in ((p, kc), (pv, vc)):
                new.values.view(torch.uint8)[page, :w] = old.values.view(torch.uint8)[b, j:j + w]
                new.scales[page, :w] = old.scales[b, j:j + w]
            table[b, j // 4] = page
    t = dict(s, k_cache=p, v_cache=pv, block_table=table)
    assert torch.equal(llima_amd.tree_attention(tree_mask=mask, **t), a)
    t["block_table"] = torch.stack((table, table), 2).transpose(0, 1).contiguous().transpose(0, 1)[:, :, 0]
    assert torch.equal(llima_amd.tree_attention(tree_mask=mask, **t), a)
    t["block_table"] = table.clone()
    t["block_table"][1, :5] = table[0, :5]                   # a shared prefix of 20 tokens
    check(llima_amd.tree_attention(tree_mask=mask, **t), t, mask)


def test_bad_lengths_and_pages_are_nan_for_their_sequence_alone(gpu):
    import llima_amd
    for page in (32, 16, 5):
        lens = [700, 500, 200, 64, 1]
        s, g = make8(gpu, 5, 3, 4, 2, 64, lens, page, seed=8)
        a = llima_amd.tree_attention(**s)
        check(a, s)
        t = dict(s, block_table=s["block_table"].clone(), cache_lens=s["cache_lens"].clone())
        t["block_table"][0, 699 // page] = s["k_cache"].shape[0]          # one past the last page, at the last token
        t["block_table"][1, 0] = -1
        t["block_table"][2, 199 // page + 1:] = 99999        # past its length
        t["cache_lens"][3] = -1
        t["cache_lens"][4] = s["block_table"].shape[1] * page + 1
        got = llima_amd.tree_attention(**t)
        assert all(torch.isnan(got[b]).all() for b in (0, 1, 3, 4)), page
        ref, tol = definition(s, None)
        assert ((got[2].double() - ref[2]).abs() <= tol[2]).all()


def test_no_room_no_blocks_and_no_sequences(gpu):
    """A cache without a block or a page: every length must be 0."""
    import llima_amd
    s, g = make8(gpu, 2, 4, 4, 2, 64, [0, 0], 0, seed=1)
    ref = llima_amd.tree_attention(**s)
    check(ref, s)
    t = dict(s, block_table=torch.zeros(2, 0, dtype=torch.int32, device=gpu))
    assert torch.equal(llima_amd.tree_attention(**t), ref)
    none = llima_amd.Fp8Cache.empty(0, 4, 2, 64, device=gpu)
    t = dict(s, block_table=torch.zeros(2, 3, dtype=torch.int32, device=gpu), k_cache=none, v_cache=none)
    assert torch.equal(llima_amd.tree_attention(**t), ref)
    t["cache_lens"] = torch.tensor([0, 1], dtype=torch.int32, device=gpu)
    got = llima_amd.tree_attention(**t)
    assert torch.equal(got[0], ref[0]) and torch.isnan(got[1]).all()
    z = {k: v[:0] for k, v in s.items() if not isinstance(v, llima_amd.Fp8Cache)}
    assert llima_amd.tree_attention(k_cache=none, v_cache=none, **z).shape == (0, 4, 4, 64)


def test_a_cache_past_32_bits(gpu):
    """Keys at offsets above 2^32 bytes: a long contiguous cache, and pages at the end of a large one."""
    import llima_amd
    L, Hkv, D = 2_200_000, 8, 256                            # 4.5 GB each of K and V
    kc, vc = (llima_amd.Fp8Cache(torch.zeros(1, L, Hkv, D, dtype=torch.uint8, device=gpu).view(F8),
                                 torch.full((1, L, Hkv), 2.0, device=gpu)) for _ in range(2))
    q = torch.zeros(1, 2, 8, D, dtype=torch.bfloat16, device=gpu)
    q[..., 0] = 16.0
    k = torch.zeros(1, 2, Hkv, D, dtype=torch.bfloat16, device=gpu)
    for h in range(8):                                       # head h finds its key near the end, weight 1 - 2e-8 L e-9
        kc.values[0, L - 1 - h, h, 0] = 20.0
        vc.values[0, L - 1 - h, h] = float(h + 1) / 2
    want = torch.arange(1.0, 9.0, device=gpu).to(torch.bfloat16)[:, None].expand(8, D)
    out = llima_amd.tree_attention(q, k, k, kc, vc, torch.tensor([L], dtype=torch.int32, device=gpu))
    assert torch.equal(out[0, 0], want)
    n = 5000
    for page in (100, 8):
        table = torch.arange(L // page - n // page, L // page, dtype=torch.int32, device=gpu).view(1, -1)
        kp, vp = (llima_amd.Fp8Cache(c.values.view(torch.uint8).view(L // page, page, Hkv, D).view(F8), c.scales.view(L // page, page, Hkv))
                  for c in (kc, vc))
        out = llima_amd.tree_attention(q, k, k, kp, vp, torch.tensor([n], dtype=torch.int32, device=gpu), block_table=table)
        assert torch.equal(out[0, 1], want)


@pytest.mark.parametrize("B,N,Hq,Hkv,D,page", [(40, 1, 64, 64, 64, 0), (21, 3, 128, 64, 64, 16), (30, 40, 64, 8, 128, 64),
                                               (33, 2, 512, 512, 64, 0), (18, 9, 48, 24, 256, 5), (200, 1, 32, 8, 128, 64)])
def test_more_sequences_than_shares(gpu, monkeypatch, B, N, Hq, Hkv, D, page):
    """Sequences that begin, end and lie inside a share, or span several, and nothing written past the workspace's size."""
    import llima_amd
    from llima_amd import attention
    lens = [(7 * b * b) % 500 for b in range(B)]
    lens[3], lens[B // 2], lens[B - 1] = 9000, 0, 4000
    if Hkv == 512 or B == 200:
        lens[3], lens[B - 1] = 3000, 1000
    s, g = make8(gpu, B, N, Hq, Hkv, D, lens, page, seed=B)
    bufs = []

    def scratch(dev, kind, nbytes):
        bufs.append((torch.full((nbytes + 4096,), 0x7F, dtype=torch.uint8, device=dev), nbytes))
        return bufs[-1][0][:nbytes]
    monkeypatch.setattr(attention, "_scratch", scratch)
    mask = tree_mask(g, B, N).to(gpu)
    check(llima_amd.tree_attention(tree_mask=mask, **s), s, mask)
    buf, n = bufs[0]
    assert (buf[n:] == 0x7F).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [0, 5, 6000])
def test_scores_that_are_all_minus_infinity(gpu, n, dtype):
    """The softmax over visible scores of minus infinity alone is NaN, as by the formula (0 / 0); beside a finite score
    they weigh nothing."""
    import llima_amd
    s, g = make8(gpu, 2, 4, 4, 2, 64, [n, n], 0, dtype=dtype, seed=n + 1)
    mask = tree_mask(g, 2, 4).to(gpu)
    mask[1, 2] = False
    s["q"][:, :, :2] = 0.0
    s["q"][:, :, 0, 7] = 1.0                                  # head 0 of key head 0
    s["k"][0, :, 0, 7] = -math.inf
    got = llima_amd.tree_attention(tree_mask=mask, **s)
    if n == 0:
        assert torch.isnan(got[0, :, 0]).all() and (got[1, 2] == 0).all()
    else:
        assert torch.isfinite(got[0, :, 0]).all()
    assert torch.isfinite(got[1]).all()
    s["k"][0, 0, 0, 7] = 0.5                                  # node 0, which all see, has a finite score
    got = llima_amd.tree_attention(tree_mask=mask, **s)
    if n == 0:
        assert torch.equal(got[0, :, 0], s["v"][0, 0, 0].expand(4, 64))


def test_same_call_twice_other_streams_and_graph_replays(gpu):
    """Bit-identical again, on another stream, and in two graphs captured on one stream and replayed on two, with other
    lengths."""
    import llima_amd
    s, g = make8(gpu, 3, 8, 8, 2, 128, [3000, 10, 800], 16, seed=12)
    mask = tree_mask(g, 3, 8).to(gpu)
    a = llima_amd.tree_attention(tree_mask=mask, **s)
    assert torch.equal(a, llima_amd.tree_attention(tree_mask=mask, **s))
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        assert torch.equal(a, llima_amd.tree_attention(tree_mask=mask, **s))
    s2, _ = make8(gpu, 3, 8, 8, 2, 128, [2000, 1000, 8], 16, seed=13)
    graphs = []
    torch.cuda.synchronize()
    for t in (s, s2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = llima_amd.tree_attention(tree_mask=mask, **t)
        graphs.append((gr, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(5):
        for t in (s, s2):                                    # lengths are read on the device, at each replay
            t["cache_lens"].sub_(1 if i else 0)
        expect = [llima_amd.tree_attention(tree_mask=mask, **t) for t in (s, s2)]
        for _, out in graphs:
            out.fill_(7.0)
        torch.cuda.synchronize()
        for st, (gr, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for (_, out), e in zip(graphs, expect):
            assert torch.equal(out, e)
