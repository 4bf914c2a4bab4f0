"""tree_attention and tree_commit against their definitions in 64 bits.

Tolerance of an output: u = 2^-8 (bf16) or 2^-11 (fp16).  The weights are rounded for their
product with v (u of sum p |v|; fp16 weights below 2^-24 of the largest by 2^-35 of it), the
output once (u of it); a score of D products and its scaling is off by (D + 4) 2^-23 of
scale sum |q k|, which moves its weight by as much again in the sum it is divided by; the sums over
n keys, the exponentials and the rescaling add (n + 64) 2^-23.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def tree_mask(g, B, N):
    mask = torch.eye(N, dtype=torch.bool).repeat(B, 1, 1)
    for b in range(B):
        for i in range(1, N):
            mask[b, i] |= mask[b, int(torch.randint(0, i, (1,), generator=g))]
    return mask


def make(dev, B, N, Hq, Hkv, D, lens, page=0, dtype=torch.bfloat16, seed=0, qscale=2.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    gc = torch.Generator().manual_seed(seed)

    def rnd(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dtype)
    S = max(max(lens), 1)
    s = dict(q=qscale * rnd(B, N, Hq, D), k=rnd(B, N, Hkv, D), v=rnd(B, N, Hkv, D),
             cache_lens=torch.tensor(lens, dtype=torch.int32, device=dev))
    if page:
        nblk = -(-S // page)
        perm = torch.randperm(B * nblk + 3, generator=gc)[:B * nblk]
        s["block_table"] = perm.view(B, nblk).to(torch.int32).to(dev)
        shape = (B * nblk + 3, page, Hkv, D)
    else:
        shape = (B, S, Hkv, D)
    s["k_cache"], s["v_cache"] = rnd(*shape), rnd(*shape)
    # what no sequence has is NaN: it must not be read into a result
    used = torch.zeros(shape[:2], dtype=torch.bool, device=dev)
    for b, n in enumerate(lens):
        for j0 in range(0, n, page or max(n, 1)):
            if page:
                used[int(s["block_table"][b, j0 // page]), :min(page, n - j0)] = True
            else:
                used[b, :n] = True
    s["k_cache"][~used] = float("nan")
    s["v_cache"][~used] = float("nan")
    return s, gc


def definition(s, mask, scale=None):
    """(out, tolerance) in 64 bits; mask bool [B, N, N] or None."""
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    B, N, Hq, D = q.shape
    Hkv = k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    u = U[s["q"].dtype]
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    table = s.get("block_table")
    for b, n in enumerate(s["cache_lens"].tolist()):
        def keys(cache, new):
            rows = cache[b] if table is None else cache[table[b].long()].flatten(0, 1)
            return torch.cat((rows[:n].double(), new[b]))
        kb, vb = keys(s["k_cache"], k), keys(s["v_cache"], v)
        see = torch.ones(N, n + N, dtype=torch.bool, device=q.device)
        see[:, n:] = torch.ones(N, N, device=q.device).tril().bool() if mask is None else mask[b]
        for h in range(Hq):
            kh, vh = kb[:, h // (Hq // Hkv)], vb[:, h // (Hq // Hkv)]
            t = (q[b, :, h] @ kh.t() * scale).masked_fill(~see, -math.inf)
            p = torch.softmax(t, 1).masked_fill(~see.any(1, keepdim=True), 0.0)
            seen = torch.where(see.any(0)[:, None], vh, 0.0)
            o = p @ seen
            mag = p @ seen.abs()
            es = (D + 4) * 2.0 ** -23 * abs(scale) * (q[b, :, h].abs() @ torch.where(see.any(0)[:, None], kh, 0.0).abs().t()).amax(1, keepdim=True)
            a = (u + 2 * es + (n + N + 64) * 2.0 ** -23) * mag + u * o.abs()
            if u < 2.0 ** -8:                                # subnormal weights and outputs of fp16
                a = a + 2.0 ** -35 * seen.abs().sum(0) + 2.0 ** -25
            out[b, :, h], tol[b, :, h] = o, a
    return out, tol


def check(got, s, mask=None, scale=None):
    ref, tol = definition(s, mask, scale)
    err = (got.double() - ref).abs()
    assert got.dtype == s["q"].dtype and torch.isfinite(got).all()
    assert (err <= tol + 1e-30).all(), (float((err / (tol + 1e-30)).max()), (err > tol + 1e-30).nonzero()[:4].tolist())


CASES = [  # B, N, Hq, Hkv, D, lens, page, mask
    (1, 1, 1, 1, 64, [0], 0, None), (1, 1, 4, 1, 64, [1], 0, None), (1, 1, 8, 8, 128, [63], 0, None),
    (1, 1, 32, 8, 128, [64], 0, None), (1, 1, 8, 2, 256, [65], 0, None), (2, 1, 6, 2, 128, [0, 1000], 16, None),
    (1, 16, 8, 2, 128, [500], 0, "tree"), (1, 16, 8, 2, 128, [512], 1, "tree"), (3, 5, 4, 4, 64, [0, 17, 300], 7, "tree"),
    (1, 33, 8, 2, 128, [129], 64, "tree"), (2, 33, 16, 2, 64, [31, 32], 100, "tree"), (1, 64, 8, 1, 128, [200], 48, "tree"),
    (1, 64, 3, 1, 128, [63], 64, "tree"), (2, 8, 8, 4, 256, [300, 5], 16, None), (1, 40, 16, 4, 256, [77], 0, "tree"),
    (1, 70, 12, 3, 256, [130], 32, "tree"), (1, 200, 2, 1, 64, [90], 0, "tree"), (1, 300, 4, 1, 128, [1000], 128, None),
    (5, 3, 10, 2, 128, [2000, 0, 1, 999, 64], 33, "tree"), (1, 9, 28, 4, 128, [1500], 0, "tree"),
    (70, 2, 4, 2, 64, list(range(0, 280, 4)), 5, "tree"), (1, 1, 16, 16, 128, [9000], 256, None),
    (1, 17, 32, 8, 128, [6001], 64, "tree"), (1, 1024, 1, 1, 64, [10], 0, None), (1, 2, 1024, 1024, 64, [3], 0, None),
    (2, 128, 4, 2, 128, [700, 64], 64, "tree"),
]


@pytest.mark.parametrize("B,N,Hq,Hkv,D,lens,page,kind", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_is_its_definition(gpu, B, N, Hq, Hkv, D, lens, page, kind, dtype):
    import llima_amd
    s, g = make(gpu, B, N, Hq, Hkv, D, lens, page, dtype, seed=B + N + Hq + D)
    mask = tree_mask(g, B, N).to(gpu) if kind else None
    check(llima_amd.tree_attention(tree_mask=mask, **s), s, mask)


def test_masks_of_every_kind(gpu):
    """bool, bytes, float32, one for all sequences, strided, and rows that see nothing of the tree."""
    import llima_amd
    s, g = make(gpu, 3, 12, 8, 2, 128, [0, 40, 130], 16, seed=4)
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
    assert torch.equal(one[2], a[2])
    causal = torch.ones(12, 12, dtype=torch.bool, device=gpu).tril()
    assert torch.equal(llima_amd.tree_attention(tree_mask=causal, **s), llima_amd.tree_attention(**s))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [0, 50, 2000])
def test_what_a_row_does_not_see_does_not_reach_it(gpu, n, dtype):
    """Infinities and NaN in drafted tokens' keys and values: rows that see them get them, others do not."""
    import llima_amd
    s, g = make(gpu, 1, 10, 4, 2, 128, [n], 16 if n else 0, dtype, seed=9)
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


def test_large_scores_and_scales(gpu):
    """Scores far apart (all weight on one key), equal scores, negative and zero scales."""
    import llima_amd
    s, g = make(gpu, 2, 4, 4, 2, 64, [300, 77], 16, seed=2, qscale=60.0)
    for scale in (None, 1.0, -0.3, 0.0, 1e-4):
        check(llima_amd.tree_attention(scale=scale, **s), s, scale=scale)
    s["k_cache"][:] = torch.where(torch.isnan(s["k_cache"]), s["k_cache"], 1.0)
    check(llima_amd.tree_attention(**s), s)


def test_strides_and_layouts(gpu):
    """Head-major caches as views, sliced q, k, v, tables wider than needed, shared pages."""
    import llima_amd
    s, g = make(gpu, 2, 6, 8, 2, 128, [100, 33], 0, seed=3)
    mask = tree_mask(g, 2, 6).to(gpu)
    a = llima_amd.tree_attention(tree_mask=mask, **s)
    t = dict(s)
    t["k_cache"] = s["k_cache"].transpose(1, 2).contiguous().transpose(1, 2)
    both = torch.stack((s["v_cache"], s["k_cache"]), 3)
    t["v_cache"] = both[:, :, :, 0]
    qkv = torch.randn(2, 6, 12, 128, device=gpu).to(torch.bfloat16)
    qkv[:, :, :8], qkv[:, :, 8:10], qkv[:, :, 10:] = s["q"], s["k"], s["v"]
    t["q"], t["k"], t["v"] = qkv[:, :, :8], qkv[:, :, 8:10], qkv[:, :, 10:]
    assert torch.equal(llima_amd.tree_attention(tree_mask=mask, **t), a)
    odd = torch.empty(2, 6, 8, 129, device=gpu, dtype=torch.bfloat16)[..., 1:]
    odd.copy_(s["q"])
    t["q"] = odd
    assert torch.equal(llima_amd.tree_attention(tree_mask=mask, **t), a)
    # the same cache in pages of 4, the second sequence's first pages the first one's
    p = torch.full((60, 4, 2, 128), math.nan, device=gpu, dtype=torch.bfloat16)
    pv = p.clone()
    table = torch.full((2, 40), 12345, dtype=torch.int32, device=gpu)     # entries past the length are not read
    ids = torch.randperm(60)[:34].tolist()
    for b, n in ((0, 100), (1, 33)):
        for j in range(0, n, 4):
            page = ids.pop()
            w = min(4, n - j)
            p[page, :w], pv[page, :w] = s["k_cache"][b, j:j + w], s["v_cache"][b, j:j + w]
            table[b, j // 4] = page
    t = dict(s, k_cache=p, v_cache=pv, block_table=table)
    assert torch.equal(llima_amd.tree_attention(tree_mask=mask, **t), a)
    t["block_table"] = torch.stack((table, table), 2).transpose(0, 1).contiguous().transpose(0, 1)[:, :, 0]
    assert torch.equal(llima_amd.tree_attention(tree_mask=mask, **t), a)
    t["block_table"] = table.clone()
    t["block_table"][1, :5] = table[0, :5]                   # a shared prefix of 20 tokens
    s["k_cache"][1, :20], s["v_cache"][1, :20] = s["k_cache"][0, :20], s["v_cache"][0, :20]
    check(llima_amd.tree_attention(tree_mask=mask, **t), s, mask)


def test_bad_lengths_and_pages_are_nan_for_their_sequence_alone(gpu):
    import llima_amd
    s, g = make(gpu, 5, 3, 4, 2, 64, [700, 500, 200, 64, 1], 16, seed=8)
    a = llima_amd.tree_attention(**s)
    check(a, s)
    t = dict(s, block_table=s["block_table"].clone(), cache_lens=s["cache_lens"].clone())
    t["block_table"][0, 43] = s["k_cache"].shape[0]          # one past the last page, in the last tile
    t["block_table"][1, 0] = -1
    t["block_table"][2, 13] = 99999                          # tokens 208 .. 223: past its length
    t["cache_lens"][3] = -1
    t["cache_lens"][4] = s["block_table"].shape[1] * 16 + 1
    got = llima_amd.tree_attention(**t)
    assert all(torch.isnan(got[b]).all() for b in (0, 1, 3, 4))
    ref, tol = definition(dict(s), None)
    assert ((got[2].double() - ref[2]).abs() <= tol[2]).all()


def test_no_room_no_blocks_and_no_sequences(gpu):
    """A cache without a block or a page: every length must be 0."""
    import llima_amd
    s, g = make(gpu, 2, 4, 4, 2, 64, [0, 0], 0, seed=1)
    ref = llima_amd.tree_attention(**s)
    check(ref, s)
    t = dict(s, block_table=torch.zeros(2, 0, dtype=torch.int32, device=gpu))
    assert torch.equal(llima_amd.tree_attention(**t), ref)
    t = dict(s, block_table=torch.zeros(2, 3, dtype=torch.int32, device=gpu), k_cache=s["k_cache"][:0], v_cache=s["v_cache"][:0])
    assert torch.equal(llima_amd.tree_attention(**t), ref)
    t["cache_lens"] = torch.tensor([0, 1], dtype=torch.int32, device=gpu)
    got = llima_amd.tree_attention(**t)
    assert torch.equal(got[0], ref[0]) and torch.isnan(got[1]).all()
    z = {k: v[:0] for k, v in s.items()}
    assert llima_amd.tree_attention(**z).shape == (0, 4, 4, 64)


def test_a_cache_past_32_bits(gpu):
    """Keys at offsets above 2^32 bytes: a long contiguous cache, and pages at the end of a large one."""
    import llima_amd
    L, Hkv, D = 1_100_000, 8, 256                            # 4.5 GB each of K and V
    kc = torch.zeros(1, L, Hkv, D, dtype=torch.bfloat16, device=gpu)
    vc = torch.zeros_like(kc)
    q = torch.zeros(1, 2, 8, D, dtype=torch.bfloat16, device=gpu)
    q[..., 0] = 16.0
    k = torch.zeros(1, 2, Hkv, D, dtype=torch.bfloat16, device=gpu)
    for h in range(8):                                       # head h finds its key near the end, weight 1 - 1e-8 L
        kc[0, L - 1 - h, h, 0] = 30.0
        vc[0, L - 1 - h, h] = float(h + 1)
    out = llima_amd.tree_attention(q, k, k, kc, vc, torch.tensor([L], dtype=torch.int32, device=gpu))
    assert torch.equal(out[0, 0], torch.arange(1.0, 9.0, device=gpu).to(torch.bfloat16)[:, None].expand(8, D))
    n = 5000
    page = 100
    table = torch.arange(L // page - n // page, L // page, dtype=torch.int32, device=gpu).view(1, -1)
    out = llima_amd.tree_attention(q, k, k, kc.view(L // page, page, Hkv, D), vc.view(L // page, page, Hkv, D),
                                   torch.tensor([n], dtype=torch.int32, device=gpu), block_table=table)
    assert torch.equal(out[0, 1], torch.arange(1.0, 9.0, device=gpu).to(torch.bfloat16)[:, None].expand(8, D))


def test_many_small_pages_in_one_chunk(gpu):
    """More table entries in a chunk of keys than a workgroup keeps: pages of one token, one long sequence among
    many heads (few chunks)."""
    import llima_amd
    s, g = make(gpu, 1, 2, 128, 64, 64, [30000], 1, seed=6, qscale=1.0)
    check(llima_amd.tree_attention(**s), s)
    s["block_table"][0, 29999] = -5
    assert torch.isnan(llima_amd.tree_attention(**s)).all()


def test_same_call_twice_and_graph_replays(gpu):
    """Bit-identical again; two graphs captured on one stream, replayed on two, with other lengths."""
    import llima_amd
    s, g = make(gpu, 3, 8, 8, 2, 128, [3000, 10, 800], 16, seed=12)
    mask = tree_mask(g, 3, 8).to(gpu)
    a = llima_amd.tree_attention(tree_mask=mask, **s)
    assert torch.equal(a, llima_amd.tree_attention(tree_mask=mask, **s))
    s2, _ = make(gpu, 3, 8, 8, 2, 128, [2000, 1000, 8], 16, seed=13)
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


# ------------------------------------------------------------------ commit


def plain_commit(k, v, nodes, counts, kc, vc, lens, table):
    kc, vc, new = kc.clone(), vc.clone(), []
    page = kc.shape[2]
    for b in range(k.shape[1]):
        n, c = int(lens[b]), int(counts[b])
        cap = page * (table.shape[1] if table is not None else 1)
        path = nodes[b, :max(c, 0)].tolist() if c <= nodes.shape[1] else [-1]
        pages = []
        ok = 0 <= n and 0 <= c <= nodes.shape[1] and n + c <= cap and all(0 <= x < k.shape[2] for x in path)
        if ok and table is not None:
            pages = [int(table[b, (n + j) // page]) for j in range(c)]
            ok = all(0 <= p < kc.shape[1] for p in pages)
        new.append(n + c if ok else -2)
        for j in range(c if ok else 0):
            p, o = (pages[j], (n + j) % page) if table is not None else (b, n + j)
            kc[:, p, o], vc[:, p, o] = k[:, b, path[j]], v[:, b, path[j]]
    return kc, vc, new


@pytest.mark.parametrize("layers,B,N,L,Hkv,D,page,blocks", [
    (1, 1, 1, 1, 1, 64, 0, 0), (32, 1, 16, 5, 8, 128, 0, 0), (3, 9, 33, 8, 2, 128, 16, 6), (2, 5, 7, 7, 3, 256, 1, 40),
    (5, 3, 64, 64, 1, 8, 7, 20), (1, 2, 4, 3, 40, 128, 64, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_commit_is_its_definition(gpu, layers, B, N, L, Hkv, D, page, blocks, dtype):
    import llima_amd
    g = torch.Generator().manual_seed(layers + B + N)
    k, v = (torch.randn(layers, B, N, Hkv, D, generator=g).to(dtype) for _ in range(2))
    if page:
        shape, cap = (layers, B * blocks + 2, page, Hkv, D), page * blocks
        table = torch.randperm(B * blocks + 2, generator=g)[:B * blocks].view(B, blocks).to(torch.int32)
    else:
        shape, cap, table = (layers, B, 77, Hkv, D), 77, None
    kc, vc = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    nodes = torch.randint(0, N, (B, L), generator=g).to(torch.int32)      # a node may come twice
    counts = torch.randint(0, L + 1, (B,), generator=g).to(torch.int32)
    lens = torch.tensor([int(torch.randint(0, cap - int(c) + 1, (1,), generator=g)) if int(c) <= cap else 0 for c in counts],
                        dtype=torch.int32)
    lens[0] = max(0, cap - int(counts[0]))                   # fills its room
    nodes[-1, int(counts[-1]):] = -1                         # what lies past the count is not read
    for bad in range(-1, 6):
        n2, c2, l2, t2 = nodes.clone(), counts.clone(), lens.clone(), None if table is None else table.clone()
        b = B // 2
        if bad == 0:
            c2[b] = L + 1
        elif bad == 1:
            c2[b] = -1
        elif bad == 2:
            c2[b], n2[b, 0], l2[b] = 1, N, 0
        elif bad == 3:
            l2[b] = -1
        elif bad == 4:
            c2[b], l2[b] = 1, cap
        elif bad == 5 and t2 is not None:
            c2[b], l2[b], t2[b, 0] = 1, 0, shape[1]
        ek, ev, en = plain_commit(k, v, n2, c2, kc, vc, l2, t2)
        dk, dv = kc.to(gpu), vc.to(gpu)
        new = llima_amd.tree_commit(k.to(gpu), v.to(gpu), n2.to(gpu), c2.to(gpu), dk, dv, l2.to(gpu),
                                    block_table=None if t2 is None else t2.to(gpu))
        assert new.tolist() == en, bad
        assert torch.equal(dk.cpu(), ek) and torch.equal(dv.cpu(), ev), bad


def test_commit_without_layers_dimension_and_with_views(gpu):
    import llima_amd
    k, v = (torch.randn(2, 5, 2, 64, device=gpu).to(torch.bfloat16) for _ in range(2))
    both = torch.randn(2, 2, 2, 30, 64, device=gpu).to(torch.bfloat16)     # [B, K or V, heads, tokens, D]
    kc, vc = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    before = both.clone()
    nodes = torch.tensor([[0, 3, 4], [0, 1, 2]], dtype=torch.int32, device=gpu)
    lens = torch.tensor([4, 27], dtype=torch.int32, device=gpu)
    new = llima_amd.tree_commit(k, v, nodes, torch.tensor([2, 3], dtype=torch.int32, device=gpu), kc, vc, lens)
    assert new.tolist() == [6, 30]
    before[0, 0, :, 4:6], before[0, 1, :, 4:6] = k[0, [0, 3]].transpose(0, 1), v[0, [0, 3]].transpose(0, 1)
    before[1, 0, :, 27:30], before[1, 1, :, 27:30] = k[1, :3].transpose(0, 1), v[1, :3].transpose(0, 1)
    assert torch.equal(both, before)
    with pytest.raises(ValueError):                          # a cache that would have to be copied
        llima_amd.tree_commit(k, v, nodes, lens, torch.zeros(2, 30, 2, 65, device=gpu, dtype=torch.bfloat16)[..., 1:],
                              vc, lens)


@pytest.mark.parametrize("page", [0, 64, 24, 7])
@pytest.mark.parametrize("N,Hq,Hkv", [(3, 4, 2), (11, 8, 2), (20, 4, 1), (30, 8, 2), (33, 8, 2), (64, 16, 4), (65, 16, 2)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_kernel(gpu, dtype, D, N, Hq, Hkv, page):
    """Every number of row tiles in a workgroup (1, 2, 3, 4, 5, 8, and more than one group of them) with every way of
    addressing the cache, short and longer sequences together, with and without a mask."""
    import llima_amd
    lens = [0, 130, 700, 63]
    s, g = make(gpu, 4, N, Hq, Hkv, D, lens, page, dtype, seed=N + D)
    mask = tree_mask(g, 4, N).to(gpu)
    check(llima_amd.tree_attention(tree_mask=mask, **s), s, mask)
    check(llima_amd.tree_attention(scale=-0.05, **s), s, scale=-0.05)


def test_commit_refuses_keys_inside_the_cache(gpu):
    """Drafted tokens kept in the cache itself: copies in no order would read what others wrote."""
    import llima_amd
    buf = torch.randn(2, 2, 40, 4, 64, device=gpu).to(torch.bfloat16)      # K and V in one allocation
    kc, vc = buf[0], buf[1]
    nodes = torch.tensor([[0, 2], [1, 2]], dtype=torch.int32, device=gpu)
    counts = torch.tensor([2, 2], dtype=torch.int32, device=gpu)
    lens = torch.tensor([10, 10], dtype=torch.int32, device=gpu)
    before = buf.clone()
    for k, v in ((kc[:, 10:13], vc[:, 10:13]), (vc[:, 10:13], vc[:, 10:13])):
        with pytest.raises(ValueError, match="overlap"):
            llima_amd.tree_commit(k, v, nodes, counts, kc, vc, lens)
    assert torch.equal(buf, before)
    k, v = kc[:, 10:13].clone(), vc[:, 10:13].clone()
    assert llima_amd.tree_commit(k, v, nodes, counts, kc, vc, lens).tolist() == [12, 12]
    assert torch.equal(kc[0, 11], k[0, 2]) and torch.equal(vc[1, 10], v[1, 1])


@pytest.mark.parametrize("B,N,Hq,Hkv,D,page", [(40, 1, 64, 64, 64, 0), (21, 3, 128, 64, 64, 16), (30, 40, 64, 8, 128, 64),
                                               (33, 2, 512, 512, 64, 0), (18, 9, 48, 24, 256, 5)])
def test_more_sequences_than_shares(gpu, monkeypatch, B, N, Hq, Hkv, D, page):
    """Batches above the number of shares, where partial sums stand two to a share: sequences that begin, end and lie inside a
    share, or span several, and nothing written past the workspace's size."""
    import llima_amd
    from llima_amd import attention
    lens = [(7 * b * b) % 500 for b in range(B)]
    lens[3], lens[B // 2], lens[B - 1] = 9000, 0, 4000
    s, g = make(gpu, B, N, Hq, Hkv, D, lens, page, seed=B)
    bufs = []

    def scratch(dev, kind, nbytes):
        bufs.append((torch.full((nbytes + 4096,), 0x7F, dtype=torch.uint8, device=dev), nbytes))
        return bufs[-1][0][:nbytes]
    monkeypatch.setattr(attention, "_scratch", scratch)
    mask = tree_mask(g, B, N).to(gpu)
    check(llima_amd.tree_attention(tree_mask=mask, **s), s, mask)
    buf, n = bufs[0]
    assert (buf[n:] == 0x7F).all()


def test_commit_of_drafts_behind_the_cached_tokens(gpu):
    """One buffer per step: the drafts stand behind each sequence's cached tokens, K and V side by side."""
    import llima_amd
    buf = torch.randn(3, 2, 24, 2, 2, 64, device=gpu).to(torch.bfloat16)   # [layers, B, tokens + drafts, K or V, heads, D]
    k, v, kc, vc = buf[:, :, 20:, 0], buf[:, :, 20:, 1], buf[:, :, :20, 0], buf[:, :, :20, 1]
    want = buf.clone()
    for b, (n, path) in enumerate(((3, [0, 2]), (17, [1, 2, 3]))):
        for j, node in enumerate(path):
            want[:, b, n + j] = buf[:, b, 20 + node]
    nodes = torch.tensor([[0, 2, 0], [1, 2, 3]], dtype=torch.int32, device=gpu)
    new = llima_amd.tree_commit(k, v, nodes, torch.tensor([2, 3], dtype=torch.int32, device=gpu), kc, vc,
                                torch.tensor([3, 17], dtype=torch.int32, device=gpu))
    assert new.tolist() == [5, 20] and torch.equal(buf, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [0, 5, 6000])
def test_scores_that_are_all_minus_infinity(gpu, n, dtype):
    """The softmax over visible scores of minus infinity alone is NaN, as by the formula (0 / 0), not the 0 of a row that sees
    nothing; beside a finite score they weigh nothing."""
    import llima_amd
    s, g = make(gpu, 2, 4, 4, 2, 64, [n, n], 0, dtype, seed=n + 1)
    mask = tree_mask(g, 2, 4).to(gpu)
    mask[1, 2] = False
    s["q"][:, :, 0] = s["q"][:, :, 0].abs() + 1.0             # head 0 of key head 0: positive, times -inf
    s["k"][0, :, 0, 7] = -math.inf
    s["k_cache"][0, :n, 0, 7] = -math.inf
    got = llima_amd.tree_attention(tree_mask=mask, **s)
    ref, tol = definition(s, mask)
    assert torch.isnan(ref[0, :, 0]).all() and torch.isnan(got[0, :, 0]).all()
    assert torch.isfinite(got[1]).all() and ((got[1].double() - ref[1]).abs() <= tol[1] + 1e-30).all()
    assert ((got[0, :, 2:].double() - ref[0, :, 2:]).abs() <= tol[0, :, 2:] + 1e-30).all()
    if n == 0:
        assert (got[1, 2] == 0).all()
    s["k"][0, 0, 0, 7] = 0.5                                  # node 0, which all see, has a finite score
    got = llima_amd.tree_attention(tree_mask=mask, **s)
    want = s["v"][0, 0, 0].expand(4, 64)
    assert torch.equal(got[0, :, 0], want)
