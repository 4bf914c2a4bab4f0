"""Steps over an 8-bit KV cache in the order a serving loop calls them.

prompt into the cache -> draft tree -> attention under its mask -> projection -> the norms around the residual stream,
to 8 bits -> 8-bit LM head with tree verification -> the accepted path into the cache -> the next step; at the end
the sequence back in 16 bits.
"""
import math

import pytest
import torch

from .test_gpu_attention8 import F8, cache8, definition, quantize
from .test_gpu_cache8 import same as equal
from .test_gpu_norm import plain_blocks, same
from .test_gpu_sandwich import plain
from .test_gpu_verification_step import draft_tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [0, 16, 64])
def test_steps_of_one_stream(gpu, page):
    import llima_amd
    bf = torch.bfloat16
    g = torch.Generator(device=gpu).manual_seed(14 + page)
    Hq, Hkv, D, H, V, layers, room, prompt = 8, 2, 128, 512, 700, 3, 448, 150

    def rnd(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=gpu) * scale).to(bf)
    if page:
        n = room // page
        table = torch.randperm(n + 5, generator=torch.Generator().manual_seed(1))[:n].to(torch.int32).to(gpu)[None]
        shape = (layers, n + 5, page, Hkv, D)
    else:
        table, shape = None, (layers, 1, room, Hkv, D)
    kc, vc = llima_amd.Fp8Cache.empty(*shape, device=gpu), llima_amd.Fp8Cache.empty(*shape, device=gpu)
    for c in (kc, vc):                                       # what is not written is NaN
        c.values.view(torch.uint8).fill_(0x7F)
        c.scales.fill_(math.nan)
    dense = [rnd(layers, 1, prompt, Hkv, D) for _ in range(2)]   # what the cache should hold, before its 8 bits
    lens = torch.zeros(1, dtype=torch.int32, device=gpu)
    for at in range(0, prompt, 64):                          # the prompt in chunks, the last one padded
        k, v = (torch.nn.functional.pad(d[:, :, at:at + 64], (0, 0, 0, 0, 0, max(0, at + 64 - prompt)), value=math.nan) for d in dense)
        lens = llima_amd.cache_write(k, v, kc, vc, lens, torch.tensor([min(64, prompt - at)], dtype=torch.int32, device=gpu),
                                     block_table=table)
    assert lens.tolist() == [prompt]
    wo, gate, post, pre = rnd(Hq * D, H, scale=(Hq * D) ** -0.5), rnd(H), rnd(H, scale=0.1), rnd(H, scale=0.1)
    head = llima_amd.lm_head_quantize(rnd(V, H, scale=H ** -0.5))
    token, kw = 3, dict(gate=gate, residual_scale=0.9, eps=1e-5, weight_offset=1.0)
    for step in range(4):
        out = draft_tree(gpu, g, token)
        N = out["tokens"].numel()
        q, k, v = rnd(1, N, Hq, D, scale=2.0), rnd(layers, 1, N, Hkv, D), rnd(layers, 1, N, Hkv, D)
        res = rnd(N, H)
        for layer in range(layers):
            o = llima_amd.tree_attention(q, k[layer], v[layer], kc[layer], vc[layer], lens, tree_mask=out["tree_mask"], block_table=table)
            s = dict(q=q, k=k[layer], v=v[layer], cache_lens=lens, k_cache=cache8(dense[0][layer]), v_cache=cache8(dense[1][layer]))
            ref, tol = definition(s, out["tree_mask"][None] > 0)
            assert ((o.double() - ref).abs() <= tol).all(), (step, layer)
            x = (o.reshape(N, Hq * D).float() @ wo.float()).to(bf)
            y, new_res = llima_amd.sandwich_norm(x, post, res, pre, out="fp8", **kw)
            ey, er = plain(x.cpu(), post.cpu(), res.cpu(), pre.cpu(), gate.cpu(), 0.9, float(torch.tensor(1e-5)), 1.0)
            eq, es = plain_blocks(ey)
            same(new_res, er)
            same(y.values, eq)
            same(y.scales, es)
            res = new_res
        # candidates of each path, the accepted ones planted from the head's own choice
        ids, _, logits = llima_amd.lm_head_argmax(y, head, return_logits=True)
        retrieve = out["retrieve"].cpu()
        cand = torch.where(retrieve >= 0, out["tokens"].cpu()[retrieve.clamp_min(0).long()], -1)
        want = retrieve.shape[0] // 2
        for i in range(1, int((retrieve[want] >= 0).sum())):
            cand[retrieve == int(retrieve[want, i])] = int(ids[int(retrieve[want, i - 1])])
        cand = cand.to(torch.int32)
        best, accepted, token = llima_amd.lm_head_verify_tree(y, head, out["retrieve"], cand)
        assert (best, accepted, token) == llima_amd.verify_tree(logits, out["retrieve"], cand) and accepted >= 1
        nodes = out["retrieve"][best:best + 1, :accepted + 1].to(torch.int32).contiguous()
        counts = torch.tensor([accepted + 1], dtype=torch.int32, device=gpu)
        new = llima_amd.tree_commit(k, v, nodes, counts, kc, vc, lens, block_table=table)
        assert new.tolist() == [int(lens[0]) + accepted + 1]
        path = nodes[0].long()
        dense = [torch.cat((d, t[:, :, path]), 2) for d, t in zip(dense, (k, v))]
        lens = new
    n = int(lens[0])
    for r, d in zip(llima_amd.cache_read(kc, vc, lens, block_table=table), dense):
        qd, sd = quantize(d)
        assert r.shape == (layers, 1, room, Hkv, D) and (r[:, :, n:] == 0).all()
        assert equal(r[:, :, :n], (qd.float() * sd[..., None]).to(bf))


def test_a_step_in_a_graph(gpu):
    """Attention over the 8-bit cache, the norms, the 8-bit head with chain verification and the path's write captured together;
    replayed with new inputs and lengths, eager work between the replays, every replay against the eager calls."""
    import llima_amd
    bf = torch.bfloat16
    g = torch.Generator(device=gpu).manual_seed(9)
    B, D1, Hq, Hkv, D, V, page = 3, 4, 4, 2, 64, 500, 16
    H = Hq * D

    def rnd(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=gpu) * scale).to(bf)
    table = torch.arange(B * 20, dtype=torch.int32, device=gpu).view(B, 20)
    kc, vc = cache8(rnd(B * 20, page, Hkv, D)), cache8(rnd(B * 20, page, Hkv, D))
    lens = torch.tensor([5, 100, 0], dtype=torch.int32, device=gpu)
    q, k, v, res = rnd(B, D1, Hq, D), rnd(B, D1, Hkv, D), rnd(B, D1, Hkv, D), rnd(B * D1, H)
    post, pre = rnd(H), rnd(H)
    head = llima_amd.lm_head_quantize(rnd(V, H))
    drafts = torch.zeros(B, D1 - 1, dtype=torch.int32, device=gpu)
    nodes = torch.arange(D1, dtype=torch.int32, device=gpu).expand(B, D1).contiguous()

    def copy(c):
        n = llima_amd.Fp8Cache.empty(*c.shape, device=gpu)
        n.values.view(torch.uint8).copy_(c.values.view(torch.uint8))
        n.scales.copy_(c.scales)
        return n

    def step(kc, vc):
        o = llima_amd.tree_attention(q, k, v, kc, vc, lens, block_table=table)
        y, r = llima_amd.sandwich_norm(o.reshape(B * D1, H), post, res, pre, gate=0.5, out="fp8")
        acc, em = llima_amd.lm_head_verify_greedy(y, head, drafts)
        new = llima_amd.tree_commit(k, v, nodes, acc + 1, kc, vc, lens, block_table=table)
        return [o, y.values.view(torch.uint8), y.scales, r, acc, em, new]

    step(copy(kc), copy(vc))
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = step(kc, vc)
    for i in range(5):
        q.copy_(rnd(B, D1, Hq, D))
        lens.copy_(torch.tensor([5 + i, 100 - 7 * i, 31 * i], dtype=torch.int32))
        o = step(copy(kc), copy(vc))
        drafts.copy_(o[5][:, :1].expand(B, D1 - 1).clamp_min(0))     # the first draft is accepted
        ek, ev = copy(kc), copy(vc)
        want = step(ek, ev)
        gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i
        assert equal(kc.values, ek.values) and equal(vc.values, ev.values)
        assert torch.equal(kc.scales, ek.scales) and torch.equal(vc.scales, ev.scales)
        assert (want[4] >= 1).all()


def test_calls_of_one_form_with_other_tensors(gpu):
    """The checks of a call are kept by its tensors' forms: other tensors of the same form, others of another, and
    refusals after accepted calls."""
    import llima_amd
    bf = torch.bfloat16
    outs = []
    for seed in range(2):
        g = torch.Generator(device=gpu).manual_seed(seed)
        q = torch.randn(2, 3, 4, 64, generator=g, device=gpu).to(bf)
        k, v = (torch.randn(2, 3, 2, 64, generator=g, device=gpu).to(bf) for _ in range(2))
        kc, vc = (cache8(torch.randn(2, 50, 2, 64, generator=g, device=gpu)) for _ in range(2))
        lens = torch.tensor([50, 7], dtype=torch.int32, device=gpu)
        s = dict(q=q, k=k, v=v, k_cache=kc, v_cache=vc, cache_lens=lens)
        o = llima_amd.tree_attention(**s)
        ref, tol = definition(s, None)
        assert ((o.double() - ref).abs() <= tol).all()
        wide = torch.zeros(2, 3, 9, 64, dtype=bf, device=gpu)
        wide[:, :, 2:6] = q
        assert torch.equal(llima_amd.tree_attention(**dict(s, q=wide[:, :, 2:6])), o)
        assert torch.equal(llima_amd.tree_attention(**dict(s, q=q.transpose(1, 2).contiguous().transpose(1, 2))), o)
        odd = torch.zeros(q.numel() + 1, dtype=bf, device=gpu)[1:].view(q.shape)
        odd.copy_(q)
        assert torch.equal(llima_amd.tree_attention(**dict(s, q=odd)), o)
        for bad in (dict(q=q.half()), dict(cache_lens=lens.long()), dict(q=q.cpu()), dict(v_cache=llima_amd.Fp8Cache(vc.values[:, :49], vc.scales[:, :49]))):
            with pytest.raises(ValueError):
                llima_amd.tree_attention(**dict(s, **bad))
        outs.append(o)
    assert not torch.equal(*outs)


def test_a_scale_is_its_value_at_the_call(gpu):
    """A scale or a number of tokens given as a tensor of one element, changed between two calls."""
    import llima_amd
    q, k, v = (torch.randn(1, 2, 2, 64, device=gpu).bfloat16() for _ in range(3))
    kc, vc = (cache8(torch.randn(1, 50, 2, 64, device=gpu)) for _ in range(2))
    lens = torch.tensor([50], dtype=torch.int32, device=gpu)
    scale, tokens = torch.tensor(0.1), torch.tensor(3)
    for s, n in ((0.1, 3), (0.7, 5)):
        scale.fill_(s)
        tokens.fill_(n)
        assert torch.equal(llima_amd.tree_attention(q, k, v, kc, vc, lens, scale=scale),
                           llima_amd.tree_attention(q, k, v, kc, vc, lens, scale=float(scale)))
        assert llima_amd.cache_read(kc, vc, lens, tokens=tokens)[0].shape == (1, n, 2, 64)
