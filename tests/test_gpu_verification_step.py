"""The operators of a verification step in the order a serving loop calls them.

draft tree -> attention under its mask over a paged cache -> projection -> residual norm to 8 bits
-> 8-bit LM head with tree verification -> the accepted path into the cache -> the next step.
"""
import pytest
import torch

from .test_gpu_attention import definition
from .test_gpu_norm import plain_blocks, plain_norm, same

pytestmark = pytest.mark.gpu


def draft_tree(gpu, g, token):
    import llima_amd
    Vd, K, depth = 400, 4, 3
    d2t = torch.zeros(Vd, dtype=torch.int32, device=gpu)
    tree = llima_amd.Eagle3DraftTree(d2t, topk=K, depth=depth)
    tree.begin(torch.randn(Vd, generator=g, device=gpu))
    for _ in range(depth - 1):
        tree.grow(torch.randn(K, Vd, generator=g, device=gpu))
    return tree.finish(11, token)


@pytest.mark.parametrize("page", [0, 16])
def test_steps_of_one_stream(gpu, page):
    import llima_amd
    bf = torch.bfloat16
    g = torch.Generator(device=gpu).manual_seed(4 + page)
    Hq, Hkv, D, H, V, layers, room = 8, 2, 128, 512, 700, 3, 400

    def rnd(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=gpu) * scale).to(bf)
    if page:
        table = torch.randperm(room // page + 5, generator=torch.Generator().manual_seed(1))[:room // page].to(torch.int32).to(gpu)[None]
        shape = (layers, room // page + 5, page, Hkv, D)
    else:
        table, shape = None, (layers, 1, room, Hkv, D)
    kc, vc = torch.full(shape, float("nan"), device=gpu, dtype=bf), torch.full(shape, float("nan"), device=gpu, dtype=bf)
    dense = [torch.zeros(layers, 0, Hkv, D, dtype=bf, device=gpu) for _ in range(2)]   # what the cache should hold
    lens = torch.zeros(1, dtype=torch.int32, device=gpu)
    wo, wn = rnd(Hq * D, H, scale=(Hq * D) ** -0.5), rnd(H, scale=0.1) + 1
    head = llima_amd.lm_head_quantize(rnd(V, H, scale=H ** -0.5))
    token = 3
    for step in range(4):
        out = draft_tree(gpu, g, token)
        N = out["tokens"].numel()
        q, k, v = rnd(1, N, Hq, D, scale=2.0), rnd(layers, 1, N, Hkv, D), rnd(layers, 1, N, Hkv, D)
        res = rnd(N, H)
        for layer in range(layers):
            s = dict(q=q, k=k[layer], v=v[layer], cache_lens=lens, k_cache=kc[layer], v_cache=vc[layer])
            if page:
                s["block_table"] = table
            o = llima_amd.tree_attention(tree_mask=out["tree_mask"], **s)
            plain = dict(s, k_cache=dense[0][layer][None], v_cache=dense[1][layer][None])
            plain.pop("block_table", None)
            ref, tol = definition(plain, out["tree_mask"][None] > 0)
            assert ((o.double() - ref).abs() <= tol).all(), (step, layer)
            x = (o.reshape(N, Hq * D).float() @ wo.float()).to(bf)
            y, new_res = llima_amd.add_rms_norm(x, wn, res, out="fp8")
            ey, er = plain_norm(x.cpu(), wn.cpu(), res.cpu(), 1e-6, 0.0)
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
        depth = int((retrieve[want] >= 0).sum())
        for i in range(1, depth):
            node = int(retrieve[want, i])
            cand[retrieve == node] = int(ids[int(retrieve[want, i - 1])])
        cand = cand.to(torch.int32)
        got = llima_amd.lm_head_verify_tree(y, head, out["retrieve"], cand)
        assert got == llima_amd.verify_tree(logits, out["retrieve"], cand)
        best, accepted, token = got
        assert accepted >= 1
        # the accepted path (its root is the sampled token) goes into every layer's cache
        nodes = out["retrieve"][best:best + 1, :accepted + 1].to(torch.int32).contiguous()
        counts = torch.tensor([accepted + 1], dtype=torch.int32, device=gpu)
        new = llima_amd.tree_commit(k, v, nodes, counts, kc, vc, lens, block_table=table)
        assert new.tolist() == [int(lens[0]) + accepted + 1]
        path = nodes[0].long()
        dense = [torch.cat((d, t[:, 0, path]), 1) for d, t in zip(dense, (k, v))]
        # the last accepted node as a decode step over the cache without it: the row that the tree gave it
        s = dict(q=q[:, path[-1:]], k=k[-1][:, path[-1:]], v=v[-1][:, path[-1:]], cache_lens=new - 1, k_cache=kc[-1], v_cache=vc[-1])
        one = llima_amd.tree_attention(block_table=table, **s)
        ref, tol = definition(dict(s, k_cache=dense[0][-1][None], v_cache=dense[1][-1][None]), None)
        assert ((one.double() - ref).abs() <= tol).all()
        assert ((one[0, 0].double() - o[0, path[-1]].double()).abs() <= 2 * tol[0, 0]).all()
        lens = new


def test_a_step_in_a_graph(gpu):
    """Attention, norm, 8-bit head with chain verification and commit captured together; replayed with new inputs and
    lengths, eager work between the replays, every replay against the eager calls."""
    import llima_amd
    bf = torch.bfloat16
    g = torch.Generator(device=gpu).manual_seed(9)
    B, D1, Hq, Hkv, D, V, page = 3, 4, 4, 2, 64, 500, 16
    H = Hq * D

    def rnd(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=gpu) * scale).to(bf)
    table = torch.arange(B * 20, dtype=torch.int32, device=gpu).view(B, 20)
    kc, vc = rnd(B * 20, page, Hkv, D), rnd(B * 20, page, Hkv, D)
    lens = torch.tensor([5, 100, 0], dtype=torch.int32, device=gpu)
    q, k, v, res, wn = rnd(B, D1, Hq, D), rnd(B, D1, Hkv, D), rnd(B, D1, Hkv, D), rnd(B * D1, H), rnd(H)
    head = llima_amd.lm_head_quantize(rnd(V, H))
    drafts = torch.zeros(B, D1 - 1, dtype=torch.int32, device=gpu)
    nodes = torch.arange(D1, dtype=torch.int32, device=gpu).expand(B, D1).contiguous()

    def step(kc, vc):
        o = llima_amd.tree_attention(q, k, v, kc, vc, lens, block_table=table)
        y, r = llima_amd.add_rms_norm(o.reshape(B * D1, H), wn, res, out="fp8")
        acc, em = llima_amd.lm_head_verify_greedy(y, head, drafts)
        new = llima_amd.tree_commit(k, v, nodes, acc + 1, kc, vc, lens, block_table=table)
        return [o, y.values.view(torch.uint8), y.scales, r, acc, em, new]

    step(kc.clone(), vc.clone())
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = step(kc, vc)
    for i in range(5):
        q.copy_(rnd(B, D1, Hq, D))
        lens.copy_(torch.tensor([5 + i, 100 - 7 * i, 31 * i], dtype=torch.int32))
        o = step(kc.clone(), vc.clone())
        drafts.copy_(o[5][:, :1].expand(B, D1 - 1).clamp_min(0))     # the first draft is accepted
        ek, ev = kc.clone(), vc.clone()
        want = step(ek, ev)
        gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i
        assert torch.equal(kc, ek) and torch.equal(vc, ev)
        assert (want[4] >= 1).all()
