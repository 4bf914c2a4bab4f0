"""cache_write, tree_commit and cache_read over Fp8Cache against their definitions, bit for bit: a value is 448 x / max
by one division rounded to nearest and then to e4m3, a scale max / 448, and read back q scale is one product rounded to
fp32 and then to the type."""
import math

import pytest
import torch

from .test_gpu_attention8 import F8, cache8, quantize

pytestmark = pytest.mark.gpu


def same(a, b):
    """Equal bits; NaN of any sign and payload are one."""
    if a.dtype == F8:
        a, b = a.float(), b.float()
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def plain_write(k, v, nodes, counts, kc, vc, lens, table):
    """New (values, scales) of both caches and the lengths, on the CPU."""
    (kq, ks), (vq, vs) = ((c.values.cpu().view(torch.uint8).clone(), c.scales.cpu().clone()) for c in (kc, vc))
    page, new = kq.shape[2], []
    for b in range(k.shape[1]):
        n, c, L = int(lens[b]), int(counts[b]), k.shape[2] if nodes is None else nodes.shape[1]
        cap = page * (table.shape[1] if table is not None else 1)
        path = [-1] if c > L else list(range(max(c, 0))) if nodes is None else nodes[b, :max(c, 0)].tolist()
        pages = []
        ok = 0 <= n and 0 <= c <= L and n + c <= cap and all(0 <= x < k.shape[2] for x in path)
        if ok and table is not None:
            pages = [int(table[b, (n + j) // page]) for j in range(c)]
            ok = all(0 <= p < kq.shape[1] for p in pages)
        new.append(n + c if ok else -2)
        for j in range(c if ok else 0):
            p, o = (pages[j], (n + j) % page) if table is not None else (b, n + j)
            for x, q8, s8 in ((k, kq, ks), (v, vq, vs)):
                q, s = quantize(x[:, b, path[j]])
                q8[:, p, o], s8[:, p, o] = q.view(torch.uint8), s
    return kq.view(F8), ks, vq.view(F8), vs, new


@pytest.mark.parametrize("layers,B,N,L,Hkv,D,page,blocks", [
    (1, 1, 1, 0, 1, 64, 0, 0), (1, 1, 1, 1, 1, 64, 0, 0), (32, 1, 16, 5, 8, 128, 0, 0), (3, 9, 33, 8, 2, 128, 16, 6),
    (2, 5, 7, 7, 3, 256, 1, 40), (1, 3, 300, 0, 5, 128, 7, 90), (5, 3, 64, 64, 1, 64, 7, 20), (1, 2, 4, 0, 40, 128, 64, 2),
    (2, 2, 70, 0, 1, 256, 16, 9)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_write_is_its_definition(gpu, layers, B, N, L, Hkv, D, page, blocks, dtype):
    import llima_amd
    g = torch.Generator().manual_seed(layers + B + N)
    wide = torch.exp2(torch.randint(-9, 10, (N, 1, 1), generator=g).float())
    k, v = ((torch.randn(layers, B, N, Hkv, D, generator=g) * wide).to(dtype) for _ in range(2))
    k[0, 0, 0, 0] = 0.0                                      # a row of zeros has the smallest scale
    if page:
        shape, cap = (layers, B * blocks + 2, page, Hkv, D), page * blocks
        table = torch.randperm(B * blocks + 2, generator=g)[:B * blocks].view(B, blocks).to(torch.int32)
    else:
        shape, cap, table = (layers, B, 77, Hkv, D), 77, None
    old = [torch.randn(shape, generator=g) for _ in range(2)]
    places = L or N
    nodes = torch.randint(0, N, (B, L), generator=g).to(torch.int32) if L else None     # a node may come twice
    counts = torch.randint(0, places + 1, (B,), generator=g).clamp_max(cap).to(torch.int32)
    lens = torch.tensor([int(torch.randint(0, cap - int(c) + 1, (1,), generator=g)) for c in counts], dtype=torch.int32)
    lens[0] = cap - int(counts[0])                           # fills its room
    if nodes is not None:
        nodes[-1, int(counts[-1]):] = -1                     # what lies past the count is not read
    for bad in range(-1, 6):
        n2, c2, l2, t2 = None if nodes is None else nodes.clone(), counts.clone(), lens.clone(), None if table is None else table.clone()
        b = B // 2
        if bad == 0:
            c2[b] = places + 1
        elif bad == 1:
            c2[b] = -1
        elif bad == 2 and n2 is not None:
            c2[b], n2[b, 0], l2[b] = 1, N, 0
        elif bad == 3:
            l2[b] = -1
        elif bad == 4:
            c2[b], l2[b] = 1, cap
        elif bad == 5 and t2 is not None:
            c2[b], l2[b], t2[b, 0] = 1, 0, shape[1]
        kc, vc = (cache8(o.to(gpu), head_major=bad != 0) for o in old)
        want = plain_write(k, v, n2, c2, kc, vc, l2, t2)
        tg = None if t2 is None else t2.to(gpu)
        if n2 is not None:
            new = llima_amd.tree_commit(k.to(gpu), v.to(gpu), n2.to(gpu), c2.to(gpu), kc, vc, l2.to(gpu), block_table=tg)
        else:
            new = llima_amd.cache_write(k.to(gpu), v.to(gpu), kc, vc, l2.to(gpu), c2.to(gpu), block_table=tg)
        assert new.tolist() == want[4], bad
        for got, w in zip((kc.values, kc.scales, vc.values, vc.scales), want):
            assert same(got.cpu(), w), bad


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_value_of_a_row(gpu, dtype):
    """All finite values of the type, and rows with NaN and infinities, through writing and reading back."""
    import llima_amd
    every = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype)
    every = every[torch.isfinite(every)]
    n = every.numel() // 128
    rows = every[torch.randperm(every.numel(), generator=torch.Generator().manual_seed(1))][:n * 128].view(1, n, 1, 128)
    order = every.float().abs().argsort()
    near = every[order][:n * 128].view(1, n, 1, 128)         # rows of values of about one size
    special = torch.randn(1, 4, 1, 128).to(dtype)
    special[0, 0, 0, 5], special[0, 1, 0, 9], special[0, 2, 0, 0], special[0, 2, 0, 1] = math.nan, -math.inf, math.inf, math.nan
    x = torch.cat((rows, near, special), 1).to(gpu)
    T = x.shape[1]
    kc, vc = llima_amd.Fp8Cache.empty(1, T, 1, 128, device=gpu), llima_amd.Fp8Cache.empty(1, T, 1, 128, device=gpu)
    lens = llima_amd.cache_write(x, -x, kc, vc, torch.zeros(1, dtype=torch.int32, device=gpu))
    assert lens.tolist() == [T]
    q, s = quantize(x.cpu())
    assert same(kc.values.cpu()[0, :-4], q[0, :-4]) and same(kc.scales.cpu()[0, :-4], s[0, :-4])
    assert torch.equal(vc.values.float(), -kc.values.float()) or same(vc.values.float(), -kc.values.float())
    # NaN: that scale and NaN values; an infinity: an infinite scale, NaN where it stood and 0 elsewhere
    assert kc.scales[0, -4:, 0].isnan().tolist() == [True, False, True, False] and torch.isinf(kc.scales[0, -3, 0])
    odd = kc.values[0, -4:, 0].float()
    assert odd[0].isnan().all() and odd[2].isnan().all() and odd[1].isnan().sum() == 1 and odd[1, 9].isnan()
    assert (odd[1].nan_to_num(0.0) == 0).all()
    for out in (torch.bfloat16, torch.float16):
        rk, rv = llima_amd.cache_read(kc, vc, lens, dtype=out)
        for r, c in ((rk, kc), (rv, vc)):
            assert r.dtype == out and same(r, (c.values.float() * c.scales[..., None]).to(out))


@pytest.mark.parametrize("layers,B,Hkv,D,page,lens,tokens", [
    (0, 1, 1, 64, 0, [0], None), (0, 1, 1, 64, 0, [1], 1), (0, 3, 5, 128, 16, [0, 77, 33], None), (3, 2, 2, 256, 7, [50, 1], 64),
    (0, 4, 8, 128, 64, [300, 5, 0, 129], 200), (2, 2, 1, 64, 1, [9, 30], 33), (0, 1, 40, 128, 0, [70], 100), (0, 2, 2, 64, 8, [4, 4], 0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_read_is_its_definition(gpu, layers, B, Hkv, D, page, lens, tokens, dtype):
    import llima_amd
    g = torch.Generator().manual_seed(B + D)
    front = (layers,) if layers else ()
    S = max(max(lens), 1)
    nblk = -(-S // page) if page else 1
    shape = front + ((B * nblk + 1, page) if page else (B, S)) + (Hkv, D)
    table = torch.randperm(B * nblk + 1, generator=g)[:B * nblk].view(B, nblk).to(torch.int32).to(gpu) if page else None
    kc, vc = (cache8((100.0 * torch.randn(shape, generator=g)).to(gpu), head_major=h) for h in (True, False))
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    rk, rv = llima_amd.cache_read(kc, vc, n, block_table=table, dtype=dtype, tokens=tokens)
    T = tokens if tokens is not None else (nblk * page if page else S)
    for got, c in ((rk, kc), (rv, vc)):
        x = (c.values.float() * c.scales[..., None]).to(dtype)
        want = torch.zeros(front + (B, T, Hkv, D), dtype=dtype, device=gpu)
        for b in range(B):
            rows = x[..., table[b].long(), :, :, :].flatten(-4, -3) if page else x[..., b, :, :, :]
            w = min(lens[b], T)
            want[..., b, :w, :, :] = rows[..., :w, :, :]
        assert got.shape == want.shape and same(got, want)


def test_read_of_bad_sequences(gpu):
    """A length or page out of range makes that sequence NaN, entries past a length do not."""
    import llima_amd
    kc, vc = (cache8(torch.randn(30, 4, 2, 64, device=gpu)) for _ in range(2))
    table = torch.arange(20, dtype=torch.int32, device=gpu).view(5, 4).contiguous()
    lens = torch.tensor([16, 17, -1, 9, 9], dtype=torch.int32, device=gpu)
    table[3, 2], table[4, 3], table[0, 0] = 30, -7, 29
    rk, rv = llima_amd.cache_read(kc, vc, lens, block_table=table, tokens=20)
    for r, c in ((rk, kc), (rv, vc)):
        assert r[1].isnan().all() and r[2].isnan().all() and r[3].isnan().all()
        x = (c.values.float() * c.scales[..., None]).bfloat16()
        assert torch.equal(r[0, :4], x[29]) and torch.equal(r[0, 4:16], x[1:4].flatten(0, 1)) and (r[0, 16:] == 0).all()
        assert torch.equal(r[4, :9], x[[16, 17, 18]].flatten(0, 1)[:9]) and (r[4, 9:] == 0).all()


def test_layers_by_index_and_views(gpu):
    """One layer of a cache of layers; k and v sliced from one tensor; all of a cache's parts in one storage."""
    import llima_amd
    kc, vc = llima_amd.Fp8Cache.empty(3, 2, 40, 2, 128, device=gpu), llima_amd.Fp8Cache.empty(3, 2, 40, 2, 128, device=gpu)
    for c in (kc, vc):
        c.values.view(torch.uint8).zero_()
        c.scales.zero_()
    qkv = torch.randn(2, 5, 6, 128, device=gpu).bfloat16()
    lens = torch.tensor([3, 35], dtype=torch.int32, device=gpu)
    new = llima_amd.cache_write(qkv[:, :, 2:4], qkv[:, :, 4:], kc[1], vc[1], lens)
    assert new.tolist() == [8, 40]
    q, s = quantize(qkv)
    assert same(kc.values[1, 0, 3:8], q[0, :, 2:4]) and same(vc.values[1, 1, 35:], q[1, :, 4:])
    assert torch.equal(kc.scales[1, 0, 3:8], s[0, :, 2:4]) and torch.equal(vc.scales[1, 1, 35:], s[1, :, 4:])
    assert (kc.scales[0] == 0).all() and (vc.scales[2] == 0).all() and (kc.scales[1, 0, 8:] == 0).all()
    one, s1 = kc[0], kc.scales[0]
    assert one.values.data_ptr() == kc.values.data_ptr() and torch.equal(one.scales, s1)
    buf = torch.zeros(2, 2, 40, 2, 128 + 16, dtype=torch.uint8, device=gpu)       # values, then the scale, of each row
    sc = buf.view(torch.float32)[..., 32:33].squeeze(-1)
    k8, v8 = (llima_amd.Fp8Cache(buf[i, ..., :128].view(F8), sc[i]) for i in range(2))
    new = llima_amd.cache_write(qkv[:, :, 2:4], qkv[:, :, 4:], k8, v8, lens)
    assert same(k8.values[0, 3:8], q[0, :, 2:4]) and torch.equal(v8.scales[1, 35:], s[1, :, 4:])
    assert (buf[..., 132:] == 0).all() and (buf[0, 0, 8:] == 0).all()


def test_write_in_a_graph(gpu):
    import llima_amd
    kc, vc = llima_amd.Fp8Cache.empty(4, 2, 300, 2, 64, device=gpu), llima_amd.Fp8Cache.empty(4, 2, 300, 2, 64, device=gpu)
    for c in (kc, vc):
        c.values.view(torch.uint8).zero_()
        c.scales.zero_()
    k, v = (torch.randn(4, 2, 3, 2, 64, device=gpu).bfloat16() for _ in range(2))
    lens, counts = torch.tensor([0, 100], dtype=torch.int32, device=gpu), torch.tensor([3, 1], dtype=torch.int32, device=gpu)
    llima_amd.cache_write(k, v, kc, vc, lens, counts)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        new = llima_amd.cache_write(k, v, kc, vc, lens, counts)
        rk, rv = llima_amd.cache_read(kc, vc, new, tokens=130)
    for i in range(4):
        k.normal_()
        v.normal_()
        counts.copy_(torch.tensor([i % 4, 3 - i % 4], dtype=torch.int32))
        ek, ev = (llima_amd.Fp8Cache(c.values.view(torch.uint8).clone().view(F8), c.scales.clone()) for c in (kc, vc))
        want = llima_amd.cache_write(k, v, ek, ev, lens, counts)
        wk, wv = llima_amd.cache_read(ek, ev, want, tokens=130)
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(new, want) and torch.equal(rk, wk) and torch.equal(rv, wv)
        assert same(kc.values, ek.values) and torch.equal(vc.scales, ev.scales)
        lens.copy_(want)


def test_overlaps_are_refused(gpu):
    import llima_amd
    lens = torch.zeros(2, dtype=torch.int32, device=gpu)
    buf = torch.zeros(2, 2, 40, 2, 64, dtype=torch.uint8, device=gpu)
    sc = torch.zeros(2, 2, 40, 2, device=gpu)
    kc, vc = llima_amd.Fp8Cache(buf[0].view(F8), sc[0]), llima_amd.Fp8Cache(buf[1].view(F8), sc[1])
    k = torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16, device=gpu)
    inside = buf.view(torch.bfloat16).view(2, 2, 40, 64)[:, :, :3].view(2, 2, 3, 64)[0]
    for call in (lambda: llima_amd.cache_write(k, k.clone(), kc, kc, lens),
                 lambda: llima_amd.cache_write(k, k.clone(), kc, llima_amd.Fp8Cache(buf[1].view(F8), sc[0]), lens),
                 lambda: llima_amd.cache_write(k, k, kc, llima_amd.Fp8Cache(buf[1, :1].expand(2, 40, 2, 64).view(F8), sc[1]), lens),
                 lambda: llima_amd.cache_write(k, k, kc, llima_amd.Fp8Cache(buf[1].view(F8), sc[1, :1].expand(2, 40, 2)), lens),
                 lambda: llima_amd.cache_write(inside[:, :, None, :].expand(2, 3, 2, 64), k, kc, vc, lens)):
        with pytest.raises(ValueError, match="overlap"):
            call()
    assert (buf == 0).all() and (sc == 0).all()
    assert llima_amd.cache_write(k, k, kc, kc, lens).tolist() == [3, 3]           # keys that are the values


def test_strides_and_places_past_32_bits(gpu):
    """Sequences 4.5 GB apart, and a page behind as many bytes."""
    import llima_amd
    L, Hkv, D = 2_200_000, 8, 256

    def cache():
        return llima_amd.Fp8Cache(torch.empty(2, L, Hkv, D, dtype=torch.uint8, device=gpu).view(F8), torch.empty(2, L, Hkv, device=gpu))
    kc, vc = cache(), cache()
    k, v = (torch.randn(2, 3, Hkv, D, device=gpu).bfloat16() for _ in range(2))
    lens = torch.tensor([0, L - 3], dtype=torch.int32, device=gpu)
    assert llima_amd.cache_write(k, v, kc, vc, lens).tolist() == [3, L]
    for c, x in ((kc, k), (vc, v)):
        q, s = quantize(x)
        assert same(c.values[0, :3], q[0]) and same(c.values[1, -3:], q[1])
        assert torch.equal(c.scales[0, :3], s[0]) and torch.equal(c.scales[1, -3:], s[1])
    page = 100
    kp, vp = (llima_amd.Fp8Cache(c.values.view(torch.uint8).view(2 * L // page, page, Hkv, D).view(F8), c.scales.view(2 * L // page, page, Hkv))
              for c in (kc, vc))
    table = torch.tensor([[5, 2 * L // page - 1]], dtype=torch.int32, device=gpu)
    kp.values.view(torch.uint8)[5].zero_()
    kp.scales[5].zero_()
    vp.values.view(torch.uint8)[5].zero_()
    vp.scales[5].zero_()
    n = torch.tensor([197], dtype=torch.int32, device=gpu)
    new = llima_amd.cache_write(k[:1], v[:1], kp, vp, n, block_table=table)
    assert new.tolist() == [200]
    rk, rv = llima_amd.cache_read(kp, vp, new, block_table=table)
    for r, c, x in ((rk, kp, k), (rv, vp, v)):
        q, s = quantize(x[0])
        assert same(c.values[-1, -3:], q) and torch.equal(r[0, 197:], (q.float() * s[..., None]).bfloat16()) and (r[0, :100] == 0).all()
