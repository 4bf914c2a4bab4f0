"""The LM head over an 8-bit weight against its definition in 64 bits.

Tolerance of a logit: the e4m3 products are exact in fp32, so a logit carries at most 128 roundings
within a block, two of the scales, and one per block's addition, each at most 2^-23 of the sum of
the terms' magnitudes (2^-24 where the matrix core rounds to nearest): (130 + NK) 2^-23 of it.
These bounds add up; roundings of either sign do not, so the whole of many logits is off by far
less (test_error_of_many_logits).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


def make(B, H, V, seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    NK = -(-H // 128)
    xq = torch.randn(B, H, generator=g, device=dev).mul_(60.0).clamp_(-448, 448).to(F8)
    wq = torch.randn(V, H, generator=g, device=dev).mul_(60.0).clamp_(-448, 448).to(F8)
    xs = torch.rand(B, NK, generator=g, device=dev).add_(0.5).mul_(0.01)
    ws = torch.rand(-(-V // 128), NK, generator=g, device=dev).add_(0.5).mul_(1e-3)
    return xq, xs, wq, ws


def definition(xq, xs, wq, ws):
    """(logits, bound) in 64 bits: each block's sum times its two scales, added up."""
    B, V = xq.shape[0], wq.shape[0]
    ref = torch.zeros(B, V, dtype=torch.float64, device=xq.device)
    mag = torch.zeros_like(ref)
    at = torch.arange(V, device=xq.device) // 128
    for kb in range(xs.shape[1]):
        x, w = (t[:, kb * 128:(kb + 1) * 128].double() for t in (xq, wq))
        s = xs[:, kb, None].double() * ws[at, kb].double()
        ref += (x @ w.t()) * s
        mag += (x.abs() @ w.abs().t()) * s.abs()
    return ref, (130 + xs.shape[1]) * 2.0 ** -23 * mag


def check_ids(ids, vals, ref, tol):
    """The id's logit is the row's greatest but for the tolerance, the value its own."""
    at = ref.gather(1, ids.long()[:, None])[:, 0]
    t = tol.amax(1)
    assert (at >= ref.amax(1) - 2 * t).all()
    assert ((vals.double() - at).abs() <= t).all()


CASES = [(1, 64, 1), (1, 128, 63), (2, 192, 64), (1, 4096, 1000), (31, 512, 200), (32, 576, 130),
         (33, 1024, 1024), (64, 640, 257), (65, 512, 4100), (96, 704, 129), (128, 4096, 300),
         (129, 256, 700), (200, 1088, 513), (300, 512, 300), (513, 2048, 1111), (7, 8192, 260), (5, 65536, 70)]


@pytest.mark.parametrize("B,H,V", CASES)
def test_logits_and_ids(gpu, B, H, V):
    import llima_amd
    xq, xs, wq, ws = make(B, H, V, B + H + V, gpu)
    ref, tol = definition(xq, xs, wq, ws)
    head, rows = llima_amd.Fp8LmHead(wq, ws), llima_amd.Fp8Rows(xq, xs)
    ids, vals, logits = llima_amd.lm_head_argmax(rows, head, return_logits=True, logit_dtype="f32")
    assert ((logits.double() - ref).abs() <= tol).all(), ((logits.double() - ref).abs() / tol).max()
    check_ids(ids, vals, ref, tol)
    assert torch.equal(vals, logits.amax(1)) and torch.equal(vals, logits.gather(1, ids.long()[:, None])[:, 0])
    # without logits, and as bf16 values: the same sums
    i2, v2 = llima_amd.lm_head_argmax(rows, head, logit_dtype="f32")
    assert torch.equal(i2, ids) and torch.equal(v2, vals)
    i3, v3, l3 = llima_amd.lm_head_argmax(rows, head, return_logits=True, logits_out="bf16")
    assert torch.equal(l3, logits.to(torch.bfloat16)) and torch.equal(v3, l3.amax(1).float())
    first = torch.where(l3 == l3.amax(1, keepdim=True), torch.arange(V, device=gpu), V).amin(1)
    assert torch.equal(i3.long(), first)


@pytest.mark.parametrize("B", [1, 60, 128, 200])
def test_error_of_many_logits(gpu, B):
    """Roundings of either sign: the root mean square over many logits is within 2^-24 sqrt(130 + NK) of the terms'
    magnitude each, also where one product of a block is 2^11 times the others and cancels in pairs."""
    import llima_amd
    H, V = 1024, 2000
    xq, xs, wq, ws = make(B, H, V, 21, gpu)
    for spread in (False, True):
        if spread:
            x = xq.float() / 2048.0
            x[:, ::64] *= 2048.0
            xq = x.to(F8)
        ref, tol = definition(xq, xs, wq, ws)
        _, _, logits = llima_amd.lm_head_argmax(llima_amd.Fp8Rows(xq, xs), llima_amd.Fp8LmHead(wq, ws),
                                                return_logits=True, logit_dtype="f32")
        mag = tol / ((130 + 8) * 2.0 ** -23)
        rel = ((logits.double() - ref) / mag).square().mean().sqrt()
        assert rel < 2.0 ** -24 * 138 ** 0.5


@pytest.mark.parametrize("B", [1, 40, 100, 140, 260])
def test_integers_with_ties_are_exact(gpu, B):
    """Small integers and scales of powers of two: every sum is exact, equal logits tie, the lowest id wins."""
    import llima_amd
    H, V = 320, 777
    g = torch.Generator(device=gpu).manual_seed(B)
    xq = torch.randint(-2, 3, (B, H), generator=g, device=gpu).float().to(F8)
    wq = torch.randint(-1, 2, (V, H), generator=g, device=gpu).float().to(F8)
    wq[500:] = wq[:277]                                      # each of these logits twice, up to the scales
    xs = torch.full((B, 3), 0.5, device=gpu)
    ws = torch.full((7, 3), 2.0, device=gpu)
    ref, _ = definition(xq, xs, wq, ws)
    ids, vals, logits = llima_amd.lm_head_argmax(llima_amd.Fp8Rows(xq, xs), llima_amd.Fp8LmHead(wq, ws),
                                                 return_logits=True, logit_dtype="f32")
    assert torch.equal(logits.double(), ref)
    first = torch.where(ref == ref.amax(1, keepdim=True), torch.arange(V, device=gpu), V).amin(1)
    assert torch.equal(ids.long(), first) and torch.equal(vals.double(), ref.amax(1))


def test_extreme_scales_and_subnormal_values(gpu):
    """The smallest e4m3 values (2^-9), the largest, and scales far apart in one row."""
    import llima_amd
    H, V, B = 256, 130, 3
    xq = torch.full((B, H), 2.0 ** -9, device=gpu).to(F8)
    wq = torch.full((V, H), 448.0, device=gpu).to(F8)
    xs = torch.tensor([[2.0 ** 40, 2.0 ** -40], [1.0, 1.0], [2.0 ** -60, 2.0 ** -60]], device=gpu)
    ws = torch.tensor([[2.0 ** -20, 2.0 ** 20], [2.0 ** -50, 2.0 ** -50]], device=gpu)
    ref, tol = definition(xq, xs, wq, ws)
    _, _, logits = llima_amd.lm_head_argmax(llima_amd.Fp8Rows(xq, xs), llima_amd.Fp8LmHead(wq, ws),
                                            return_logits=True, logit_dtype="f32")
    assert ((logits.double() - ref).abs() <= tol).all() and (ref > 0).all() and (logits > 0).all()


@pytest.mark.parametrize("B", [3, 70, 150])
def test_nan_and_infinite_scales(gpu, B):
    """A NaN value or scale spoils its logits alone; they never win, and a row of NaN gives id 0 and NaN."""
    import llima_amd
    H, V = 256, 300
    xq, xs, wq, ws = make(B, H, V, 5, gpu)
    q = wq.view(torch.uint8)
    q[10, 3] = 0x7F                                          # NaN: logit 10 of every row
    ws[1, 0] = float("nan")                                  # ids 128 .. 255
    xs[1, 1] = float("nan")                                  # all of row 1
    xs[2, 0] = float("inf")                                  # row 2: infinite or NaN
    ids, vals, logits = llima_amd.lm_head_argmax(llima_amd.Fp8Rows(xq, xs), llima_amd.Fp8LmHead(wq, ws),
                                                 return_logits=True, logit_dtype="f32")
    ref, tol = definition(xq, xs, wq, ws)
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(logits), nan)
    assert nan[0, 10] and nan[0, 128:256].all() and nan[1].all() and not nan[0, 11:128].any()
    assert ids[1] == 0 and torch.isnan(vals[1])
    fin = torch.isfinite(ref)
    assert ((logits.double() - ref).abs()[fin] <= tol[fin]).all()
    r0 = torch.where(nan[0], -float("inf"), ref[0])
    assert r0[ids[0].long()] >= r0.max() - 2 * tol[0][fin[0]].max()
    assert torch.isinf(vals[2]) and vals[2] > 0


@pytest.mark.parametrize("B,H,V,cap", [(1, 512, 1000, 30.0), (20, 256, 333, 0.0), (130, 320, 900, 5.0)])
def test_score_and_verification_are_those_of_the_logits(gpu, B, H, V, cap):
    import llima_amd
    xq, xs, wq, ws = make(B, H, V, 11, gpu)
    head, rows = llima_amd.Fp8LmHead(wq, ws), llima_amd.Fp8Rows(xq, xs)
    for ld in ("f32", "bf16"):
        ids, vals, logits = llima_amd.lm_head_argmax(rows, head, softcap=cap, return_logits=True, logit_dtype=ld)
        tg = torch.where(torch.arange(B, device=gpu) % 2 == 0, ids, (ids + 1) % V).to(torch.int32)
        lp, greedy = llima_amd.lm_head_score(rows, head, tg, softcap=cap, logit_dtype=ld)
        elp, egr = llima_amd.score_logits(logits, tg)
        # fp32 exponentials (2^-22 relative each, their argument's rounding 2^-24 of the logits' range)
        assert ((lp - elp).abs() <= 1e-5).all() and torch.equal(greedy, egr)
        if B > 1:
            D = 4 if B % 5 == 0 else 1
            n = B // (D + 1)
            sub = llima_amd.Fp8Rows(xq[:n * (D + 1)], xs[:n * (D + 1)])
            i2, _, l2 = llima_amd.lm_head_argmax(sub, head, softcap=cap, return_logits=True, logit_dtype=ld)
            drafts = i2.view(n, D + 1)[:, :D].clone()
            drafts[n // 2:, D // 2] += 1
            acc, em = llima_amd.lm_head_verify_greedy(sub, head, drafts, softcap=cap, logit_dtype=ld)
            eacc, eem = llima_amd.verify_greedy(l2.view(n, D + 1, V), drafts)
            assert torch.equal(acc, eacc) and torch.equal(em, eem)
            ret = torch.tensor([[0, 1, 3, -1], [0, 2, 4, 5], [0, 1, -1, -1]], dtype=torch.int32)
            tok = ids.cpu()
            cand = torch.stack([tok.new_tensor([9, int(tok[0]), int(tok[1]), -1]),
                                tok.new_tensor([9, int(tok[0]), int(tok[2]), int(tok[4])]),
                                tok.new_tensor([9, int(tok[0]), -1, -1])])
            assert (llima_amd.lm_head_verify_tree(rows, head, ret, cand, softcap=cap, logit_dtype=ld)
                    == llima_amd.verify_tree(logits, ret, cand))


def test_bf16_hidden_goes_through_quantize_rows(gpu):
    import llima_amd
    g = torch.Generator(device=gpu).manual_seed(3)
    w = torch.randn(500, 448, generator=g, device=gpu).to(torch.bfloat16)
    x = torch.randn(6, 448, generator=g, device=gpu).to(torch.bfloat16)
    head = llima_amd.lm_head_quantize(w)
    a = llima_amd.lm_head_argmax(x, head, return_logits=True)
    b = llima_amd.lm_head_argmax(llima_amd.quantize_rows(x), head, return_logits=True)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    one = llima_amd.lm_head_argmax(x[0], head)
    assert one[0].shape == (1,) and one[0][0] == a[0][0]
    lp, gr = llima_amd.lm_head_score(x[0], head, int(a[0][0]))
    assert gr and lp < 0
    with pytest.raises(RuntimeError):
        llima_amd.lm_head_score(x, head, torch.tensor([0, 1, 2, 3, 4, 500]))
    # 8 bits are near the bf16 head: two roundings of 2^-4 relative each, independent over 448 terms
    full = x.double() @ w.double().t()
    err = (a[2].double() - full).norm() / full.norm()
    assert err < 2 * 2.0 ** -4
    # strided rows, an unaligned weight, no rows
    big = torch.randn(9, 1000, generator=g, device=gpu).to(torch.bfloat16)
    v = big[::2, 7:455]
    assert torch.equal(llima_amd.lm_head_argmax(v, head)[0], llima_amd.lm_head_argmax(v.contiguous().clone(), head)[0])
    flat = torch.empty(500 * 448 + 3, dtype=torch.uint8, device=gpu)
    off = flat[3:].view(500, 448).view(F8)
    off.view(torch.uint8).copy_(head.values.view(torch.uint8))
    again = llima_amd.lm_head_argmax(x, llima_amd.Fp8LmHead(off, head.scales), return_logits=True)
    assert torch.equal(again[2], a[2])
    assert llima_amd.lm_head_argmax(x[:0], head)[0].shape == (0,)


def test_weight_past_32_bits(gpu):
    """A weight of more than 2^32 bytes: its first and last rows are right."""
    import llima_amd
    H, V, B = 16384, 262400, 130
    g = torch.Generator(device=gpu).manual_seed(2)
    wq = torch.randint(0, 127, (V, H), generator=g, device=gpu, dtype=torch.uint8)
    wq[:, ::2] |= 0x80
    wq = wq.view(F8)
    xq = torch.randn(B, H, generator=g, device=gpu).to(F8)
    xs = torch.full((B, 128), 2.0 ** -8, device=gpu)
    ws = torch.full((2050, 128), 2.0 ** -8, device=gpu)
    _, _, logits = llima_amd.lm_head_argmax(llima_amd.Fp8Rows(xq, xs), llima_amd.Fp8LmHead(wq, ws),
                                            return_logits=True, logit_dtype="f32")
    for lo in (0, V - 384):
        ref, tol = definition(xq, xs, wq[lo:lo + 384], ws[:3])
        assert ((logits[:, lo:lo + 384].double() - ref).abs() <= tol).all()


def test_two_graphs_on_one_stream_have_their_own_scratch(gpu):
    """Two captured heads replayed at once on two streams, several times, with eager work between."""
    import llima_amd
    H, V = 512, 20000
    a, b = make(4, H, V, 1, gpu), make(90, H, V, 2, gpu)
    eager, graphs = [], []
    for xq, xs, wq, ws in (a, b):
        rows, head = llima_amd.Fp8Rows(xq, xs), llima_amd.Fp8LmHead(wq, ws)
        eager.append([t.clone() for t in llima_amd.lm_head_argmax(rows, head, logit_dtype="f32")])
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = llima_amd.lm_head_argmax(rows, head, logit_dtype="f32")
        graphs.append((gr, out, rows, head))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for gr, out, _, _ in graphs:
            out[0].zero_()
            out[1].zero_()
        torch.cuda.synchronize()
        for s, (gr, _, _, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for (gr, out, _, _), e in zip(graphs, eager):
            assert torch.equal(out[0], e[0]) and torch.equal(out[1], e[1])
        llima_amd.lm_head_argmax(llima_amd.Fp8Rows(*a[:2]), llima_amd.Fp8LmHead(*a[2:]))


@pytest.mark.parametrize("B", [1, 32, 33, 64, 65, 128, 140, 200])
@pytest.mark.parametrize("H", [64, 320, 512, 1984, 4096])
def test_equal_rows_have_equal_logits(gpu, B, H):
    """Equal weight rows under equal scales, 256 rows apart over the whole vocabulary: the same bits wherever a row lies, so
    the lowest id wins; a part of the vocabulary gives the whole's logits, and equal hidden rows of a batch equal ones."""
    import llima_amd
    T = 36
    xq, xs, wq, ws = make(B, H, 256, B + H, gpu)
    xq.view(torch.uint8)[-1], xs[-1] = xq.view(torch.uint8)[0], xs[0]
    rows = llima_amd.Fp8Rows(xq, xs)
    whole = llima_amd.Fp8LmHead(wq.view(torch.uint8).repeat(T, 1).view(F8), ws.repeat(T, 1))
    for ld in ("f32", "bf16"):
        ids, vals, logits = llima_amd.lm_head_argmax(rows, whole, return_logits=True, logit_dtype=ld)
        first = logits[:, :256]
        assert torch.equal(logits.view(B, T, 256), first[:, None].expand(B, T, 256))
        assert torch.equal(logits[0], logits[-1])
        lowest = torch.where(first == first.amax(1, keepdim=True), torch.arange(256, device=gpu), 256).amin(1)
        assert torch.equal(ids.long(), lowest)
        part = llima_amd.lm_head_argmax(rows, llima_amd.Fp8LmHead(wq, ws), return_logits=True, logit_dtype=ld)
        assert torch.equal(part[2], first) and torch.equal(part[0], ids) and torch.equal(part[1], vals)
        _, greedy = llima_amd.lm_head_score(rows, whole, ids, logit_dtype=ld)
        assert greedy.all()
        _, greedy = llima_amd.lm_head_score(rows, whole, ids + 256 * (T - 1), logit_dtype=ld)
        assert not greedy.any()
