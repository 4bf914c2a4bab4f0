"""What the norm, the 8-bit head and the attention over a cache refuse, before any launch (no GPU)."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(16)
ODD = ctypes.c_void_p(24)
N = None
BIG = 1 << 30


def L():
    from llima_amd._lib import lib
    return lib()


def norm(x=P, res=P, w=P, dt=1, B=2, H=64, xs=64, rs=64, eps=1e-6, off=0.0, out=P, sc=N, ro=P):
    return L().llima_add_rms_norm(x, res, w, dt, B, H, xs, rs, eps, off, out, sc, ro, None)


@pytest.mark.parametrize("bad", [dict(dt=3), dict(dt=-1), dict(H=0), dict(H=12), dict(H=65544), dict(B=-1), dict(x=N),
                                 dict(x=ODD), dict(xs=60), dict(xs=68), dict(xs=56), dict(res=ODD), dict(rs=56),
                                 dict(rs=65), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
                                 dict(off=float("nan")), dict(off=float("inf")), dict(w=N), dict(w=ODD), dict(out=N),
                                 dict(out=ODD), dict(ro=ODD), dict(res=N)])
def test_norm_refuses(bad):
    assert norm(**bad) == -1                                 # (res=N: a residual output without a residual)


def test_no_rows_launch_nothing():
    assert norm(B=0) == 0 and norm(B=0, x=N, out=N, w=N, res=N, ro=N) == 0
    assert L().llima_quantize_rows(N, 1, 0, 64, 64, N, N, None) == 0
    assert L().llima_lm_head_argmax_fp8(N, N, P, P, 0, 64, 100, 0.0, 1, N, N, N, N, 0, None) == 0


def test_quantize_refuses():
    q = L().llima_quantize_rows
    assert q(P, 1, 2, 64, 64, N, P, None) == -1 and q(P, 1, 2, 64, 64, P, N, None) == -1
    assert q(P, 1, 2, 60, 64, P, P, None) == -1 and q(P, 1, 2, 64, 60, P, P, None) == -1
    assert q(ODD, 1, 2, 64, 64, P, P, None) == -1 and q(P, 4, 2, 64, 64, P, P, None) == -1
    assert q(P, 0, 2, 64, 66, P, P, None) == -1              # fp32 rows 264 bytes apart
    w = L().llima_lm_head_quantize
    assert w(P, 0, 64, P, P, None) == -1 and w(P, 10, 96, P, P, None) == -1 and w(P, 10, 65600, P, P, None) == -1
    assert w(N, 10, 64, P, P, None) == -1 and w(P, 10, 64, ODD, P, None) == -1 and w(P, 10, 64, P, N, None) == -1


def head(x=P, xs=P, w=P, ws=P, B=2, H=64, V=100, cap=0.0, ld=1, ids=P, vals=N, logits=N, wsp=P, n=BIG):
    return L().llima_lm_head_argmax_fp8(x, xs, w, ws, B, H, V, cap, ld, ids, vals, logits, wsp, n, None)


@pytest.mark.parametrize("bad,status", [
    (dict(x=N), -1), (dict(xs=N), -1), (dict(w=N), -1), (dict(ws=N), -1), (dict(B=-1), -1), (dict(H=0), -1),
    (dict(H=96), -1), (dict(H=65600), -1), (dict(V=0), -1), (dict(cap=float("nan")), -1), (dict(cap=float("inf")), -1),
    (dict(ld=2), -1), (dict(ld=0x100), -1), (dict(ids=N), -1), (dict(x=ODD), -1), (dict(w=ODD), -1),
    (dict(wsp=N), -4), (dict(n=8), -4)])
def test_fp8_head_refuses(bad, status):
    assert head(**bad) == status


def test_fp8_score_and_verification_refuse():
    l = L()
    for f in (l.llima_lm_head_score_fp8,):
        assert f(P, P, P, P, 2, 64, 100, 0.0, 0x101, P, P, P, P, BIG, None) == -1
        assert f(P, P, P, P, 2, 64, 100, 0.0, 1, N, P, P, P, BIG, None) == -1
        assert f(P, P, P, P, 2, 64, 100, 0.0, 1, P, P, P, P, 0, None) == -4
    g = l.llima_lm_head_verify_greedy_fp8
    assert g(P, P, P, P, 2, -1, 64, 100, 0.0, 1, P, P, P, P, BIG, None) == -1
    assert g(P, P, P, P, 2, 3, 64, 100, 0.0, 1, N, P, P, P, BIG, None) == -1
    assert g(P, P, P, P, 1 << 20, 1 << 12, 64, 100, 0.0, 1, P, P, P, P, BIG, None) == -1   # rows past 2^31
    assert g(P, P, P, P, 2, 3, 64, 100, 0.0, 1, P, P, P, P, 0, None) == -4
    t = l.llima_lm_head_verify_tree_fp8
    assert t(P, P, P, P, 0, 64, 100, 0.0, 1, P, P, 2, 3, P, P, BIG, None) == -1
    assert t(P, P, P, P, 4, 64, 100, 0.0, 1, P, P, 0, 3, P, P, BIG, None) == -1
    assert t(P, P, P, P, 4, 64, 100, 0.0, 1, P, P, 2, 3, P, P, 0, None) == -4
    assert l.llima_lm_head_argmax_fp8_workspace_bytes(0, 10) == 0
    assert l.llima_lm_head_argmax_fp8_workspace_bytes(3, 65) >= 3 * 8


def test_python_refuses_on_host_tensors_and_shapes():
    import llima_amd
    F8 = torch.float8_e4m3fn
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.bfloat16)
    for call in (lambda: llima_amd.add_rms_norm(x, w),                                # not on the GPU
                 lambda: llima_amd.add_rms_norm(x, w[:32]), lambda: llima_amd.add_rms_norm(x, w.float()),
                 lambda: llima_amd.add_rms_norm(x, w, x[:1]), lambda: llima_amd.add_rms_norm(x, w, x.float()),
                 lambda: llima_amd.add_rms_norm(x, w, out="int8"),
                 lambda: llima_amd.add_rms_norm(x.double(), w.double()),
                 lambda: llima_amd.quantize_rows(x), lambda: llima_amd.quantize_rows(torch.zeros(())),
                 lambda: llima_amd.quantize_rows(x[:, :60]), lambda: llima_amd.lm_head_quantize(x),
                 lambda: llima_amd.lm_head_quantize(x.float()),
                 lambda: llima_amd.Fp8Rows(x, torch.zeros(2, 1)),
                 lambda: llima_amd.Fp8Rows(x.to(F8), torch.zeros(2, 2)),
                 lambda: llima_amd.Fp8Rows(x.to(F8), torch.zeros(2, 1, dtype=torch.float64)),
                 lambda: llima_amd.Fp8LmHead(x.to(F8), torch.zeros(2, 1))):
        with pytest.raises(ValueError):
            call()


def attention_args(**kw):
    from llima_amd import _lib
    a = _lib.TreeAttentionArgsC()
    for n in ("q", "k", "v", "k_cache", "v_cache", "out", "cache_lens", "mask", "block_table"):
        setattr(a, n, 4096)
    for n in ("q_strides", "k_strides", "v_strides", "out_strides", "k_cache_strides", "v_cache_strides"):
        getattr(a, n)[:] = (4096, 512, 128)
    a.mask_strides[:] = (16, 4)
    a.table_stride = 8
    for n, x in dict(dtype=1, mask_dtype=0, B=2, N=4, Hq=8, Hkv=4, D=128, page_size=16, pages=20, max_blocks=8,
                     scale=0.1).items():
        setattr(a, n, x)
    for n, x in kw.items():
        if isinstance(x, tuple):
            getattr(a, n)[:] = x
        else:
            setattr(a, n, x)
    return a


@pytest.mark.parametrize("bad", [
    dict(dtype=0), dict(dtype=3), dict(B=-1), dict(N=0), dict(N=1025), dict(Hq=0), dict(Hq=9), dict(Hkv=0),
    dict(Hq=1028), dict(D=96), dict(D=0), dict(page_size=0), dict(pages=-1), dict(max_blocks=-1),
    dict(block_table=None), dict(block_table=None, max_blocks=1, pages=1), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(mask_dtype=2), dict(q_strides=(4096, 512, 129)), dict(k_strides=(-8, 512, 128)),
    dict(out_strides=(4, 512, 128)), dict(k_cache_strides=(4096, 511, 128)), dict(mask_strides=(-1, 4)),
    dict(table_stride=-1), dict(q=None), dict(q=4104), dict(k=None), dict(v=4100), dict(out=None), dict(cache_lens=None),
    dict(k_cache=None), dict(v_cache=4097), dict(page_size=1 << 28, max_blocks=4), dict(B=1 << 20, N=1024)])
def test_attention_refuses(bad):
    a = attention_args(**bad)
    assert L().llima_tree_attention(ctypes.byref(a), P, BIG << 10, None) == -1


def test_attention_workspace_and_empty_batch():
    l = L()
    a = attention_args()
    need = l.llima_tree_attention_workspace_bytes(2, 4, 8, 4, 128)
    assert need > 0 and l.llima_tree_attention_workspace_bytes(2, 4, 8, 4, 96) == 0
    assert l.llima_tree_attention(ctypes.byref(a), N, need, None) == -4
    assert l.llima_tree_attention(ctypes.byref(a), P, need - 1, None) == -4
    assert l.llima_tree_attention(ctypes.byref(a), ctypes.c_void_p(24), need, None) == -1
    assert l.llima_tree_attention(None, P, need, None) == -1
    a = attention_args(B=0, q=None, k=None, v=None, out=None, cache_lens=None)
    assert l.llima_tree_attention(ctypes.byref(a), N, 0, None) == 0


def commit_args(**kw):
    from llima_amd import _lib
    a = _lib.TreeCommitArgsC()
    for n in ("k", "v", "k_cache", "v_cache", "nodes", "counts", "cache_lens", "block_table", "new_lens"):
        setattr(a, n, 4096)
    for n in ("k_strides", "v_strides", "k_cache_strides", "v_cache_strides"):
        getattr(a, n)[:] = (65536, 4096, 512, 128)
    a.nodes_stride, a.table_stride = 3, 8
    for n, x in dict(layers=2, B=2, N=4, L=3, Hkv=4, D=128, page_size=16, pages=20, max_blocks=8).items():
        setattr(a, n, x)
    for n, x in kw.items():
        if isinstance(x, tuple):
            getattr(a, n)[:] = x
        else:
            setattr(a, n, x)
    return a


@pytest.mark.parametrize("bad", [
    dict(layers=0), dict(layers=65536), dict(B=-1), dict(N=0), dict(L=0), dict(Hkv=0), dict(D=0), dict(D=12), dict(D=131072),
    dict(page_size=0), dict(pages=-1), dict(max_blocks=-1), dict(block_table=None), dict(k=None), dict(v=None),
    dict(k_cache=None), dict(v_cache=4104), dict(k=4104), dict(nodes=None), dict(counts=None), dict(cache_lens=None),
    dict(new_lens=None), dict(k_strides=(65536, 4096, 512, 4)), dict(v_cache_strides=(65536, -8, 512, 128)),
    dict(nodes_stride=-1), dict(table_stride=-1), dict(page_size=1 << 30, max_blocks=2), dict(B=1 << 20, L=1 << 12)])
def test_commit_refuses(bad):
    assert L().llima_tree_commit(ctypes.byref(commit_args(**bad)), None) == -1
    assert L().llima_tree_commit(None, None) == -1


def test_commit_of_no_sequences():
    a = commit_args(B=0, k=None, v=None, nodes=None, counts=None, cache_lens=None, new_lens=None)
    assert L().llima_tree_commit(ctypes.byref(a), None) == 0


def test_python_attention_refuses():
    import llima_amd
    bf = torch.bfloat16
    q, k = torch.zeros(2, 3, 8, 64, dtype=bf), torch.zeros(2, 3, 4, 64, dtype=bf)
    c, n = torch.zeros(2, 10, 4, 64, dtype=bf), torch.zeros(2, dtype=torch.int32)
    f, g = llima_amd.tree_attention, llima_amd.tree_commit
    p, m = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    for call in (lambda: f(q, k, k, c, c, n), lambda: f(q[0], k, k, c, c, n), lambda: f(q[:1], k, k, c, c, n),
                 lambda: f(q, k, k[:, :2], c, c, n), lambda: f(q.float(), k, k, c, c, n), lambda: f(q, k.half(), k, c, c, n),
                 lambda: f(q[..., :32], k[..., :32], k[..., :32], c, c, n), lambda: f(q[:, :, :6], k, k, c, c, n),
                 lambda: f(q[:, :0], k[:, :0], k[:, :0], c, c, n), lambda: g(k, k, p, m, c, c, n),
                 lambda: g(k, k[:, :2], p, m, c, c, n), lambda: g(k, k, p[:, :0], m, c, c, n),
                 lambda: g(k, k, p.long(), m, c, c, n), lambda: g(k[None], k[None], p, m, c, c, n),
                 lambda: g(k.float(), k.float(), p, m, c, c, n), lambda: g(k[0], k[0], p, m, c, c, n),
                 lambda: g(k[None].expand(2, 2, 3, 4, 64), k[None].expand(2, 2, 3, 4, 64), p, m, c[None], c[None], n)):
        with pytest.raises(ValueError):
            call()


def test_packed_arguments_are_the_structures():
    """The byte layouts that the Python calls pack are those of the C structures, field by field."""
    from llima_amd import _lib
    for fmt, cls in ((_lib.TREE_ATTENTION_ARGS, _lib.TreeAttentionArgsC), (_lib.TREE_COMMIT_ARGS, _lib.TreeCommitArgsC)):
        assert fmt.size == ctypes.sizeof(cls)
        n = sum(getattr(t, "_length_", 1) for _, t in cls._fields_)
        a = cls.from_buffer_copy(fmt.pack(*range(1, n + 1)))
        got = []
        for name, t in cls._fields_:
            v = getattr(a, name)
            got += list(v) if hasattr(t, "_length_") else [v]
        assert got == list(range(1, n + 1))


def test_batches_past_one_launch_are_refused():
    a = attention_args(B=1 << 19, N=16)                      # 2^26 rows
    assert L().llima_tree_attention(ctypes.byref(a), P, BIG << 20, None) == -1
    assert L().llima_tree_attention_workspace_bytes(1 << 19, 16, 8, 4, 128) == 0
    assert L().llima_tree_attention_workspace_bytes((1 << 19) - 1, 16, 8, 4, 128) > 0
    assert L().llima_tree_commit(ctypes.byref(commit_args(B=1 << 20, L=1 << 4)), None) == -1


def test_8_bit_rows_need_an_8_bit_weight():
    import llima_amd
    x = llima_amd.Fp8Rows.__new__(llima_amd.Fp8Rows)          # (the constructor refuses host tensors)
    x.values, x.scales = torch.zeros(2, 64).to(torch.float8_e4m3fn), torch.zeros(2, 1)
    h = llima_amd.Fp8LmHead.__new__(llima_amd.Fp8LmHead)
    h.values, h.scales, h.V, h.H = torch.zeros(100, 64).to(torch.float8_e4m3fn), torch.zeros(1, 1), 100, 64
    w, i = torch.zeros(100, 64, dtype=torch.bfloat16), torch.zeros(2, 2, dtype=torch.int32)
    for call in (lambda: llima_amd.lm_head_argmax(x, w), lambda: llima_amd.lm_head_score(x, w, i[0]),
                 lambda: llima_amd.lm_head_verify_greedy(x, w, i[:1, :1]),
                 lambda: llima_amd.lm_head_verify_tree(x, w, i, i), lambda: llima_amd.lm_head_pack(h)):
        with pytest.raises(ValueError, match="bf16"):
            call()


def host_head():
    """An 8-bit head on the host (the constructor refuses host tensors): H 64, V 100."""
    import llima_amd
    h = llima_amd.Fp8LmHead.__new__(llima_amd.Fp8LmHead)
    h.values, h.scales, h.V, h.H = torch.zeros(100, 64).to(torch.float8_e4m3fn), torch.zeros(1, 1), 100, 64
    return h


@pytest.mark.parametrize("shape", [(2, 3, 64), (2, 1, 64), (1, 1, 2, 64), ()])
def test_scoring_over_an_8_bit_head_takes_rows(shape):
    """Two targets for [2, 3, H]: one target per leading index is not one per row, and the rows past them would be scored
    against what lies behind the targets."""
    import llima_amd
    with pytest.raises(ValueError, match="hidden must be"):
        llima_amd.lm_head_score(torch.zeros(shape, dtype=torch.bfloat16), host_head(), torch.tensor([1, 2]))


@pytest.mark.parametrize("shape", [(2, 3, 64), (1, 1, 64), ()])
def test_argmax_over_an_8_bit_head_takes_rows(shape):
    """As over a bf16 weight: rows or one row, not rows of rows flattened."""
    import llima_amd
    x = torch.zeros(shape, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="hidden must be"):
        llima_amd.lm_head_argmax(x, host_head())
    if x.dim():
        with pytest.raises(ValueError):
            llima_amd.lm_head_argmax(x, torch.zeros(100, 64, dtype=torch.bfloat16))


def test_attention_workspace_is_bounded_by_the_shares():
    """A share of the keys leaves the parts of two sequences at most, its first and its last: the workspace stops growing with
    the batch (8 key heads of 264 rows: two row groups, 16 shares)."""
    l = L()
    size = [l.llima_tree_attention_workspace_bytes(B, 33, 64, 8, 128) for B in (1, 8, 16, 32, 64, 1024, 4096)]
    row = 33 * 64 * (128 + 2) * 4
    assert size[0] < size[1] <= 2 * size[0]
    assert size[3:] == [size[3]] * 4 and size[3] <= 64 * row + 256


def offsets(t):
    at = torch.zeros(t.shape, dtype=torch.int64) + t.storage_offset()
    for d, (n, s) in enumerate(zip(t.shape, t.stride())):
        at += (torch.arange(n) * s).view([-1 if i == d else 1 for i in range(t.dim())])
    return set(at.flatten().tolist())


def test_drafts_beside_the_cache_in_one_storage_are_apart():
    """Drafted tokens behind or between the cached ones of the same storage, without a value in common, are not refused."""
    from llima_amd.attention import _shared
    bf = torch.bfloat16
    buf = torch.empty(3, 2, 20 + 4, 2, 8, dtype=bf)           # [layers, B, tokens + drafts, heads, D]
    assert not _shared(buf[:, :, 20:], buf[:, :, :20])
    assert _shared(buf[:, :, 19:23], buf[:, :, :20]) and _shared(buf[1:2, :, 5:9], buf[:, :, :20])
    assert not _shared(buf[:, :, 20:].transpose(2, 3), buf[:, :, :20]) and not _shared(buf[:1], buf[1:])
    both = torch.empty(2, 24, 2, 2, 8, dtype=bf)              # K and V side by side per token
    for k, c in ((0, 1), (1, 0)):
        assert not _shared(both[:, 20:, k], both[:, :20, c]) and not _shared(both[:, 20:, k], both[:, :20, k])
        assert not _shared(both[:, :, k], both[:, :, c]) and _shared(both[:, :, k], both[:, :, k])
    heads = torch.empty(2, 6, 30, 8, dtype=bf)                # K's heads, then V's, tokens inside
    assert not _shared(heads[:, :3].transpose(1, 2), heads[:, 3:].transpose(1, 2))
    assert _shared(heads[:, :3].transpose(1, 2), heads[:, 2:5].transpose(1, 2))
    assert not _shared(torch.empty(2, 3), torch.empty(2, 3)) and not _shared(buf[:, :0], buf)


def test_whether_two_views_share_values_is_never_denied_wrongly():
    from llima_amd.attention import _shared
    g = torch.Generator().manual_seed(3)
    base = torch.empty(4000, dtype=torch.bfloat16)
    r = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))
    apart = 0
    for _ in range(3000):
        views = []
        for _ in range(2):
            shape = [r(1, 5) for _ in range(3)]
            views.append(base.as_strided(shape, [r(0, 60), r(0, 40), r(0, 12)], r(0, 400)))
        common = bool(offsets(views[0]) & offsets(views[1]))
        assert _shared(*views) or not common, views
        apart += not _shared(*views)
    assert apart > 100


def test_commit_refuses_caches_in_one_memory(monkeypatch):
    """Two writes to one place in no order: K's and V's cache the same, or overlapping, or one that repeats its memory."""
    import llima_amd
    from llima_amd import attention
    monkeypatch.setattr(attention, "_on_gpu", lambda *t: None)
    launched = []
    monkeypatch.setattr(attention, "lib", lambda: launched.append(1) or (_ for _ in ()).throw(AssertionError("launched")))
    bf = torch.bfloat16
    k, v = torch.zeros(2, 3, 4, 64, dtype=bf), torch.zeros(2, 3, 4, 64, dtype=bf)
    c, o = torch.zeros(2, 10, 4, 64, dtype=bf), torch.zeros(2, 10, 4, 64, dtype=bf)
    wide = torch.zeros(2, 15, 4, 64, dtype=bf)
    p, m, n = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    one = torch.zeros(1, 10, 4, 64, dtype=bf)
    for kc, vc in ((c, c), (wide[:, :10], wide[:, 5:]), (one.expand(2, 10, 4, 64), o), (c, one.expand(2, 10, 4, 64)),
                   (c, o[:, :, :1].expand(2, 10, 4, 64)), (o.view(-1).as_strided((2, 10, 4, 64), (2048, 128, 64, 1)), c)):
        with pytest.raises(ValueError, match="overlap"):
            llima_amd.tree_commit(k, v, p, m, kc, vc, n)
    layers = torch.zeros(1, 2, 10, 4, 64, dtype=bf).expand(3, 2, 10, 4, 64)
    k3 = torch.zeros(3, 2, 3, 4, 64, dtype=bf)
    with pytest.raises(ValueError, match="overlap"):
        llima_amd.tree_commit(k3, k3, p, m, layers, torch.zeros(3, 2, 10, 4, 64, dtype=bf), n)
    assert not launched
    both = torch.zeros(2, 10, 4, 128, dtype=bf)               # K and V of a head side by side, head-major caches, tied K and V
    major = torch.zeros(2, 2, 4, 10, 64, dtype=bf).transpose(2, 3)
    odd = torch.zeros(2, 3, 4, 65, dtype=bf)[..., 1:]         # (copied to aligned rows)
    for kc, vc, w, x in ((both[..., :64], both[..., 64:], k, v), (major[0], major[1], k, v), (major[:, 0], major[:, 1], k, v),
                         (c, c, k, k), (c, c, odd, odd)):
        with pytest.raises((AssertionError, RuntimeError)):   # (past the checks: no GPU here)
            llima_amd.tree_commit(w, x, p, m, kc, vc, n)


def test_more_rows_than_a_count_holds_are_refused(monkeypatch):
    """2^32 + 5 rows of 8 (69 GB): the count given to the library has 32 bits, and 5 rows would be computed."""
    import llima_amd
    from llima_amd import sampler
    monkeypatch.setattr(sampler, "_on_gpu", lambda *t: None)
    counts = []

    class Library:
        def __getattr__(self, name):
            return lambda *a: counts.append(ctypes.c_int32(a[2 if "quantize" in name else 4]).value) or 0
    monkeypatch.setattr(sampler, "lib", Library)
    monkeypatch.setattr(sampler, "_on", lambda dev: __import__("contextlib").nullcontext())
    monkeypatch.setattr(sampler, "_stream", lambda dev: 0)
    for rows in ((1 << 32) + 5, 1 << 31):
        x = torch.empty(rows, 8, dtype=torch.bfloat16, device="meta")
        w = torch.empty(8, dtype=torch.bfloat16, device="meta")
        for call in (lambda: llima_amd.quantize_rows(x), lambda: llima_amd.add_rms_norm(x, w),
                     lambda: llima_amd.add_rms_norm(x, w, x, out="fp8")):
            with pytest.raises(ValueError, match="rows"):
                call()
    assert not counts
    llima_amd.quantize_rows(torch.empty((1 << 31) - 1, 8, dtype=torch.bfloat16, device="meta"))
    assert counts == [(1 << 31) - 1]
