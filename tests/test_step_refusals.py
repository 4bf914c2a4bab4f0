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
    assert l.llima_lm_head_argmax_fp8_workspace_bytes(3, 65) >= 3 * 2 * 8


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
