"""What the operators over an 8-bit cache and the norm around a block refuse, before any launch (no GPU)."""
import ctypes

import pytest
import torch

from .test_step_refusals import BIG, L, N, P, attention_args


def fill(a, bad, **base):
    for n, x in {**base, **bad}.items():
        if isinstance(x, tuple):
            getattr(a, n)[:] = x
        else:
            setattr(a, n, x)
    return a


def attention8(**bad):
    from llima_amd import _lib
    x = _lib.TreeAttentionFp8ArgsC()
    own = {n: bad.pop(n) for n in list(bad) if "scale" in n and n != "scale"}
    x.a = attention_args(**bad)
    return fill(x, own, k_scales=4096, v_scales=4096, k_scale_strides=(128, 8, 1), v_scale_strides=(128, 1, 16))


@pytest.mark.parametrize("bad", [
    dict(dtype=0), dict(dtype=3), dict(B=-1), dict(N=0), dict(N=1025), dict(Hq=9), dict(Hkv=0), dict(D=96), dict(D=0),
    dict(page_size=0), dict(pages=-1), dict(max_blocks=-1), dict(block_table=None), dict(scale=float("nan")),
    dict(mask_dtype=2), dict(q_strides=(4096, 512, 129)), dict(k_cache_strides=(4096, 512, 136)),
    dict(v_cache_strides=(4096, 520, 128)), dict(k_cache_strides=(-16, 512, 128)), dict(table_stride=-1), dict(q=None),
    dict(q=4104), dict(out=None), dict(cache_lens=None), dict(k_cache=None), dict(v_cache=4104), dict(k_scales=None),
    dict(v_scales=None), dict(k_scales=4098), dict(v_scale_strides=(128, -1, 1)), dict(page_size=1 << 28, max_blocks=4),
    dict(B=1 << 20, N=1024)])
def test_attention_refuses(bad):
    assert L().llima_tree_attention_fp8(ctypes.byref(attention8(**bad)), P, BIG << 10, None) == -1


def test_attention_workspace_and_empty_batch():
    l = L()
    a = attention8()
    need = l.llima_tree_attention_fp8_workspace_bytes(2, 4, 8, 4, 128)
    assert need > 0 and l.llima_tree_attention_fp8_workspace_bytes(2, 4, 8, 4, 96) == 0
    assert l.llima_tree_attention_fp8_workspace_bytes(0, 4, 8, 4, 128) == 0
    assert l.llima_tree_attention_fp8(ctypes.byref(a), N, need, None) == -4
    assert l.llima_tree_attention_fp8(ctypes.byref(a), P, need - 1, None) == -4
    assert l.llima_tree_attention_fp8(ctypes.byref(a), ctypes.c_void_p(24), need, None) == -1
    assert l.llima_tree_attention_fp8(None, P, need, None) == -1
    a = attention8(B=0, q=None, k=None, v=None, out=None, cache_lens=None, k_scales=None)
    assert l.llima_tree_attention_fp8(ctypes.byref(a), N, 0, None) == 0
    # bounded by the device's workgroups, not by the batch
    assert l.llima_tree_attention_fp8_workspace_bytes(4096, 1, 32, 8, 128) == l.llima_tree_attention_fp8_workspace_bytes(8192, 1, 32, 8, 128)


def write(**bad):
    from llima_amd import _lib
    a = _lib.CacheWriteFp8ArgsC()
    base = dict.fromkeys(("k", "v", "k_cache", "v_cache", "k_scales", "v_scales", "nodes", "counts", "cache_lens",
                          "block_table", "new_lens"), 4096)
    base.update(dict.fromkeys(("k_strides", "v_strides", "k_cache_strides", "v_cache_strides", "k_scale_strides",
                               "v_scale_strides"), (65536, 4096, 512, 128)))
    base.update(nodes_stride=3, table_stride=8, dtype=1, layers=2, B=2, N=4, L=3, Hkv=4, D=128, page_size=16, pages=20, max_blocks=8)
    return L().llima_cache_write_fp8(ctypes.byref(fill(a, bad, **base)), None)


@pytest.mark.parametrize("bad", [
    dict(dtype=0), dict(dtype=3), dict(layers=0), dict(layers=65536), dict(B=-1), dict(N=0), dict(L=0), dict(Hkv=0),
    dict(Hkv=1025), dict(D=96), dict(D=8), dict(page_size=0), dict(pages=-1), dict(max_blocks=-1), dict(block_table=None),
    dict(nodes=None), dict(nodes_stride=-1), dict(table_stride=-1), dict(k=None), dict(v=None), dict(k=4104), dict(k_cache=None),
    dict(v_cache=None), dict(k_cache=4104), dict(k_scales=None), dict(v_scales=4097), dict(cache_lens=None), dict(new_lens=None),
    dict(k_strides=(65536, 4096, 512, 4)), dict(v_cache_strides=(65536, 4096, 512, 8)), dict(k_scale_strides=(1, 1, 1, -1)),
    dict(page_size=1 << 28, max_blocks=5), dict(L=(1 << 30) + 1), dict(B=1 << 20, L=1 << 10)])
def test_write_refuses(bad):
    assert write(**bad) == -1


def read(**bad):
    from llima_amd import _lib
    a = _lib.CacheReadFp8ArgsC()
    base = dict.fromkeys(("k", "v", "k_cache", "v_cache", "k_scales", "v_scales", "cache_lens", "block_table"), 4096)
    base.update(dict.fromkeys(("k_strides", "v_strides", "k_cache_strides", "v_cache_strides", "k_scale_strides",
                               "v_scale_strides"), (65536, 4096, 512, 128)))
    base.update(table_stride=8, dtype=1, layers=2, B=2, L=3, Hkv=4, D=128, page_size=16, pages=20, max_blocks=8)
    return L().llima_cache_read_fp8(ctypes.byref(fill(a, bad, **base)), None)


@pytest.mark.parametrize("bad", [
    dict(dtype=0), dict(layers=0), dict(B=-1), dict(L=-1), dict(Hkv=0), dict(D=32), dict(page_size=0), dict(block_table=None),
    dict(k=None), dict(v=4100), dict(k_cache=None), dict(v_scales=None), dict(k_scales=4098), dict(cache_lens=None),
    dict(k_strides=(65536, 4096, 516, 128)), dict(k_cache_strides=(65536, 4096, 24, 128)), dict(L=(1 << 30) + 1),
    dict(B=1 << 22, L=1 << 20)])
def test_read_refuses(bad):
    assert read(**bad) == -1


def test_nothing_to_do_launches_nothing():
    assert write(B=0, k=None, new_lens=None) == 0 and read(B=0, k=None) == 0 and read(L=0) == 0
    assert L().llima_cache_write_fp8(None, None) == -1 and L().llima_cache_read_fp8(None, None) == -1


def sandwich(**bad):
    from llima_amd import _lib
    a = _lib.SandwichNormArgsC()
    base = dict.fromkeys(("x", "residual", "gate", "post_weight", "pre_weight", "out", "out_residual"), 4096)
    base.update(out_scales=None, x_stride=64, residual_stride=64, gate_stride=64, dtype=1, B=2, H=64, eps=1e-6,
                weight_offset=0.0, residual_scale=1.0, gate_scale=1.0)
    return L().llima_sandwich_norm(ctypes.byref(fill(a, bad, **base)), None)


@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(dtype=-1), dict(B=-1), dict(H=0), dict(H=12), dict(H=65544), dict(x=None), dict(x=4104),
    dict(x_stride=56), dict(x_stride=68), dict(residual=None), dict(residual=4100), dict(residual_stride=60), dict(gate=4104),
    dict(gate_stride=56), dict(gate_stride=-64), dict(post_weight=4104), dict(pre_weight=None), dict(pre_weight=4104),
    dict(out=None), dict(out=4104), dict(out_residual=None), dict(out_residual=4104), dict(eps=-1.0), dict(eps=float("nan")),
    dict(weight_offset=float("inf")), dict(residual_scale=float("nan")), dict(gate_scale=float("inf")), dict(dtype=0, x_stride=66)])
def test_sandwich_refuses(bad):
    assert sandwich(**bad) == -1


def test_sandwich_of_no_rows():
    assert sandwich(B=0, x=None, residual=None, gate=None, out=None, out_residual=None) == 0
    assert L().llima_sandwich_norm(None, None) == -1


def test_packed_arguments_have_the_structures_sizes():
    from llima_amd import _lib
    for packed, c in ((_lib.TREE_ATTENTION_FP8_ARGS, _lib.TreeAttentionFp8ArgsC), (_lib.CACHE_WRITE_FP8_ARGS, _lib.CacheWriteFp8ArgsC),
                      (_lib.CACHE_READ_FP8_ARGS, _lib.CacheReadFp8ArgsC), (_lib.SANDWICH_NORM_ARGS, _lib.SandwichNormArgsC)):
        assert packed.size == ctypes.sizeof(c)
    whole = _lib.TREE_ATTENTION_ARGS.size
    assert _lib.NINE_POINTERS.size + _lib.TREE_ATTENTION_SIZES.size == whole == ctypes.sizeof(_lib.TreeAttentionArgsC)
    assert whole + _lib.TWO_POINTERS.size + _lib.SIX_STRIDES.size == _lib.TREE_ATTENTION_FP8_ARGS.size
    assert _lib.ELEVEN_POINTERS.size + _lib.CACHE_WRITE_FP8_SIZES.size == _lib.CACHE_WRITE_FP8_ARGS.size
    assert _lib.EIGHT_POINTERS.size + _lib.CACHE_READ_FP8_SIZES.size == _lib.CACHE_READ_FP8_ARGS.size


def test_python_refuses(monkeypatch):
    """Shapes, types and mixed caches, on host tensors that only the last check would take for the GPU's."""
    import llima_amd
    from llima_amd import attention
    F8 = torch.float8_e4m3fn

    def cache(*shape):
        return llima_amd.Fp8Cache(torch.zeros(shape, dtype=torch.uint8).view(F8), torch.zeros(shape[:-1]))
    with pytest.raises(ValueError):                          # not on the GPU
        cache(2, 30, 2, 64)
    monkeypatch.setattr(attention, "_on_gpu", lambda *t: None)
    c, c5 = cache(2, 30, 2, 64), cache(3, 2, 30, 2, 64)
    bf = torch.bfloat16
    k, q = torch.zeros(2, 3, 2, 64, dtype=bf), torch.zeros(2, 3, 4, 64, dtype=bf)
    i2 = torch.zeros(2, dtype=torch.int32)
    nodes = torch.zeros(2, 2, dtype=torch.int32)
    t16 = torch.zeros(2, 30, 2, 64, dtype=bf)
    for call in (lambda: llima_amd.Fp8Cache(torch.zeros(2, 30, 2, 64), torch.zeros(2, 30, 2)),
                 lambda: llima_amd.Fp8Cache(c.values, c.scales.double()), lambda: llima_amd.Fp8Cache(c.values, c.scales[:1]),
                 lambda: cache(2, 30, 2, 96), lambda: cache(30, 2, 64), lambda: c[0], lambda: llima_amd.Fp8Cache.empty(3, 2, 64),
                 lambda: llima_amd.tree_attention(q, k, k, c, t16, i2), lambda: llima_amd.tree_attention(q, k, k, t16, c, i2),
                 lambda: llima_amd.tree_attention(q, k, k, c5, c5, i2), lambda: llima_amd.tree_attention(q, k, k, c, cache(2, 29, 2, 64), i2),
                 lambda: llima_amd.tree_attention(q, k, k, cache(2, 30, 2, 128), cache(2, 30, 2, 128), i2),
                 lambda: llima_amd.tree_commit(k, k, nodes, i2, c, t16, i2), lambda: llima_amd.tree_commit(k, k, nodes.long(), i2, c, c, i2),
                 lambda: llima_amd.tree_commit(k, k, nodes[:, :0], i2, c, c, i2), lambda: llima_amd.tree_commit(k, k, nodes[:1], i2, c, c, i2),
                 lambda: llima_amd.cache_write(k, k, t16, t16, i2), lambda: llima_amd.cache_write(k, k, c5, c5, i2),
                 lambda: llima_amd.cache_write(k.float(), k.float(), c, c, i2), lambda: llima_amd.cache_write(k, k[:, :2], c, c, i2),
                 lambda: llima_amd.cache_write(k, k, c, c, i2.long()), lambda: llima_amd.cache_write(k, k, c, c, i2, i2[:1]),
                 lambda: llima_amd.cache_write(k[:, :0], k[:, :0], c, c, i2),
                 lambda: llima_amd.cache_write(k[None], k[None], c5, c5, i2), lambda: llima_amd.cache_read(t16, t16, i2),
                 lambda: llima_amd.cache_read(c, c, i2, dtype=torch.float32), lambda: llima_amd.cache_read(c, c, i2[:1]),
                 lambda: llima_amd.cache_read(c, c, i2, tokens=-1), lambda: llima_amd.cache_read(c, c5, i2),
                 lambda: llima_amd.cache_read(c, c, i2, block_table=nodes.long())):
        with pytest.raises(ValueError):
            call()


def test_sandwich_python_refuses():
    import llima_amd
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.bfloat16)
    for call in (lambda: llima_amd.sandwich_norm(x, w, x, w), lambda: llima_amd.sandwich_norm(x, w, x[:1], w),
                 lambda: llima_amd.sandwich_norm(x, w, x.float(), w), lambda: llima_amd.sandwich_norm(x, w, x, w, out="int8")):
        with pytest.raises(ValueError):
            call()
