"""Attention of drafted tokens over a KV cache, and the commit of an accepted path.

  tree_attention(q, k, v, k_cache, v_cache, cache_lens, tree_mask, block_table)
  tree_commit(k, v, nodes, counts, k_cache, v_cache, cache_lens, block_table)

The step of a draft tree around the token selection: the attention reads the mask
that Eagle3DraftTree.finish makes, the commit keeps the path that verify_tree or
lm_head_verify_tree accepted.  No counterpart in the reference, whose attention and
caches are on the NPU.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._lib import check, lib
from .sampler import FLOAT_CODES, _on, _on_gpu, _scratch, _stream

__all__ = ["tree_attention", "tree_commit"]


def _heads(t: torch.Tensor) -> torch.Tensor:
    """[..., D] that 16-byte accesses can read: D adjacent, the other strides multiples
    of 8 and not negative, 16-byte aligned (copied when it is not)."""
    if t.is_contiguous() and t.shape[-1] % 8 == 0 and t.data_ptr() % 16 == 0:
        return t
    st = t.stride()
    if st[-1] == 1 and t.data_ptr() % 16 == 0:
        if not any([s % 8 for s in st[:-1]]):
            return t
        if not any([s % 8 and n > 1 for s, n in zip(st[:-1], t.shape[:-1])]):
            return t.as_strided(t.shape, [0 if n <= 1 else s for s, n in zip(st[:-1], t.shape[:-1])] + [1])
    return t.clone(memory_format=torch.contiguous_format)


def _in_place(t: torch.Tensor, name: str) -> torch.Tensor:
    """A cache as the kernels can use it where it is (it is never copied)."""
    h = _heads(t)
    if h is not t and h.data_ptr() != t.data_ptr():
        raise ValueError(f"{name}: head values must be adjacent, other strides multiples of 8, "
                         "and the first 16-byte aligned")
    return h


def _shared(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors may have memory in common: False where their strides show that they
    have none.  Either the spans from their first to their last value do not meet, or, for one of
    the strides, the places of a's values modulo that stride (an interval) are not those of b's,
    as in views that differ in one index or range of a dimension of a larger tensor."""
    sa, sb = a.untyped_storage(), b.untyped_storage()        # first, as the usual case: 0.6 us
    ba, bb = sa.data_ptr(), sb.data_ptr()
    if ba >= bb + sb.nbytes() or bb >= ba + sa.nbytes() or not a.numel() or not b.numel():
        return False

    def span(t, period=0):
        return t.element_size() * (1 + sum([(n - 1) * s for n, s in zip(t.shape, t.stride())
                                            if not period or s * t.element_size() % period]))
    pa, pb = a.data_ptr(), b.data_ptr()
    if pa >= pb + span(b) or pb >= pa + span(a):
        return False
    for t in (a, b):
        for n, s in zip(t.shape, t.stride()):
            period = s * t.element_size()
            if n > 1 and period:
                d = (pb - pa) % period
                if d >= span(a, period) and period - d >= span(b, period):
                    return False
    return True


def _same(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and a.stride() == b.stride()


def _folded(t: torch.Tensor) -> bool:
    """Whether values of a tensor may share memory: a stride less than what the smaller ones span."""
    if t.is_contiguous():
        return False
    end = 1
    for s, n in sorted([(s, n) for n, s in zip(t.shape, t.stride()) if n > 1]):
        if s < end:
            return t.numel() > 0
        end += (n - 1) * s
    return False


def _cache(k_cache, v_cache, Hkv, D, dtype, block_table, B, dev):
    """Checks of a cache [..., page_size, Hkv, D] and its table -> (page size, pages, blocks per
    sequence, table)."""
    for t in (k_cache, v_cache):
        if t.dtype != dtype or tuple(t.shape[-2:]) != (Hkv, D) or t.shape != k_cache.shape:
            raise ValueError("k_cache and v_cache must both be [..., tokens, Hkv, D] of k's type")
    pages, page = k_cache.shape[-4], k_cache.shape[-3]
    if page == 0:
        raise ValueError("the cache has no room for a token")
    if block_table is None:
        if pages != B:
            raise ValueError("without a block table the cache must be [B, tokens, Hkv, D]")
        return page, pages, 1, None
    if block_table.dim() != 2 or block_table.shape[0] != B or block_table.dtype != torch.int32:
        raise ValueError("block_table must be int32 [B, blocks]")
    if block_table.device != dev:
        raise ValueError("block_table must be on the cache's device")
    t = block_table if block_table.stride(1) == 1 or block_table.shape[1] == 1 else block_table.contiguous()
    if t.shape[1] and page * t.shape[1] > 1 << 30:
        raise ValueError("a sequence's blocks hold more than 2^30 tokens")
    return page, pages, t.shape[1], t


def _ints(t: torch.Tensor, B: int, name: str, dev) -> torch.Tensor:
    if tuple(t.shape) != (B,) or t.dtype != torch.int32 or t.device != dev:
        raise ValueError(f"{name} must be int32 [{B}] on the cache's device")
    return t.contiguous()


def tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                   v_cache: torch.Tensor, cache_lens: torch.Tensor,
                   tree_mask: Optional[torch.Tensor] = None,
                   block_table: Optional[torch.Tensor] = None,
                   scale: Optional[float] = None) -> torch.Tensor:
    """Attention of N drafted tokens of B sequences over the sequences' caches and, under the
    tree mask, over each other (llima_tree_attention) -> [B, N, Hq, D] of q's type.

    q [B, N, Hq, D], k and v [B, N, Hkv, D] (the drafted tokens' own, not in the cache yet;
    Hq a multiple of Hkv), bf16 or fp16, D 64, 128 or 256.  k_cache, v_cache: [B, tokens, Hkv,
    D], or pages [pages, page_size, Hkv, D] with block_table int32 [B, blocks]; cache_lens
    int32 [B]: the cached tokens, which every node sees.  tree_mask [N, N] or [B, N, N],
    bool (or uint8, nonzero) or float32 (above 0, as Eagle3DraftTree.finish's): node n sees
    drafted token m where mask[n, m]; None: m <= n, the chain of drafts, or with N = 1 a
    decode step.  A row that sees nothing is 0; a sequence with a length or a page out of
    range is NaN.  scale defaults to D^-0.5.  Strides are free where values of a head are
    adjacent (head-major caches as transposed views).  Nothing waits for the device, and the
    call can be captured into a graph."""
    if q.dim() != 4 or k.dim() != 4 or k_cache.dim() != 4 or v_cache.dim() != 4:
        raise ValueError("q [B, N, Hq, D], k and v [B, N, Hkv, D] and 4-dimensional caches are needed")
    B, N, Hq, D = q.shape
    Hkv = k.shape[2]
    if tuple(k.shape) != (B, N, Hkv, D) or v.shape != k.shape:
        raise ValueError("k and v must be [B, N, Hkv, D] with q's B, N and D")
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must be bfloat16 or float16, of one type")
    if D not in (64, 128, 256):
        raise ValueError("the head size must be 64, 128 or 256")
    if N == 0 or N > 1024 or Hkv == 0 or Hq == 0 or Hq % Hkv or Hq > 1024:
        raise ValueError("1 to 1024 drafted tokens and query heads, a multiple of the key heads, are supported")
    _on_gpu(q, k, v, k_cache, v_cache, cache_lens, tree_mask, block_table)
    dev = q.device
    if not (k.device == v.device == k_cache.device == v_cache.device == dev):
        raise ValueError("tree_attention: tensors must be on one device")
    page, pages, blocks, table = _cache(k_cache, v_cache, Hkv, D, q.dtype, block_table, B, dev)
    lens = _ints(cache_lens, B, "cache_lens", dev)
    mask, mask_dtype, ms = tree_mask, _lib.LLIMA_MASK_U8, (0, 0)
    if mask is not None:
        if tuple(mask.shape) not in ((N, N), (B, N, N)) or mask.device != dev:
            raise ValueError("tree_mask must be [N, N] or [B, N, N] on q's device")
        if mask.dtype not in (torch.bool, torch.uint8, torch.float32):
            raise ValueError("tree_mask must be bool, uint8 or float32")
        if mask.stride(-1) != 1:
            mask = mask.contiguous()
        if mask.dtype == torch.float32:
            mask_dtype = _lib.LLIMA_MASK_F32
        ms = (mask.stride(0) if mask.dim() == 3 else 0, mask.stride(-2))
    q, k, v = _heads(q), _heads(k), _heads(v)
    kc, vc = _in_place(k_cache, "k_cache"), _in_place(v_cache, "v_cache")
    out = torch.empty((B, N, Hq, D), dtype=q.dtype, device=dev)
    if B == 0:
        return out
    L = lib()
    ws = _scratch(dev, "tree_attention", L.llima_tree_attention_workspace_bytes(B, N, Hq, Hkv, D))
    # a table of no blocks is not read
    tp, ts = (0, 0) if table is None else (table.data_ptr() or lens.data_ptr(), table.stride(0))
    a = _lib.TREE_ATTENTION_ARGS.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), kc.data_ptr(), vc.data_ptr(), out.data_ptr(), lens.data_ptr(),
        0 if mask is None else mask.data_ptr(), tp, *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
        *out.stride()[:3], *kc.stride()[:3], *vc.stride()[:3], *ms, ts, FLOAT_CODES[q.dtype], mask_dtype, B, N, Hq,
        Hkv, D, page, pages, blocks, D ** -0.5 if scale is None else float(scale))
    with _on(dev):
        check(L.llima_tree_attention(a, ws.data_ptr(), ws.numel(), _stream(dev)), "llima_tree_attention")
    return out


def tree_commit(k: torch.Tensor, v: torch.Tensor, nodes: torch.Tensor, counts: torch.Tensor,
                k_cache: torch.Tensor, v_cache: torch.Tensor, cache_lens: torch.Tensor,
                block_table: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Keeps the accepted path of each sequence in its cache, in place (llima_tree_commit), and
    returns the new lengths int32 [B]: token cache_lens[b] + j becomes drafted token
    nodes[b, j], j < counts[b].

    k, v [B, N, Hkv, D] or, for every layer at once, [layers, B, N, Hkv, D], with caches
    [B, tokens, Hkv, D] or [pages, page_size, Hkv, D] (and the layers' dimension in front);
    bf16 or fp16, D a multiple of 8.  nodes int32 [B, L], counts int32 [B] (a row of
    Eagle3DraftTree's retrieve indices and the accept length + 1; arange and accepted_len + 1
    for a chain).  k and v may stand beside the caches in one storage, but not in them, and the
    caches not in each other (unless keys and values are the same tensors).  A sequence with a
    count, node, length or page out of range, or no room for its path, is left as it is and its
    new length is -2 (LLIMA_E_RANGE).  Nothing waits for the device, and the call can be captured
    into a graph."""
    if k.dim() == 4:
        if k_cache.dim() != 4 or v_cache.dim() != 4 or v.dim() != 4:
            raise ValueError("k and v [B, N, Hkv, D] need 4-dimensional caches")
        k, v, k_cache, v_cache = k[None], v[None], k_cache[None], v_cache[None]
    if k.dim() != 5 or k_cache.dim() != 5 or v_cache.dim() != 5:
        raise ValueError("k and v must be [B, N, Hkv, D] or [layers, B, N, Hkv, D], the caches likewise")
    layers, B, N, Hkv, D = k.shape
    if v.shape != k.shape or v.dtype != k.dtype or k.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("k and v must have one shape and type, bfloat16 or float16")
    if k_cache.shape[0] != layers or v_cache.shape[0] != layers:
        raise ValueError("k, v and the caches must have the same number of layers")
    if N == 0 or Hkv == 0 or D == 0 or D % 8 or layers == 0 or layers > 65535:
        raise ValueError("1 to 65535 layers, tokens, and heads of a multiple of 8 values are needed")
    if nodes.dim() != 2 or nodes.shape[0] != B or nodes.shape[1] == 0 or nodes.dtype != torch.int32:
        raise ValueError("nodes must be int32 [B, L], L at least 1")
    _on_gpu(k, v, nodes, counts, k_cache, v_cache, cache_lens, block_table)
    dev = k.device
    if not (v.device == k_cache.device == v_cache.device == nodes.device == dev):
        raise ValueError("tree_commit: tensors must be on one device")
    page, pages, blocks, table = _cache(k_cache, v_cache, Hkv, D, k.dtype, block_table, B, dev)
    counts, lens = _ints(counts, B, "counts", dev), _ints(cache_lens, B, "cache_lens", dev)
    nodes = nodes if nodes.stride(1) == 1 or nodes.shape[1] == 1 else nodes.contiguous()
    tied = _same(k, v)
    k, v = _heads(k), _heads(v)
    kc, vc = _in_place(k_cache, "k_cache"), _in_place(v_cache, "v_cache")
    if _shared(k, kc) or _shared(k, vc) or _shared(v, kc) or _shared(v, vc):
        raise ValueError("tree_commit: k and v must not overlap the caches (copy them first)")
    if _folded(kc) or _folded(vc):
        raise ValueError("tree_commit: a cache's own values must not overlap (expanded dimensions)")
    if _shared(kc, vc) and not (tied and _same(kc, vc)):
        raise ValueError("tree_commit: k_cache and v_cache must not overlap")
    new = torch.empty(B, dtype=torch.int32, device=dev)
    if B == 0:
        return new
    tp, ts = (0, 0) if table is None else (table.data_ptr() or lens.data_ptr(), table.stride(0))
    a = _lib.TREE_COMMIT_ARGS.pack(
        k.data_ptr(), v.data_ptr(), kc.data_ptr(), vc.data_ptr(), nodes.data_ptr(), counts.data_ptr(), lens.data_ptr(),
        tp, new.data_ptr(), *k.stride()[:4], *v.stride()[:4], *kc.stride()[:4], *vc.stride()[:4], nodes.stride(0), ts,
        layers, B, N, nodes.shape[1], Hkv, D, page, pages, blocks)
    with _on(dev):
        check(lib().llima_tree_commit(a, _stream(dev)), "llima_tree_commit")
    return new
