"""Attention of drafted tokens over a KV cache, and the commit of an accepted path.

  tree_attention(q, k, v, k_cache, v_cache, cache_lens, tree_mask, block_table)
  tree_commit(k, v, nodes, counts, k_cache, v_cache, cache_lens, block_table)
  Fp8Cache(values, scales), cache_write(k, v, k_cache, v_cache, cache_lens, counts, block_table)
  cache_read(k_cache, v_cache, cache_lens, block_table, dtype, tokens)

The step of a draft tree around the token selection: the attention reads the mask
that Eagle3DraftTree.finish makes, the commit keeps the path that verify_tree or
lm_head_verify_tree accepted.  The caches are in 16 bits, or Fp8Cache: in e4m3 with a
scale per token and head, quantised as they are written.  No counterpart in the reference, whose attention and
caches are on the NPU.
"""
from __future__ import annotations

from functools import lru_cache
from typing import Optional

import torch

from . import _lib
from ._lib import check, lib
from .sampler import _PLANS, FLOAT_CODES, _form, _on, _on_gpu, _planned, _scratch, _stream

F8 = torch.float8_e4m3fn

__all__ = ["Fp8Cache", "cache_read", "cache_write", "tree_attention", "tree_commit"]


class Fp8Cache:
    """The keys or the values of an 8-bit KV cache: `values` float8_e4m3fn [..., tokens, Hkv, D]
    (D 64, 128 or 256) and `scales` float32 [..., tokens, Hkv], one per token and head: a head's
    row is values * scales.  In front stand B or, with a block table, pages, and in front of those
    the layers where every layer's cache is one tensor; cache[i] is layer i's.  tree_attention,
    tree_commit, cache_write and cache_read take it; a scale is max(max |x|, 2^-100) / 448 of the
    row that was written.  Strides are free where values of a head are adjacent; `empty` gives
    the order that is read fastest."""
    __slots__ = ("values", "scales")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor):
        if values.dtype != F8 or scales.dtype != torch.float32:
            raise ValueError("Fp8Cache: values must be float8_e4m3fn and scales float32")
        shape = values.shape
        if len(shape) < 4 or shape[:-1] != scales.shape or shape[-1] not in (64, 128, 256):
            raise ValueError("Fp8Cache: values [..., tokens, Hkv, D], D 64, 128 or 256, and scales [..., tokens, Hkv] are needed")
        _on_gpu(values, scales)
        if values.device != scales.device:
            raise ValueError("Fp8Cache: values and scales must be on one device")
        self.values, self.scales = values, scales

    @classmethod
    def empty(cls, *shape: int, device=None) -> "Fp8Cache":
        """A cache [..., tokens, Hkv, D] whose values are not set; in memory a head's tokens follow
        each other: [..., Hkv, tokens, D]."""
        if len(shape) < 4:
            raise ValueError("Fp8Cache.empty takes [..., tokens, Hkv, D]")
        n = (*shape[:-3], shape[-2], shape[-3])
        dev = device if device is not None else "cuda"
        return cls(torch.empty((*n, shape[-1]), dtype=F8, device=dev).transpose(-3, -2),
                   torch.empty(n, dtype=torch.float32, device=dev).transpose(-2, -1))

    @property
    def shape(self):
        return self.values.shape

    def dim(self) -> int:
        return self.values.dim()

    def __getitem__(self, layer) -> "Fp8Cache":
        if self.values.dim() < 5:
            raise ValueError("Fp8Cache: only a cache of layers is indexed")
        return Fp8Cache(self.values[layer], self.scales[layer])


def _heads(t: torch.Tensor, align: int = 8) -> torch.Tensor:
    """[..., D] that 16-byte accesses can read: D adjacent, the other strides multiples
    of 8 (of 16 for bytes) and not negative, 16-byte aligned (copied when it is not).  The
    stride of a dimension of one, which may be any number also where is_contiguous() holds, becomes 0."""
    st = t.stride()
    if st[-1] == 1 and t.data_ptr() % 16 == 0:
        bits = 0
        for n in st[:-1]:                                    # align is a power of two
            bits |= n
        if not bits % align:
            return t
        if not any([s % align and n > 1 for s, n in zip(st[:-1], t.shape[:-1])]):
            return t.as_strided(t.shape, [0 if n <= 1 else s for s, n in zip(st[:-1], t.shape[:-1])] + [1])
    return t.clone(memory_format=torch.contiguous_format)


def _in_place(t: torch.Tensor, name: str, align: int = 8) -> torch.Tensor:
    """A cache as the kernels can use it where it is (it is never copied)."""
    h = _heads(t, align)
    if h is not t and h.data_ptr() != t.data_ptr():
        raise ValueError(f"{name}: head values must be adjacent, other strides multiples of {align}, "
                         "and the first 16-byte aligned")
    return h


def _eight_bits(k_cache, v_cache) -> bool:
    """Whether both caches are Fp8Cache; one alone is refused."""
    f = isinstance(k_cache, Fp8Cache)
    if f != isinstance(v_cache, Fp8Cache):
        raise ValueError("k_cache and v_cache must both be tensors, or both Fp8Cache")
    return f


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
    return not t.is_contiguous() and _folds(t.shape, t.stride())


@lru_cache(256)
def _folds(shape, stride) -> bool:
    end = 1
    for s, n in sorted([(s, n) for n, s in zip(shape, stride) if n > 1]):
        if s < end:
            return 0 not in shape
        end += (n - 1) * s
    return False


def _apart(ts) -> bool:
    """Whether no two of the tensors' storages meet (then none shares memory with another)."""
    spans = sorted([(s.data_ptr(), s.nbytes()) for s in [t.untyped_storage() for t in ts]])
    return all([a + n <= b for (a, n), (b, _) in zip(spans, spans[1:])])


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
    D], or pages [pages, page_size, Hkv, D] with block_table int32 [B, blocks], of q's type or
    both Fp8Cache (llima_tree_attention_fp8); cache_lens
    int32 [B]: the cached tokens, which every node sees.  tree_mask [N, N] or [B, N, N],
    bool (or uint8, nonzero) or float32 (above 0, as Eagle3DraftTree.finish's): node n sees
    drafted token m where mask[n, m]; None: m <= n, the chain of drafts, or with N = 1 a
    decode step.  A row that sees nothing is 0; a sequence with a length or a page out of
    range is NaN.  scale defaults to D^-0.5.  Strides are free where values of a head are
    adjacent (head-major caches as transposed views).  Nothing waits for the device, and the
    call can be captured into a graph."""
    scale = None if scale is None else float(scale)
    if _eight_bits(k_cache, v_cache):
        return _attend(q, k, v, k_cache.values, v_cache.values, cache_lens, tree_mask, block_table, k_cache.scales,
                       v_cache.scales, scale)
    return _attend(q, k, v, k_cache, v_cache, cache_lens, tree_mask, block_table, None, None, scale)


def _attend(q, k, v, kc, vc, lens, mask, table, k8, v8, scale):
    form = (scale, _form(q), _form(k), _form(v), _form(kc), _form(vc), _form(lens), _form(mask), _form(table), _form(k8), _form(v8))
    plan = _PLANS.get(form)
    if plan is None:
        given = (q, k, v, kc, vc, lens, mask, table)
        used = _attend_checks(*given, k8, v8)
        if any([x is not y for x, y in zip(given, used)]):   # copies, or views with other strides
            return _attend(*used, k8, v8, scale)
        plan = _planned(form, _attend_plan(*given, k8, v8, scale))
    like, dev, nbytes, sizes, scales = plan
    out = torch.empty_like(q) if like else torch.empty(q.shape, dtype=q.dtype, device=dev)
    if nbytes == 0:                                          # no sequences
        return out
    ws = _scratch(dev, "tree_attention", nbytes)
    ptrs = _lib.NINE_POINTERS.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), kc.data_ptr(), vc.data_ptr(), out.data_ptr(), lens.data_ptr(),
        0 if mask is None else mask.data_ptr(),
        0 if table is None else table.data_ptr() or lens.data_ptr())     # a table of no blocks is not read
    with _on(dev):
        if k8 is None:
            check(lib().llima_tree_attention(ptrs + sizes, ws.data_ptr(), ws.numel(), _stream(dev)), "llima_tree_attention")
        else:
            a = ptrs + sizes + _lib.TWO_POINTERS.pack(k8.data_ptr(), v8.data_ptr()) + scales
            check(lib().llima_tree_attention_fp8(a, ws.data_ptr(), ws.numel(), _stream(dev)), "llima_tree_attention_fp8")
    return out


def _attend_checks(q, k, v, k_cache, v_cache, cache_lens, mask, block_table, k8, v8):
    """The call's tensors as the kernels can read them, or ValueError."""
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
    if B * N * Hq >= 1 << 26:
        raise ValueError("fewer than 2^26 rows (sequences, drafted tokens and query heads) are supported")
    _on_gpu(q, k, v, k_cache, v_cache, cache_lens, mask, block_table)
    dev = q.device
    if not (k.device == v.device == k_cache.device == v_cache.device == dev):
        raise ValueError("tree_attention: tensors must be on one device")
    if k8 is not None and not (k8.shape == v8.shape == k_cache.shape[:-1] and k8.device == v8.device == dev):
        raise ValueError("tree_attention: an Fp8Cache's scales must be [..., tokens, Hkv] beside its values")
    table = _cache(k_cache, v_cache, Hkv, D, q.dtype if k8 is None else F8, block_table, B, dev)[3]
    lens = _ints(cache_lens, B, "cache_lens", dev)
    if mask is not None:
        if tuple(mask.shape) not in ((N, N), (B, N, N)) or mask.device != dev:
            raise ValueError("tree_mask must be [N, N] or [B, N, N] on q's device")
        if mask.dtype not in (torch.bool, torch.uint8, torch.float32):
            raise ValueError("tree_mask must be bool, uint8 or float32")
        if mask.stride(-1) != 1:
            mask = mask.clone(memory_format=torch.contiguous_format)
    align = 8 if k8 is None else 16
    return (_heads(q), _heads(k), _heads(v), _in_place(k_cache, "k_cache", align), _in_place(v_cache, "v_cache", align),
            lens, mask, table)


def _attend_plan(q, k, v, kc, vc, lens, mask, table, k8, v8, scale):
    """(whether the output is laid out as q, device, workspace bytes, the arguments behind the pointers, the scales' strides)."""
    B, N, Hq, D = q.shape
    Hkv, dev = k.shape[2], q.device
    page, pages, blocks, _ = _cache(kc, vc, Hkv, D, kc.dtype, table, B, dev)
    bytes_of = lib().llima_tree_attention_workspace_bytes if k8 is None else lib().llima_tree_attention_fp8_workspace_bytes
    os = (N * Hq * D, Hq * D, D)
    ms = (0, 0) if mask is None else (mask.stride(0) if mask.dim() == 3 else 0, mask.stride(-2))
    sizes = _lib.TREE_ATTENTION_SIZES.pack(
        *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *os, *kc.stride()[:3], *vc.stride()[:3], *ms,
        0 if table is None else table.stride(0), FLOAT_CODES[q.dtype],
        _lib.LLIMA_MASK_F32 if mask is not None and mask.dtype == torch.float32 else _lib.LLIMA_MASK_U8, B, N, Hq, Hkv, D,
        page, pages, blocks, D ** -0.5 if scale is None else scale)
    scales = b"" if k8 is None else _lib.SIX_STRIDES.pack(*k8.stride(), *v8.stride())
    return q.is_contiguous(), dev, bytes_of(B, N, Hq, Hkv, D), sizes, scales


def tree_commit(k: torch.Tensor, v: torch.Tensor, nodes: torch.Tensor, counts: torch.Tensor,
                k_cache: torch.Tensor, v_cache: torch.Tensor, cache_lens: torch.Tensor,
                block_table: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Keeps the accepted path of each sequence in its cache, in place (llima_tree_commit), and
    returns the new lengths int32 [B]: token cache_lens[b] + j becomes drafted token
    nodes[b, j], j < counts[b].

    k, v [B, N, Hkv, D] or, for every layer at once, [layers, B, N, Hkv, D], with caches
    [B, tokens, Hkv, D] or [pages, page_size, Hkv, D] (and the layers' dimension in front);
    bf16 or fp16, D a multiple of 8; or both Fp8Cache, which the path is quantised into
    (llima_cache_write_fp8).  nodes int32 [B, L], counts int32 [B] (a row of
    Eagle3DraftTree's retrieve indices and the accept length + 1; arange and accepted_len + 1
    for a chain).  k and v may stand beside the caches in one storage, but not in them, and the
    caches not in each other (unless keys and values are the same tensors).  A sequence with a
    count, node, length or page out of range, or no room for its path, is left as it is and its
    new length is -2 (LLIMA_E_RANGE).  Nothing waits for the device, and the call can be captured
    into a graph."""
    if _eight_bits(k_cache, v_cache):
        if nodes.dim() != 2 or nodes.shape[1] == 0 or nodes.dtype != torch.int32:
            raise ValueError("nodes must be int32 [B, L], L at least 1")
        return _write8("tree_commit", k, v, k_cache, v_cache, cache_lens, nodes, counts, block_table)
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


def _layers(k_cache: Fp8Cache, v_cache: Fp8Cache):
    """Values and scales of both caches with the layers' dimension in front."""
    ts = (k_cache.values, v_cache.values, k_cache.scales, v_cache.scales)
    return [t[None] for t in ts] if k_cache.dim() == 4 else ts


def _write8(name, k, v, k_cache, v_cache, cache_lens, nodes, counts, block_table):
    """Keys and values into an Fp8Cache (llima_cache_write_fp8)."""
    if k.dim() == 4:
        if k_cache.dim() != 4 or v_cache.dim() != 4 or v.dim() != 4:
            raise ValueError("k and v [B, N, Hkv, D] need 4-dimensional caches")
        k, v = k[None], v[None]
    elif k.dim() != 5 or k_cache.dim() != 5 or v_cache.dim() != 5 or v.dim() != 5:
        raise ValueError("k and v must be [B, N, Hkv, D] or [layers, B, N, Hkv, D], the caches likewise")
    return _put8(name, k, v, *_layers(k_cache, v_cache), cache_lens, nodes, counts, block_table)


def _put8(name, k, v, kq, vq, ks, vs, lens, nodes, counts, table):
    form = (_form(k), _form(v), _form(kq), _form(vq), _form(ks), _form(vs), _form(lens), _form(nodes), _form(counts), _form(table))
    plan = _PLANS.get(form)
    if plan is None:
        given = (k, v, kq, vq, ks, vs, lens, nodes, counts, table)
        used = _put8_checks(name, *given)
        if any([x is not y for x, y in zip(given, used)]):   # copies, or views with other strides
            return _put8(name, *used)
        plan = _planned(form, _put8_plan(*given))
    B, dev, sizes = plan
    outs = (kq, vq, ks, vs)
    if not _apart((k, v, *outs)):                            # (the usual case: no two in one storage)
        if any([_shared(a, o) for a in (k, v) for o in outs]):
            raise ValueError(f"{name}: k and v must not overlap the caches (copy them first)")
        tied = _same(k, v) and _same(kq, vq) and _same(ks, vs)
        if not tied and (_shared(kq, vq) or _shared(ks, vs)) or \
                _shared(kq, ks) or _shared(vq, vs) or _shared(kq, vs) or _shared(vq, ks):
            raise ValueError(f"{name}: k_cache and v_cache, values and scales, must not overlap")
    new = torch.empty(B, dtype=torch.int32, device=dev)
    if B == 0:
        return new
    ptrs = _lib.ELEVEN_POINTERS.pack(
        k.data_ptr(), v.data_ptr(), kq.data_ptr(), vq.data_ptr(), ks.data_ptr(), vs.data_ptr(),
        0 if nodes is None else nodes.data_ptr(), 0 if counts is None else counts.data_ptr(), lens.data_ptr(),
        0 if table is None else table.data_ptr() or lens.data_ptr(), new.data_ptr())
    with _on(dev):
        check(lib().llima_cache_write_fp8(ptrs + sizes, _stream(dev)), "llima_cache_write_fp8")
    return new


def _put8_checks(name, k, v, kq, vq, ks, vs, cache_lens, nodes, counts, block_table):
    """The call's tensors as the kernel can use them, or ValueError."""
    layers, B, N, Hkv, D = k.shape
    if v.shape != k.shape or v.dtype != k.dtype or k.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("k and v must have one shape and type, bfloat16 or float16")
    if kq.shape[0] != layers or vq.shape[0] != layers:
        raise ValueError("k, v and the caches must have the same number of layers")
    if N == 0 or Hkv == 0 or Hkv > 1024 or layers == 0 or layers > 65535:
        raise ValueError("1 to 65535 layers, tokens, and 1 to 1024 heads are needed")
    _on_gpu(k, v, nodes, counts, cache_lens, block_table)
    dev = k.device
    if not (v.device == kq.device == vq.device == dev):
        raise ValueError(f"{name}: tensors must be on one device")
    table = _cache(kq, vq, Hkv, D, F8, block_table, B, dev)[3]
    lens = _ints(cache_lens, B, "cache_lens", dev)
    if counts is not None:
        counts = _ints(counts, B, "counts", dev)
    if nodes is not None:
        if nodes.shape[0] != B or nodes.device != dev:
            raise ValueError("nodes must be int32 [B, L] on the cache's device")
        nodes = nodes if nodes.stride(1) == 1 or nodes.shape[1] == 1 else nodes.contiguous()
    kq, vq = _in_place(kq, "k_cache", 16), _in_place(vq, "v_cache", 16)
    if any([_folded(o) for o in (kq, vq, ks, vs)]):
        raise ValueError(f"{name}: a cache's own values must not overlap (expanded dimensions)")
    if not _same(k, v):
        return _heads(k), _heads(v), kq, vq, ks, vs, lens, nodes, counts, table
    k = _heads(k)                                            # (keys that are the values stay so)
    return k, k, kq, vq, ks, vs, lens, nodes, counts, table


def _put8_plan(k, v, kq, vq, ks, vs, lens, nodes, counts, table):
    """(sequences, device, the arguments behind the pointers)."""
    layers, B, N, Hkv, D = k.shape
    page, pages, blocks, _ = _cache(kq, vq, Hkv, D, F8, table, B, k.device)
    L, ns = (N, 0) if nodes is None else (nodes.shape[1], nodes.stride(0))
    return B, k.device, _lib.CACHE_WRITE_FP8_SIZES.pack(
        *k.stride()[:4], *v.stride()[:4], *kq.stride()[:4], *vq.stride()[:4], *ks.stride(), *vs.stride(), ns,
        0 if table is None else table.stride(0), FLOAT_CODES[k.dtype], layers, B, N, L, Hkv, D, page, pages, blocks)


def cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: Fp8Cache, v_cache: Fp8Cache, cache_lens: torch.Tensor,
                counts: Optional[torch.Tensor] = None, block_table: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Quantises the first counts[b] (None: all) of N new tokens' keys and values into 8-bit caches,
    in place, behind the cache_lens[b] tokens that they hold (llima_cache_write_fp8), and returns the
    new lengths int32 [B].  For prompts, chunks of them, and decoded tokens; tree_commit keeps an
    accepted path.

    k, v [B, N, Hkv, D] or [layers, B, N, Hkv, D], bf16 or fp16, D 64, 128 or 256; the caches
    [B, tokens, Hkv, D] or pages [pages, page_size, Hkv, D] with block_table int32 [B, blocks] (and the
    layers' dimension in front).  A sequence with a count outside [0, N], a length or page out of range,
    or no room is left as it is and its new length is -2 (LLIMA_E_RANGE).  The caches may not overlap k,
    v or each other, and no two sequences may write to one page's token.  Nothing waits for the
    device, and the call can be captured into a graph."""
    if not _eight_bits(k_cache, v_cache):
        raise ValueError("cache_write takes Fp8Cache")
    return _write8("cache_write", k, v, k_cache, v_cache, cache_lens, None, counts, block_table)


def cache_read(k_cache: Fp8Cache, v_cache: Fp8Cache, cache_lens: torch.Tensor,
               block_table: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16,
               tokens: Optional[int] = None):
    """The first `tokens` tokens (None: all that there is room for) of B sequences of 8-bit caches, in
    16 bits and in order (llima_cache_read_fp8) -> keys and values [B, tokens, Hkv, D], or [layers, B,
    tokens, Hkv, D] of caches with the layers' dimension: round(values * scales) of the cache_lens[b]
    cached tokens, 0 behind them.  dtype bfloat16 or float16.  A sequence with a length or a page out
    of range is NaN.  For programs that know no 8-bit cache.  Nothing waits for the device, and
    the call can be captured into a graph."""
    if not _eight_bits(k_cache, v_cache):
        raise ValueError("cache_read takes Fp8Cache")
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("cache_read gives bfloat16 or float16")
    if k_cache.dim() not in (4, 5) or v_cache.shape != k_cache.shape:
        raise ValueError("both caches must be [B, tokens, Hkv, D] or pages, with or without layers, of one shape")
    k, v = _get8(*_layers(k_cache, v_cache), cache_lens, block_table, dtype, None if tokens is None else int(tokens))
    return (k[0], v[0]) if k_cache.dim() == 4 else (k, v)


def _get8(kq, vq, ks, vs, lens, table, dtype, tokens):
    form = (dtype, tokens, _form(kq), _form(vq), _form(ks), _form(vs), _form(lens), _form(table))
    plan = _PLANS.get(form)
    if plan is None:
        given = (kq, vq, ks, vs, lens, table)
        used = _get8_checks(*given, tokens)
        if any([x is not y for x, y in zip(given, used)]):   # copies, or views with other strides
            return _get8(*used, dtype, tokens)
        plan = _planned(form, _get8_plan(*given, dtype, tokens))
    shape, dev, sizes = plan
    k, v = torch.empty(shape, dtype=dtype, device=dev), torch.empty(shape, dtype=dtype, device=dev)
    if sizes:
        ptrs = _lib.EIGHT_POINTERS.pack(
            k.data_ptr(), v.data_ptr(), kq.data_ptr(), vq.data_ptr(), ks.data_ptr(), vs.data_ptr(), lens.data_ptr(),
            0 if table is None else table.data_ptr() or lens.data_ptr())
        with _on(dev):
            check(lib().llima_cache_read_fp8(ptrs + sizes, _stream(dev)), "llima_cache_read_fp8")
    return k, v


def _get8_checks(kq, vq, ks, vs, cache_lens, block_table, tokens):
    layers, Hkv = kq.shape[0], kq.shape[3]
    if layers == 0 or layers > 65535 or Hkv == 0 or Hkv > 1024:
        raise ValueError("1 to 65535 layers and 1 to 1024 heads are needed")
    _on_gpu(cache_lens, block_table)
    dev = kq.device
    if vq.device != dev:
        raise ValueError("cache_read: tensors must be on one device")
    B = cache_lens.shape[0] if cache_lens.dim() == 1 else -1
    table = _cache(kq, vq, Hkv, kq.shape[4], F8, block_table, B, dev)[3]
    lens = _ints(cache_lens, B, "cache_lens", dev)
    if tokens is not None and not 0 <= tokens <= 1 << 30:
        raise ValueError("0 to 2^30 tokens can be read")
    return _in_place(kq, "k_cache", 16), _in_place(vq, "v_cache", 16), ks, vs, lens, table


def _get8_plan(kq, vq, ks, vs, lens, table, dtype, tokens):
    """(outputs' shape, device, the arguments behind the pointers or nothing where there is nothing to read)."""
    layers, Hkv, D, B = kq.shape[0], kq.shape[3], kq.shape[4], lens.shape[0]
    page, pages, blocks, _ = _cache(kq, vq, Hkv, D, F8, table, B, kq.device)
    n = page * blocks if tokens is None else tokens
    os = (B * n * Hkv * D, n * Hkv * D, Hkv * D, D)
    sizes = b"" if B * n == 0 else _lib.CACHE_READ_FP8_SIZES.pack(
        *os, *os, *kq.stride()[:4], *vq.stride()[:4], *ks.stride(), *vs.stride(), 0 if table is None else table.stride(0),
        FLOAT_CODES[dtype], layers, B, n, Hkv, D, page, pages, blocks)
    return (layers, B, n, Hkv, D), kq.device, sizes
