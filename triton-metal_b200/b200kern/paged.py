"""What a serving step does to a paged KV cache before attention reads it
(torch tensors in, torch tensors out, libb2.so compute).

  * build_page_table: page table and slot map of the step, on the GPU from the
    request lengths;
  * store_kv: the step's K/V rows into the cache, by slot.
Both work on the cache of decode_attention / tree_attention: pages
[n_pages, page_size, Hkv, D] and page_table int32 [B, max_pages] (the layout
of the reference's paged_attention, _msl_templates.py:2279-2532; it has no
counterpart of these two, its host fills the buffers).
"""
import ctypes

import torch

from . import _lib
from .errors import B2DtypeError, B2ShapeError

_DT = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_pi64x2 = ctypes.c_int64 * 2


def _lens(t, name):
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
        raise B2ShapeError(f"{name} must be a contiguous int32 vector, got {t.dtype} {tuple(t.shape)}")


def build_page_table(context_lens, new_lens, page_size, free_pages, page_table, max_tokens):
    """Pages and slots for the new tokens of a step.

    context_lens, new_lens: int32 [B], tokens that each request has in the
    cache and gets now.  free_pages: int32 [n_free], physical pages to take
    from, in order.  page_table: int32 [B, max_pages], rows may be strided; it
    is updated in place: the pages opened by request b go behind the
    ceil(context_lens[b] / page_size) pages that it holds.

    Returns (page_table, slots, offsets, pages_used): slots int64 [max_tokens]
    holds page * page_size + offset of every new token, request after request,
    then -1; offsets int32 [B + 1] the first token of each request and their
    number; pages_used int32 [1] how many free pages the step wanted.  With too
    few of them, or with a request beyond max_pages, the tokens concerned get
    slot -1 (store_kv passes them over) and the missing pages entry -1; compare
    pages_used with n_free before the cache is read.  max_tokens has to be at
    least sum(new_lens), which stays on the GPU: tokens beyond it are dropped
    with the pages they would open.  One launch, no synchronisation; a step
    captured in a CUDA graph follows the lengths of each replay.
    """
    r = _lib.fast_call("build_page_table", "b2_build_page_table", context_lens, new_lens, page_size, free_pages,
                       page_table, max_tokens)
    if r is not None:
        return r
    _lens(context_lens, "context_lens")
    _lens(new_lens, "new_lens")
    _lens(free_pages, "free_pages")
    B = context_lens.shape[0]
    if new_lens.shape[0] != B:
        raise B2ShapeError(f"context_lens and new_lens differ in length: {B} and {new_lens.shape[0]}")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != B:
        raise B2ShapeError(f"page_table must be int32 [{B}, max_pages], got {page_table.dtype} "
                           f"{tuple(page_table.shape)}")
    max_pages = page_table.shape[1]
    stride = page_table.stride(0) if B > 1 else max(max_pages, 1)
    if (max_pages > 1 and page_table.stride(1) != 1) or (B > 1 and stride < max_pages):
        raise B2ShapeError("page_table rows must be contiguous and must not overlap")
    if page_size <= 0 or max_tokens < 0:
        raise B2ShapeError("page_size must be positive and max_tokens not negative")
    _lib.check_device(context_lens, new_lens=new_lens, free_pages=free_pages, page_table=page_table)
    dev = context_lens.device
    slots = torch.empty(max_tokens, dtype=torch.int64, device=dev)
    offsets = torch.empty(B + 1, dtype=torch.int32, device=dev)
    used = torch.empty(1, dtype=torch.int32, device=dev)
    with _lib.on_device(context_lens):
        _lib.call("b2_build_page_table", context_lens.data_ptr(), new_lens.data_ptr(), free_pages.data_ptr(),
                  page_table.data_ptr(), slots.data_ptr(), offsets.data_ptr(), used.data_ptr(), B, page_size,
                  free_pages.shape[0], max_pages, stride, max_tokens, _lib.current_stream())
    return page_table, slots, offsets, used


def _overlaps_itself(t):
    """Whether two indices of t may share an element (strides of 0, windows)."""
    need = 1
    for n, s in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n > 1), key=lambda x: x[1]):
        if s < need:
            return True
        need = s * n
    return False


def store_kv(k, v, k_pages, v_pages, slots):
    """Writes row r of k and v ([N, Hkv, D]) to slot slots[r] of the cache.

    k_pages, v_pages: [n_pages, page_size, Hkv, D], written in place and
    returned; slots: int64 [N], as build_page_table makes them.  Any strides
    with a contiguous last dimension (a contiguous cache [B, Hkv, S, D] is
    k_cache.transpose(1, 2): pages of size S, slot b * S + position).  The rows
    have the cache's dtype, or are fp32 and rounded into an fp16 / bf16 cache.
    Slots outside the cache (the -1 of padding) are passed over.  A slot may
    occur once in a call; which of several rows for one slot stays is not
    defined.  Nothing else of the cache is touched.
    """
    r = _lib.fast_call("store_kv", "b2_store_kv", k, v, k_pages, v_pages, slots)
    if r is not None:
        return r
    for name, t in (("k", k), ("v", v)):
        if t.dim() != 3 or t.shape != k.shape or t.dtype != k.dtype:
            raise B2ShapeError("k and v must be [N, Hkv, D] of one shape and dtype")
        if t.stride(2) != 1 and t.shape[2] > 1:
            raise B2ShapeError(f"{name} must have a contiguous last dimension")
    N, Hkv, D = k.shape
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if t.dim() != 4 or t.shape != k_pages.shape or tuple(t.shape[2:]) != (Hkv, D):
            raise B2ShapeError(f"k_pages and v_pages must be [n_pages, page_size, {Hkv}, {D}] of one shape")
        if t.dtype != k_pages.dtype:
            raise B2DtypeError("k_pages and v_pages must share one dtype")
        if (t.stride(3) != 1 and D > 1) or _overlaps_itself(t):
            raise B2ShapeError(f"{name} must have a contiguous last dimension and must not overlap itself")
    if k.dtype not in _DT or k_pages.dtype not in _DT or (k.dtype != k_pages.dtype and k.dtype != torch.float32):
        raise B2DtypeError(f"store_kv: {k.dtype} rows into a {k_pages.dtype} cache")
    if slots.dtype != torch.int64 or slots.dim() != 1 or slots.shape[0] != N or not slots.is_contiguous():
        raise B2ShapeError(f"slots must be a contiguous int64 [{N}]")
    if k_pages.shape[1] == 0 or Hkv == 0 or D == 0:
        raise B2ShapeError("empty pages")
    _lib.check_device(k, v=v, k_pages=k_pages, v_pages=v_pages, slots=slots)
    with _lib.on_device(k):
        _lib.call("b2_store_kv", k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                  slots.data_ptr(), N, Hkv, D, k_pages.shape[0], k_pages.shape[1], _pi64x2(*k.stride()[:2]),
                  _pi64x2(*v.stride()[:2]), _lib.strides_arg(k_pages.stride()[:3]),
                  _lib.strides_arg(v_pages.stride()[:3]), _DT[k.dtype], _DT[k_pages.dtype], _lib.current_stream())
    return k_pages, v_pages
