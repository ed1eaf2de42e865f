"""Attention over a paged cache, beside the packed projections (the C ABI's lloom_hip_paged_* calls).

A layer's cache is two f16 tensors of pages, k [pages, kv_heads, page_size, head_dim] and v [pages, kv_heads, head_dim,
page_size] (a page's tokens innermost, as the second product of attention reads them).  A step of a server is

    plan = paged_plan(cached, new, tokens, block_tables, free_pages, page_size)      # once
    cache.append(k, v, plan.slots)                                                   # each layer
    y = cache.attention(q, plan, window=..., sinks=...)                              # each layer

with one new token of each request (decode), chunks of prompts, or both.  Nothing here waits for the GPU: what only the
GPU can see (a page or slot out of range, no free page, lengths that do not fit) is left out of the result and raised by
the next paged_check().
"""
import ctypes
import math
from typing import NamedTuple

import torch

from .lib import LloomHipError, check, lib
from .quantized import _ACT_IDS, _ctx, _ctxs, _stream_of

HEAD_DIMS = (64, 96, 128, 256)


class PagedPlan(NamedTuple):
    """One step's bookkeeping, int32 on the GPU but for the slots (int64)."""
    q_start: torch.Tensor       # [requests + 1]: the requests' first rows among the step's tokens
    seq_lens: torch.Tensor      # [requests]: cached + new
    positions: torch.Tensor     # [tokens]
    slots: torch.Tensor         # [tokens]: page * page_size + place, -1 for rows of no request
    taken: torch.Tensor         # [1]: pages taken from the front of the free list
    block_tables: torch.Tensor  # the caller's, with the new pages in it


def _need(ok, code, msg):
    if not ok:
        raise LloomHipError(code, msg)


def _ints(index, dtype, **tensors):
    """Each tensor (by its argument's name, with its dimensions) is of dtype, on GPU `index`, dense in its last."""
    for what, (t, dim) in tensors.items():
        if t.dtype is not dtype or t.dim() != dim or t.get_device() != index or (t.stride(-1) != 1 and t.numel()):
            raise LloomHipError(1, f"{what}: {tuple(t.shape)} {t.dtype} on {t.device} is not a {dtype} tensor of {dim} "
                                   f"dimension(s), dense in its last, on GPU {index}")


def _gpu(t, what):
    """The GPU that t is on, and the handle of its context."""
    i = t.get_device()
    if i < 0:
        raise LloomHipError(1, f"{what}: the cache is not on a HIP device")
    return i, _ctxs.get(i) or _ctx(i)


def paged_plan(cached, new, tokens, block_tables, free_pages, page_size):
    """Block tables, slots and positions of a step from the requests' lengths: cached [requests] tokens each has in the
    cache, new [requests] more, `tokens` rows in all (more than their sum: a padded batch).  block_tables [requests,
    max_blocks] is updated in place with pages from the front of free_pages; all int32 on one GPU."""
    i, ctx = _gpu(cached, "paged_plan")
    _ints(i, torch.int32, cached=(cached, 1), new=(new, 1), block_tables=(block_tables, 2), free_pages=(free_pages, 1))
    n = cached.shape[0]
    _need(new.shape[0] == n and block_tables.shape[0] == n, 3,
          f"paged_plan: {n} cached lengths, {new.shape[0]} new ones and {block_tables.shape[0]} tables")
    # one allocation for the five small outputs, the slots (8 bytes each) first
    at = 2 * tokens
    buf = cached.new_empty(at + tokens + 2 * n + 2)
    base = buf.data_ptr()
    p_pos = base + 4 * at
    p_start = p_pos + 4 * tokens
    p_seq = p_start + 4 * (n + 1)
    check(lib().lloom_hip_paged_plan(ctx, cached.data_ptr(), new.data_ptr(), n, tokens, block_tables.data_ptr(),
                                     _table_stride(block_tables), block_tables.shape[1], free_pages.data_ptr(),
                                     free_pages.shape[0], page_size, p_start, p_seq, p_pos, base, p_seq + 4 * n,
                                     _stream_of(i)))
    slots, positions, q_start, seq_lens, taken = buf.split((at, tokens, n + 1, n, 1))
    return PagedPlan(q_start, seq_lens, positions, slots.view(torch.int64), taken, block_tables)


def _table_stride(t):
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _cache_dims(k_cache, v_cache, what):
    pages, heads, page, dim = k_cache.shape if k_cache.dim() == 4 else (0, 0, 0, 0)
    if (k_cache.dtype is not torch.float16 or v_cache.dtype is not torch.float16 or not k_cache.is_contiguous()
            or not v_cache.is_contiguous() or v_cache.shape != (pages, heads, dim, page)
            or v_cache.get_device() != k_cache.get_device()):
        raise LloomHipError(3, f"{what}: k {tuple(k_cache.shape)} {k_cache.dtype} and v {tuple(v_cache.shape)} "
                               f"{v_cache.dtype} are not one cache: contiguous f16 [pages, heads, page, dim] and "
                               f"[pages, heads, dim, page]")
    return pages, heads, page, dim


def _rows(t, heads, dim, what):
    """t [tokens, heads, dim] with its heads dense; rows may be apart (slices of one projection).  A layout that the
    kernels do not read (heads apart, rows not 16-byte aligned) is copied."""
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != dim:
        raise LloomHipError(3, f"{what}: {tuple(t.shape)} is not [tokens, {heads}, {dim}]")
    if t.dtype not in _ACT_IDS:
        raise LloomHipError(2, f"{what}: {t.dtype} is not an activation dtype of the HIP arm (F32 or F16)")
    s = t.stride()
    if ((s[2] != 1 or s[1] != dim or s[0] < heads * dim or s[0] * t.element_size() % 16 or t.data_ptr() % 16)
            and t.numel()):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def paged_append(k_cache, v_cache, k, v, slots):
    """Rows k and v [tokens, kv_heads, head_dim] (f32 or f16) into the cache at slots [tokens] (int64; negative: not
    stored).  No two rows of a call share a slot."""
    pages, heads, page, dim = _cache_dims(k_cache, v_cache, "paged_append")
    i = k_cache.get_device()
    k, v = _rows(k, heads, dim, "paged_append k"), _rows(v, heads, dim, "paged_append v")
    _ints(i, torch.int64, slots=(slots, 1))
    if k.dtype is not v.dtype or k.get_device() != i or v.get_device() != i:
        raise LloomHipError(2, f"paged_append: k {k.dtype} on {k.device} and v {v.dtype} on {v.device} differ, or the cache "
                               f"is on {k_cache.device}")
    n = slots.shape[0]
    if k.shape[0] != n or v.shape[0] != n:
        raise LloomHipError(3, f"paged_append: {k.shape[0]} and {v.shape[0]} rows, {n} slots")
    i, ctx = _gpu(k_cache, "paged_append")
    check(lib().lloom_hip_paged_append(ctx, _ACT_IDS[k.dtype], k.data_ptr(),
                                       max(k.stride(0), heads * dim), v.data_ptr(), max(v.stride(0), heads * dim),
                                       slots.data_ptr(), n, k_cache.data_ptr(), v_cache.data_ptr(), pages, heads, dim,
                                       page, _stream_of(i)))


def paged_attention(q, k_cache, v_cache, block_tables, q_start, seq_lens, scale=None, window=0, sinks=0, max_new=None,
                    out=None):
    """Causal attention of q [tokens, heads, head_dim] (f32 or f16) over the cache; out is of q's type and shape.  Rows
    q_start[b] .. q_start[b + 1] are request b's last tokens, the last at position seq_lens[b] - 1; query head h reads key
    head h // (heads // kv_heads).  The token at position p sees position j <= p with window = 0, j > p - window or
    j < sinks.  A q_start that falls anywhere or is negative leaves the call out (out is zero, paged_check() raises);
    one that passes the number of rows leaves out those that are not there (paged_check() raises).  scale: 1 / sqrt(head_dim) by default.  max_new: the most new tokens of any request, where the caller
    knows it (1 for a decode step): only speed and roundings depend on it."""
    pages, heads, page, dim = _cache_dims(k_cache, v_cache, "paged_attention")
    if q.dim() != 3 or heads == 0 or q.shape[1] == 0 or q.shape[1] % heads:
        raise LloomHipError(3, f"paged_attention: q {tuple(q.shape)} is not [tokens, heads, {dim}] with a multiple of "
                               f"{heads} heads")
    q = _rows(q, q.shape[1], dim, "paged_attention q")
    i = k_cache.get_device()
    _ints(i, torch.int32, block_tables=(block_tables, 2), q_start=(q_start, 1), seq_lens=(seq_lens, 1))
    n, (tokens, all_heads, _) = seq_lens.shape[0], q.shape
    if q_start.shape[0] != n + 1 or block_tables.shape[0] != n or q.get_device() != i:
        raise LloomHipError(3, f"paged_attention: {n} lengths, {q_start.shape[0]} starts, {block_tables.shape[0]} tables; q "
                               f"on {q.device}, cache on {k_cache.device}")
    i, ctx = _gpu(k_cache, "paged_attention")
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.dtype is not q.dtype or out.shape != q.shape or not out.is_contiguous() or out.get_device() != i:
        raise LloomHipError(3, f"paged_attention: out {tuple(out.shape)} {out.dtype} does not fit the contiguous {q.dtype} "
                               f"output {tuple(q.shape)}")
    check(lib().lloom_hip_paged_attention(ctx, _ACT_IDS[q.dtype], q.data_ptr(),
                                          max(q.stride(0), all_heads * dim), tokens, k_cache.data_ptr(),
                                          v_cache.data_ptr(), pages, heads, all_heads // heads, dim, page, block_tables.data_ptr(),
                                          _table_stride(block_tables), block_tables.shape[1],
                                          q_start.data_ptr(), seq_lens.data_ptr(), n,
                                          1.0 / math.sqrt(dim) if scale is None else scale, window, sinks,
                                          max_new or 0, out.data_ptr(), _stream_of(i)))
    return out


def paged_attention_workspace_bytes(tokens, requests, kv_heads, group, head_dim, max_new=None):
    """The workspace an attention call of these sizes takes (reserve_workspace it before a capture)."""
    out = ctypes.c_size_t()
    check(lib().lloom_hip_paged_attention_workspace_bytes(tokens, requests, kv_heads, group, head_dim, max_new or 0,
                                                          ctypes.byref(out)))
    return out.value


def paged_check(device=0):
    """Wait for the device and raise what its calls have recorded since the last check (EPAGE: a page, slot or length
    that a paged call could not serve; EEXPERT: an id out of range)."""
    check(lib().lloom_hip_ctx_sync(_ctx(device)))


class PagedCache:
    """One layer's cache: the two page tensors and the calls on them."""

    def __init__(self, pages, page_size, kv_heads, head_dim, device="cuda"):
        _need(head_dim in HEAD_DIMS, 3, f"PagedCache: head_dim {head_dim} is none of {HEAD_DIMS}")
        _need(16 <= page_size <= 4096 and page_size & (page_size - 1) == 0, 3,
              f"PagedCache: page_size {page_size} is no power of two from 16 to 4096")
        _need(pages > 0 and kv_heads > 0, 1, f"PagedCache: {pages} pages of {kv_heads} heads")
        self.page_size = page_size
        self.k = torch.zeros(pages, kv_heads, page_size, head_dim, dtype=torch.float16, device=device)
        self.v = torch.zeros(pages, kv_heads, head_dim, page_size, dtype=torch.float16, device=device)

    def append(self, k, v, slots):
        paged_append(self.k, self.v, k, v, slots)

    def attention(self, q, plan, scale=None, window=0, sinks=0, max_new=None, out=None):
        return paged_attention(q, self.k, self.v, plan.block_tables, plan.q_start, plan.seq_lens, scale, window, sinks,
                               max_new, out)
