"""Paged KV cache for the decode path.

The reference's decode reads a dense, padded [B,H,N,D] cache
(src/pallas_flash/kernels/decoding.py:86-103) and has no cache update.  Here
the cache can also live in fixed-size pages, so sequences grow token by
token without re-allocating or copying:

  k_pool, v_pool  [num_pages, H_kv, page_size, D]  fp16/bf16, or fp8 (e4m3)
                  with per-tensor scales; H_kv divides the query heads
  page_table      int32 [B, max_pages_per_seq]  physical page of each
                  logical page of a sequence (-1 = unmapped)
  kv_lens         int32 [B]                     tokens held per sequence

`paged_decode` (pu_decode_paged) gives the same result as
`pallas_flash_decoding` on the dense cache the pages describe;
`kv_append` (pu_kv_append) writes one token per sequence and advances
kv_lens on the device.  `PageAllocator` keeps the host-side free list and
table; `PagedKVCache` ties the pieces together.

A serving loop that never leaves the device uses `DevicePagedKVCache`: per
step, `plan_append` (pu_page_plan) makes table rows, slots and positions of
the next tokens from lengths alone, `qk_norm_rope_append`
(pu_qk_norm_rope_append) norms and rotates q and k and writes keys and values
to their slots, and `paged_decode` attends; the three calls can be captured
into a CUDA graph and replayed.

Long contexts are served with less reading:

  - `page_bounds` (pu_page_bounds) keeps the elementwise minimum and maximum of
    each page's keys, `select_pages` (pu_select_pages) lists for each K/V head
    the pages whose bound of the scores is highest, and `paged_decode` over such
    lists (pu_decode_paged_heads) reads those pages only.
  - `paged_decode` with `shared_lens` (pu_decode_paged_shared) reads pages that
    sequences have in common once for all of them.
"""
from __future__ import annotations

import functools
import math
from typing import NamedTuple, Optional, Sequence

import numpy as np
import torch

from .. import _lib
from ..ops.rotary import _DT as _DT_ROPE, _NONE, _check_angles, _check_weight, _pack, _refuse_tangents, _rows
from .decoding import _DT, _DT_KV, DecodeWorkspace

__all__ = ["PageAllocator", "PagedKVCache", "DevicePagedKVCache", "AppendPlan", "PageSelection", "paged_decode",
           "kv_append", "plan_append", "qk_norm_rope_append", "empty_bounds", "page_bounds", "select_pages"]


def _check_pool(k_pool: torch.Tensor, v_pool: torch.Tensor, page_table: torch.Tensor,
                kv_lens: torch.Tensor, kinds=_DT):
    shape, kind, rows = k_pool.shape, k_pool.dtype, page_table.shape
    if shape != v_pool.shape or len(shape) != 4:
        raise ValueError("k_pool and v_pool must both be [num_pages, H, page_size, D]")
    if kind != v_pool.dtype or kind not in kinds:
        raise ValueError("pools must share one dtype, fp16 or bf16" + (" or fp8 (e4m3)" if kinds is _DT_KV else ""))
    if len(rows) == 3 and kinds is _DT_KV and page_table.dtype == torch.int32:
        if rows[1] != shape[1]:
            raise ValueError(f"page lists of each K/V head must be int32 [B, {shape[1]}, pages]")
        if kv_lens.dtype != torch.int32 or kv_lens.shape != rows[:2]:
            raise ValueError("kv_lens of page lists must be int32 [B, H_kv]")
    else:
        if page_table.dtype != torch.int32 or len(rows) != 2:
            raise ValueError("page_table must be int32 [B, max_pages_per_seq]")
        if kv_lens.dtype != torch.int32 or kv_lens.numel() != rows[0]:
            raise ValueError("kv_lens must be int32 [B]")
    at = k_pool.get_device()             # -1 on the host
    if not (at >= 0 and v_pool.get_device() == at and page_table.get_device() == at and kv_lens.get_device() == at
            and k_pool.is_contiguous() and v_pool.is_contiguous() and page_table.is_contiguous()
            and kv_lens.is_contiguous()):
        raise ValueError("pools, page table and lengths must be contiguous CUDA tensors on one device")


@functools.lru_cache(maxsize=256)
def _gqa_bytes(device: int, B: int, H: int, H_kv: int, max_pages: int, page_size: int, D: int) -> int:
    return int(_lib.lib().pu_decode_paged_gqa_workspace_size(B, H, H_kv, max_pages, page_size, D))


@functools.lru_cache(maxsize=64)
def _cta_counters(device: int) -> int:
    return 4 * torch.cuda.get_device_properties(device).multi_processor_count


@functools.lru_cache(maxsize=256)
def _shared_bytes(device: int, B: int, H: int, H_kv: int, groups: int, D: int) -> int:
    return int(_lib.lib().pu_decode_paged_shared_workspace_size(B, H, H_kv, groups, D))


def paged_decode(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                 page_table: torch.Tensor, kv_lens: torch.Tensor, *,
                 sm_scale: Optional[float] = None, return_lse: bool = False,
                 k_scale: float = 1.0, v_scale: float = 1.0,
                 shared_lens: Optional[torch.Tensor] = None, shared_groups: Optional[torch.Tensor] = None):
    """One decode step over a paged cache -> o bf16 [B,H,1,D] (and lse fp32 [B,H]).

    q [B,H,1,D] fp16/bf16; the pools hold H_kv heads, H a multiple of H_kv,
    in fp16, bf16 or fp8 (e4m3; keys and values are the stored values times
    k_scale and v_scale).  A sequence of length 0 gives o = 0, lse = -inf.

    page_table [B,H_kv,pages] with kv_lens [B,H_kv] are lists of their own for
    each K/V head, as `select_pages` makes them: the head's queries attend the
    first kv_lens tokens of its list and read no other page.

    shared_lens int32 [n] (n up to 64) says that sequences hold the same pages:
    those of group i, sequences shared_groups[i] <= b < shared_groups[i + 1] (int32
    [n + 1]; without it one group is the whole batch), have the same first
    shared_lens[i] tokens, which are then read once for the group, through the
    table row of one of its sequences.  Only whole pages are shared.  A sequence
    that holds fewer tokens than that attends them by itself; a group in which too few
    hold as many shares nothing, nor does a call where that would save little or
    whose scale is not positive.
    The result is that of the call without it, up to the order of sums and the rounding of the
    softmax weights: those of shared tokens are rounded once to the pools' 16-bit type, to
    f16 over fp8 pools (which keep three e4m3 parts without it), and so are all tokens' of 16-bit
    pools, as in the grouped decode (with a query head to each K/V head the call
    without it keeps them in fp32).  Where q and the pools have different 16-bit
    types, or e4m3 pools heads of 64, it is that call.  Up to 8192 sequences; the scratch, kept for
    the stream, is 39 MB at D = 128 and more for larger batches (pu_decode_paged_shared)."""
    _check_pool(k_pool, v_pool, page_table, kv_lens, _DT_KV)
    P, H_kv, page_size, D = k_pool.shape
    rows = page_table.shape
    by_head = len(rows) == 3
    B, max_pages = rows[0], rows[-1]
    qs, dev = q.shape, k_pool.device
    H = qs[1] if len(qs) == 4 else 0
    if qs != (B, H, 1, D) or H == 0 or H_kv == 0 or H % H_kv or q.dtype not in _DT or q.device != dev:
        raise ValueError(f"q must be fp16/bf16 CUDA [{B}, multiple of {H_kv}, 1, {D}] on {dev}")
    if shared_lens is not None:
        _check_shared(shared_lens, shared_groups, by_head, dev)
    elif shared_groups is not None:
        raise ValueError("shared_groups without shared_lens")
    if not q.is_contiguous():
        q = q.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(D)
    lib = _lib.lib()
    with _lib.on_device(dev) as stream:
        o = _lib.empty((B, H, 1, D), (H * D, D, D, 1), torch.bfloat16, dev)
        lse = _lib.empty((B, H), (H, 1), torch.float32, dev)
        if B == 0:
            return (o, lse) if return_lse else o
        if shared_lens is not None and (k_pool.dtype == q.dtype or (D == 128 and k_pool.dtype not in _DT)):
            groups = shared_lens.numel()
            ws = DecodeWorkspace.get(dev, _shared_bytes(dev.index, B, H, H_kv, groups, D), _cta_counters(dev.index))
            _lib.check(lib.pu_call_packed(_lib.DECODE_PAGED_SHARED, _lib.pack_shared(
                q.data_ptr(), _DT[q.dtype], k_pool.data_ptr(), v_pool.data_ptr(), _DT_KV[k_pool.dtype],
                page_table.data_ptr(), max_pages, P, page_size, kv_lens.data_ptr(), shared_lens.data_ptr(),
                0 if shared_groups is None else shared_groups.data_ptr(), groups, o.data_ptr(), lse.data_ptr(),
                ws.data_ptr(), ws.numel(), B, H, H_kv, D, sm_scale, k_scale, v_scale, stream)),
                "pu_decode_paged_shared")
        elif not by_head and H == H_kv and k_pool.dtype in _DT and k_scale == 1.0 and v_scale == 1.0:
            need = int(lib.pu_decode_paged_workspace_size(B, H, max_pages, page_size, D))
            ws = DecodeWorkspace.get(dev, need, 4 * B * H)
            _lib.check(lib.pu_decode_paged(q.data_ptr(), _DT[q.dtype], k_pool.data_ptr(),
                                           v_pool.data_ptr(), _DT[k_pool.dtype], page_table.data_ptr(),
                                           max_pages, P, page_size, kv_lens.data_ptr(), o.data_ptr(),
                                           lse.data_ptr(), ws.data_ptr(), ws.numel(), B, H, D,
                                           float(sm_scale), stream), "pu_decode_paged")
        else:
            # a counter for each CTA (one an SM), or in the query-head kernel for each head
            ws = DecodeWorkspace.get(dev, _gqa_bytes(dev.index, B, H, H_kv, max_pages, page_size, D),
                                     max(4 * B * H, _cta_counters(dev.index)))
            _lib.check(lib.pu_call_packed(
                _lib.DECODE_PAGED_HEADS if by_head else _lib.DECODE_PAGED_GQA, _lib.pack_decode(
                    q.data_ptr(), _DT[q.dtype], k_pool.data_ptr(), v_pool.data_ptr(), _DT_KV[k_pool.dtype],
                    page_table.data_ptr(), max_pages, P, page_size, kv_lens.data_ptr(), o.data_ptr(), lse.data_ptr(),
                    ws.data_ptr(), ws.numel(), B, H, H_kv, D, sm_scale, k_scale, v_scale, stream)),
                "pu_decode_paged_heads" if by_head else "pu_decode_paged_gqa")
    return (o, lse) if return_lse else o


def _check_shared(shared_lens: torch.Tensor, shared_groups: Optional[torch.Tensor], by_head: bool, dev: torch.device):
    if by_head:
        raise ValueError("page lists of each K/V head have no shared prefix")
    n = shared_lens.numel()
    if shared_lens.dtype != torch.int32 or shared_lens.dim() != 1 or not 1 <= n <= 64:
        raise ValueError("shared_lens must be int32 [n], n from 1 to 64")
    if shared_groups is None:
        if n != 1:
            raise ValueError("more than one shared prefix needs shared_groups")
    elif shared_groups.dtype != torch.int32 or shared_groups.shape != (n + 1,):
        raise ValueError(f"shared_groups must be int32 [{n + 1}]")
    if shared_lens.device != dev or not shared_lens.is_contiguous() or \
            (shared_groups is not None and (shared_groups.device != dev or not shared_groups.is_contiguous())):
        raise ValueError(f"shared_lens and shared_groups must be contiguous on {dev}")


class PageSelection(NamedTuple):
    """Pages chosen for each K/V head (select_pages), as `paged_decode` takes them."""
    pages: torch.Tensor        # int32 [B, H_kv, count]  pool pages in the sequence's order; -1 behind the last
    lens: torch.Tensor         # int32 [B, H_kv]  tokens in them


def _check_bounds_size(D: int):
    if D != 128 and D != 64:
        raise ValueError(f"page bounds of head size {D} (supported: 64, 128)")


def empty_bounds(k_pool: torch.Tensor) -> torch.Tensor:
    """Room for the bounds of a pool's pages: [num_pages, H_kv, 2, D] in the pool's
    16-bit type, fp16 for an fp8 pool (which holds every e4m3 value).  [..., 0, :] is
    the minimum and [..., 1, :] the maximum of a page's keys as stored.  D is 64 or 128."""
    P, H_kv, _, D = k_pool.shape
    _check_bounds_size(D)
    return torch.zeros((P, H_kv, 2, D), dtype=k_pool.dtype if k_pool.dtype in _DT else torch.float16,
                       device=k_pool.device)


def _check_bounds(bounds: torch.Tensor, shape):
    if len(shape) != 4 or shape[2] != 2 or bounds.dtype not in _DT:
        raise ValueError("bounds must be fp16/bf16 [num_pages, H_kv, 2, D]")
    _check_bounds_size(shape[3])
    if bounds.get_device() < 0 or not bounds.is_contiguous():
        raise ValueError("bounds must be a contiguous CUDA tensor")


def page_bounds(k_pool: torch.Tensor, slots: torch.Tensor, bounds: torch.Tensor) -> None:
    """Bring the pages' bounds up to date with keys that were written to `slots`.

    slots int32 [T] as `plan_append` makes them (negative: no key): the rows of a
    page stand together and in order, and a page begins with its row 0.  For each
    page that a slot names, `bounds` (empty_bounds) becomes the elementwise minimum
    and maximum of the keys in these rows, and of what it was where the page's row 0
    is not among them.  A NaN makes its element's bounds NaN.  A slot past the pool is
    reported (device_status detail 309) and left out."""
    shape, pool, kind = bounds.shape, k_pool.shape, k_pool.dtype
    _check_bounds(bounds, shape)
    P, H_kv, _, D = shape
    if len(pool) != 4 or pool[0] != P or pool[1] != H_kv or pool[3] != D or kind not in _DT_KV:
        raise ValueError(f"k_pool must be fp16, bf16 or fp8 (e4m3) [{P}, {H_kv}, page_size, {D}]")
    if bounds.dtype != (kind if kind in _DT else torch.float16):
        raise ValueError("bounds must have the pool's 16-bit dtype, fp16 for an fp8 pool")
    if slots.dtype != torch.int32 or slots.dim() != 1 or not slots.is_contiguous():
        raise ValueError("slots must be a contiguous int32 [T]")
    at = bounds.get_device()
    if k_pool.get_device() != at or slots.get_device() != at or not k_pool.is_contiguous():
        raise ValueError("pool, slots and bounds must be contiguous CUDA tensors on one device")
    if (k_pool.requires_grad or bounds.requires_grad) and torch.is_grad_enabled():
        raise ValueError("page_bounds writes a cache's bounds and has no gradient")
    with _lib.on_device(bounds.device) as stream:
        _lib.check(_lib.lib().pu_call_packed(_lib.PAGE_BOUNDS, _lib.pack_bounds(
            k_pool.data_ptr(), _DT_KV[kind], slots.data_ptr(), bounds.data_ptr(), P, pool[2], H_kv, D, slots.numel(),
            stream)), "pu_page_bounds")


def select_pages(q: torch.Tensor, bounds: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor, count: int, *,
                 page_size: int, first: int = 1, last: int = 1) -> PageSelection:
    """The pages that each K/V head's queries attend, `count` of them at most.

    A page's score is sum over the head's queries and their elements of
    max(q_d lo_d, q_d hi_d): no key of the page scores higher, summed over the
    queries.  The first `first` and the last `last` pages of a sequence are always
    chosen, then those with the highest scores (the lowest index among equals), all
    in the sequence's order; a sequence of no more than `count` pages keeps all of
    them.  Scores are summed in 64 bits.  Table entries outside the pool are never
    chosen and reported (device_status detail 310); queries and bounds are finite.

    q [B,H,1,D] fp16/bf16, bounds of `page_bounds`, page_table int32
    [B,max_pages_per_seq] (up to 24576), kv_lens int32 [B].  The scores' scale and
    the scale of an fp8 pool change nothing.  The result goes into
    `paged_decode(q, k_pool, v_pool, chosen.pages, chosen.lens)`."""
    shape, rows, qs, kind = bounds.shape, page_table.shape, q.shape, q.dtype
    _check_bounds(bounds, shape)
    P, H_kv, _, D = shape
    if page_table.dtype != torch.int32 or len(rows) != 2:
        raise ValueError("page_table must be int32 [B, max_pages_per_seq]")
    B, max_pages = rows
    if kv_lens.dtype != torch.int32 or kv_lens.shape != (B,):
        raise ValueError(f"kv_lens must be int32 [{B}]")
    dev, at = bounds.device, bounds.get_device()
    H = qs[1] if len(qs) == 4 else 0
    if qs != (B, H, 1, D) or H == 0 or H_kv == 0 or H % H_kv or kind not in _DT or q.get_device() != at:
        raise ValueError(f"q must be fp16/bf16 CUDA [{B}, multiple of {H_kv}, 1, {D}] on {dev}")
    if page_table.get_device() != at or kv_lens.get_device() != at or not page_table.is_contiguous() \
            or not kv_lens.is_contiguous():
        raise ValueError("page table and lengths must be contiguous and on the bounds' device")
    if count < 1 or first < 0 or last < 0 or first + last > count:
        raise ValueError(f"{first} first and {last} last of {count} pages")
    if not q.is_contiguous():
        q = q.contiguous()
    with _lib.on_device(dev) as stream:
        pages = _lib.empty((B, H_kv, count), (H_kv * count, count, 1), torch.int32, dev)
        lens = _lib.empty((B, H_kv), (H_kv, 1), torch.int32, dev)
        if B:
            _lib.check(_lib.lib().pu_call_packed(_lib.SELECT_PAGES, _lib.pack_select(
                q.data_ptr(), _DT[kind], bounds.data_ptr(), _DT[bounds.dtype], page_table.data_ptr(), max_pages, P,
                page_size, kv_lens.data_ptr(), pages.data_ptr(), lens.data_ptr(), count, first, last, B, H, H_kv, D,
                stream)), "pu_select_pages")
    return PageSelection(pages, lens)


def kv_append(k_new: torch.Tensor, v_new: torch.Tensor, k_pool: torch.Tensor,
              v_pool: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor) -> None:
    """Write k_new/v_new [B,H,1,D] at position kv_lens[b] and advance kv_lens (on the device)."""
    _check_pool(k_pool, v_pool, page_table, kv_lens)
    P, H, page_size, D = k_pool.shape
    B, max_pages = page_table.shape
    for t in (k_new, v_new):
        if t.shape != (B, H, 1, D) or t.dtype != k_pool.dtype or not t.is_cuda:
            raise ValueError(f"new k/v must be CUDA {k_pool.dtype} [{B}, {H}, 1, {D}]")
    k_new, v_new = k_new.contiguous(), v_new.contiguous()
    _lib.check(_lib.lib().pu_kv_append(k_new.data_ptr(), v_new.data_ptr(), _DT[k_pool.dtype],
                                       k_pool.data_ptr(), v_pool.data_ptr(),
                                       page_table.data_ptr(), max_pages, P, page_size,
                                       kv_lens.data_ptr(), B, H, D,
                                       torch.cuda.current_stream().cuda_stream),
               "pu_kv_append")


class AppendPlan(NamedTuple):
    """Where a batch's new tokens go (plan_append); row t is a row of the packed batch."""
    slots: torch.Tensor        # int32 [T]  page * page_size + row in the page; -1: none
    positions: torch.Tensor    # int32 [T]
    seq_ids: torch.Tensor      # int32 [T]  sequence of the row; -1 behind the last token
    cu_new: torch.Tensor       # int32 [B+1]  first row of each sequence
    kv_lens: torch.Tensor      # int32 [B]  lengths with the new tokens
    cursor: torch.Tensor       # int64 [2]  head and tail of the ring after
    page_table: torch.Tensor   # int32 [B, max_pages_per_seq] after


def plan_append(page_table: torch.Tensor, kv_lens: torch.Tensor, new_lens: torch.Tensor,
                free_ring: torch.Tensor, cursor: torch.Tensor, *, page_size: int, num_tokens: int,
                release: Optional[torch.Tensor] = None, inplace: bool = False,
                shared_lens: Optional[torch.Tensor] = None, sources: Optional[torch.Tensor] = None) -> AppendPlan:
    """Table rows, slots and positions of a batch's next tokens, on the device.

    kv_lens, new_lens int32 [B]: tokens held, and tokens that each sequence
    gets now; num_tokens: rows of the packed batch (sequence after sequence),
    at least the sum of new_lens, the rest are padding rows.  The free pages
    are free_ring[i % num_pages] for cursor[0] <= i < cursor[1]; pages are
    taken from its head in sequence order.  Where `release` [B] (bool) is set,
    a sequence's pages (which no other may share) go to the ring's tail first and
    it starts empty; they are handed out from the next call on.

    A sequence that does not fit its table row or the batch's rows, or for
    which the free pages do not last, is refused: it stays as it is (empty, if
    it was released in the call), its rows get slot -1, and device_status()
    reports it (detail 307 or 308).  Pages are counted in sequence order, those
    that a refused sequence asked for as well, so later ones that need a page are
    refused with it.  Where the ring has no room for what is released, released
    sequences are refused and keep pages and lengths (detail 308); entries of a
    released row that name no page are reported (307) and left out of the ring.

    With `inplace` the table, lengths and cursor are advanced where they are
    (the same tensors come back); otherwise new ones are returned and only the
    ring's places behind its tail are written.

    shared_lens and sources int32 [B] (with `inplace`) say which sequences begin with
    pages of another one: sequence b's first shared_lens[b] tokens are sources[b]'s
    (DevicePagedKVCache.share).  A release then returns only a sequence's own pages and
    clears its entries; a sequence whose pages others hold that are not
    released with it is not released, its rows get slot -1, and it is reported (detail 311)."""
    if page_table.dim() != 2 or page_table.dtype != torch.int32:
        raise ValueError("page_table must be int32 [B, max_pages_per_seq]")
    B, max_pages = page_table.shape
    dev = page_table.device
    if kv_lens.dtype != torch.int32 or new_lens.dtype != torch.int32 or kv_lens.shape != (B,) or new_lens.shape != (B,):
        raise ValueError(f"kv_lens and new_lens must be int32 [{B}]")
    if cursor.dtype != torch.int64 or cursor.shape != (2,):
        raise ValueError("cursor must be int64 [2]")
    if free_ring.dim() != 1 or free_ring.dtype != torch.int32:
        raise ValueError("free_ring must be int32 [num_pages]")
    if not (page_table.is_cuda and kv_lens.device == dev and new_lens.device == dev and free_ring.device == dev
            and cursor.device == dev and page_table.is_contiguous() and kv_lens.is_contiguous()
            and new_lens.is_contiguous() and free_ring.is_contiguous() and cursor.is_contiguous()):
        raise ValueError("the plan's tensors must be contiguous CUDA tensors on one device")
    if release is not None and (release.dtype not in (torch.bool, torch.uint8) or release.shape != (B,)
                                or release.device != dev or not release.is_contiguous()):
        raise ValueError(f"release must be a contiguous bool [{B}] on {dev}")
    if shared_lens is not None or sources is not None:
        if not inplace or shared_lens is None or sources is None:
            raise ValueError("shared_lens and sources come together, with inplace")
        for t in (shared_lens, sources):
            if t.dtype != torch.int32 or t.shape != (B,) or t.device != dev or not t.is_contiguous():
                raise ValueError(f"shared_lens and sources must be contiguous int32 [{B}] on {dev}")
    if inplace and abs(new_lens.data_ptr() - kv_lens.data_ptr()) < 4 * B:
        raise ValueError("new_lens must not overlap kv_lens when they are advanced in place")
    T = int(num_tokens)
    if T < 0:
        raise ValueError("num_tokens must not be negative")
    with _lib.on_device(dev) as stream:
        slots, positions, seq_ids, cu, lens_out = torch.split_with_sizes(
            torch.empty(3 * T + 2 * B + 1, dtype=torch.int32, device=dev), (T, T, T, B + 1, B))
        if inplace:
            table_out, lens_out, cursor_out = page_table, kv_lens, cursor
        else:
            table_out, cursor_out = torch.empty_like(page_table), torch.empty_like(cursor)
        if shared_lens is not None and release is not None:
            _lib.check(_lib.lib().pu_page_plan_shared(
                page_table.data_ptr(), max_pages, kv_lens.data_ptr(), new_lens.data_ptr(), release.data_ptr(),
                free_ring.data_ptr(), free_ring.numel(), cursor.data_ptr(), int(page_size), slots.data_ptr(),
                positions.data_ptr(), seq_ids.data_ptr(), cu.data_ptr(), shared_lens.data_ptr(), sources.data_ptr(),
                B, T, stream), "pu_page_plan_shared")
            return AppendPlan(slots, positions, seq_ids, cu, lens_out, cursor_out, table_out)
        _lib.check(_lib.lib().pu_page_plan(
            page_table.data_ptr(), table_out.data_ptr(), max_pages, kv_lens.data_ptr(), lens_out.data_ptr(),
            new_lens.data_ptr(), None if release is None else release.data_ptr(), free_ring.data_ptr(),
            free_ring.numel(), cursor.data_ptr(), cursor_out.data_ptr(), int(page_size), slots.data_ptr(),
            positions.data_ptr(), seq_ids.data_ptr(), cu.data_ptr(), B, T, stream), "pu_page_plan")
    return AppendPlan(slots, positions, seq_ids, cu, lens_out, cursor_out, table_out)


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, inv_freq: torch.Tensor,
                        positions: torch.Tensor, slots: torch.Tensor, k_pool: torch.Tensor,
                        v_pool: torch.Tensor, *, q_weight: Optional[torch.Tensor] = None,
                        k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                        sections: Optional[Sequence[int]] = None, interleaved: bool = False,
                        k_scale: float = 1.0, v_scale: float = 1.0) -> torch.Tensor:
    """`ops.rotary.qk_norm_rope` of packed new tokens, keys and values written to the cache.

    q [T,H,D], k and v [T,H_kv,D] (views of one projection are read where they
    are); positions [T] or [axes,T]; slots int32 [T] as `plan_append` makes
    them: token t's normed and rotated key and its value go to row slots[t] %
    page_size of page slots[t] // page_size, divided by k_scale and v_scale
    (an fp8 pool saturates); a negative slot writes nothing, one past the pool
    is reported (device_status detail 306).  No slot may occur twice.  Returns
    the normed and rotated q, dense [T,H,D] (`.unsqueeze(2)` for a decode)."""
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError("q must be [T, H, D], k and v [T, H_kv, D]")
    T, H, D = q.shape
    H_kv, dev = k.shape[1], q.device
    if k_pool.dim() != 4 or k_pool.shape != v_pool.shape or k_pool.shape[1] != H_kv or k_pool.shape[3] != D:
        raise ValueError(f"pools must both be [num_pages, {H_kv}, page_size, {D}]")
    if k_pool.dtype != v_pool.dtype or k_pool.dtype not in _DT_KV:
        raise ValueError("pools must share one dtype: fp16, bf16 or fp8 (e4m3)")
    if q.dtype not in _DT_ROPE or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k and v must share one dtype: bf16, fp16 or fp32")
    if slots.dtype != torch.int32 or slots.shape != (T,) or not slots.is_contiguous():
        raise ValueError("slots must be a contiguous int32 [T]")
    if not (q.is_cuda and k.device == dev and v.device == dev and slots.device == dev and k_pool.device == dev
            and v_pool.device == dev):
        raise ValueError("q, k, v, slots and pools must be CUDA tensors on one device")
    if not k_pool.is_contiguous() or not v_pool.is_contiguous():
        raise ValueError("pools must be contiguous")
    if D % 16 or not 16 <= D <= 128 or H == 0 or H_kv == 0:
        raise ValueError(f"{H} and {H_kv} heads of size {D} (at least one head, a multiple of 16 up to 128)")
    if (q.requires_grad or k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        raise ValueError("qk_norm_rope_append writes a cache and has no gradient")
    _refuse_tangents(q, k, v, inv_freq, q_weight, k_weight)
    wq, wk = _check_weight(q_weight, D, dev, "q_weight"), _check_weight(k_weight, D, dev, "k_weight")
    if positions is None:
        raise ValueError("appended tokens need their positions")
    f, R, pos_st, axes, sizes = _check_angles(inv_freq, positions, sections, D, (T,), dev)
    with _lib.on_device(dev) as stream:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if T:
            q, k, v = _rows(q), _rows(k), _rows(v)
            by = lambda t: (0, t.stride(1), t.stride(0))     # noqa: E731
            desc = _pack(1, T, H, H_kv, D, q.dtype, R, interleaved, f, positions, (pos_st[0], 0, pos_st[1]), axes,
                         sizes, wq, wk, float(eps), by(q), by(k), by(v))
            _lib.check(_lib.lib().pu_qk_norm_rope_append(
                desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr(), slots.data_ptr(),
                k_pool.data_ptr(), v_pool.data_ptr(), _DT_KV[k_pool.dtype], k_pool.shape[0], k_pool.shape[2],
                float(k_scale), float(v_scale), stream), "pu_qk_norm_rope_append")
    return q_out


class PageAllocator:
    """Host-side page bookkeeping: a free list over `num_pages` physical pages
    and the [batch, max_pages_per_seq] table (-1 where unmapped).

    `reserve(b, n)` maps pages so that sequence b can hold n tokens;
    `release(b)` returns its pages.  Pure host logic (no device calls)."""

    def __init__(self, num_pages: int, page_size: int, batch: int, max_pages_per_seq: int):
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two >= 16")
        self.num_pages = int(num_pages)
        self.page_size = int(page_size)
        self.table = np.full((batch, max_pages_per_seq), -1, dtype=np.int32)
        self.mapped = np.zeros(batch, dtype=np.int64)   # table entries in use per sequence
        self._free = list(range(self.num_pages - 1, -1, -1))

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def reserve(self, b: int, n_tokens: int) -> bool:
        """Map pages for tokens [0, n_tokens) of sequence b; True if the table changed."""
        need = -(-int(n_tokens) // self.page_size)
        if need > self.table.shape[1]:
            raise ValueError(f"sequence {b}: {n_tokens} tokens exceed "
                             f"{self.table.shape[1]} pages of {self.page_size}")
        have = int(self.mapped[b])
        if need <= have:
            return False
        if need - have > len(self._free):
            raise MemoryError(f"page pool exhausted ({self.num_pages} pages)")
        for i in range(have, need):
            self.table[b, i] = self._free.pop()
        self.mapped[b] = need
        return True

    def release(self, b: int) -> None:
        for i in range(int(self.mapped[b]) - 1, -1, -1):
            self._free.append(int(self.table[b, i]))
            self.table[b, i] = -1
        self.mapped[b] = 0

    def shuffle(self, seed: int) -> None:
        """Randomise the order in which free pages are handed out."""
        np.random.Generator(np.random.PCG64(seed)).shuffle(self._free)


class PagedKVCache:
    """A paged KV cache on one GPU: pools, device page table and lengths.

    cache = PagedKVCache(B, H, D, num_pages=..., page_size=64, max_seq_len=...)
    cache.append(k_new, v_new)       # one token per sequence
    o = cache.decode(q)              # attention of q over every held token
    """

    def __init__(self, batch: int, heads: int, head_dim: int, *, num_pages: int,
                 page_size: int = 64, max_seq_len: int, dtype=torch.bfloat16, device=None):
        if dtype not in _DT:
            raise ValueError("cache dtype must be fp16 or bf16")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None \
            else torch.device(device)
        max_pages = -(-int(max_seq_len) // page_size)
        self.alloc = PageAllocator(num_pages, page_size, batch, max_pages)
        self.k_pool = torch.zeros((num_pages, heads, page_size, head_dim), dtype=dtype, device=device)
        self.v_pool = torch.zeros_like(self.k_pool)
        self.page_table = torch.from_numpy(self.alloc.table.copy()).to(device)
        self.kv_lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.host_lens = np.zeros(batch, dtype=np.int64)

    @property
    def page_size(self) -> int:
        return self.alloc.page_size

    def _push_table(self) -> None:
        self.page_table.copy_(torch.from_numpy(self.alloc.table))

    @classmethod
    def from_dense(cls, k: torch.Tensor, v: torch.Tensor, kv_lens, *, page_size: int = 64,
                   num_pages: Optional[int] = None, shuffle_seed: Optional[int] = None):
        """Pack dense caches [B,H,N,D] (first kv_lens[b] tokens of each sequence)."""
        B, H, N, D = k.shape
        lens = np.asarray(torch.as_tensor(kv_lens).cpu(), dtype=np.int64)
        pages_needed = int(sum(-(-int(n) // page_size) for n in lens))
        cache = cls(B, H, D, num_pages=num_pages or max(1, pages_needed), page_size=page_size,
                    max_seq_len=N, dtype=k.dtype, device=k.device)
        if shuffle_seed is not None:
            cache.alloc.shuffle(shuffle_seed)
        for b in range(B):
            n = int(lens[b])
            cache.alloc.reserve(b, n)
            for i in range(-(-n // page_size)):
                t0, t1 = i * page_size, min(n, (i + 1) * page_size)
                pg = int(cache.alloc.table[b, i])
                cache.k_pool[pg, :, :t1 - t0] = k[b, :, t0:t1]
                cache.v_pool[pg, :, :t1 - t0] = v[b, :, t0:t1]
        cache.host_lens[:] = lens
        cache.kv_lens.copy_(torch.from_numpy(lens.astype(np.int32)))
        cache._push_table()
        return cache

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor) -> None:
        """Append one token [B,H,1,D] to every sequence, mapping pages as needed."""
        changed = False
        for b in range(self.host_lens.shape[0]):
            changed |= self.alloc.reserve(b, int(self.host_lens[b]) + 1)
        if changed:
            self._push_table()
        kv_append(k_new, v_new, self.k_pool, self.v_pool, self.page_table, self.kv_lens)
        self.host_lens += 1

    def release(self, b: int) -> None:
        """Drop sequence b and return its pages to the pool."""
        self.alloc.release(b)
        self.host_lens[b] = 0
        self.kv_lens[b] = 0
        self._push_table()

    def decode(self, q: torch.Tensor, *, sm_scale: Optional[float] = None,
               return_lse: bool = False):
        return paged_decode(q, self.k_pool, self.v_pool, self.page_table, self.kv_lens,
                            sm_scale=sm_scale, return_lse=return_lse)


class DevicePagedKVCache:
    """A paged KV cache whose bookkeeping stays on the GPU: pools, page table,
    lengths and the ring of free pages.

    cache = DevicePagedKVCache(B, H_kv, D, num_pages=..., page_size=64, max_seq_len=...)
    plan = cache.plan(new_lens, num_tokens=T)                  # rows, slots, positions
    q = cache.append(q, k, v, plan, inv_freq, q_weight=wq, k_weight=wk)
    o = cache.decode(q)                                        # one new token each

    Nothing here reads from the device, so a step can be captured into a CUDA
    graph (new_lens, release, q, k and v in fixed buffers) and replayed.

    With `bounds=True` the cache keeps its pages' bounds (every `append` brings them
    up to date), and a step over a long context reads the pages that matter:

    o = cache.decode(q, pages=cache.select(q, 64))

    Sequences may begin with the pages of another one (`share`); `decode` reads them
    once where `shared_lens` says so.

    This is one layer's cache.  A model of several layers plans once a step
    (`plan_append`) and gives every layer the same slots, positions, table and
    lengths with pools of its own (`qk_norm_rope_append`, `paged_decode`): L of these
    caches would plan L times.  `decode` attends one token a sequence; a prompt's
    own attention runs on dense tensors (`qk_norm_rope`, whose keys are those
    that `append` stores, then `pallas_flash_attention`)."""

    def __init__(self, batch: int, kv_heads: int, head_dim: int, *, num_pages: int, page_size: int = 64,
                 max_seq_len: int, dtype=torch.bfloat16, k_scale: float = 1.0, v_scale: float = 1.0,
                 bounds: bool = False, device=None):
        if dtype not in _DT_KV:
            raise ValueError("cache dtype must be fp16, bf16 or fp8 (e4m3)")
        if page_size < 16 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two in [16, 4096]")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None \
            else torch.device(device)
        max_pages = -(-int(max_seq_len) // page_size)
        self.page_size, self.k_scale, self.v_scale = int(page_size), float(k_scale), float(v_scale)
        self.k_pool = torch.zeros((num_pages, kv_heads, page_size, head_dim), dtype=dtype, device=device)
        self.v_pool = torch.zeros_like(self.k_pool)
        self.bounds = empty_bounds(self.k_pool) if bounds else None
        self.page_table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=device)
        self.kv_lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.free_ring = torch.arange(num_pages, dtype=torch.int32, device=device)
        self.cursor = torch.tensor([0, num_pages], dtype=torch.int64, device=device)
        # tokens at the front of each sequence that are another one's, and whose (share)
        self.shared_lens, self.sources = torch.zeros_like(self.kv_lens), torch.full_like(self.kv_lens, -1)

    def plan(self, new_lens: torch.Tensor, *, num_tokens: int,
             release: Optional[torch.Tensor] = None) -> AppendPlan:
        """Map pages for new_lens [B] more tokens and advance the lengths (plan_append in place).
        A released sequence that shares pages gives them up; one whose pages others share stays
        until they are released or `unshare` (or are in the same call), and is reported (detail 311)."""
        return plan_append(self.page_table, self.kv_lens, new_lens, self.free_ring, self.cursor,
                           page_size=self.page_size, num_tokens=num_tokens, release=release, inplace=True,
                           shared_lens=self.shared_lens, sources=self.sources)

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: AppendPlan, inv_freq: torch.Tensor, *,
               positions: Optional[torch.Tensor] = None, **norm) -> torch.Tensor:
        """Norm and rotate the plan's tokens and write their keys and values
        (qk_norm_rope_append); positions [axes,T] replace the plan's where they have axes."""
        q = qk_norm_rope_append(q, k, v, inv_freq, plan.positions if positions is None else positions, plan.slots,
                                self.k_pool, self.v_pool, k_scale=self.k_scale, v_scale=self.v_scale, **norm)
        if self.bounds is not None:
            page_bounds(self.k_pool, plan.slots, self.bounds)
        return q

    def share(self, source: int, sequences: torch.Tensor, tokens: int) -> None:
        """Let empty `sequences` (int64, on the cache's device) begin with the first `tokens`
        of sequence `source`: whole pages of it, which they read and never write.  The pages stay
        `source`'s, which is not released before the sequences that share them.  A sequence
        that holds something, or for which `source` does not hold that many tokens, stays
        as it is and is reported (device_status detail 311)."""
        B = self.kv_lens.shape[0]
        if not -B <= int(source) < B:
            raise ValueError(f"sequence {source} of {B}")
        self._share(int(source) % B, sequences, tokens)

    def unshare(self, sequences: torch.Tensor, tokens: int) -> None:
        """Take the first `tokens`, shared with another sequence, out of `sequences`: what is left of
        them are their own pages (and what else they share).  A release does the same.  A sequence
        that shares fewer tokens, or whose pages others share, stays as it is and
        is reported (device_status detail 311)."""
        self._share(-1, sequences, tokens)

    def _share(self, source: int, sequences: torch.Tensor, tokens: int) -> None:
        B, max_pages = self.page_table.shape
        dev = self.page_table.device
        if tokens % self.page_size or not 0 <= tokens <= max_pages * self.page_size:
            raise ValueError(f"{tokens} tokens are not whole pages of {self.page_size} that a table row holds")
        at = torch.as_tensor(sequences, device=dev)
        if at.dtype == torch.bool:
            at = at.nonzero()
        elif at.numel() and (at.is_floating_point() or at.is_complex()):
            raise ValueError("sequences must be whole numbers")
        at = at.to(torch.int64).reshape(-1).contiguous()
        if not at.is_cuda:
            raise ValueError("the cache must be on a CUDA device")
        with _lib.on_device(dev) as stream:
            _lib.check(_lib.lib().pu_page_share(
                self.page_table.data_ptr(), max_pages, self.page_size, self.kv_lens.data_ptr(),
                self.shared_lens.data_ptr(), self.sources.data_ptr(), at.data_ptr(), at.numel(), source, int(tokens), B,
                stream), "pu_page_share")

    def select(self, q: torch.Tensor, count: int, *, first: int = 1, last: int = 1) -> PageSelection:
        """The pages that q [B,H,1,D] or [B,H,D] attends, for each K/V head (select_pages)."""
        if self.bounds is None:
            raise ValueError("this cache keeps no bounds of its pages (bounds=True)")
        return select_pages(q.unsqueeze(2) if q.dim() == 3 else q, self.bounds, self.page_table, self.kv_lens, count,
                            page_size=self.page_size, first=first, last=last)

    def decode(self, q: torch.Tensor, *, sm_scale: Optional[float] = None, return_lse: bool = False,
               pages: Optional[PageSelection] = None, shared_lens: Optional[torch.Tensor] = None,
               shared_groups: Optional[torch.Tensor] = None):
        """Attention of one token a sequence, q [B,H,1,D] or the appended [B,H,D], over all held tokens,
        or over `pages` that `select` chose; `shared_lens` and `shared_groups` as in paged_decode."""
        if q.dim() == 3:
            q = q.unsqueeze(2)
        table, lens = (self.page_table, self.kv_lens) if pages is None else pages
        return paged_decode(q, self.k_pool, self.v_pool, table, lens, sm_scale=sm_scale,
                            return_lse=return_lse, k_scale=self.k_scale, v_scale=self.v_scale,
                            shared_lens=shared_lens, shared_groups=shared_groups)
