"""The order of a paged cache between steps (libkvrepair kvr_keep_rows, kvr_fork_requests, kvr_free_pages).

A step plan hands pages out; what happens to them afterwards stands here, all on the
GPU, on the current stream, without a copy to or from the host: ``keep_rows_`` moves a
step's accepted rows together, ``fork_`` continues requests as several, or in another
order, and ``FreePages.collect`` makes the free list anew from what requests still
hold, so that the pages of rejected rows, finished requests and dropped beams
come back, and a page that several requests share stays until the last lets it go.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Sequence

import torch

from .. import _native
from .step_plan import MAX_REQUESTS, StepPlan, _host_int
from .writeback import _nonoverlapping_layout


def _device_of(device) -> torch.device:
    device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
    if device.type != "cuda":
        raise ValueError("paged caches require a CUDA (ROCm) device")
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    from .indexed_attention import _require_gfx950

    _require_gfx950(device)
    return device


def _ints(name: str, t, count: int | None, device) -> tuple[int, int]:
    """Where an int32 tensor of one dimension begins and ends."""
    if (not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != device or t.ndim != 1
            or (count is not None and t.shape[0] != count) or not t.is_contiguous()):
        size = "any number of" if count is None else str(count)
        raise ValueError(f"{name} must be a contiguous int32 tensor of {size} values on {device}")
    at = t.data_ptr()
    return at, at + 4 * t.shape[0]


def _tables(name: str, t, requests: int | None, device) -> tuple[int, int, int]:
    """(address, end, row stride) of block tables."""
    if (not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != device or t.ndim != 2
            or (requests is not None and t.shape[0] != requests) or not 1 <= t.shape[0] <= MAX_REQUESTS
            or not t.shape[1]):
        size = f"1 to {MAX_REQUESTS}" if requests is None else str(requests)
        raise ValueError(f"{name} must be int32 [{size}, pages] on {device}")
    rows, width = t.shape
    stride, one = t.stride()
    stride = stride if rows > 1 else width
    if (width > 1 and one != 1) or stride < width:
        raise ValueError(f"{name} must have contiguous rows")
    at = t.data_ptr()
    return at, at + 4 * ((rows - 1) * stride + width), stride


class Fork(NamedTuple):
    """What ``PagedCache.fork_`` gives: lengths int32 [n] and block_tables int32 [n, pages] of the new requests,
    status int32 [n] (OK, NO_PAGES, TOO_LONG or INVALID of step_plan) and pages_taken int32 [1] of the free list."""

    lengths: torch.Tensor
    block_tables: torch.Tensor
    status: torch.Tensor
    pages_taken: torch.Tensor


class PagedCache:
    """The K and V pools of a model's layers, [1, Hkv, n_slots, D] each, of one layout.

    keys, values: one tensor a layer, any type of 1, 2 or 4 bytes, contiguous dims of a
    multiple of 16 bytes on 16-byte aligned rows; all keys share their strides, and all
    values theirs; no element belongs to two of them. Keeps the tensors; one that was given other storage (``.data``) needs a
    new PagedCache: calls of this one are refused."""

    def __init__(self, keys: Sequence[torch.Tensor], values: Sequence[torch.Tensor], *, page_size: int):
        keys, values = list(keys), list(values)
        if not keys or len(keys) != len(values):
            raise ValueError("a paged cache needs a K and a V pool for each layer")
        first = keys[0]
        if any(not isinstance(t, torch.Tensor) for t in (*keys, *values)) or first.ndim != 4 or first.shape[0] != 1:
            raise ValueError("pools must be [1, heads, n_slots, D] tensors")
        self.page_size = _host_int("page_size", page_size, 16, 1 << 30)
        _, heads, n_slots, dim = first.shape
        if self.page_size & (self.page_size - 1):
            raise ValueError("page_size must be a power of two")
        if not n_slots or n_slots % self.page_size or n_slots // self.page_size > (1 << 31) - 1:
            raise ValueError("n_slots must be a whole number of pages, fewer than 2^31")
        size = first.element_size()
        if size not in (1, 2, 4) or not heads or not dim or dim * size % 16:
            raise ValueError("a token of one head must be a multiple of 16 bytes, of elements of 1, 2 or 4")
        if heads * (dim * size // 16) * self.page_size > (1 << 31) - 1:
            raise ValueError("a page of one layer's K or V must be smaller than 32 GiB")
        device = _device_of(first.device)

        def strides(t) -> tuple[int, int]:
            head, row = t.stride()[1:3]
            return (head if heads > 1 else n_slots * row) * size, row * size  # a single head's may be anything

        for tensors in (keys, values):
            for t in tensors:
                if t.shape != first.shape or t.dtype != first.dtype or t.device != first.device:
                    raise ValueError("pools must share shape, dtype and device")
                if strides(t) != strides(tensors[0]):
                    raise ValueError("the K pools, and the V pools, must share their strides")
                if (t.stride(3) != 1 or any(s <= 0 or s % 16 for s in strides(t)) or t.data_ptr() % 16
                        or not _nonoverlapping_layout(t)):
                    raise ValueError("pools need contiguous dims, 16-byte aligned rows and elements of their own")
                if t.requires_grad:
                    raise ValueError("paged caches are inference-only; detach gradient-bearing pools")
        self.device, self.n_slots, self.layers = device, int(n_slots), len(keys)
        self._all = (*keys, *values)
        self._at = tuple(map(torch.Tensor.data_ptr, self._all))
        if len(set(self._at)) != len(self._at):
            raise ValueError("every pool must be a tensor of its own")
        n = len(keys)
        self._k = (ctypes.c_void_p * n)(*self._at[:n])
        self._v = (ctypes.c_void_p * n)(*self._at[n:])
        pools = self._pools = _native.Pools()
        pools.k, pools.v = self._k, self._v
        pools.k_head, pools.k_row = strides(keys[0])
        pools.v_head, pools.v_row = strides(values[0])
        pools.n_slots, pools.layers, pools.kv_heads = self.n_slots, n, int(heads)
        pools.row_bytes, pools.page_size = int(dim) * size, self.page_size
        self._ref = ctypes.byref(pools)

    def _same(self) -> None:
        if tuple(map(torch.Tensor.data_ptr, self._all)) != self._at:
            raise ValueError("a pool of the cache has other storage now: make a new PagedCache")

    def keep_rows_(self, plan: StepPlan, path, kept) -> None:
        """Move each request's accepted rows behind its committed tokens, in all layers: one launch a 64 layers.

        path: int32 [rows], kept: int32 [requests], as ``verify_drafts`` gives them: of
        request r the rows path[row_starts[r]] .. + kept[r], ascending nodes of the
        plan's step, become tokens length, length + 1, ...; then ``lengths += kept``
        commits them, before the plan's next update. A path counts up to its first entry
        that is not above the one before it or no node of its request."""
        if not isinstance(plan, StepPlan) or plan.device != self.device:
            raise ValueError("plan must be a StepPlan on the cache's device")
        if not plan.planned:
            raise ValueError("plan has not been updated")
        if plan.page_size != self.page_size or plan.n_slots != self.n_slots:
            raise ValueError("plan must be one of the cache's pages")
        path_at, _ = _ints("path", path, plan.rows, self.device)
        kept_at, _ = _ints("kept", kept, plan.requests, self.device)
        self._same()
        status = _native.launch(self.device, _native.lib().kvr_keep_rows, self._ref, plan._desc_ref, path_at, kept_at)
        _native.check(status, "kvr_keep_rows")

    def fork_(self, sources, lengths, block_tables, free_pages=None, free_start=None) -> Fork:
        """New requests that continue others: copies of one, the beams that are left, another order.

        sources: int32 [n], the request that each new one continues, -1 for an empty one;
        any may be named more than once, or not at all. lengths: int32 [requests],
        block_tables: int32 [requests, pages]; both are left as they were. Full pages
        are shared. A partly filled last page stays with the first request that continues
        its owner; every later one gets a page of free_pages (int32, from free_start (int32
        [1]) on), with the tokens copied in all layers, so that each can go on by itself.
        Behind a new request's pages its row of the tables is -1. Once the free list ends,
        later ones that need a page fail (NO_PAGES); they are empty, as those whose source
        is none (INVALID) or does not fit its table (TOO_LONG). A page of free_pages outside
        the pool is entered as it is and holds no copy, as in a step's plan: the list of a
        ``FreePages`` goes with its ``start``."""
        device = self.device
        at, end, stride = _tables("block_tables", block_tables, None, device)
        requests, width = block_tables.shape
        if width * self.page_size > 1 << 30:
            raise ValueError("block tables take at most 2^30 tokens a request")
        sources_at, _ = _ints("sources", sources, None, device)
        count = sources.shape[0]
        if not 1 <= count <= MAX_REQUESTS:
            raise ValueError(f"sources must be 1 to {MAX_REQUESTS} requests")
        lengths_at, _ = _ints("lengths", lengths, requests, device)
        free, given, start = None, 0, None
        if free_pages is not None:
            free, given = _ints("free_pages", free_pages, None, device)[0], free_pages.shape[0]
        if free_start is not None:
            start = _ints("free_start", free_start, 1, device)[0]
        self._same()
        flat = torch.empty(count * (width + 2) + 1, dtype=torch.int32, device=device)
        new, status, taken, pages = flat.split((count, count, 1, count * width))
        done = Fork(new, pages.view(count, width), status, taken)
        base = flat.data_ptr()
        desc = _native.ForkDesc(sources_at, lengths_at, at, free, start, base, base + 8 * count + 4, base + 4 * count,
                                base + 8 * count, stride, width, count, requests, width, given)
        status = _native.launch(device, _native.lib().kvr_fork_requests, self._ref, desc)
        _native.check(status, "kvr_fork_requests")
        return done


class FreePages:
    """The free list of a pool of ``count`` pages, as ``StepPlan.update`` and ``PagedCache.fork_`` take it:
    ``pages`` int32 [count], of which those from ``start`` int32 [1] on are free (all of them at first)."""

    def __init__(self, count: int, device: torch.device | str | int = "cuda"):
        self.count = _host_int("count", count, 1, (1 << 31) - 1)
        self.device = device = _device_of(device)
        need = int(_native.lib().kvr_free_pages_workspace_bytes(self.count))
        _native.check(need, "kvr_free_pages_workspace_bytes")
        with torch.inference_mode(False):
            self.pages = torch.arange(self.count, dtype=torch.int32, device=device)
            self.start = torch.empty(1, dtype=torch.int32, device=device).zero_()
            self._workspace = torch.empty(need, dtype=torch.uint8, device=device).zero_()
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(device).synchronize()  # the first use may be on any stream
        self._own = (self.pages.data_ptr(), self.start.data_ptr(), self._workspace.data_ptr())

    def collect(self, lengths, block_tables, *, page_size: int) -> "FreePages":
        """Make the list of the pages that no request holds, ascending, at the end of ``pages`` (-1 before them).

        lengths: int32 [requests], block_tables: int32 [requests, pages]. Request r holds the
        first ceil(lengths[r] / page_size) entries of its row; what stands behind them is not read, so a
        request that is done is one of length 0. Entries outside the pool hold nothing.
        The list and the memory that it is made in are this object's: collect, and
        what reads the list, must be ordered on one stream or by events. Returns itself."""
        device = self.device
        at, end, stride = _tables("block_tables", block_tables, None, device)
        requests, width = block_tables.shape
        page_size = _host_int("page_size", page_size, 16, 1 << 30)
        if page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two")
        first, last = _ints("lengths", lengths, requests, device)
        pages, start = self.pages.data_ptr(), self.start.data_ptr()
        for name, lo, hi in (("lengths", first, last), ("block_tables", at, end)):
            if lo < pages + 4 * self.count and hi > pages or lo < start + 4 and hi > start:
                raise ValueError(f"{name} must not be a tensor that the free list writes")
        if (pages, start, self._workspace.data_ptr()) != self._own:
            raise ValueError("the free list has other storage now: make a new FreePages")
        status = _native.launch(device, _native.lib().kvr_free_pages, first, at, stride, requests, width, page_size,
                                self.count, pages, start, self._own[2], self._workspace.shape[0])
        _native.check(status, "kvr_free_pages")
        return self
