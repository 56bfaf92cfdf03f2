"""The plan of one step of several requests over one paged cache (libkvrepair kvr_step_plan).

``IndexedPlan`` holds the selected rows of one request, validated on the host.
A ``StepPlan`` holds the rows that several requests add in one step (a prompt's
rows paged in, one new token each, trees of drafted tokens) and is built on the
GPU from the requests' lengths, so a step needs no copy to or from the host and
can be captured in a graph: new pages are taken from a free list and entered in
the block tables, and every row gets its slot, its position and the mask of its
ancestors. ``indexed_kv_scatter_`` and ``rope_indexed_kv_scatter_`` write a
step's fresh rows by its slots, ``tree_attention`` attends with it.

A pool is a cache tensor [1, Hkv, n_slots, D]; page p is its slots
[p * page_size, (p + 1) * page_size). Token j of request r lies in slot
``block_tables[r, j // page_size] * page_size + j % page_size``.
"""

from __future__ import annotations

import ctypes
from numbers import Integral

import torch

from .. import _native

MAX_REQUESTS = 4096
MAX_NODES = 64  # rows of one request that attend
OK, NO_PAGES, TOO_LONG, INVALID = range(4)  # StepPlan.status


def _host_int(name: str, value, low: int, high: int) -> int:
    if isinstance(value, bool) or not isinstance(value, Integral) or not low <= value <= high:
        raise ValueError(f"{name} must be a host integer in [{low}, {high}]")
    return int(value)


class StepPlan:
    """Sizes and device metadata of a step; ``update`` builds the plan of one.

    ``requests`` requests with at most ``max_rows`` rows each and room for
    ``rows`` packed rows in all; ``heads`` = (query heads, KV heads) makes it a
    plan for ``tree_attention`` too (``max_rows`` at most 64). The tensors are
    allocated once, as a plan without requests, and rewritten by every ``update``:

    row_starts   int32 [requests + 1]: request r's rows are [row_starts[r], row_starts[r + 1])
    request      int32 [rows]: each row's request, -1 behind the last
    slots        int64 [rows]: where the row's K/V go; -1: nowhere
    positions    int64 [rows]: the row's position, committed tokens plus ancestors; -1: none
    masks        int64 [rows]: the row's ancestors and itself, one bit a node; None above 64 rows a request
    status       int32 [requests]: OK, NO_PAGES (the free list ended), TOO_LONG (for its row of the
                 table) or INVALID (negative length, count outside [0, max_rows], rows past ``rows``)
    pages_taken  int32 [1]: pages of the free list that went to requests

    A request that fails takes no page, and its rows get no slot and attend to
    nothing; once the free list ends, later requests that need a page fail too.
    Requests may share pages of committed tokens (a common prefix), but not a page
    that a step writes: the partly filled last one is each request's own.
    An update, and everything that reads the plan, must be ordered on one
    stream or by events, like any tensor that is rewritten; calls that only read it
    may run at once. One thread at a time may update it. Attention reads the block
    tables of the last ``update`` call, a captured one too, and the rest of the plan
    of the last that ran: a plan that a graph updates takes its eager updates with
    the tables that the graph has.
    """

    def __init__(self, requests: int, rows: int, *, page_size: int, n_slots: int, table_width: int,
                 max_rows: int = 1, heads: tuple[int, int] | None = None, device: torch.device | str | int = "cuda"):
        self.requests = _host_int("requests", requests, 1, MAX_REQUESTS)
        self.rows = _host_int("rows", rows, 1, (1 << 31) - 1)
        self.max_rows = _host_int("max_rows", max_rows, 1, (1 << 30))
        self.page_size = _host_int("page_size", page_size, 16, 1 << 30)
        self.n_slots = _host_int("n_slots", n_slots, 1, (1 << 62))
        self.table_width = _host_int("table_width", table_width, 1, (1 << 30) // self.page_size)
        if self.page_size & (self.page_size - 1):
            raise ValueError("page_size must be a power of two")
        if self.n_slots % self.page_size or self.n_slots // self.page_size > (1 << 31) - 1:
            raise ValueError("n_slots must be a whole number of pages, fewer than 2^31")
        if self.table_width * self.requests > (1 << 31) - 1:
            raise ValueError("block tables must have fewer than 2^31 entries")
        self.heads = None
        if heads is not None:
            if not isinstance(heads, (tuple, list)) or len(heads) != 2:
                raise ValueError("heads must be (query heads, KV heads)")
            q_heads, kv_heads = heads
            self.heads = (_host_int("query heads", q_heads, 1, 1 << 16), _host_int("KV heads", kv_heads, 1, 1 << 16))
            if q_heads % kv_heads:
                raise ValueError("query head count must be divisible by KV head count")
            if self.max_rows > MAX_NODES:
                raise ValueError(f"attention takes at most {MAX_NODES} rows of a request")
            if self.requests * (-(-self.table_width * self.page_size // 128) + 1) > 1 << 30:
                raise ValueError("attention takes block tables of at most 2^37 tokens in all")
        device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if device.type != "cuda":
            raise ValueError("step plans require a CUDA (ROCm) device")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        from .indexed_attention import _require_gfx950

        _require_gfx950(device)
        self.device = device
        lib = _native.lib()
        schedule = 0
        if self.heads:
            schedule = int(lib.kvr_step_schedule_ints(self.requests, self.max_rows, *self.heads))
            _native.check(schedule, "kvr_step_schedule_ints")
        masks = self.rows if self.max_rows <= MAX_NODES else 0
        wide = 2 * (2 * self.rows + masks)  # int32 of the int64 tensors
        with torch.inference_mode(False):
            # one allocation, the schedule first (32-byte aligned, whole 16 bytes). What an update that has only
            # been captured leaves is a plan without requests: no row, no work
            flat = torch.empty(schedule + wide + self.rows + 2 * self.requests + 2, dtype=torch.int32, device=device)
            flat.zero_()
            flat[schedule:schedule + wide + self.rows] = -1
            longs, rest = flat[schedule:schedule + wide].view(torch.int64), flat[schedule + wide:]
            self.slots, self.positions = longs[:self.rows], longs[self.rows:2 * self.rows]
            self.masks = longs[2 * self.rows:].zero_() if masks else None
            self._schedule = flat[:schedule] if schedule else None
            self.request, rest = rest[:self.rows], rest[self.rows:]
            self.row_starts, rest = rest[:self.requests + 1], rest[self.requests + 1:]
            self.status, self.pages_taken = rest[:self.requests], rest[self.requests:]
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(device).synchronize()  # the first update may be on any stream
        self._own = (flat.data_ptr(), flat.data_ptr() + 4 * flat.shape[0])
        self.block_tables = None  # the tables of the last update
        self.planned = False
        desc = self._desc = _native.StepDesc()
        for name in ("row_starts", "request", "slots", "positions", "status", "pages_taken"):
            setattr(desc, name, getattr(self, name).data_ptr())
        desc.masks = self.masks.data_ptr() if masks else None
        desc.schedule = self._schedule.data_ptr() if schedule else None
        desc.n_slots, desc.requests, desc.rows, desc.max_rows = self.n_slots, self.requests, self.rows, self.max_rows
        desc.page_size, desc.table_width = self.page_size, self.table_width
        desc.q_heads, desc.kv_heads = self.heads or (0, 0)
        self._desc_ref = ctypes.byref(desc)
        self._workspace_bytes: dict[int, int] = {}
        self._layouts: dict = {}  # tree_attention's checked layouts

    def _vector(self, name: str, tensor, count: int | None, tables: int, end: int) -> int:
        """The address of an input beside block tables at [tables, end)."""
        if (not isinstance(tensor, torch.Tensor) or tensor.dtype != torch.int32 or tensor.device != self.device
                or tensor.ndim != 1 or (count is not None and tensor.shape[0] != count) or not tensor.is_contiguous()):
            size = "any number of" if count is None else str(count)
            raise ValueError(f"{name} must be a contiguous int32 tensor of {size} values on {self.device}")
        address = tensor.data_ptr()
        first, last = self._own
        if address < last and address + 4 * tensor.shape[0] > first:
            raise ValueError(f"{name} must not be a tensor that the plan writes")
        if address < end and address + 4 * tensor.shape[0] > tables:
            raise ValueError(f"{name} must not overlap block_tables")
        return address

    def update(self, lengths, counts, block_tables, free_pages=None, parents=None, free_start=None) -> "StepPlan":
        """Plan a step on the current stream: one launch, no host synchronisation.

        lengths, counts: int32 [requests], tokens in the cache and rows of this
        step. block_tables: int32 [requests, table_width], whose first
        ceil(length / page_size) entries are the request's pages; the entries
        after them that this step's rows need are written, with the pages of
        free_pages (int32) from free_start (int32 [1], on the device) on. What
        stands behind a request's length is not read: the pages of rows that were not
        accepted go to waste unless they are put on the free list again.
        parents: int32 [rows], each packed row's parent as a node index within
        its request, -1 for one that hangs on the cache; None: each row follows
        the one before it. A parent that is neither -1 nor an earlier node marks a
        padding node: it and its descendants get no slot and attend to nothing.
        Returns the plan itself."""
        requests, width = self.requests, self.table_width
        if (not isinstance(block_tables, torch.Tensor) or block_tables.dtype != torch.int32
                or block_tables.device != self.device or block_tables.shape != (requests, width)):
            raise ValueError(f"block_tables must be int32 [{requests}, {width}] on {self.device}")
        stride, one = block_tables.stride()
        stride = stride if requests > 1 else width
        if (width > 1 and one != 1) or stride < width:
            raise ValueError("block_tables must have contiguous rows")
        if parents is not None and self.masks is None:
            raise ValueError(f"trees have at most {MAX_NODES} nodes")
        tables = block_tables.data_ptr()
        end = tables + 4 * ((requests - 1) * stride + width)
        if tables < self._own[1] and end > self._own[0]:
            raise ValueError("block_tables must not be a tensor that the plan writes")
        at = (self._vector("lengths", lengths, requests, tables, end),
              self._vector("counts", counts, requests, tables, end))
        free, given = None, 0
        if free_pages is not None:
            free, given = self._vector("free_pages", free_pages, None, tables, end), free_pages.shape[0]
        start = None if free_start is None else self._vector("free_start", free_start, 1, tables, end)
        tree = None if parents is None else self._vector("parents", parents, self.rows, tables, end)
        # from here on the plan is the new step's
        self.planned = False
        desc = self._desc
        desc.lengths, desc.counts = at
        desc.tables, desc.table_stride = tables, stride
        desc.free_pages, desc.free_count, desc.free_start, desc.parents = free, given, start, tree
        self.block_tables = block_tables
        status = _native.launch(self.device, _native.lib().kvr_step_plan, self._desc_ref)
        _native.check(status, "kvr_step_plan")
        self.planned = True
        return self

    def workspace_bytes(self, head_dim: int) -> int:
        """Bytes of the partial results of ``tree_attention`` calls with this plan."""
        need = self._workspace_bytes.get(head_dim)
        if need is None:
            need = int(_native.lib().kvr_tree_workspace_bytes(self._desc_ref, head_dim))
            _native.check(need, "kvr_tree_workspace_bytes")
            self._workspace_bytes[head_dim] = need
        return need
