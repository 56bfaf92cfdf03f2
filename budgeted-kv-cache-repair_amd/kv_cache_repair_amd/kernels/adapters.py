"""Projections with a low-rank adapter of each row's own (libkvrepair kvr_adapter_linear).

Beside ``ProjectionPlan`` (one projection's weights, the same for all rows):
the rows of a step belong to many requests, each with an adapter of its own or
none, and share one projection:

  y[m] = W x[m] + scales[a] * up[a] (down[a] x[m])       a = ids[m]

for one weight or up to three concatenated ones (q/k/v), each with pools of its
own. A StepPlan's ``request`` gives the ids: ``adapter_of_request[plan.request]``, with one
entry more at the end, -1, for the rows of no request.
"""

from __future__ import annotations

import ctypes
from typing import Sequence

import torch

from .. import _native
from .projection import supported_weight

MAX_ROWS = 1 << 20
MAX_RANK = 512


class AdapterProjectionPlan:
    """Bound ctypes arguments of one projection and its adapters.

    weights: 1-3 [rows_i, k] (as ProjectionPlan takes them); down: for each a
    pool [adapters, rank, k], up: [adapters, rows_i, rank], contiguous, in the
    weights' dtype; scales: float32 [adapters]. rank a multiple of 8, at most 512
    (pad with zeros). An infinity in an up pool makes its columns of that
    adapter's rows infinite or NaN. Keeps the tensors; rows of the pools may be rewritten in
    place (an adapter swapped for another) between calls. A tensor that was given other storage
    (``.data``, a module moved or cast) needs a new plan: calls of this one are refused."""

    def __init__(self, weights: Sequence[torch.Tensor], down: Sequence[torch.Tensor], up: Sequence[torch.Tensor],
                 scales: torch.Tensor):
        weights, down, up = list(weights), list(down), list(up)
        if not 1 <= len(weights) <= 3 or not all(supported_weight(w) for w in weights):
            raise ValueError("adapter projection needs 1-3 supported fp16/bf16 weights")
        if len(down) != len(weights) or len(up) != len(weights):
            raise ValueError("adapter projection needs a down and an up pool for each weight")
        first = weights[0]
        k = int(first.shape[1])
        if not isinstance(down[0], torch.Tensor) or down[0].ndim != 3:
            raise ValueError("down pools must be [adapters, rank, k]")
        count, rank = int(down[0].shape[0]), int(down[0].shape[1])
        if count < 1 or rank < 8 or rank % 8 or rank > MAX_RANK:
            raise ValueError(f"adapters need a rank that is a multiple of 8, at most {MAX_RANK}")
        for w, a, b in zip(weights, down, up):
            if w.shape[1] != k or w.dtype != first.dtype or w.device != first.device:
                raise ValueError("adapter projection weights must share k, dtype and device")
            if w.shape[0] > 1 and w.stride(0) < k:
                raise ValueError("adapter projection weights must have rows of their own")
            for name, pool, shape in (("down", a, (count, rank, k)), ("up", b, (count, int(w.shape[0]), rank))):
                if (not isinstance(pool, torch.Tensor) or pool.shape != shape or pool.dtype != first.dtype
                        or pool.device != first.device or not pool.is_contiguous() or pool.data_ptr() % 16):
                    raise ValueError(f"{name} pools must be contiguous {list(shape)} tensors of the weights' dtype "
                                     "and device")
        if (not isinstance(scales, torch.Tensor) or scales.dtype != torch.float32 or scales.shape != (count,)
                or scales.device != first.device or not scales.is_contiguous()):
            raise ValueError("scales must be a contiguous float32 [adapters] tensor on the weights' device")
        if any(t.requires_grad for t in (*weights, *down, *up, scales)) and torch.is_grad_enabled():
            raise ValueError("adapter projections are inference-only; detach gradient-bearing tensors")
        self.k, self.dtype, self.device = k, first.dtype, first.device
        self.adapters, self.rank = count, rank
        self.n_out = sum(int(w.shape[0]) for w in weights)
        self._all = (*weights, *down, *up, scales)
        self._at = tuple(map(torch.Tensor.data_ptr, self._all))
        n = self._count = len(weights)
        self._w = (ctypes.c_void_p * n)(*(w.data_ptr() for w in weights))
        self._rows = (ctypes.c_int32 * n)(*(int(w.shape[0]) for w in weights))
        self._ldw = _native.i64_array([int(w.stride(0)) if w.shape[0] > 1 else k for w in weights])
        self._down = (ctypes.c_void_p * n)(*(t.data_ptr() for t in down))
        self._up = (ctypes.c_void_p * n)(*(t.data_ptr() for t in up))
        self._scales = scales.data_ptr()
        self._code = _native.DTYPE_CODES[self.dtype]
        self._workspace: dict[int, int] = {}

    def workspace_bytes(self, m: int) -> int:
        need = self._workspace.get(m)
        if need is None:
            need = int(_native.lib().kvr_adapter_linear_workspace_bytes(m, self._count, self._rows, self.k, self.rank))
            _native.check(need, "kvr_adapter_linear_workspace_bytes")
            if len(self._workspace) >= 64:
                self._workspace.clear()
            self._workspace[m] = need
        return need

    def __call__(self, x: torch.Tensor, ids: torch.Tensor) -> torch.Tensor:
        """y[..., n_out] of x[..., k] on the current stream; ids: int32, one for each row of x,
        the row's adapter, or a value outside [0, adapters) for none. Sums in fp32, rounded once."""
        if (not isinstance(x, torch.Tensor) or x.dtype != self.dtype or x.device != self.device or x.ndim < 1
                or x.shape[-1] != self.k):
            raise ValueError(f"x must be [..., {self.k}] in the weights' dtype and device")
        if tuple(map(torch.Tensor.data_ptr, self._all)) != self._at:
            raise ValueError("a weight, pool or scale of the plan has other storage now: make a new plan")
        if torch.is_grad_enabled() and (x.requires_grad or any(t.requires_grad for t in self._all)):
            raise ValueError("adapter projections are inference-only; detach gradient-bearing tensors")
        m = x.numel() // self.k
        if m > MAX_ROWS:
            raise ValueError(f"adapter projections take at most {MAX_ROWS} rows, got {m}")
        if (not isinstance(ids, torch.Tensor) or ids.dtype != torch.int32 or ids.device != self.device
                or ids.numel() != m or not ids.is_contiguous()):
            raise ValueError("ids must be a contiguous int32 tensor with one value for each row of x")
        y = torch.empty((*x.shape[:-1], self.n_out), dtype=self.dtype, device=self.device)
        if m == 0:
            return y
        rows = x if x.ndim == 2 else x.reshape(m, self.k)
        stride, one = rows.stride()
        ldx = stride if m > 1 else self.k
        at = rows.data_ptr()
        if (self.k > 1 and one != 1) or ldx % 8 or ldx < self.k or at % 16:
            raise ValueError("x needs contiguous rows at a stride of a multiple of 8, on a 16-byte aligned base")
        need = self.workspace_bytes(m)
        workspace = torch.empty(need, dtype=torch.uint8, device=self.device)
        status = _native.launch(
            self.device, _native.lib().kvr_adapter_linear, at, self._count, self._w, self._rows, self._ldw, self._down,
            self._up, self._scales, self.adapters, self.rank, ids.data_ptr(), y.data_ptr(), m, self.k, ldx, self.n_out,
            workspace.data_ptr(), need, self._code)
        _native.check(status, "kvr_adapter_linear")
        return y


def adapter_linear(x, weight, down, up, scales, ids) -> torch.Tensor:
    """``AdapterProjectionPlan([weight], [down], [up], scales)(x, ids)``."""
    return AdapterProjectionPlan([weight], [down], [up], scales)(x, ids)
