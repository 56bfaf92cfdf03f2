"""Attention of a step's rows over a paged cache (libkvrepair kvr_tree_attention).

Beside ``indexed_causal_attention`` (selected rows of one request over its own
cache tensor): rows of many requests, each over its request's pages of one pool,
the new rows attending among themselves as the plan's masks say, causally or
along the branches of a tree of drafted tokens.
"""

from __future__ import annotations

import ctypes
import math
from numbers import Real

import torch

from .. import _native
from .step_plan import StepPlan
from .writeback import _nonoverlapping_layout

_DTYPES = (torch.float16, torch.bfloat16)


def _check(name: str, t, heads: int, rows: int, dim: int, like, unit: int) -> None:
    if not isinstance(t, torch.Tensor) or t.shape != (1, heads, rows, dim):
        raise ValueError(f"{name} must be a [1, {heads}, {rows}, {dim}] tensor")
    if t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must share the queries' dtype and device")
    head, row, one = t.stride()[1:]
    if one != 1 or row < dim or row % unit or row > 1 << 26 or head % unit or head <= 0 or \
            t.data_ptr() % (2 * unit):
        raise ValueError(f"{name} needs contiguous dims, head and row strides of {unit} elements and a "
                         f"{2 * unit}-byte aligned base")


def tree_attention(q, keys, values, plan: StepPlan, scale=None, out=None):
    """Attend a step's rows to their requests' caches and to their own ancestors.

    q=[1,Hq,rows,D] packed as the plan's rows, keys/values=[1,Hkv,n_slots,D]
    pools that already hold the step's fresh rows, result=[1,Hq,rows,D] (or
    ``out``, any layout of such a shape). Row t of request r attends to the
    request's committed tokens and to the nodes of its mask. Rows that see
    nothing (padding nodes, failed requests) get zeros; rows behind the last
    request are zeros in a fresh result and left as they were in ``out``. What
    stands in a key that a row does not see, NaN and infinities included, does
    not reach it. float16 or bfloat16, D 64 or 128, scale > 0; inference only.
    QK^T and PV run on the MFMA with fp32 statistics and sums, probabilities as
    a hi + lo pair of 16-bit values (not rounded to the input dtype).
    """
    if not isinstance(plan, StepPlan) or plan.heads is None:
        raise ValueError("plan must be a StepPlan with heads")
    if not plan.planned:
        raise ValueError("plan has not been updated")
    q_heads, kv_heads = plan.heads
    if not isinstance(q, torch.Tensor) or q.ndim != 4 or q.dtype not in _DTYPES or q.device != plan.device:
        raise ValueError("q must be a four-dimensional float16 or bfloat16 tensor on the plan's device")
    dim = q.shape[3]
    if dim not in (64, 128):
        raise ValueError("head dimension must be 64 or 128")
    _check("q", q, q_heads, plan.rows, dim, q, 8)
    _check("keys", keys, kv_heads, plan.n_slots, dim, q, 8)
    _check("values", values, kv_heads, plan.n_slots, dim, q, 8)
    if max(keys.stride(2), values.stride(2)) * 2 * plan.page_size > (1 << 32) - 1:
        raise ValueError("a page of keys or values must span less than 4 GiB")
    if scale is None:
        scale = dim ** -0.5
    if isinstance(scale, bool) or not isinstance(scale, Real) or not 0 < scale < math.inf:
        raise ValueError("attention scale must be a positive finite host real number")
    fresh = out is None
    if fresh:
        out = torch.empty((1, plan.rows, q_heads, dim), dtype=q.dtype, device=q.device).transpose(1, 2)
    else:
        _check("out", out, q_heads, plan.rows, dim, q, 4)
        mine = out.untyped_storage().data_ptr()
        if not _nonoverlapping_layout(out) or any(mine == t.untyped_storage().data_ptr() for t in (q, keys, values)):
            raise ValueError("out must have storage of its own")
    if q.requires_grad or keys.requires_grad or values.requires_grad or out.requires_grad:
        raise ValueError("tree attention is inference-only; detach gradient-bearing inputs")
    need = plan.workspace_bytes(dim)
    workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    strides = (ctypes.c_int64 * 12)(*q.stride()[1:], *keys.stride()[1:], *values.stride()[1:], *out.stride()[1:])
    with torch.cuda.device(q.device):
        status = _native.lib().kvr_tree_attention(
            q.data_ptr(), keys.data_ptr(), values.data_ptr(), out.data_ptr(), ctypes.byref(plan._desc), dim,
            float(scale), strides, fresh, workspace.data_ptr(), need, _native.DTYPE_CODES[q.dtype],
            _native.stream_handle(q.device))
    _native.check(status, "kvr_tree_attention")
    return out
