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


def _check(name: str, t, heads: int, rows: int, dim: int, like, unit: int) -> tuple[int, int, int]:
    """The strides of a tensor, those of a single head or row (which may be anything) as dense ones."""
    if not isinstance(t, torch.Tensor) or t.shape != (1, heads, rows, dim):
        raise ValueError(f"{name} must be a [1, {heads}, {rows}, {dim}] tensor")
    if t.dtype != like.dtype:
        raise ValueError(f"{name} must share the queries' dtype")
    head, row, one = t.stride()[1:]
    row = row if rows > 1 else dim
    head = head if heads > 1 else rows * row
    if one != 1 or row < dim or row % unit or row > 1 << 26 or head % unit or head <= 0:
        raise ValueError(f"{name} needs contiguous dims, and head and row strides of {unit} elements")
    return head, row, one


def _layout(q, keys, values, out, plan: StepPlan, heads: tuple[int, int], workspace_bytes) -> tuple:
    """(strides for the library, workspace bytes, head_dim, strides of a fresh result) of a
    call over tensors of these shapes, types and strides, which it checks."""
    q_heads, kv_heads = heads
    if not isinstance(q, torch.Tensor) or q.ndim != 4 or q.dtype not in _DTYPES:
        raise ValueError("q must be a four-dimensional float16 or bfloat16 tensor")
    dim = q.shape[3]
    if dim not in (64, 128):
        raise ValueError("head dimension must be 64 or 128")
    of_q = _check("q", q, q_heads, plan.rows, dim, q, 8)
    of_k = _check("keys", keys, kv_heads, plan.n_slots, dim, q, 8)
    of_v = _check("values", values, kv_heads, plan.n_slots, dim, q, 8)
    if max(of_k[1], of_v[1]) * 2 * plan.page_size > (1 << 32) - 1:
        raise ValueError("a page of keys or values must span less than 4 GiB")
    to = (dim, q_heads * dim, 1)  # token-major, as the output projection reads it
    if out is not None:
        to = _check("out", out, q_heads, plan.rows, dim, q, 4)
        if not _nonoverlapping_layout(out):
            raise ValueError("out must not overlap itself")
    strides = (ctypes.c_int64 * 12)(*of_q, *of_k, *of_v, *to)
    return strides, workspace_bytes(dim), dim, (plan.rows * q_heads * dim, dim, q_heads * dim, 1)


def _prepare(q, keys, values, plan: StepPlan, scale, out, heads: tuple[int, int], workspace_bytes, layouts: dict):
    """What a call of attention over a step's plan has in hand, checked: (addresses of q, keys, values and the result,
    the result, whether it is a fresh one, head_dim, scale, strides, workspace, its bytes)."""
    if not plan.planned:
        raise ValueError("plan has not been updated")
    Tensor = torch.Tensor
    if not (isinstance(q, Tensor) and isinstance(keys, Tensor) and isinstance(values, Tensor)
            and (out is None or isinstance(out, Tensor))):
        raise ValueError("q, keys, values and out must be tensors")
    # the checks of shapes, types and strides, once for each set of them
    key = (q.shape, q.stride(), q.dtype, keys.shape, keys.stride(), keys.dtype, values.shape, values.stride(),
           values.dtype, None if out is None else (out.shape, out.stride(), out.dtype))
    layout = layouts.get(key)
    if layout is None:
        if len(layouts) >= 64:
            layouts.clear()
        layout = layouts[key] = _layout(q, keys, values, out, plan, heads, workspace_bytes)
    strides, need, dim, fresh_strides = layout
    device = plan.device
    at = [q.data_ptr(), keys.data_ptr(), values.data_ptr()]
    if (q.device != device or keys.device != device or values.device != device
            or (out is not None and out.device != device)):
        raise ValueError("q, keys, values and out must be on the plan's device")
    if (at[0] | at[1] | at[2]) & 15 or (out is not None and out.data_ptr() & 7):
        raise ValueError("q, keys and values need 16-byte, out an 8-byte aligned base")
    if q.requires_grad or keys.requires_grad or values.requires_grad or (out is not None and out.requires_grad):
        raise ValueError("attention is inference-only; detach gradient-bearing inputs")
    if scale is None:
        scale = dim ** -0.5
    elif isinstance(scale, bool) or not isinstance(scale, Real) or not 0 < scale < math.inf:
        raise ValueError("attention scale must be a positive finite host real number")
    fresh = out is None
    if fresh:
        out = torch.empty_strided(q.shape, fresh_strides, dtype=q.dtype, device=device)
    else:
        mine = out.untyped_storage().data_ptr()
        if any(mine == t.untyped_storage().data_ptr() for t in (q, keys, values)):
            raise ValueError("out must have storage of its own")
    at.append(out.data_ptr())
    workspace = torch.empty(need, dtype=torch.uint8, device=device)
    return at, out, fresh, dim, scale, strides, workspace, need


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
    a hi + lo pair of 16-bit values: off by at most 2^-16 of each in bfloat16, by
    2^-22 of each or 2^-37 of the row's largest in float16.
    """
    if not isinstance(plan, StepPlan) or plan.heads is None:
        raise ValueError("plan must be a StepPlan with heads")
    at, out, fresh, dim, scale, strides, workspace, need = _prepare(q, keys, values, plan, scale, out, plan.heads,
                                                                    plan.workspace_bytes, plan._layouts)
    status = _native.launch(plan.device, _native.lib().kvr_tree_attention, *at, plan._desc_ref, dim, scale, strides,
                            fresh, workspace.data_ptr(), need, _native.DTYPE_CODES[q.dtype])
    _native.check(status, "kvr_tree_attention")
    return out
