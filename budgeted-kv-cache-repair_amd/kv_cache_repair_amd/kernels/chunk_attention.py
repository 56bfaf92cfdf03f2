"""Attention of chunks of new tokens over a paged cache (libkvrepair kvr_chunk_attention).

Beside ``tree_attention`` (at most 64 rows of a request, trees among them, and
unrounded probabilities): the next part of a prompt, or all of it, any number of rows
of each of many requests, each row over its request's committed tokens and the new
tokens up to itself.
"""

from __future__ import annotations

from .. import _native
from .step_plan import StepPlan
from .tree_attention import _prepare


def chunk_attention(q, keys, values, plan: StepPlan, scale=None, out=None):
    """Attend a step's rows to their requests' caches and to the rows before them.

    plan: a StepPlan with ``chunk_heads``, updated without ``parents``. q=[1,Hq,rows,D]
    packed as the plan's rows, keys/values=[1,Hkv,n_slots,D] pools that already hold the
    step's fresh rows, result=[1,Hq,rows,D] (or ``out``, any layout of such a shape).
    Row t of request r attends to the request's committed tokens and to its new tokens
    0..t. Rows of failed requests get zeros, as rows none of whose keys lies in the pool
    (one whose scores are all -inf gets NaN, as the softmax has it); rows behind the last
    request are zeros in a fresh result and left as they were in ``out``. What stands in a
    key that a row does not see, NaN and infinities included, does not reach it. float16 or
    bfloat16, D 64 or 128, scale > 0; inference only. Scores, maxima and sums are fp32;
    each probability is rounded to the inputs' type, half a step of its own at most
    (in float16 2^-37 of the row's largest for small ones), and a row is divided by the
    sum of what its values were weighted with.
    """
    if not isinstance(plan, StepPlan) or plan.chunk_heads is None:
        raise ValueError("plan must be a StepPlan with chunk_heads")
    if plan._desc.parents:
        raise ValueError("chunks have no parents: trees take tree_attention")
    at, out, fresh, dim, scale, strides, workspace, need = _prepare(q, keys, values, plan, scale, out, plan.chunk_heads,
                                                                    plan.chunk_workspace_bytes, plan._chunk_layouts)
    status = _native.launch(plan.device, _native.lib().kvr_chunk_attention, *at, plan._desc_ref,
                            plan._chunks.data_ptr(), *plan.chunk_heads, dim, scale, strides, fresh,
                            workspace.data_ptr(), need, _native.DTYPE_CODES[q.dtype])
    _native.check(status, "kvr_chunk_attention")
    return out
