"""Verification of drafted tokens against the target's probabilities (libkvrepair kvr_verify_drafts).

After ``tree_attention`` has run a step's drafted rows through the target model:
which of them hold, with the distribution that the target alone would give, and
the token that follows. What is random is given, so the same numbers give the same tokens.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _native
from .step_plan import StepPlan


class Verified(NamedTuple):
    """kept: int32 [requests], how many rows of each request hold, its node 0 among them; path: int32
    [rows], their nodes in order, packed as the plan's rows, -1 behind each request's; answers:
    int64 [requests], the token after the last of them, -1 for none."""

    kept: torch.Tensor
    path: torch.Tensor
    answers: torch.Tensor


def _probabilities(name: str, t, rows: int, vocab: int | None, device) -> int:
    """The row stride of a [rows, vocab] tensor."""
    if (not isinstance(t, torch.Tensor) or t.ndim != 2 or t.dtype != torch.float32 or t.device != device
            or t.shape[0] != rows or not 1 <= t.shape[1] <= 1 << 30 or (vocab is not None and t.shape[1] != vocab)):
        raise ValueError(f"{name} must be a float32 [{rows}, {'vocabulary' if vocab is None else vocab}] tensor on {device}")
    stride, one = t.stride()
    stride = stride if rows > 1 else t.shape[1]
    if (t.shape[1] > 1 and one != 1) or stride < t.shape[1]:
        raise ValueError(f"{name} must have contiguous rows of their own")
    return stride


def _numbers(name: str, t, dtype, count: int, device) -> int:
    if (not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device or t.ndim != 1 or t.shape[0] != count
            or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {str(dtype).replace('torch.', '')} tensor of {count} values on {device}")
    return t.data_ptr()


def verify_drafts(probs, tokens, plan: StepPlan, uniforms, draws, draft_probs=None) -> Verified:
    """Keep the drafted rows of a step that hold, and draw each request's next token, in one launch or
    (rows of more than 32768 tokens) two.

    The rows of a request are its plan's nodes (``max_rows`` at most 64): node 0 a
    token that is known, the last answer, the others drafts that hang on it, a chain or
    a tree. probs: float32 [rows, vocabulary], row i the target's distribution after node
    i; tokens: int64 [rows]; uniforms: float32 [rows] in [0, 1), row i's decides among the
    nodes that hang on node i; draws: float32 [requests] in [0, 1), for the answers.

    Without draft_probs, of the nodes that hang on a kept node a the first, in order, is
    kept with uniforms[a] < the sum of probs[a] over the tokens up to its own; the answer is drawn from
    probs[a] without their tokens. With draft_probs (float32 [rows, vocabulary], row i the
    distribution that the token after node i was drawn from; plans without ``parents``), the
    node that hangs on a is kept if uniforms[a] * draft_probs[a, token] < probs[a, token];
    the answer is drawn from max(probs[a] - draft_probs[a], 0). Where nothing hangs on
    the last kept node, or nothing is left, it is drawn from probs[a]. Entries of probs
    that are negative, infinite or NaN count as zero, and so do such differences.
    Differences are of the entries as they stand, and an entry of draft_probs by itself is
    what it is: an infinite or NaN one leaves nothing of its token, a negative one adds to
    it, and a product that is NaN or +inf keeps nothing. Tokens outside the vocabulary are
    not kept, and a node whose token an earlier one on the same node has does not count
    again. Sums and comparisons are in 64 bits; drawing takes the first token whose
    running sum exceeds the draw's share of the whole. A request without rows keeps none and
    answers -1, as one that failed."""
    if not isinstance(plan, StepPlan) or plan.masks is None:
        raise ValueError("plan must be a StepPlan of at most 64 rows a request")
    if not plan.planned:
        raise ValueError("plan has not been updated")
    device, rows, requests = plan.device, plan.rows, plan.requests
    ld = _probabilities("probs", probs, rows, None, device)
    vocab = probs.shape[1]
    ldd, drafts = 0, None
    if draft_probs is not None:
        if plan._desc.parents:
            raise ValueError("draft_probs are for chains: a tree's drafts are verified without them")
        ldd, drafts = _probabilities("draft_probs", draft_probs, rows, vocab, device), draft_probs.data_ptr()
    at = (_numbers("tokens", tokens, torch.int64, rows, device),
          _numbers("uniforms", uniforms, torch.float32, rows, device),
          _numbers("draws", draws, torch.float32, requests, device))
    if torch.is_grad_enabled() and (probs.requires_grad or uniforms.requires_grad or draws.requires_grad
                                    or (draft_probs is not None and draft_probs.requires_grad)):
        raise ValueError("verification is inference-only; detach gradient-bearing inputs")
    need = plan._verify_workspace.get(vocab)
    if need is None:
        need = int(_native.lib().kvr_verify_workspace_bytes(requests, vocab))
        _native.check(need, "kvr_verify_workspace_bytes")
        if len(plan._verify_workspace) >= 64:
            plan._verify_workspace.clear()
        plan._verify_workspace[vocab] = need
    # one allocation, the workspace (16-byte aligned) and the answers (8) first
    flat = torch.empty(need // 4 + 3 * requests + rows, dtype=torch.int32, device=device)
    _, answers, kept, path = flat.split((need // 4, 2 * requests, requests, rows))
    done = Verified(kept, path, answers.view(torch.int64))
    base = flat.data_ptr()
    out = base + need
    status = _native.launch(device, _native.lib().kvr_verify_drafts, probs.data_ptr(), ld, drafts, ldd, vocab, *at,
                            plan._desc_ref, out + 8 * requests, out + 12 * requests, out, base, need)
    _native.check(status, "kvr_verify_drafts")
    return done
