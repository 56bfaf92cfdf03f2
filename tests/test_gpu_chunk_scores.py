"""chunk_attention's rows whose scores have no finite maximum, against the softmax in float64."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from test_gpu_chunk_attention import BF16, FP16, STRIDES, assert_close, exact, plan_of, tensors
from test_step_plan import _desc, walk


def exact_nan(q, k, v, plan, lengths, counts, page, pages, scale):
    """As `exact`, but a row that sees keys, all of whose scores are -inf, is NaN, as the softmax is."""
    out, size = exact(q, k, v, plan, lengths, counts, page, pages, scale)
    group = q.shape[1] // k.shape[1]
    for r in range(len(lengths)):
        length, count, start = int(lengths[r]), int(counts[r]), int(plan["row_starts"][r])
        if plan["status"][r] or not count:
            continue
        token = np.arange(length + count)
        page_of = plan["tables"][r][token // page].astype(np.int64)
        inside = torch.from_numpy((page_of >= 0) & (page_of < pages)).to(q.device)
        slot = torch.from_numpy(np.where((page_of >= 0) & (page_of < pages), page_of * page + token % page, 0)).to(q.device)
        see = torch.ones(count, length + count, dtype=torch.bool, device=q.device).tril(length) & inside
        for h in range(q.shape[1]):
            # the first dim is the only one that the queries of these tests have
            low = torch.isneginf(k[0, h // group][slot][:, 0])
            none = see.any(-1) & ~(see & ~low).any(-1)
            out[0, h, start:start + count][none] = math.nan
    return out, size


@pytest.mark.gpu
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, FP16), (64, BF16), (128, FP16)])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (32, 32)])
def test_scores_of_minus_infinity(gpu_device, dim, dtype, heads, kv_heads):
    """A row whose scores are all -inf is NaN, in whole tiles and in those that are cut between workers, and beside
    pages outside the pool; one that sees no key at all is zero; -inf among others is a weight of zero."""
    from kv_cache_repair_amd.kernels.chunk_attention import chunk_attention

    lengths, counts = np.array([0, 0, 48, 2000, 2000, 48, 300, 2000, 2000]), np.array([70, 90, 40, 96, 80, 66, 5, 30, 90])
    page, width = 16, 140
    need = -(-(lengths + counts) // page)
    pages = int(need.sum())
    order, tables, free, at = np.random.RandomState(1).permutation(pages), np.full((9, width), -1), [], 0
    for r in range(9):
        have = -(-int(lengths[r]) // page)
        tables[r, :have] = order[at:at + have]
        free += [pages] * (need[r] - have) if r == 7 else order[at + have:at + need[r]].tolist()
        at += need[r]
    tables[5, :3] = [pages, -1, 1 << 30]   # request 5's committed tokens: none of them can be read
    tables[7, :125] = pages                # no key of request 7, its new ones neither
    tables[8, :125:2] = -1                 # every other page of request 8
    rows = int(counts.sum()) + 3
    expect = walk(lengths, counts, tables, np.array(free), page, rows, 96, pages)
    assert not expect["status"].any()
    plan = plan_of(lengths, counts, tables, np.array(free), page, rows, 96, pages, (heads, kv_heads))
    q, k, v = tensors(6, heads, kv_heads, dim, rows, pages * page, dtype)
    q.zero_()
    q[..., 0] = 1.0

    def low(r, tokens):
        token = np.array(tokens)
        slot = expect["tables"][r][token // page].astype(np.int64) * page + token % page
        k[0, :, torch.from_numpy(slot[(slot >= 0) & (slot < pages * page)]).cuda(), 0] = -math.inf

    low(0, range(70))                      # no row of request 0 has a score
    low(1, range(50))                      # rows from 50 on have one
    low(2, range(0, 88, 2))                # every other key
    low(3, range(2096))                    # long, no score anywhere
    low(4, range(2040))                    # rows from 40 on have one
    low(5, range(48, 60))                  # of the keys in the pool the first 12
    low(8, range(2085))                    # the last 5 rows have one
    want, size = exact_nan(q, k, v, expect, lengths, counts, page, pages, 1.0)
    got = chunk_attention(q, k, v, plan, scale=1.0)
    starts = expect["row_starts"].tolist()
    none = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for r, n in ((0, 70), (1, 50), (3, 96), (4, 40), (5, 12), (8, 85)):
        none[starts[r]:starts[r] + n] = True
    assert torch.equal(torch.isnan(want), none[None, None, :, None].expand_as(want))
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert_close(got[:, :, ~none], want[:, :, ~none], size[:, :, ~none])
    assert not got[:, :, starts[7]:starts[8]].any()


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38, 1e39])
def test_a_scale_that_is_infinite_in_powers_of_two(scale):
    """Scores are scaled by scale * log2(e): an infinite one would make NaN of scores of zero."""
    from kv_cache_repair_amd import _native

    lib, at = _native.lib(), 1 << 30
    d = _desc(schedule=None, masks=None, parents=None, max_rows=100)
    need = lib.kvr_chunk_workspace_bytes(ctypes.byref(d), 8, 4, 64)
    assert lib.kvr_chunk_attention(at, at, at, at, ctypes.byref(d), at, 8, 4, 64, scale, _native.i64_array(STRIDES), 0, None,
                                   need, 2, None) == -1
