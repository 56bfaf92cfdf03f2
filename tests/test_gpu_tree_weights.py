"""tree_attention where small weights are all of a result: in every 32 keys one has a zero
value and a score far above the others'. Weights that fp16 would lose beside it have to
stay what they are.

Tolerance: that of test_gpu_tree_attention, of which the scores here (one product of up to 20,
exact in fp32) take less, and in fp16 what the hi + lo pair leaves of a small weight: the
largest weight stands for 2^12 or more in it, and its smallest step is 2^-24, so each weight
is off by at most 2^-37 of the largest, which is 1 here before the sum divides all of them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_tree_attention import BF16, FP16, assert_close, exact
from test_step_plan import make, plan_of, walk


@pytest.mark.gpu
@pytest.mark.parametrize("depth", [4.0, 10.0, 14.0, 17.0, 18.5])  # nats below the largest score
@pytest.mark.parametrize("dim", [64, 128])
# query rows of a KV head 4 and 20 (the ring form), 36 to 256 (shared stages), one wave or several a row
@pytest.mark.parametrize("most,group", [(1, 4), (5, 4), (9, 4), (26, 4), (64, 4)])
@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_small_weights_beside_a_large_one_of_zero_value(gpu_device, dtype, most, group, dim, depth):
    from kv_cache_repair_amd.kernels.tree_attention import tree_attention

    rs = np.random.RandomState(5)
    lengths, counts, tables, free, pages, rows, parents = make(rs, 2, 1500, 1700, most, 32, True, most)
    expect = walk(lengths, counts, tables, free, 32, rows, most, pages, parents)
    plan, _ = plan_of(lengths, counts, tables, free, 32, rows, most, pages, parents, heads=(2 * group, 2))
    gen = torch.Generator(device="cuda").manual_seed(3)
    slots = pages * 32
    q = torch.zeros(1, 2 * group, rows, dim, dtype=dtype, device="cuda")
    q[..., 7] = 8.0
    k = torch.zeros(1, 2, slots, dim, dtype=dtype, device="cuda")
    far = -(depth + torch.rand(2, slots, device="cuda", generator=gen)) / 8
    # values so large that a result of the far keys alone is an ordinary fp16 number
    v = ((torch.rand(1, 2, slots, dim, device="cuda", generator=gen) + 0.5) * 2.0 ** 14).to(dtype)
    top = torch.arange(slots, device="cuda") % 32 == 5
    k[0, :, :, 7] = torch.where(top, 0.0, far).to(dtype)
    v[:, :, top] = 0.0
    want, size = exact(q, k, v, expect, lengths, counts, 32, pages, 1.0)
    if dtype == FP16:
        # every weight's 2^-37 over the sum of them, which has a largest one in each 32 keys
        most_keys, fewest_keys = int((lengths + counts).max()), int(lengths.min())
        size = size + 2.0 ** 12 * 2.0 ** -37 * most_keys * 1.5 * 2.0 ** 14 / (fewest_keys // 32)
    assert_close(tree_attention(q, k, v, plan, scale=1.0), want, size)
