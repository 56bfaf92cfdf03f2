"""A step of several requests over repaired caches, as a program runs it: the
caches of two edited prompts paged into one pool by a plan's slots, then drafted
trees through a layer's q/k/v projection with each request's adapter, the rotary
scatter into new pages, tree attention and the output projection, every stage
against a plain restatement on what the stage before it gave; then the next step
with single tokens, whose captured form must give the same bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import test_gpu_adapters
import test_gpu_tree_attention
from test_step_plan import gpu, walk

PAGE, PAGES, WIDTH, HEADS, KV, DIM, HIDDEN = 16, 64, 24, 4, 2, 64, 256


def repaired_caches(device):
    """Shifted caches of two prompts, edited in different places (a tiny random Llama)."""
    from transformers import LlamaConfig, LlamaForCausalLM

    from kv_cache_repair_amd.cache import OperatorShim, build_halo_cache
    from kv_cache_repair_amd.kernels.packed_cache import packed_refresh_owned_

    torch.manual_seed(0)
    model = LlamaForCausalLM(LlamaConfig(
        vocab_size=128, hidden_size=HIDDEN, intermediate_size=256, num_hidden_layers=2, num_attention_heads=HEADS,
        num_key_value_heads=KV, head_dim=DIM, rope_theta=10000.0)).to(device=device, dtype=torch.bfloat16).eval()
    shim, caches = OperatorShim(model), []
    for length, cut, span in ((203, 40, 11), (150, 100, 30)):
        old_ids = torch.randint(0, 128, (1, length), device=device)
        new_ids = torch.cat((old_ids[:, :cut], old_ids[:, cut + span:]), 1)
        with torch.no_grad():
            old = model(input_ids=old_ids, use_cache=True).past_key_values
        cache, _ = build_halo_cache(shim, old, old_ids, new_ids, 0)
        packed_refresh_owned_(shim, cache, new_ids, [(cut + 5, cut + 9)])
        caches.append(cache)
    return model, caches


def rotary(model, positions, like):
    # rows of no request have position -1; what they get is never used
    return model.model.rotary_emb(like, positions.clamp(min=0)[None])


@pytest.mark.gpu
def test_a_step_over_repaired_caches(gpu_device):
    from transformers.models.llama.modeling_llama import apply_rotary_pos_emb

    from kv_cache_repair_amd.kernels.adapters import AdapterProjectionPlan
    from kv_cache_repair_amd.kernels.indexed_attention import indexed_kv_scatter_, rope_indexed_kv_scatter_
    from kv_cache_repair_amd.kernels.step_plan import StepPlan
    from kv_cache_repair_amd.kernels.tree_attention import tree_attention

    model, caches = repaired_caches(gpu_device)
    sizes = [c.layers[0].keys.shape[2] for c in caches]
    tables = torch.full((2, WIDTH), -1, dtype=torch.int32, device=gpu_device)
    free = gpu(np.random.RandomState(0).permutation(PAGES))
    taken = torch.zeros(1, dtype=torch.int32, device=gpu_device)
    zero = torch.zeros(2, dtype=torch.int32, device=gpu_device)

    # ---- the prompts into the pools, layer by layer ----
    total = sum(sizes)
    paging = StepPlan(2, total, page_size=PAGE, n_slots=PAGES * PAGE, table_width=WIDTH, max_rows=max(sizes))
    paging.update(zero, gpu(sizes), tables, free, free_start=taken)
    taken += paging.pages_taken
    assert paging.status.tolist() == [0, 0]
    assert taken.item() == sum(-(-n // PAGE) for n in sizes)
    pools = []
    for layer in range(2):
        rows = [torch.cat([getattr(c.layers[layer], name) for c in caches], 2) for name in ("keys", "values")]
        pool = [torch.full((1, KV, PAGES * PAGE, DIM), float("nan"), dtype=torch.bfloat16, device=gpu_device)
                for _ in rows]
        indexed_kv_scatter_(*pool, *rows, paging)
        for p, r in zip(pool, rows):
            assert torch.equal(p[:, :, paging.slots], r)
            assert torch.isnan(p).sum().item() == p.numel() - r.numel()
        pools.append(pool)

    # ---- drafted trees through one layer ----
    most = 7
    step = StepPlan(2, 2 * most, page_size=PAGE, n_slots=PAGES * PAGE, table_width=WIDTH, max_rows=most,
                    heads=(HEADS, KV), device=gpu_device)
    lengths, counts = gpu(sizes), gpu([7, 5])
    tree = [-1, 0, 0, 1, 1, -2, 5] + [-1, -1, 1, 2, 0] + [-1, -1]
    parents = gpu(tree)
    before = tables.clone()
    step.update(lengths, counts, tables, free, parents, free_start=taken)
    expect = walk(sizes, [7, 5], before.cpu().numpy(), free.cpu().numpy(), PAGE, 14, most, PAGES, tree,
                  free_start=int(taken))
    for name in ("slots", "positions", "request"):
        assert np.array_equal(getattr(step, name).cpu().numpy(), expect[name])
    gen = torch.Generator(device=gpu_device).manual_seed(3)
    hidden = torch.randn(14, HIDDEN, device=gpu_device, generator=gen).to(torch.bfloat16)
    attention = model.model.layers[1].self_attn
    weights = [m.weight.detach() for m in (attention.q_proj, attention.k_proj, attention.v_proj)]
    shape = test_gpu_adapters.make(4, 1, HIDDEN, [w.shape[0] for w in weights], 5, 8, torch.bfloat16)
    qkv = AdapterProjectionPlan(weights, shape[2], shape[3], shape[4])
    adapter_of_request = gpu([3, -1])
    ids = torch.where(step.request < 0, -1, adapter_of_request[step.request.clamp(min=0)]).int()
    assert torch.equal(gpu([3, -1, -1])[step.request], ids)  # one entry more, for the rows of no request
    fresh = qkv(hidden, ids)
    test_gpu_adapters.assert_close(fresh, *test_gpu_adapters.exact(hidden, weights, shape[2], shape[3], shape[4], ids))

    split = [t.view(1, 14, -1, DIM).transpose(1, 2) for t in fresh.split([w.shape[0] for w in weights], 1)]
    cos, sin = rotary(model, step.positions, fresh)
    query = torch.zeros_like(split[0])
    keys, values = pools[1]
    held = [keys.clone(), values.clone()]
    rope_indexed_kv_scatter_(split[0], query, keys, values, split[1], split[2], cos, sin, step)
    want_q, want_k = apply_rotary_pos_emb(split[0], split[1], cos, sin)
    live = step.slots >= 0
    assert torch.equal(query[:, :, live], want_q[:, :, live])
    held[0][:, :, step.slots[live]] = want_k[:, :, live]
    held[1][:, :, step.slots[live]] = split[2][:, :, live]
    for got, want in zip((keys, values), held):
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))

    got = tree_attention(query, keys, values, step)
    want, size = test_gpu_tree_attention.exact(query, keys, values, expect, sizes, [7, 5], PAGE, PAGES, DIM ** -0.5)
    test_gpu_tree_attention.assert_close(got, want, size)
    assert (got[:, :, ~live] == 0).all() and live.tolist() == [True] * 5 + [False] * 2 + [True] * 5 + [False] * 2

    weight = [attention.o_proj.weight.detach()]
    shape = test_gpu_adapters.make(5, 1, HEADS * DIM, [HIDDEN], 5, 8, torch.bfloat16)
    flat = got.transpose(1, 2).reshape(14, HEADS * DIM)
    out = AdapterProjectionPlan(weight, shape[2], shape[3], shape[4])(flat, ids)
    test_gpu_adapters.assert_close(out, *test_gpu_adapters.exact(flat, weight, shape[2], shape[3], shape[4], ids))

    # ---- one token each after the first nodes were accepted: eager, and captured ----
    accepted = gpu([2, 1])  # nodes 0, 1 and 0: the rows after the prompts, already in place
    taken += step.pages_taken
    lengths += accepted
    one = StepPlan(2, 2, page_size=PAGE, n_slots=PAGES * PAGE, table_width=WIDTH, heads=(HEADS, KV), device=gpu_device)
    single = gpu([1, 1])
    x = hidden[:2].clone()

    def decode():
        one.update(lengths, single, tables, free, free_start=taken)
        mine = adapter_of_request[one.request].int()
        parts = [t.view(1, 2, -1, DIM).transpose(1, 2) for t in qkv(x, mine).split([w.shape[0] for w in weights], 1)]
        c, s = rotary(model, one.positions, x)
        q = torch.empty_like(parts[0])
        rope_indexed_kv_scatter_(parts[0], q, keys, values, parts[1], parts[2], c, s, one)
        return q, tree_attention(q, keys, values, one)

    query, eager = decode()
    expect = walk(lengths.tolist(), [1, 1], tables.cpu().numpy(), free.cpu().numpy(), PAGE, 2, 1, PAGES,
                  free_start=int(taken))
    want, size = test_gpu_tree_attention.exact(query, keys, values, expect, lengths.tolist(), [1, 1], PAGE, PAGES,
                                               DIM ** -0.5)
    test_gpu_tree_attention.assert_close(eager, want, size)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, captured = decode()
    for turn in range(3):
        x.copy_(hidden[2 * turn:2 * turn + 2])
        lengths.copy_(gpu([sizes[0] + 2 + turn, sizes[1] + 1 - turn]))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _, eager = decode()
        assert torch.equal(captured, eager)


@pytest.mark.gpu
def test_scatter_by_a_step_plan_checks_it(gpu_device):
    from kv_cache_repair_amd.kernels.indexed_attention import indexed_kv_scatter_
    from kv_cache_repair_amd.kernels.step_plan import StepPlan

    plan = StepPlan(1, 4, page_size=16, n_slots=64, table_width=4, max_rows=4)
    pool = [torch.zeros(1, 2, 64, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    fresh = [torch.ones(1, 2, 4, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    with pytest.raises(ValueError, match="updated"):
        indexed_kv_scatter_(*pool, *fresh, plan)
    plan.update(gpu([14]), gpu([4]), gpu([[2, 9, 9, 9]]), gpu([1]))
    with pytest.raises(ValueError, match="plan"):
        indexed_kv_scatter_(*[p[:, :, :48] for p in pool], *fresh, plan)
    with pytest.raises(ValueError, match="selected_count"):
        indexed_kv_scatter_(*pool, *[f[:, :, :3] for f in fresh], plan)
    indexed_kv_scatter_(*pool, *fresh, plan)
    assert [(p[0, 0, :, 0] != 0).nonzero()[:, 0].tolist() for p in pool] == [[16, 17, 46, 47]] * 2
