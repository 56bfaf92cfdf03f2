"""Step plans (kvr_step_plan, kernels/step_plan.py): pages, slots, positions,
masks and the attention work list against a plain restatement that walks request
by request and node by node; requests that fail; what is refused before any
launch."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

NO_PAGES, TOO_LONG, INVALID = 1, 2, 3


def walk(lengths, counts, tables, free, page, rows, max_rows, pages, parents=None, free_start=0):
    """The plan by its definition."""
    R, width = tables.shape
    out = {"row_starts": np.zeros(R + 1, np.int32), "request": np.full(rows, -1, np.int32),
           "slots": np.full(rows, -1, np.int64), "positions": np.full(rows, -1, np.int64),
           "masks": np.zeros(rows, np.uint64), "status": np.zeros(R, np.int32), "tables": tables.copy()}
    given = len(free) - free_start if 0 <= free_start <= len(free) else 0
    start, asked, taken = 0, 0, 0
    for r in range(R):
        length, count = int(lengths[r]), int(counts[r])
        out["row_starts"][r] = min(start, rows)
        end = start + max(count, 0)
        mine = range(min(start, rows), min(end, rows))
        out["request"][mine.start:mine.stop] = r
        fits = end <= rows
        start = end
        if length < 0 or not 0 <= count <= max_rows or not fits:
            out["status"][r] = INVALID
            continue
        if length + count > width * page:
            out["status"][r] = TOO_LONG
            continue
        have, want = -(-length // page), -(-(length + count) // page)
        first, asked = asked, asked + want - have
        if want > have and asked > given:
            out["status"][r] = NO_PAGES
            continue
        if want > have:
            taken = asked
        for j in range(want - have):
            out["tables"][r, have + j] = free[free_start + first + j]
        seen = {}
        for t in range(count):
            up = int(parents[mine.start + t]) if parents is not None else t - 1
            if parents is None and max_rows > 64:
                seen[t] = range(t + 1)
            else:
                seen[t] = {t} if up == -1 else seen[up] | {t} if 0 <= up < t and seen[up] else set()
            if not seen[t]:
                continue
            row, token = mine.start + t, length + t
            p = int(out["tables"][r, token // page])
            out["slots"][row] = p * page + token % page if 0 <= p < pages else -1
            out["positions"][row] = length + len(seen[t]) - 1
            if max_rows <= 64:
                out["masks"][row] = sum(1 << u for u in seen[t])
    out["row_starts"][R] = min(start, rows)
    out["pages_taken"] = np.array([taken], np.int32)
    return out


def make(rs, R, low, high, most, page, tree, fewest=0, extra_pages=3, spare_rows=5, padded=0.1):
    lengths = rs.randint(low, high + 1, R)
    counts = rs.randint(fewest, most + 1, R)
    width = -(-(high + most) // page) + 1
    pages = int((-(-(lengths + counts) // page)).sum()) + extra_pages
    order = rs.permutation(pages).astype(np.int32)
    tables, at = np.full((R, width), -9, np.int32), 0
    for r in range(R):
        have = -(-int(lengths[r]) // page)
        tables[r, :have] = order[at:at + have]
        at += have
    rows = int(counts.sum()) + spare_rows
    parents = None
    if tree:
        parents = np.full(rows, 7, np.int32)
        at_row = 0
        for r in range(R):
            for t in range(counts[r]):
                parents[at_row + t] = rs.randint(-1, t) if t else -1
                if rs.uniform() < padded:
                    parents[at_row + t] = rs.choice([-2, t, t + 1, 1 << 30, -(1 << 31)])
            at_row += counts[r]
    return lengths, counts, tables, order[at:], pages, rows, parents


def gpu(x):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def plan_of(lengths, counts, tables, free, page, rows, max_rows, pages, parents=None, heads=None, free_start=None,
            stride=0):
    from kv_cache_repair_amd.kernels.step_plan import StepPlan

    R, width = tables.shape
    plan = StepPlan(R, rows, page_size=page, n_slots=pages * page, table_width=width, max_rows=max_rows, heads=heads,
                    device="cuda")
    wide = torch.full((R, width + stride), -5, dtype=torch.int32, device="cuda")
    wide[:, :width] = gpu(tables)
    plan.update(gpu(lengths), gpu(counts), wide[:, :width], gpu(free), gpu(parents),
                None if free_start is None else gpu([free_start]))
    return plan, wide


def check(plan, wide, expect, width):
    for name in ("row_starts", "request", "slots", "positions", "status", "pages_taken"):
        got = getattr(plan, name).cpu().numpy()
        assert np.array_equal(got, expect[name]), name
    if plan.masks is not None:
        assert np.array_equal(plan.masks.cpu().numpy().view(np.uint64), expect["masks"])
    got = wide.cpu().numpy()
    assert np.array_equal(got[:, :width], expect["tables"])
    assert (got[:, width:] == -5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("R,low,high,most,page,tree", [
    (1, 0, 0, 1, 16, False), (1, 0, 40, 64, 16, True), (3, 15, 17, 1, 16, False), (7, 0, 100, 13, 32, True),
    (64, 0, 3000, 5, 64, False), (65, 0, 500, 64, 16, True), (1024, 0, 200, 3, 16, True), (4096, 0, 90, 2, 32, False),
    (4095, 0, 60, 4, 16, True), (2, 0, 1, 64, 256, False), (5, 0, 700, 3001, 16, False), (16, 100, 100, 16, 16, True)])
def test_plan_matches_its_definition(gpu_device, R, low, high, most, page, tree):
    rs = np.random.RandomState(R * 1000 + most)
    lengths, counts, tables, free, pages, rows, parents = make(rs, R, low, high, most, page, tree)
    expect = walk(lengths, counts, tables, free, page, rows, most, pages, parents)
    assert not expect["status"].any()
    plan, wide = plan_of(lengths, counts, tables, free, page, rows, most, pages, parents, stride=3)
    check(plan, wide, expect, tables.shape[1])
    # the same step again finds its pages entered already and gives the same plan
    plan.update(gpu(lengths), gpu(counts), wide[:, :tables.shape[1]], gpu(free), gpu(parents))
    check(plan, wide, expect, tables.shape[1])


@pytest.mark.gpu
def test_deepest_chain_and_star(gpu_device):
    """64 nodes in a row, and 64 on the cache: every bit of a mask, every depth."""
    lengths, counts = np.array([5, 5]), np.array([64, 64])
    parents = np.concatenate((np.arange(64) - 1, np.full(64, -1)))
    tables, free = np.array([[0, 9, 9, 9, 9], [1, 9, 9, 9, 9]]), np.arange(2, 10)
    expect = walk(lengths, counts, tables, free, 16, 128, 64, 10, parents)
    plan, wide = plan_of(lengths, counts, tables, free, 16, 128, 64, 10, parents)
    check(plan, wide, expect, 5)
    assert plan.masks[63].item() == -1 and plan.positions[63].item() == 68
    chain, wide = plan_of(lengths, counts, tables, free, 16, 128, 64, 10)
    assert torch.equal(chain.masks[:64], plan.masks[:64]) and torch.equal(chain.masks[64:], plan.masks[:64])


@pytest.mark.gpu
@pytest.mark.parametrize("tree", [False, True])
def test_requests_that_fail_take_nothing_and_leave_the_others(gpu_device, tree):
    rs = np.random.RandomState(3)
    lengths, counts, tables, free, pages, rows, parents = make(rs, 12, 1, 120, 9, 16, tree, fewest=2)
    lengths[2], counts[5], counts[7], lengths[8] = -4, -1, 40, 16 * tables.shape[1]
    tables[9, 0] = pages            # a page outside the pool: its rows have no slot, the request is fine
    lengths[9], counts[9] = 4, 3
    starts = np.concatenate(([0], np.cumsum(np.maximum(counts, 0))))
    rows = int(starts[-1]) - 1      # the last request's rows do not fit
    parents = None if parents is None else np.resize(parents, rows)
    if parents is not None:
        for r in range(12):
            parents[starts[r]:starts[r + 1]] = np.arange(len(parents[starts[r]:starts[r + 1]])) - 1
    expect = walk(lengths, counts, tables, free, 16, rows, 9, pages, parents)
    assert expect["status"][[2, 5, 7, 8, 11]].tolist() == [INVALID, INVALID, INVALID, TOO_LONG, INVALID]
    assert expect["status"][9] == 0 and (expect["slots"][expect["request"] == 9] == -1).all()
    plan, wide = plan_of(lengths, counts, tables, free, 16, rows, 9, pages, parents)
    check(plan, wide, expect, tables.shape[1])


@pytest.mark.gpu
@pytest.mark.parametrize("given", [0, 1, 2, 4, 7])
def test_the_free_list_ends(gpu_device, given):
    lengths, counts = np.array([16, 5, 32, 16, 0]), np.array([17, 1, 16, 0, 40])
    tables, free = np.full((5, 6), -1), np.arange(20, 20 + given + 2)
    expect = walk(lengths, counts, tables, free, 16, 80, 40, 40, free_start=2)
    plan, wide = plan_of(lengths, counts, tables, free, 16, 80, 40, 40, free_start=2)
    check(plan, wide, expect, 6)
    assert (expect["status"] == NO_PAGES).sum() == {0: 3, 1: 3, 2: 2, 4: 1, 7: 0}[given]


@pytest.mark.gpu
@pytest.mark.parametrize("free_start", [-1, 5, 1 << 30])
def test_a_start_outside_the_free_list_gives_no_pages(gpu_device, free_start):
    lengths, counts, tables = np.array([0, 3]), np.array([2, 2]), np.zeros((2, 2), np.int32)
    expect = walk(lengths, counts, tables, np.arange(4), 16, 4, 2, 9, free_start=free_start)
    plan, wide = plan_of(lengths, counts, tables, np.arange(4), 16, 4, 2, 9, free_start=free_start)
    check(plan, wide, expect, 2)
    assert expect["status"].tolist() == [NO_PAGES, 0]


def schedule_of(plan):
    """(items, units of a share, first item of each worker, items, split requests) of a plan's work list."""
    from kv_cache_repair_amd import _native

    s = plan._schedule.cpu().numpy()
    q, kv = plan.heads
    m = plan.max_rows * (q // kv)
    group_rows = next(g for g in (16, 32, 64, 128, 256) if m <= g or g == 256)
    wide = -(-m // group_rows) * kv
    workers = 256 // wide if wide <= 128 else 512 // wide if wide <= 256 else 1
    lists, room = -(-(workers + 1) // 8) * 8, plan.requests + workers
    assert len(s) == _native.lib().kvr_step_schedule_ints(plan.requests, plan.max_rows, q, kv) \
        == 8 + lists + 8 * room + 4 * min(plan.requests, workers)
    n, n_split, share = (int(v) for v in s[:3])
    assert n <= room and n_split <= min(plan.requests, workers)
    work = s[8 + lists:8 + lists + 8 * n].reshape(n, 8)
    at = 8 + lists + 8 * room
    return n, share, s[8:8 + workers + 1].tolist(), work, s[at:at + 4 * n_split].reshape(n_split, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("R,low,high,most,heads", [
    (1, 0, 0, 1, (8, 8)), (1, 130000, 131000, 64, (32, 8)), (1, 130000, 131000, 64, (1, 1)), (8, 0, 8000, 1, (32, 8)),
    (48, 64, 16384, 3, (32, 8)), (300, 0, 4000, 20, (28, 4)), (1000, 0, 300, 2, (64, 1)), (5, 2000, 2000, 64, (64, 1)),
    (3, 0, 50000, 1, (512, 256)), (4096, 0, 700, 1, (8, 2)), (1025, 0, 5, 1, (16, 16)), (2, 0, 900, 3, (200, 200)),
    (3, 0, 9, 2, (300, 300)), (31, 0, 0, 1, (8, 8)), (40, 100, 140, 1, (8, 1))])
@pytest.mark.parametrize("failing", [False, True])
def test_schedule_gives_every_key_to_one_worker(gpu_device, R, low, high, most, heads, failing):
    rs = np.random.RandomState(R)
    lengths, counts, tables, free, pages, rows, _ = make(rs, R, low, high, most, 16, False)
    if failing:
        lengths[rs.randint(0, R, max(1, R // 3))] = -1
        lengths[-1] = -1
    plan, _ = plan_of(lengths, counts, tables, free, 16, rows, most, pages, heads=heads)
    n, share, first, work, splits = schedule_of(plan)
    workers = len(first) - 1
    live = [r for r in range(R) if counts[r]]
    steps = {r: -(-int(lengths[r] + counts[r]) // 128) if lengths[r] >= 0 else 0 for r in live}
    units = sum(s + 1 for s in steps.values())
    assert share == max(1, -(-units // workers))
    assert first == sorted(first) and first[0] == 0 and first[-1] == n
    worker_of = {i: k for k in range(workers) for i in range(first[k], first[k + 1])}
    assert sorted(worker_of) == list(range(n))  # every item has one worker
    starts, by, parts = plan.row_starts.cpu().numpy(), {}, []
    for i, (r, begin, end, part, length, nodes, row0, n_rows) in enumerate(work.tolist()):
        by.setdefault(r, []).append((begin, end, part, worker_of[i]))
        failed = lengths[r] < 0
        assert (length, nodes, row0, n_rows) == (max(lengths[r], 0), 0 if failed else counts[r], starts[r], counts[r])
    assert list(by) == live
    split = {}
    for worker, pieces, n_rows, row0 in splits.tolist():
        r = [r for r in live if starts[r] == row0][0]
        assert n_rows == counts[r]
        split[r] = (worker, pieces)
    for r, chunks in by.items():
        assert [b for b, _, _, _ in chunks] == [0] + [e for _, e, _, _ in chunks][:-1]
        assert chunks[-1][1] == (lengths[r] + counts[r] if lengths[r] >= 0 else 0)
        assert all(b % 128 == 0 and (e > b or not steps[r]) for b, e, _, _ in chunks)
        if len(chunks) > 1:
            worker, pieces = split.pop(r)
            assert pieces == len(chunks)
            assert [k for _, _, _, k in chunks] == list(range(worker, worker + pieces))
            expect = [2 * worker + 1] + [2 * (worker + p) for p in range(1, pieces)]
            assert [p for _, _, p, _ in chunks] == expect
            parts += expect
        else:
            assert chunks[0][2] == -1
    assert not split and len(set(parts)) == len(parts) and all(p < 2 * workers for p in parts)
    for k in range(workers):  # no worker has more than its share and a start
        mine = work[first[k]:first[k + 1]]
        assert sum(-(-(e - b) // 128) + 1 for b, e in mine[:, 1:3].tolist()) <= share + 1


@pytest.mark.gpu
def test_captured_plan_follows_its_inputs(gpu_device):
    """A captured update replayed on other lengths, with eager work between the replays."""
    from kv_cache_repair_amd.kernels.step_plan import StepPlan

    rs = np.random.RandomState(5)
    R, page, most, width, pages = 9, 16, 11, 40, 400
    plan = StepPlan(R, R * most, page_size=page, n_slots=pages * page, table_width=width, max_rows=most, heads=(8, 4))
    state = {n: torch.zeros(R, dtype=torch.int32, device="cuda") for n in ("lengths", "counts")}
    tables = torch.zeros(R, width, dtype=torch.int32, device="cuda")
    free = torch.zeros(pages, dtype=torch.int32, device="cuda")
    parents = torch.full((R * most,), -1, dtype=torch.int32, device="cuda")
    plan.update(state["lengths"], state["counts"], tables, free, parents)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.update(state["lengths"], state["counts"], tables, free, parents)
    for _ in range(4):
        lengths, counts = rs.randint(0, 500, R), rs.randint(0, most + 1, R)
        table, order = rs.randint(0, pages, (R, width)), rs.permutation(pages)
        tree = np.array([rs.randint(-2, 3) for _ in range(R * most)])
        for tensor, value in ((state["lengths"], lengths), (state["counts"], counts), (tables, table), (free, order),
                              (parents, tree)):
            tensor.copy_(gpu(value))
        expect = walk(lengths, counts, table, order, page, R * most, most, pages, tree)
        graph.replay()
        torch.cuda.synchronize()
        check(plan, tables, expect, width)


@pytest.mark.gpu
def test_a_refused_update_leaves_the_plan_as_it_was(gpu_device):
    """Attention after an update that was refused is that of the last plan, over its tables."""
    from kv_cache_repair_amd.kernels.tree_attention import tree_attention

    gen = torch.Generator(device="cuda").manual_seed(2)
    tables = np.array([[0, 1, 9], [2, 3, 9]])
    plan, wide = plan_of(np.array([20, 30]), np.array([2, 1]), tables, np.arange(4, 8), 16, 4, 2, 8, heads=(4, 2))
    q = torch.randn(1, 4, 4, 64, device="cuda", generator=gen).bfloat16()
    k, v = (torch.randn(1, 2, 128, 64, device="cuda", generator=gen).bfloat16() for _ in range(2))
    before = tree_attention(q, k, v, plan)
    other = gpu(tables[::-1])
    with pytest.raises(ValueError, match="free_pages"):
        plan.update(gpu([9, 9]), gpu([1, 1]), other, free_pages=torch.zeros(4, device="cuda"))
    assert plan.planned and plan.block_tables.data_ptr() == wide.data_ptr()
    assert torch.equal(tree_attention(q, k, v, plan), before)


@pytest.mark.gpu
def test_a_plan_that_was_only_captured_has_no_requests(gpu_device):
    from kv_cache_repair_amd.kernels.step_plan import StepPlan
    from kv_cache_repair_amd.kernels.tree_attention import tree_attention

    plan = StepPlan(3, 6, page_size=16, n_slots=160, table_width=4, max_rows=2, heads=(4, 2))
    assert (plan.slots == -1).all() and (plan.request == -1).all() and not plan.row_starts.any()
    lengths, counts, tables = gpu([20, 3, 9]), gpu([2, 1, 2]), gpu(np.arange(12).reshape(3, 4) % 10)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.update(lengths, counts, tables)
    q = torch.ones(1, 4, 6, 64, device="cuda", dtype=torch.bfloat16)
    k = torch.ones(1, 2, 160, 64, device="cuda", dtype=torch.bfloat16)
    assert not tree_attention(q, k, k.clone(), plan).any()
    graph.replay()
    got = tree_attention(q, k, k.clone(), plan)
    assert (got[:, :, :5] == 1).all() and not got[:, :, 5:].any()


def _desc(**changes):
    from kv_cache_repair_amd import _native

    desc = _native.StepDesc()
    for i, (name, kind) in enumerate(desc._fields_):
        if kind is ctypes.c_void_p:
            setattr(desc, name, (i + 1) << 20)  # aligned, never read: every call below is refused
    desc.n_slots, desc.table_stride, desc.requests, desc.rows, desc.max_rows = 1024, 8, 4, 16, 4
    desc.page_size, desc.table_width, desc.free_count, desc.q_heads, desc.kv_heads = 16, 8, 3, 8, 4
    for name, value in changes.items():
        setattr(desc, name, value)
    return desc


@pytest.mark.parametrize("status,changes", [
    (-3, {"requests": 0}), (-3, {"requests": 4097}), (-3, {"rows": 0}), (-3, {"max_rows": 0}), (-3, {"page_size": 8}),
    (-3, {"page_size": 48}), (-3, {"n_slots": 0}), (-3, {"n_slots": 1000}), (-3, {"table_width": 0}),
    (-3, {"table_width": 1 << 27, "table_stride": 1 << 27}), (-3, {"free_count": -1}), (-4, {"table_stride": 7}),
    (-3, {"max_rows": 65}), (-3, {"requests": 4096, "page_size": 4096, "n_slots": 4096, "table_width": 1 << 14,
                                  "table_stride": 1 << 14}), (-3, {"q_heads": 6}), (-3, {"kv_heads": 0}), (-4, {"schedule": (1 << 20) + 16}),
    (-5, {"lengths": None}), (-5, {"counts": None}), (-5, {"tables": None}), (-5, {"row_starts": None}),
    (-5, {"request": None}), (-5, {"slots": None}), (-5, {"positions": None}), (-5, {"masks": None}),
    (-5, {"status": None}), (-5, {"pages_taken": None}), (-5, {"free_pages": None}),
    (-5, {"schedule": None, "max_rows": 65}), (-3, {"schedule": None, "max_rows": 65, "masks": None})])
def test_plan_refuses_before_any_launch(status, changes):
    from kv_cache_repair_amd import _native

    assert _native.lib().kvr_step_plan(ctypes.byref(_desc(**changes)), None) == status


def test_header_symbols_are_exported():
    import re
    from pathlib import Path

    from kv_cache_repair_amd import _native

    text = (Path(__file__).resolve().parents[1] / "include" / "kvrepair_step.h").read_text()
    names = set(re.findall(r"\b(kvr_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    assert names == {"kvr_step_desc_size", "kvr_step_schedule_ints", "kvr_step_plan", "kvr_tree_workspace_bytes",
                     "kvr_tree_attention", "kvr_adapter_linear_workspace_bytes", "kvr_adapter_linear"}
    for name in names:
        assert hasattr(_native.lib(), name), name


def test_plan_refuses_no_descriptor_and_bad_schedules():
    from kv_cache_repair_amd import _native

    lib = _native.lib()
    assert lib.kvr_step_plan(None, None) == -5
    assert lib.kvr_step_desc_size() == ctypes.sizeof(_native.StepDesc)
    assert lib.kvr_step_schedule_ints(1, 1, 8, 4) > 0
    for args in ((0, 1, 8, 4), (4097, 1, 8, 4), (1, 0, 8, 4), (1, 65, 8, 4), (1, 1, 0, 4), (1, 1, 8, 0), (1, 1, 6, 4)):
        assert lib.kvr_step_schedule_ints(*args) == -3


@pytest.mark.parametrize("changes", [
    {"requests": 0}, {"requests": 4097}, {"requests": True}, {"rows": 0}, {"rows": 1.5}, {"page_size": 8},
    {"page_size": 24}, {"n_slots": 100}, {"n_slots": 0}, {"table_width": 0}, {"max_rows": 0}, {"heads": (6, 4)},
    {"heads": (0, 1)}, {"heads": (8, 4), "max_rows": 65}, {"heads": 8}, {"heads": (8, 4, 2)}, {"device": "cpu"},
    {"heads": (8, 4), "requests": 4096, "page_size": 4096, "n_slots": 4096, "table_width": 1 << 14}])
def test_step_plan_checks_its_sizes(changes):
    from kv_cache_repair_amd.kernels.step_plan import StepPlan

    sizes = {"requests": 2, "rows": 4, "page_size": 16, "n_slots": 64, "table_width": 4, "max_rows": 2,
             "heads": None, "device": "cuda:0"} | changes
    with pytest.raises(ValueError):
        StepPlan(sizes.pop("requests"), sizes.pop("rows"), **sizes)


@pytest.mark.gpu
def test_update_checks_its_tensors(gpu_device):
    from kv_cache_repair_amd.kernels.step_plan import StepPlan

    plan = StepPlan(3, 6, page_size=16, n_slots=160, table_width=4, max_rows=2)
    ok = {"lengths": torch.zeros(3, dtype=torch.int32, device="cuda"),
          "counts": torch.zeros(3, dtype=torch.int32, device="cuda"),
          "block_tables": torch.zeros(3, 4, dtype=torch.int32, device="cuda"),
          "free_pages": torch.zeros(5, dtype=torch.int32, device="cuda"),
          "parents": torch.zeros(6, dtype=torch.int32, device="cuda")}
    plan.update(**ok)
    for name, bad in (("lengths", ok["lengths"].long()), ("lengths", ok["lengths"][:2]), ("lengths", [0, 0, 0]),
                      ("counts", ok["counts"].cpu()), ("counts", torch.zeros(6, dtype=torch.int32, device="cuda")[::2]),
                      ("block_tables", ok["block_tables"][:, :3]), ("block_tables", ok["block_tables"].t()),
                      ("block_tables", ok["block_tables"][:1].expand(3, 4)), ("free_pages", ok["free_pages"].float()),
                      ("parents", ok["parents"][:5]), ("free_start", ok["lengths"])):
        with pytest.raises(ValueError):
            plan.update(**(ok | {name: bad}))
    # what the plan writes is no input, and what it reads no table
    own = plan.request
    for name, bad in (("free_start", plan.pages_taken), ("lengths", plan.status), ("counts", own[3:6]),
                      ("free_pages", own[4:]), ("parents", own)):
        with pytest.raises(ValueError, match="the plan writes"):
            plan.update(**(ok | {name: bad}))
    many = torch.zeros(64, dtype=torch.int32, device="cuda")
    for name, size in (("lengths", 3), ("counts", 3), ("free_pages", 9), ("parents", 6), ("free_start", 1)):
        with pytest.raises(ValueError, match="overlap"):
            plan.update(**(ok | {"block_tables": many[:12].view(3, 4), name: many[11:11 + size]}))
        plan.update(**(ok | {"block_tables": many[:12].view(3, 4), name: many[12:12 + size]}))
    with pytest.raises(ValueError, match="nodes"):
        StepPlan(3, 600, page_size=16, n_slots=160, table_width=40, max_rows=65).update(
            ok["lengths"], ok["counts"], torch.zeros(3, 40, dtype=torch.int32, device="cuda"),
            parents=torch.zeros(600, dtype=torch.int32, device="cuda"))
