"""PagedCache.keep_rows_ and fork_, FreePages.collect (kvr_keep_rows, kvr_fork_requests,
kvr_free_pages) against plain loops over requests, rows and pages: every bit of the pools,
what moved and what did not, at odd sizes, layouts and types; bad paths, full free lists,
requests that fail; captured calls; what is refused."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from test_step_plan import _desc, gpu, make, plan_of, walk

TYPES = {torch.bfloat16: torch.int16, torch.float16: torch.int16, torch.float32: torch.int32, torch.float8_e4m3fn: torch.uint8}


def pools(seed, layers, heads, slots, dim, dtype, layout="heads"):
    """Any bits, NaN's among them: copies have to keep them."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for _ in range(2 * layers):
        shape = (1, heads, slots, dim) if layout == "heads" else (1, slots, heads, dim)
        if layout == "sliced":
            shape = (1, heads, slots, dim * 3)
        bits = torch.randint(0, 256, (*shape[:-1], shape[-1] * dtype.itemsize), device="cuda", generator=gen, dtype=torch.uint8)
        t = bits.view(dtype)
        out.append(t if layout == "heads" else t[..., dim:2 * dim] if layout == "sliced" else t.transpose(1, 2))
    return out[:layers], out[layers:]


def bits(t):
    return t.view(TYPES[t.dtype])


def cache_of(keys, values, page):
    from kv_cache_repair_amd.kernels.pages import PagedCache

    return PagedCache(keys, values, page_size=page)


# ----------------------------------------------------------------------------- accepted rows
def moved(expect, path, kept, page, pages, width):
    """(from, to) slots, in order, by the definition."""
    out = []
    for r in range(len(kept)):
        start, n = int(expect["row_starts"][r]), int(expect["row_starts"][r + 1] - expect["row_starts"][r])
        length, before = (int(expect["positions"][start]) if n else -1), -1
        if length < 0:
            continue
        for i in range(min(int(kept[r]), n)):
            node, token = int(path[start + i]), length + i
            if not before < node < n:
                break
            before = node
            held = int(expect["tables"][r, token // page]) if token // page < width else -1
            slot = int(expect["slots"][start + node])
            if node != i and slot >= 0 and 0 <= held < pages:
                out.append((slot, held * page + token % page))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("R,low,high,most,page,layers,heads,dim,dtype,layout", [
    (1, 0, 0, 1, 16, 1, 1, 8, torch.bfloat16, "heads"), (1, 5, 5, 64, 16, 2, 8, 128, torch.bfloat16, "heads"),
    (9, 0, 70, 13, 32, 3, 2, 64, torch.float16, "tokens"), (30, 0, 50, 64, 16, 1, 3, 40, torch.float32, "sliced"),
    (5, 0, 40, 20, 16, 65, 1, 16, torch.float8_e4m3fn, "heads"), (4, 3, 300, 500, 64, 2, 2, 16, torch.bfloat16, "heads"),
    (300, 0, 40, 5, 16, 1, 1, 64, torch.bfloat16, "tokens"), (2, 0, 900, 129, 256, 2, 9, 136, torch.float16, "heads")])
def test_kept_rows_move_together(gpu_device, R, low, high, most, page, layers, heads, dim, dtype, layout):
    rs = np.random.RandomState(R + most)
    lengths, counts, tables, free, pages, rows, _ = make(rs, R, low, high, most, page, False, fewest=1 if R == 1 else 0)
    expect = walk(lengths, counts, tables, free, page, rows, most, pages)
    plan, _ = plan_of(lengths, counts, tables, free, page, rows, most, pages)
    path, kept = np.full(rows, -1), np.zeros(R, int)
    for r in range(R):
        n, start = int(counts[r]), int(expect["row_starts"][r])
        kept[r] = rs.randint(0, n + 1)
        path[start:start + kept[r]] = np.sort(rs.permutation(n)[:kept[r]])
    keys, values = pools(1, layers, heads, pages * page, dim, dtype, layout)
    want = [t.clone() for t in (*keys, *values)]
    steps = moved(expect, path, kept, page, pages, tables.shape[1])
    source, target = (torch.tensor([s[i] for s in steps], dtype=torch.int64, device="cuda") for i in (0, 1))
    for t in want:  # rows move down: what one reads has not been written by one before it
        bits(t)[:, :, target] = bits(t)[:, :, source]
    assert not set(source.tolist()) & {t for i, (_, t) in enumerate(steps) for s, _ in steps[i + 1:] if s == t}
    assert cache_of(keys, values, page).keep_rows_(plan, gpu(path), gpu(kept)) is None
    for got, w in zip((*keys, *values), want):
        assert torch.equal(bits(got), bits(w))


@pytest.mark.gpu
def test_paths_that_are_none(gpu_device):
    """Entries that are no ascending nodes end a path; failed requests, padding nodes and
    pages outside the pool move nothing; more kept than rows are the rows."""
    rs = np.random.RandomState(1)
    lengths, counts, tables, free, pages, rows, parents = make(rs, 10, 20, 60, 9, 16, True, fewest=6)
    parents[:] = np.concatenate([np.arange(n) - 1 for n in counts] + [np.zeros(rows - counts.sum())])
    starts = np.concatenate(([0], np.cumsum(counts)))
    parents[starts[2] + 3] = -2          # a padding node, and those behind it
    parents[starts[3]] = -2              # node 0 itself
    lengths[4] = -1                      # failed
    tables[5, lengths[5] // 16] = pages if lengths[5] % 16 else tables[5, lengths[5] // 16]
    expect = walk(lengths, counts, tables, free, 16, rows, 9, pages, parents)
    plan, _ = plan_of(lengths, counts, tables, free, 16, rows, 9, pages, parents)
    path, kept = np.full(rows, -1), np.full(10, 4)
    for r in range(10):
        path[starts[r]:starts[r] + 4] = [0, 2, 4, 5]
    path[starts[0] + 1:starts[0] + 4] = [2, 2, 4]
    path[starts[1] + 2] = 99
    path[starts[6] + 1] = -5
    path[starts[7]] = 3                  # 3, 2: the first holds
    kept[8], kept[9] = 1 << 30, -3
    keys, values = pools(2, 2, 2, pages * 16, 64, torch.bfloat16)
    want = [t.clone() for t in (*keys, *values)]
    for source, target in moved(expect, path, kept, 16, pages, tables.shape[1]):
        for t in want:
            bits(t)[:, :, target] = bits(t)[:, :, source].clone()
    cache_of(keys, values, 16).keep_rows_(plan, gpu(path), gpu(kept))
    for got, w in zip((*keys, *values), want):
        assert torch.equal(bits(got), bits(w))


# ----------------------------------------------------------------------------- forks
def forked(sources, lengths, tables, free, page, pages, free_start=0):
    """(lengths, tables, status, taken, copied (page, page, rows)) by the definition."""
    R, width = tables.shape
    given = len(free) - free_start if 0 <= free_start <= len(free) else 0
    out_l, out_t = np.zeros(len(sources), np.int32), np.full((len(sources), width), -1, np.int32)
    status, copied, seen, asked, taken = np.zeros(len(sources), np.int32), [], set(), 0, 0
    for i, r in enumerate(sources):
        r = int(r)
        if r == -1:
            continue
        if not 0 <= r < R or lengths[r] < 0:
            status[i] = 3
            continue
        length = int(lengths[r])
        if length > width * page:
            status[i] = 2
            continue
        have, part = -(-length // page), length % page
        row = tables[r, :have].copy()
        if part and r in seen and 0 <= row[-1] < pages:
            asked += 1
            if asked > given:
                status[i] = 1
                continue
            taken, fresh = asked, int(free[free_start + asked - 1])
            if 0 <= fresh < pages:
                copied.append((int(row[-1]), fresh, part))
            row[-1] = fresh
        seen.add(r)
        out_l[i], out_t[i, :have] = length, row
    return out_l, out_t, status, np.array([taken], np.int32), copied


def fork_case(seed, R, n, low, high, page, spare=4):
    rs = np.random.RandomState(seed)
    lengths = rs.randint(low, high + 1, R)
    have = -(-lengths // page)
    width = max(1, int(have.max())) + 1
    pages = int(have.sum()) + n + spare
    order, tables, at = rs.permutation(pages), np.full((R, width), -7), 0
    for r in range(R):
        tables[r, :have[r]] = order[at:at + have[r]]
        at += have[r]
    return rs, lengths, tables, order[at:], pages, rs.randint(-1, R, n)


def check_fork(lengths, tables, free, page, pages, sources, keys, values, free_start=None, stride=0):
    want_l, want_t, status, taken, copied = forked(sources, lengths, tables, free, page, pages, free_start or 0)
    want = [t.clone() for t in (*keys, *values)]
    for source, target, rows in copied:
        for t in want:
            bits(t)[:, :, target * page:target * page + rows] = bits(t)[:, :, source * page:source * page + rows]
    wide = torch.full((tables.shape[0], tables.shape[1] + stride), -5, dtype=torch.int32, device="cuda")
    wide[:, :tables.shape[1]] = gpu(tables)
    held = wide.clone()
    lengths_in = gpu(lengths)
    done = cache_of(keys, values, page).fork_(gpu(sources), lengths_in, wide[:, :tables.shape[1]], gpu(free),
                                              None if free_start is None else gpu([free_start]))
    for got, w in zip(done, (want_l, want_t, status, taken)):
        assert got.dtype == torch.int32 and np.array_equal(got.cpu().numpy(), w)
    assert torch.equal(wide, held) and np.array_equal(lengths_in.cpu().numpy(), lengths)
    for got, w in zip((*keys, *values), want):
        assert torch.equal(bits(got), bits(w))
    return status, copied


@pytest.mark.gpu
@pytest.mark.parametrize("R,n,low,high,page,layers,heads,dim,dtype,layout", [
    (1, 1, 0, 0, 16, 1, 1, 8, torch.bfloat16, "heads"), (1, 16, 33, 33, 16, 2, 8, 128, torch.bfloat16, "heads"),
    (1, 3, 64, 64, 16, 1, 2, 64, torch.float16, "heads"), (8, 20, 0, 100, 32, 3, 2, 64, torch.float32, "tokens"),
    (40, 64, 0, 500, 128, 2, 3, 40, torch.float16, "sliced"), (3, 7, 0, 900, 256, 65, 1, 16, torch.float8_e4m3fn, "heads"),
    (700, 1500, 0, 40, 16, 1, 1, 16, torch.bfloat16, "heads"), (4096, 4096, 0, 33, 16, 1, 1, 8, torch.bfloat16, "heads"),
    (5, 4096, 1, 30, 16, 1, 1, 8, torch.bfloat16, "tokens")])
def test_forks_match_their_definition(gpu_device, R, n, low, high, page, layers, heads, dim, dtype, layout):
    _, lengths, tables, free, pages, sources = fork_case(R + n, R, n, low, high, page)
    status, _ = check_fork(lengths, tables, free, page, pages, sources, *pools(3, layers, heads, pages * page, dim, dtype, layout),
                           stride=3)
    assert not status.any()


@pytest.mark.gpu
@pytest.mark.parametrize("given", [0, 1, 3])
def test_forks_that_fail_leave_the_others(gpu_device, given):
    rs, lengths, tables, free, pages, _ = fork_case(5, 6, 12, 17, 90, 16)
    lengths[:] = lengths // 16 * 16 + 5
    lengths[2], lengths[3] = -1, tables.shape[1] * 16 + 1
    lengths[4] = lengths[4] // 16 * 16                # whole pages: needs none
    tables[5, lengths[5] // 16] = pages               # a last page outside the pool: nothing to copy
    sources = np.array([0, 0, 2, 3, -2, 6, 1 << 30, -1, 4, 4, 5, 5, 0, 1, 1, 0])
    free[2] = pages + 3                               # a page outside the pool: entered, nothing copied
    status, copied = check_fork(lengths, tables, free[:given + 2], 16, pages, sources,
                                *pools(4, 2, 2, pages * 16, 64, torch.bfloat16), free_start=2)
    assert (status == 1).sum() == 4 - min(given, 4) and status[2:7].tolist() == [3, 2, 3, 3, 3]
    check_fork(lengths, tables, free, 16, pages, sources, *pools(4, 2, 2, pages * 16, 64, torch.bfloat16), free_start=-1)
    check_fork(lengths, tables, free, 16, pages, sources, *pools(4, 2, 2, pages * 16, 64, torch.bfloat16), free_start=1 << 30)


@pytest.mark.gpu
def test_pools_past_32_bits(gpu_device):
    """Slots whose byte offsets pass 2^32: forks and kept rows near the end of a pool."""
    page, pages, dim = 256, 96 * 1024, 128   # 25 M slots of 256 bytes: 6.4 GB
    k = torch.zeros(1, 1, pages * page, dim, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(1, 1, pages * page, dim, dtype=torch.bfloat16, device="cuda")
    for t in (k, v):
        t[0, 0, -1024:] = torch.randn(1024, dim, device="cuda").bfloat16()
    cache = cache_of([k], [v], page)
    done = cache.fork_(gpu([0, 0]), gpu([100]), gpu([[pages - 1]]), gpu([pages - 4]))
    assert done.block_tables.tolist() == [[pages - 1], [pages - 4]]
    for t in (k, v):
        assert torch.equal(t[0, 0, (pages - 4) * page:(pages - 4) * page + 100], t[0, 0, (pages - 1) * page:(pages - 1) * page + 100])
    plan, _ = plan_of(np.array([3]), np.array([9]), np.array([[pages - 2]]), np.zeros(0), page, 9, 9, pages)
    row = k[0, 0, (pages - 2) * page + 3 + 8].clone()
    cache.keep_rows_(plan, gpu([0, 8] + [-1] * 7), gpu([2]))
    assert torch.equal(k[0, 0, (pages - 2) * page + 4], row) and row.any()


@pytest.mark.gpu
def test_strides_of_a_single_head_may_be_anything(gpu_device):
    keys, values = pools(5, 2, 1, 64, 64, torch.bfloat16)
    want = [t.clone() for t in (*keys, *values)]
    for t in want:
        bits(t)[:, :, 32:37] = bits(t)[:, :, 16:21]
    views = [t.as_strided(t.shape, (3, 5 + i, 64, 1)) for i, t in enumerate((*keys, *values))]
    done = cache_of(views[:2], views[2:], 16).fork_(gpu([0, 0]), gpu([21]), gpu([[0, 1]]), gpu([2]))
    assert done.block_tables.tolist() == [[0, 1], [0, 2]]
    assert all(torch.equal(bits(g), bits(w)) for g, w in zip((*keys, *values), want))


# ----------------------------------------------------------------------------- free lists
def collected(lengths, tables, page, pages):
    held = set()
    for row, length in zip(tables.tolist(), lengths.tolist()):
        held.update(row[:max(0, -(-length // page))])
    free = [p for p in range(pages) if p not in held]
    return [-1] * (pages - len(free)) + free, [pages - len(free)]


@pytest.mark.gpu
@pytest.mark.parametrize("R,low,high,page,pages", [
    (1, 0, 0, 16, 1), (1, 16, 16, 16, 1), (1, 5, 5, 16, 17), (3, 0, 500, 16, 100), (8, 0, 9000, 16, 5000),
    (70, 0, 3000, 64, 4096), (300, -5, 800, 32, 8193), (4096, 0, 100, 16, 30011), (9, 0, 70000, 256, 300000), (2, 0, 40, 16, 3000001)])
def test_free_lists_match_their_definition(gpu_device, R, low, high, page, pages):
    from kv_cache_repair_amd.kernels.pages import FreePages

    rs = np.random.RandomState(R)
    lengths = rs.randint(low, high + 1, R)
    width = max(1, -(-max(high, 1) // page))
    tables = rs.randint(0, pages, (R, width))  # shared at random
    tables[rs.uniform(0, 1, tables.shape) < 0.05] = rs.choice([-1, pages, 1 << 30, -(1 << 31)])
    wide = torch.full((R, width + 3), 0, dtype=torch.int32, device="cuda")
    wide[:, :width] = gpu(tables)
    free = FreePages(pages)
    assert free.start.tolist() == [0] and torch.equal(free.pages, torch.arange(pages, dtype=torch.int32, device="cuda"))
    for _ in range(2):  # what the list held before does not matter
        assert free.collect(gpu(lengths), wide[:, :width], page_size=page) is free
        want, start = collected(lengths, tables, page, pages)
        assert free.start.tolist() == start and np.array_equal(free.pages.cpu().numpy(), np.array(want, np.int32))
        free.pages.fill_(7)
        free.start.fill_(-3)


@pytest.mark.gpu
def test_lengths_past_their_tables(gpu_device):
    from kv_cache_repair_amd.kernels.pages import FreePages

    free = FreePages(10)
    free.collect(gpu([(1 << 31) - 1, 1]), gpu([[1, 2, 3], [9, 0, 0]]), page_size=16)
    assert free.pages.tolist() == [-1] * 4 + [0, 4, 5, 6, 7, 8] and free.start.tolist() == [4]


@pytest.mark.gpu
def test_captured_calls_follow_their_inputs(gpu_device):
    """Fork, kept rows and free list in one graph, replayed on other requests, with eager work between."""
    from kv_cache_repair_amd.kernels.pages import FreePages

    page, R, n = 16, 6, 9
    cases = [fork_case(seed, R, n, 1, 100, page) for seed in range(4)]
    width, pages = 9, max(c[4] for c in cases)
    keys, values = pools(3, 2, 2, pages * page, 64, torch.bfloat16)
    cache, free = cache_of(keys, values, page), FreePages(pages)
    lengths, tables, sources = gpu(np.zeros(R)), gpu(np.zeros((R, width))), gpu(np.zeros(n))

    def turn():
        free.collect(lengths, tables, page_size=page)
        return cache.fork_(sources, lengths, tables, free.pages, free.start)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        turn()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        done = turn()
    for _, length, table, _, _, source in cases:
        wide = np.full((R, width), -1)
        wide[:, :min(width, table.shape[1])] = table[:, :width]
        lengths.copy_(gpu(length))
        tables.copy_(gpu(wide))
        sources.copy_(gpu(source))
        held = [t.clone() for t in (*keys, *values)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want, start = collected(length, wide, page, pages)
        assert free.pages.tolist() == want and free.start.tolist() == start
        want_l, want_t, status, taken, copied = forked(source, length, wide, np.array(want), page, pages, start[0])
        for got, w in zip(done, (want_l, want_t, status, taken)):
            assert np.array_equal(got.cpu().numpy(), w)
        for a, b, rows in copied:
            for t in held:
                bits(t)[:, :, b * page:b * page + rows] = bits(t)[:, :, a * page:a * page + rows]
        assert all(torch.equal(bits(g), bits(w)) for g, w in zip((*keys, *values), held))
        turn()  # eager, between the replays: the same pages, the same copies
        assert all(torch.equal(bits(g), bits(w)) for g, w in zip((*keys, *values), held))


# ----------------------------------------------------------------------------- refusals
@pytest.mark.gpu
def test_caches_check_their_pools(gpu_device):
    keys, values = pools(1, 2, 2, 64, 64, torch.bfloat16)
    cache_of(keys, values, 16)
    other = torch.zeros(1, 2, 64, 64, dtype=torch.bfloat16, device="cuda")
    for bad in ((keys, values[:1]), ([], []), (keys, [values[0], other.float()]), (keys, [values[0], other.cpu()]),
                (keys, [values[0], other[:, :1]]), ([keys[0], keys[0]], values), ([other[0], keys[1]], values),
                ([keys[0], other.transpose(1, 2).contiguous().transpose(1, 2)], values),
                (keys, [other[:, :1].expand(1, 2, 64, 64)] * 2), ([t[..., 1:57] for t in keys], [t[..., 1:57] for t in values]),
                ([t[..., :60] for t in keys], [t[..., :60] for t in values]), ([t[:, :, :40] for t in keys], [t[:, :, :40] for t in values]),
                ([keys[0].clone().requires_grad_(), keys[1]], values), ([None, keys[1]], values),
                ([t.double() for t in keys], [t.double() for t in values])):
        with pytest.raises(ValueError):
            cache_of(*bad, 16)
    for page in (8, 24, 128, 16.0, True):
        with pytest.raises(ValueError):
            cache_of(keys, values, page)


@pytest.mark.gpu
def test_calls_check_their_tensors(gpu_device):
    from kv_cache_repair_amd.kernels.pages import FreePages
    from kv_cache_repair_amd.kernels.step_plan import StepPlan

    keys, values = pools(1, 2, 2, 64, 64, torch.bfloat16)
    cache = cache_of(keys, values, 16)
    sizes = {"page_size": 16, "n_slots": 64, "table_width": 2, "max_rows": 2}
    plan, new = StepPlan(2, 4, **sizes), StepPlan(2, 4, **sizes)
    plan.update(gpu([1, 1]), gpu([2, 2]), gpu([[0, 1], [2, 3]]))
    path, kept = gpu([0, 1, 0, 1]), gpu([2, 2])
    cache.keep_rows_(plan, path, kept)
    other = StepPlan(2, 4, **(sizes | {"page_size": 32}))
    other.update(gpu([1, 1]), gpu([2, 2]), gpu([[0, 1], [1, 0]]))
    for bad in ((new, path, kept), (other, path, kept), (None, path, kept), (plan, path[:3], kept), (plan, path.long(), kept),
                (plan, path, kept.cpu()), (plan, path, gpu([2] * 4)[::2])):
        with pytest.raises(ValueError):
            cache.keep_rows_(*bad)
    ok = {"sources": gpu([0, 0]), "lengths": gpu([5, 9]), "block_tables": gpu([[0, 9], [1, 9]]), "free_pages": gpu([2, 3]),
          "free_start": gpu([0])}
    cache.fork_(**ok)
    for name, bad in (("sources", gpu([])), ("sources", ok["sources"].long()), ("sources", gpu([0] * 4097)), ("lengths", gpu([5])),
                      ("lengths", None), ("block_tables", gpu([0, 1])), ("block_tables", ok["block_tables"].t()),
                      ("block_tables", ok["block_tables"].long()), ("block_tables", ok["block_tables"][:1].expand(2, 2)),
                      ("free_pages", ok["free_pages"].float()), ("free_start", gpu([0, 0])), ("free_start", 0)):
        with pytest.raises(ValueError):
            cache.fork_(**(ok | {name: bad}))
    free = FreePages(4)
    free.collect(ok["lengths"], ok["block_tables"], page_size=16)
    for lengths, tables, page in ((gpu([5]), ok["block_tables"], 16), (ok["lengths"], ok["block_tables"].float(), 16),
                                  (ok["lengths"], ok["block_tables"], 24), (ok["lengths"], ok["block_tables"], 8),
                                  (free.pages[:2], ok["block_tables"], 16), (ok["lengths"], free.pages.view(2, 2), 16),
                                  (free.start, ok["block_tables"][:1], 16)):
        with pytest.raises(ValueError):
            free.collect(lengths, tables, page_size=page)
    for count in (0, -1, 1 << 31, 1.5, True):
        with pytest.raises(ValueError):
            FreePages(count)
    with pytest.raises(ValueError):
        FreePages(4, device="cpu")
    # storage that was swapped under a handle
    free.pages.data = free.pages.clone()
    with pytest.raises(ValueError, match="storage"):
        free.collect(ok["lengths"], ok["block_tables"], page_size=16)
    keys[1].data = keys[1].clone()
    for call in (lambda: cache.fork_(**ok), lambda: cache.keep_rows_(plan, path, kept)):
        with pytest.raises(ValueError, match="storage"):
            call()


def _pools(**changes):
    from kv_cache_repair_amd import _native

    at = changes.pop("at", 1 << 20)
    p = _native.Pools()
    p.k, p.v = (ctypes.c_void_p * 2)(1 << 20, 1 << 21), (ctypes.c_void_p * 2)(1 << 22, at)
    p.k_head = p.v_head = 1024 * 128
    p.k_row = p.v_row = 128
    p.n_slots, p.layers, p.kv_heads, p.row_bytes, p.page_size = 1024, 2, 4, 128, 16
    for name, value in changes.items():
        setattr(p, name, value)
    return p


POOLS = [(-3, {"layers": 0}), (-3, {"kv_heads": 0}), (-3, {"row_bytes": 0}), (-3, {"row_bytes": 24}), (-3, {"n_slots": 0}),
         (-3, {"n_slots": 1000}), (-3, {"page_size": 8}), (-3, {"page_size": 48}), (-4, {"k_head": 0}), (-4, {"k_row": 120}),
         (-4, {"v_head": -16}), (-4, {"v_row": 8}), (-4, {"at": (1 << 20) + 8}), (-5, {"at": None}),
         (-3, {"kv_heads": 1 << 20, "row_bytes": 4096, "page_size": 16})]


@pytest.mark.parametrize("status,pool,desc,call", [(*p, {}, {}) for p in POOLS] + [
    (-5, {}, {}, {"path": None}), (-5, {}, {}, {"kept": None}), (-1, {"page_size": 32}, {}, {}), (-1, {"n_slots": 2048}, {}, {}),
    (-3, {}, {"requests": 0}, {})])
def test_kept_rows_refuse_before_any_launch(status, pool, desc, call):
    from kv_cache_repair_amd import _native

    p, d = _pools(**pool), _desc(**desc)
    at = 1 << 20
    assert _native.lib().kvr_keep_rows(ctypes.byref(p), ctypes.byref(d), call.get("path", at), call.get("kept", at), None) == status


@pytest.mark.parametrize("status,pool,changes", [(*p, {}) for p in POOLS] + [
    (-5, {}, {name: None}) for name in ("sources", "lengths", "tables", "free_pages", "out_lengths", "out_tables", "status",
                                       "pages_taken")] + [
    (-3, {}, {"count": 0}), (-3, {}, {"count": 4097}), (-3, {}, {"requests": 0}), (-3, {}, {"requests": 4097}),
    (-3, {}, {"table_width": 0}), (-3, {}, {"free_count": -1}), (-4, {}, {"table_stride": 7}), (-4, {}, {"out_stride": 7}),
    (-3, {}, {"table_width": 1 << 27, "table_stride": 1 << 27, "out_stride": 1 << 27})])
def test_forks_refuse_before_any_launch(status, pool, changes):
    from kv_cache_repair_amd import _native

    p, d = _pools(**pool), _native.ForkDesc()
    for name, kind in d._fields_:
        setattr(d, name, 1 << 20 if kind is ctypes.c_void_p else 8)
    for name, value in changes.items():
        setattr(d, name, value)
    assert _native.lib().kvr_fork_requests(ctypes.byref(p), ctypes.byref(d), None) == status


@pytest.mark.parametrize("status,changes", [
    (-5, {"lengths": None}), (-5, {"tables": None}), (-5, {"list": None}), (-5, {"start": None}), (-6, {"workspace": None}),
    (-6, {"workspace": (1 << 20) + 8}), (-6, {"bytes": 0}), (-4, {"stride": 7}), (-3, {"requests": 0}), (-3, {"requests": 4097}),
    (-3, {"width": 0}), (-3, {"page_size": 8}), (-3, {"page_size": 24}), (-3, {"n_pages": 0})])
def test_free_lists_refuse_before_any_launch(status, changes):
    from kv_cache_repair_amd import _native

    lib, at = _native.lib(), 1 << 20
    need = lib.kvr_free_pages_workspace_bytes(100)
    get = changes.get
    assert need > 0 and lib.kvr_free_pages_workspace_bytes(0) == -3
    assert lib.kvr_free_pages(get("lengths", at), get("tables", at), get("stride", 8), get("requests", 4), get("width", 8),
                              get("page_size", 16), get("n_pages", 100), get("list", at), get("start", at),
                              get("workspace", at), get("bytes", need), None) == status


def test_header_symbols_are_exported():
    import re
    from pathlib import Path

    from kv_cache_repair_amd import _native

    text = (Path(__file__).resolve().parents[1] / "include" / "kvrepair_serve.h").read_text()
    names = set(re.findall(r"\b(kvr_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    assert len(names) == 12
    for name in names:
        assert hasattr(_native.lib(), name), name


@pytest.mark.gpu
def test_pools_of_other_sizes_may_share_a_workspace(gpu_device):
    """Zero before its first call: no later one sees what another pool's call left there."""
    from kv_cache_repair_amd import _native

    lib, rs = _native.lib(), np.random.RandomState(9)
    sizes = [20001, 600011, 16385, 70000, 600011, 1000003, 20001, 1000003]
    need = int(lib.kvr_free_pages_workspace_bytes(max(sizes)))
    workspace = torch.zeros(need, dtype=torch.uint8, device="cuda")
    for pages in sizes:
        lengths, tables = rs.randint(0, 5000, 7), rs.randint(0, pages, (7, 313))
        wide, length = gpu(tables), gpu(lengths)
        out, start = torch.zeros(pages, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        status = _native.launch(wide.device, lib.kvr_free_pages, length.data_ptr(), wide.data_ptr(), 313, 7, 313, 16, pages,
                                out.data_ptr(), start.data_ptr(), workspace.data_ptr(), need)
        assert status == 0
        want, first = collected(lengths, tables, 16, pages)
        assert start.tolist() == first and np.array_equal(out.cpu().numpy(), np.array(want, np.int32))
