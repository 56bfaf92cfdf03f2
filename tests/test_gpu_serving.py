"""Turns of a server over one paged cache, as a program runs them: prompts in chunks
(chunk_attention), requests forked, drafted trees attended and verified, accepted rows
moved together, pages collected; every stage against books kept on the host (each request's
tokens with their K and V, layer by layer), then a turn captured in a graph against its
eager twin."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import test_gpu_chunk_attention
import test_gpu_tree_attention
import test_gpu_verification
from test_step_plan import gpu, walk

PAGE, PAGES, WIDTH, HEADS, KV, DIM, LAYERS, VOCAB = 16, 160, 30, 8, 2, 64, 2, 97


class Server:
    """Pools of all layers, requests' lengths and tables, the free list; and the books."""

    def __init__(self, requests, seed):
        from kv_cache_repair_amd.kernels.pages import FreePages, PagedCache

        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.keys, self.values = ([torch.full((1, KV, PAGES * PAGE, DIM), float("nan"), dtype=torch.bfloat16, device="cuda")
                                   for _ in range(LAYERS)] for _ in range(2))
        self.cache, self.free = PagedCache(self.keys, self.values, page_size=PAGE), FreePages(PAGES)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device="cuda")
        self.tables = torch.full((requests, WIDTH), -1, dtype=torch.int32, device="cuda")
        self.books = [[[] for _ in range(requests)] for _ in range(2 * LAYERS)]  # K of each layer, then V

    def rows(self, heads, count):
        return torch.randn(1, heads, count, DIM, device="cuda", generator=self.gen).bfloat16()

    def step(self, plan, counts, parents=None):
        """Plan a step and write its fresh rows; returns them by layer."""
        from kv_cache_repair_amd.kernels.indexed_attention import indexed_kv_scatter_

        before = self.tables.cpu().numpy()
        start = int(self.free.start)
        plan.update(self.lengths, gpu(counts), self.tables, self.free.pages, parents, self.free.start)
        expect = walk(self.lengths.tolist(), counts, before, self.free.pages.cpu().numpy(), PAGE, plan.rows, plan.max_rows,
                      PAGES, None if parents is None else parents.tolist(), free_start=start)
        assert not expect["status"].any() and np.array_equal(plan.slots.cpu().numpy(), expect["slots"])
        assert np.array_equal(self.tables.cpu().numpy(), expect["tables"])
        fresh = []
        for k, v in zip(self.keys, self.values):
            fresh.append((self.rows(KV, plan.rows), self.rows(KV, plan.rows)))
            indexed_kv_scatter_(k, v, *fresh[-1], plan)
        return expect, fresh

    def commit(self, fresh, starts, nodes):
        """Each request's nodes become tokens: in the books, and by their number."""
        for layer, (k, v) in enumerate(fresh):
            for r, mine in enumerate(nodes):
                for t in mine:
                    self.books[layer][r].append(k[0, :, starts[r] + t].clone())
                    self.books[LAYERS + layer][r].append(v[0, :, starts[r] + t].clone())
        self.lengths += gpu([len(n) for n in nodes])

    def check(self):
        """Every committed token stands where the tables say, and a page that none has is free."""
        tables, lengths = self.tables.cpu().numpy(), self.lengths.tolist()
        for i, pool in enumerate((*self.keys, *self.values)):
            for r, mine in enumerate(self.books[i]):
                assert len(mine) == lengths[r]
                token = np.arange(len(mine))
                slots = torch.from_numpy(tables[r][token // PAGE].astype(np.int64) * PAGE + token % PAGE).cuda()
                if mine:
                    assert torch.equal(pool[0][:, slots], torch.stack(mine, 1))
        self.free.collect(self.lengths, self.tables, page_size=PAGE)
        held = {int(p) for r, n in enumerate(lengths) for p in tables[r, :-(-n // PAGE)]}
        assert self.free.pages[int(self.free.start):].tolist() == sorted(set(range(PAGES)) - held)


@pytest.mark.gpu
def test_turns_of_a_server(gpu_device):
    from kv_cache_repair_amd.kernels.chunk_attention import chunk_attention
    from kv_cache_repair_amd.kernels.step_plan import StepPlan
    from kv_cache_repair_amd.kernels.tree_attention import tree_attention
    from kv_cache_repair_amd.kernels.verification import verify_drafts

    server = Server(2, 1)
    sizes = {"page_size": PAGE, "n_slots": PAGES * PAGE, "table_width": WIDTH}
    # ---- prompts, in two parts ----
    prompts = StepPlan(2, 260, max_rows=150, chunk_heads=(HEADS, KV), **sizes)
    for counts in ([150, 97], [66, 150]):
        expect, fresh = server.step(prompts, counts)
        for k, v in zip(server.keys, server.values):
            q = server.rows(HEADS, prompts.rows)
            want, size = test_gpu_chunk_attention.exact(q, k, v, expect, server.lengths.tolist(), counts, PAGE, PAGES, DIM ** -0.5)
            test_gpu_chunk_attention.assert_close(chunk_attention(q, k, v, prompts), want, size)
        server.commit(fresh, expect["row_starts"], [list(range(n)) for n in counts])
        server.check()
    # ---- three answers of the first prompt, two of the second ----
    sources = [0, 1, 0, 0, 1]
    done = server.cache.fork_(gpu(sources), server.lengths, server.tables, server.free.pages, server.free.start)
    assert done.status.tolist() == [0] * 5 and done.lengths.tolist() == [[216, 247][s] for s in sources]
    assert done.pages_taken.item() == 3  # 216 and 247 tokens both end inside a page
    server.lengths, server.tables = done.lengths, done.block_tables
    server.books = [[list(book[s]) for s in sources] for book in server.books]
    server.check()
    # ---- drafted trees, verified; then single tokens behind what was kept ----
    most, rs = 9, np.random.RandomState(4)
    drafts = StepPlan(5, 5 * most, max_rows=most, heads=(HEADS, KV), **sizes)
    kept_at_all = 0
    for turn in range(4):
        counts = [9, 7, 9, 1, 0] if turn % 2 == 0 else [1, 1, 1, 1, 1]
        parents = []
        for n in counts:  # one node of a long tree starts from the cache, and cannot hold
            parents += [-1] * (n > 0) + [rs.randint(-1 if t == 5 else 0, t) for t in range(1, n)]
        parents = gpu(parents + [-1] * (drafts.rows - len(parents)))
        expect, fresh = server.step(drafts, counts, parents)
        for k, v in zip(server.keys, server.values):
            q = server.rows(HEADS, drafts.rows)
            want, size = test_gpu_tree_attention.exact(q, k, v, expect, server.lengths.tolist(), counts, PAGE, PAGES, DIM ** -0.5)
            test_gpu_tree_attention.assert_close(tree_attention(q, k, v, drafts), want, size)
        probs = torch.softmax(torch.from_numpy(rs.standard_normal((drafts.rows, VOCAB)) * 6), -1).float()
        tokens = np.zeros(drafts.rows, np.int64)
        for row in range(drafts.rows):
            mask, start = int(expect["masks"][row]), int(expect["row_starts"][max(0, expect["request"][row])])
            above = mask & ~(1 << (row - start)) if mask else 0
            if above:
                tokens[row] = probs[start + above.bit_length() - 1].argmax()  # what the parent makes most likely
        uniforms, draws = rs.uniform(0, 1, drafts.rows).astype(np.float32), rs.uniform(0, 1, 5).astype(np.float32)
        found = verify_drafts(probs.cuda(), torch.from_numpy(tokens).cuda(), drafts, torch.from_numpy(uniforms).cuda(),
                              torch.from_numpy(draws).cuda())
        kept, path, answers = test_gpu_verification.verify(probs.numpy(), tokens, uniforms, draws, expect["masks"],
                                                           expect["row_starts"], drafts.rows)
        for got, w in zip(found, (kept, path, answers)):
            assert np.array_equal(got.cpu().numpy(), w)
        kept_at_all += int((kept - 1).clip(0).sum())
        server.cache.keep_rows_(drafts, found.path, found.kept)
        starts = expect["row_starts"]
        server.commit(fresh, starts, [path[starts[r]:starts[r] + kept[r]].tolist() for r in range(5)])
        server.check()
    assert kept_at_all >= 6  # the trees were deep enough for rows to move
    # ---- two of them go on, in another order, the others are done: their pages come back ----
    before = int(server.free.start)
    done = server.cache.fork_(gpu([3, -1, 0]), server.lengths, server.tables, server.free.pages, server.free.start)
    assert done.pages_taken.item() == 0
    server.lengths, server.tables = done.lengths, done.block_tables
    server.books = [[book[3], [], book[0]] for book in server.books]
    server.check()
    assert int(server.free.start) < before


@pytest.mark.gpu
def test_a_captured_turn(gpu_device):
    """Plan, verification, kept rows, lengths and free list in one graph: its replays leave the cache of an eager twin."""
    from kv_cache_repair_amd.kernels.step_plan import StepPlan
    from kv_cache_repair_amd.kernels.verification import verify_drafts

    R, most = 3, 6
    servers = [Server(R, 7) for _ in range(2)]
    plans = [StepPlan(R, R * most, page_size=PAGE, n_slots=PAGES * PAGE, table_width=WIDTH, max_rows=most) for _ in servers]
    probs = torch.zeros(R * most, VOCAB, device="cuda")
    tokens = torch.zeros(R * most, dtype=torch.int64, device="cuda")
    uniforms, draws = torch.zeros(R * most, device="cuda"), torch.zeros(R, device="cuda")
    counts, parents = gpu([most] * R), gpu([-1, 0, 0, 1, 2, 3] * R)
    for server in servers:
        for pool in (*server.keys, *server.values):
            pool.copy_(torch.arange(pool.numel(), device="cuda").view(pool.shape) % 251)

    def turn(server, plan):
        plan.update(server.lengths, counts, server.tables, server.free.pages, parents, server.free.start)
        done = verify_drafts(probs, tokens, plan, uniforms, draws)
        server.cache.keep_rows_(plan, done.path, done.kept)
        server.lengths.add_(done.kept)
        server.free.collect(server.lengths, server.tables, page_size=PAGE)
        return done

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for server, plan in zip(servers, plans):
            turn(server, plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = turn(servers[0], plans[0])
    rs = np.random.RandomState(3)
    moved = 0
    for _ in range(6):
        tokens.copy_(torch.from_numpy(rs.randint(0, 5, R * most)))
        probs.copy_(torch.from_numpy(np.concatenate((rs.uniform(0, 1, (R * most, 5)), np.zeros((R * most, VOCAB - 5))), 1)))
        probs.div_(probs.sum(1, keepdim=True))
        uniforms.copy_(torch.from_numpy(rs.uniform(0, 0.5, R * most)))
        draws.copy_(torch.from_numpy(rs.uniform(0, 1, R)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = turn(servers[1], plans[1])
        assert all(torch.equal(c, e) for c, e in zip(captured, eager))
        moved += int((eager.kept - 1).sum())
        for a, b in zip((*servers[0].keys, *servers[0].values, servers[0].lengths, servers[0].tables, servers[0].free.pages),
                        (*servers[1].keys, *servers[1].values, servers[1].lengths, servers[1].tables, servers[1].free.pages)):
            assert torch.equal(a, b)
    assert moved > 3


@pytest.mark.gpu
def test_a_turn_with_too_few_free_pages(gpu_device):
    """A request that finds no pages has written no rows: it keeps its length, the others go on, and its turn comes
    again. What stands in its table behind its length, another's pages here, is never attended."""
    from kv_cache_repair_amd.kernels.chunk_attention import chunk_attention
    from kv_cache_repair_amd.kernels.indexed_attention import indexed_kv_scatter_
    from kv_cache_repair_amd.kernels.step_plan import NO_PAGES, OK, StepPlan

    server = Server(4, 3)
    plan = StepPlan(4, 400, page_size=PAGE, n_slots=PAGES * PAGE, table_width=WIDTH, max_rows=150, chunk_heads=(HEADS, KV))
    expect, fresh = server.step(plan, [90, 40, 33, 0])
    server.commit(fresh, expect["row_starts"], [list(range(n)) for n in (90, 40, 33, 0)])
    server.check()
    for given, counts, status in ((4, [5, 100, 10, 100], [OK, NO_PAGES, OK, NO_PAGES]),
                                  (0, [0, 100, 5, 0], [OK, NO_PAGES, OK, OK]),
                                  (PAGES, [30, 100, 1, 150], [OK] * 4)):
        server.tables[1, 3:9] = server.tables[0, :6]     # entries that mean nothing
        before, start = server.tables.cpu().numpy(), int(server.free.start)
        lengths, pages = server.lengths.tolist(), server.free.pages[:min(PAGES, start + given)]
        plan.update(server.lengths, gpu(counts), server.tables, pages, free_start=server.free.start)
        expect = walk(lengths, counts, before, pages.cpu().numpy(), PAGE, plan.rows, plan.max_rows, PAGES, free_start=start)
        assert plan.status.tolist() == expect["status"].tolist() == status
        fresh = []
        for k, v in zip(server.keys, server.values):
            fresh.append((server.rows(KV, plan.rows), server.rows(KV, plan.rows)))
            indexed_kv_scatter_(k, v, *fresh[-1], plan)
            q = server.rows(HEADS, plan.rows)
            want, size = test_gpu_chunk_attention.exact(q, k, v, expect, lengths, counts, PAGE, PAGES, DIM ** -0.5)
            got = chunk_attention(q, k, v, plan)
            test_gpu_chunk_attention.assert_close(got, want, size)
            for r in range(4):
                if status[r] != OK:
                    assert not got[:, :, expect["row_starts"][r]:expect["row_starts"][r + 1]].any()
        # only what was planned is committed
        server.lengths += torch.where(plan.status == OK, gpu(counts), 0)
        for layer, (k, v) in enumerate(fresh):
            for r in range(4):
                rows = [expect["row_starts"][r] + t for t in range(counts[r]) if status[r] == OK]
                server.books[layer][r] += [k[0, :, row].clone() for row in rows]
                server.books[LAYERS + layer][r] += [v[0, :, row].clone() for row in rows]
        server.check()
    assert server.lengths.tolist() == [125, 140, 49, 150]
