"""verify_drafts (kvr_verify_drafts) against a plain walk from its definition, node by
node and token by token in Python's own floats (64 bits): chains and trees, with and
without the drafts' own probabilities; borders hit exactly; nothing left; entries that
do not count; failed requests and padding nodes; strides; captured calls; that answers come
from the target's distribution; what is refused.

All is decided in 64 bits, so the results have to be equal: the sums' order moves a border
by 2^-50 of the whole, and random numbers of 24 bits are not that near one."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from test_step_plan import _desc, gpu, make, plan_of, walk


def sane(w):
    return float(w) if 0 < w < math.inf else 0.0


def chosen(weights, draw):
    """The first token whose running sum exceeds the draw's share; the last that counts where none does."""
    whole, run, last = sum(weights.tolist()), 0.0, -1
    for i in np.nonzero(weights)[0].tolist():
        run += float(weights[i])
        last = i
        if run > float(draw) * whole:
            return i
    return last


def verify(probs, tokens, uniforms, draws, masks, starts, rows, drafts=None):
    """(kept, path, answers) by the definition."""
    vocab = probs.shape[1]
    path, kept, answers = np.full(rows, -1, np.int32), [], []
    for r in range(len(starts) - 1):
        start, n = int(starts[r]), int(starts[r + 1] - starts[r])
        seen = {t: {u for u in range(t + 1) if int(masks[start + t]) >> u & 1} for t in range(min(n, 64))}
        branch = [0] if n and seen[0] else []
        while branch:
            a = branch[-1]
            p = np.array([sane(w) for w in probs[start + a].astype(np.float64)])
            hang = [t for t in seen if t > a and seen[t] == set(branch) | {t}]
            u, below, names, taken = float(uniforms[start + a]), 0.0, set(), None
            for i, t in enumerate(hang):
                x = int(tokens[start + t])
                if x in names:
                    continue
                names.add(x)
                chance = p[x] if 0 <= x < vocab else 0.0
                if drafts is None:
                    below += chance
                    good = chance > 0 and u < below
                else:
                    q = float(drafts[start + a, x]) if 0 <= x < vocab else 0.0
                    good = i == 0 and chance > 0 and u * q < chance
                if good:
                    taken = t
                    break
            if taken is not None:
                branch.append(taken)
                continue
            left = p.copy()
            if hang and drafts is not None:
                with np.errstate(invalid="ignore"):
                    left = probs[start + a].astype(np.float64) - drafts[start + a].astype(np.float64)
                left = np.array([sane(w) for w in left])
            else:
                left[[int(tokens[start + t]) for t in hang if 0 <= tokens[start + t] < vocab]] = 0.0
            answers.append(chosen(left if left.any() else p, draws[r]))
            break
        if not branch:
            answers.append(-1)
        kept.append(len(branch))
        path[start:start + len(branch)] = branch
    return np.array(kept, np.int32), path, np.array(answers, np.int64)


def step(seed, R, most, tree, vocab, fewest=0, sharp=2.0, drafts=False, padded=0.1):
    rs = np.random.RandomState(seed)
    lengths, counts, tables, free, pages, rows, parents = make(rs, R, 0, 40, most, 16, tree, fewest, padded=padded)
    if tree:
        # most nodes hang on node 0 or what hangs on it: those that start from the cache cannot hold
        at = 0
        for n in counts.tolist():
            for t in range(1, n):
                if parents[at + t] == -1 and rs.uniform() < 0.8:
                    parents[at + t] = rs.randint(0, t)
            if n and rs.uniform() < 0.9:
                parents[at] = -1
            at += n
    expect = walk(lengths, counts, tables, free, 16, rows, most, pages, parents)
    plan, _ = plan_of(lengths, counts, tables, free, 16, rows, most, pages, parents)
    logits = rs.standard_normal((rows, vocab)) * sharp
    probs = torch.softmax(torch.from_numpy(logits), -1).float()
    q = torch.softmax(torch.from_numpy(logits + rs.standard_normal((rows, vocab))), -1).float() if drafts else None
    tokens = np.zeros(rows, np.int64)
    for r in range(R):
        for t in range(1, counts[r]):
            row = int(expect["row_starts"][r]) + t
            seen = int(expect["masks"][row])
            up = (seen & ~(1 << t)).bit_length() - 1
            from_ = q if drafts else probs
            tokens[row] = torch.multinomial(from_[row - t + max(up, 0)], 1,
                                            generator=torch.Generator().manual_seed(row * 7 + seed)).item()
    uniforms, draws = rs.uniform(0, 1, rows).astype(np.float32), rs.uniform(0, 1, R).astype(np.float32)
    return plan, expect, probs, tokens, uniforms, draws, q


def run(plan, probs, tokens, uniforms, draws, q=None):
    from kv_cache_repair_amd.kernels.verification import verify_drafts

    done = verify_drafts(probs.cuda(), torch.from_numpy(tokens).cuda(), plan, torch.from_numpy(uniforms).cuda(),
                         torch.from_numpy(draws).cuda(), draft_probs=None if q is None else q.cuda())
    return [t.cpu().numpy() for t in done]


def check(plan, expect, probs, tokens, uniforms, draws, q=None):
    got = run(plan, probs, tokens, uniforms, draws, q)
    want = verify(probs.numpy(), tokens, uniforms, draws, expect["masks"], expect["row_starts"], plan.rows,
                  None if q is None else q.numpy())
    for name, g, w in zip(("kept", "path", "answers"), got, want):
        assert g.dtype == w.dtype and np.array_equal(g, w), (name, np.nonzero(g != w)[0][:5])
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("R,most,tree,vocab,drafts", [
    (1, 1, False, 1, False), (1, 2, False, 3, True), (3, 5, False, 64, False), (3, 5, False, 65, True),
    (20, 6, False, 1000, True), (20, 64, False, 257, False), (9, 64, True, 100, False), (40, 13, True, 33, False),
    (5, 26, True, 4099, False), (300, 3, True, 17, False), (2, 3, False, 70001, True), (2, 4, True, 70003, False),
    (130, 4, False, 4096, True), (2000, 2, True, 11, False)])
def test_matches_its_definition(gpu_device, R, most, tree, vocab, drafts):
    s = step(R + most, R, most, tree, vocab, fewest=1 if R < 4 else 0, drafts=drafts)
    kept, _, _ = check(*s)
    if R >= 20 and most > 2:
        assert (kept > 1).any()


@pytest.mark.gpu
@pytest.mark.parametrize("draw", [0.0, 1 - 2.0 ** -24, 0.5])
@pytest.mark.parametrize("uniform", [0.0, 1 - 2.0 ** -24])
def test_first_and_last_numbers(gpu_device, draw, uniform):
    """The smallest and largest numbers: zero takes what has any chance, and no token without one."""
    plan, expect, probs, tokens, uniforms, draws, _ = step(4, 12, 8, True, 500, fewest=1)
    probs[:, ::3] = 0.0
    uniforms[:], draws[:] = uniform, draw
    _, path, answers = check(plan, expect, probs, tokens, uniforms, draws)
    assert all(answers[answers >= 0] % 3 != 0)


@pytest.mark.gpu
def test_borders_belong_to_the_next_token(gpu_device):
    """Numbers that are a running sum exactly: the sum has to exceed them."""
    lengths, counts = np.array([3] * 4), np.array([4] * 4)
    parents = np.array([-1, 0, 0, 0] * 4)
    tables = np.arange(4)[:, None]
    expect = walk(lengths, counts, tables, [], 16, 16, 4, 4, parents)
    plan, _ = plan_of(lengths, counts, tables, np.zeros(0), 16, 16, 4, 4, parents)
    probs = torch.zeros(16, 8)
    probs[:, 2], probs[:, 3], probs[:, 5], probs[:, 6] = 0.25, 0.25, 0.125, 0.375
    tokens = np.tile([0, 3, 2, 6], 4)
    uniforms, draws = np.zeros(16, np.float32), np.zeros(4, np.float32)
    uniforms[[0, 4, 8, 12]] = [0.25, 0.5, 0.875, 0.25 - 2.0 ** -26]
    uniforms[[1, 2, 3]] = 0.9
    draws[:] = [0.25, 0.5, 0.625, 0.0]
    kept, path, answers = check(plan, expect, probs, tokens, uniforms, draws)
    # 0.25 is past token 3's share: the second child; 0.5 the third; 0.875 none, the rest is token 5's; below 0.25 the first
    assert kept.tolist() == [2, 2, 1, 2] and path[[1, 5, 13]].tolist() == [2, 3, 1]
    assert answers.tolist() == [3, 5, 5, 2]


@pytest.mark.gpu
def test_nothing_left(gpu_device):
    """Children that have all of the mass, a draft equal to the target, rows without any mass."""
    lengths, counts, tables = np.array([3] * 5), np.array([2] * 5), np.arange(5)[:, None]
    expect = walk(lengths, counts, tables, [], 16, 10, 2, 5)
    plan, _ = plan_of(lengths, counts, tables, np.zeros(0), 16, 10, 2, 5)
    probs = torch.zeros(10, 300)
    probs[:, 7], probs[:, 299] = 0.5, 0.5
    tokens = np.array([0, 7] * 5)
    uniforms, draws = np.full(10, 0.75, np.float32), np.full(5, 0.75, np.float32)
    q = probs.clone()
    q[2, 7] = 0.75          # refused, and nothing above the draft's but at 299
    q[4, 7], q[4, 299] = 0.75, 0.6  # refused, and nothing left: the target's own
    probs[6] = 0.0          # no mass at all
    probs[8, 7] = math.nan  # an entry that does not count
    kept, _, answers = check(plan, expect, probs, tokens, uniforms, draws, q)
    assert kept.tolist() == [2, 1, 1, 1, 1] and answers.tolist() == [299, 299, 299, -1, 299]
    probs[:] = 0.0
    probs[:, 7] = 1.0
    uniforms[:] = 1.0       # outside [0, 1): the child is not kept though it has all of the mass
    kept, _, answers = check(plan, expect, probs, tokens, uniforms, draws)
    assert kept.tolist() == [1] * 5 and answers.tolist() == [7] * 5


@pytest.mark.gpu
@pytest.mark.parametrize("drafts", [False, True])
def test_entries_that_do_not_count(gpu_device, drafts):
    """NaN, infinities and negative values count as zero, wherever they stand; tokens outside the vocabulary are not kept."""
    plan, expect, probs, tokens, uniforms, draws, q = step(8, 30, 6, not drafts, 700, fewest=1, drafts=drafts)
    rs = np.random.RandomState(1)
    bad = torch.tensor([math.nan, math.inf, -math.inf, -0.5, -0.0])
    for t in (probs, q):
        if t is not None:
            at = torch.from_numpy(rs.uniform(0, 1, t.shape) < 0.2)
            t[at] = bad[torch.from_numpy(rs.randint(0, 5, int(at.sum())))]
    tokens[rs.uniform(0, 1, tokens.size) < 0.2] = rs.choice([-1, 700, 1 << 40, -(1 << 40)])
    check(plan, expect, probs, tokens, uniforms, draws, q)
    uniforms[::3], draws[::4] = math.nan, math.nan
    check(plan, expect, probs, tokens, uniforms, draws, q)


@pytest.mark.gpu
def test_numbers_outside_their_range(gpu_device):
    """Below 0 as 0, and 1 or more as nothing taken: the same in chains, trees and draws."""
    for drafts in (False, True):
        plan, expect, probs, tokens, uniforms, draws, q = step(12, 20, 7, not drafts, 60, fewest=1, drafts=drafts)
        uniforms[:], draws[:] = -0.5, 7.0
        uniforms[::5], draws[::3] = 1.5, -1.0
        kept, _, answers = check(plan, expect, probs, tokens, uniforms, draws, q)
        assert (kept > 1).any() and (answers[kept > 0] >= 0).all()


@pytest.mark.gpu
def test_a_tree_that_a_graph_plans(gpu_device):
    """A plan that is updated without parents and then, by a graph, with them holds a tree all the same."""
    from kv_cache_repair_amd.kernels.step_plan import StepPlan
    from kv_cache_repair_amd.kernels.verification import verify_drafts

    plan = StepPlan(1, 4, page_size=16, n_slots=16, table_width=1, max_rows=4)
    args = gpu([3]), gpu([4]), gpu([[0]])
    parents = gpu([-1, 0, 0, 0])
    plan.update(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.update(*args, parents=parents)
    plan.update(*args)
    graph.replay()
    probs = torch.tensor([[0.25, 0.25, 0.25, 0.25]] * 4, device="cuda")
    done = verify_drafts(probs, torch.tensor([0, 1, 2, 3], device="cuda"), plan, torch.full((4,), 0.6, device="cuda"),
                         torch.zeros(1, device="cuda"))
    assert done.kept.tolist() == [2] and done.path.tolist() == [0, 3, -1, -1] and done.answers.tolist() == [0]


@pytest.mark.gpu
def test_the_same_token_twice(gpu_device):
    """Siblings of one token: the second never holds, and their token leaves the row once."""
    plan, expect, probs, tokens, uniforms, draws, _ = step(2, 60, 20, True, 4, fewest=2, sharp=0.5, padded=0.0)
    kept, _, _ = check(plan, expect, probs, tokens, uniforms, draws)
    assert (kept > 2).any()


@pytest.mark.gpu
@pytest.mark.parametrize("tree", [False, True])
def test_failed_requests_and_rows_of_none(gpu_device, tree):
    rs = np.random.RandomState(3)
    lengths, counts, tables, free, pages, rows, parents = make(rs, 12, 1, 120, 9, 16, tree, fewest=2)
    lengths[2], counts[5], counts[7], lengths[8] = -4, -1, 90, 16 * tables.shape[1]
    rows = int(np.maximum(counts, 0).sum()) + 5
    parents = None if parents is None else np.resize(parents, rows)
    expect = walk(lengths, counts, tables, free, 16, rows, 9, pages, parents)
    assert (expect["status"] != 0).sum() >= 4
    plan, _ = plan_of(lengths, counts, tables, free, 16, rows, 9, pages, parents)
    probs = torch.softmax(torch.from_numpy(rs.standard_normal((rows, 50))), -1).float()
    tokens = rs.randint(0, 50, rows)
    uniforms, draws = rs.uniform(0, 0.3, rows).astype(np.float32), rs.uniform(0, 1, 12).astype(np.float32)
    kept, path, answers = check(plan, expect, probs, tokens, uniforms, draws)
    assert (kept[[2, 5, 7, 8]] == 0).all() and (answers[[2, 5, 7, 8]] == -1).all() and (path[-5:] == -1).all()


@pytest.mark.gpu
def test_rows_apart_and_odd_addresses(gpu_device):
    from kv_cache_repair_amd.kernels.verification import verify_drafts

    plan, expect, probs, tokens, uniforms, draws, q = step(6, 7, 5, False, 1001, fewest=1, drafts=True)
    args = torch.from_numpy(tokens).cuda(), plan, torch.from_numpy(uniforms).cuda(), torch.from_numpy(draws).cuda()
    want = verify_drafts(probs.cuda(), *args, draft_probs=q.cuda())
    wide = [torch.full((plan.rows, 1001 + pad + 1), math.nan, device="cuda") for pad in (2, 7)]
    views = [w[:, 1:1002] for w in wide]
    for view, t in zip(views, (probs, q)):
        view.copy_(t)
    got = verify_drafts(views[0], *args, draft_probs=views[1])
    assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.gpu
def test_rows_past_32_bits(gpu_device):
    """Rows whose element offsets pass 2^31 and 2^32."""
    from kv_cache_repair_amd.kernels.verification import verify_drafts

    R, vocab = 140, 1 << 19  # 64 rows each: 8960 rows, 4.7e9 values
    lengths, counts = np.full(R, 3), np.full(R, 64)
    tables, free = np.arange(5 * R).reshape(R, 5), np.arange(5 * R).reshape(R, 5)[:, 1:].ravel()
    plan, _ = plan_of(lengths, counts, tables, free, 16, 64 * R, 64, 5 * R)
    probs = torch.zeros(64 * R, vocab, device="cuda")
    at = torch.arange(64 * R, device="cuda")
    probs[at, at * 53 % vocab] = 1.0
    tokens = torch.cat((at.new_zeros(1), (at * 53 % vocab)[:-1]))
    tokens[64 * (R - 1) + 40] += 1
    half = torch.full((64 * R,), 0.5, device="cuda")
    done = verify_drafts(probs, tokens, plan, half, half[:R])
    want = torch.full((R,), 64, dtype=torch.int32)
    want[-1] = 40
    assert torch.equal(done.kept.cpu(), want)
    last = torch.arange(R) * 64 + want - 1
    assert torch.equal(done.answers.cpu(), last * 53 % vocab)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["chain", "drawn", "tree"])
def test_answers_come_from_the_target(gpu_device, kind):
    """The token after node 0 has the target's distribution, whatever was drafted: counts of 4000
    requests a turn, each within five standard deviations of its own."""
    R, vocab, turns = 4000, 6, 5
    n = 4 if kind == "tree" else 2
    p = torch.tensor([0.05, 0.4, 0.1, 0.25, 0.2, 0.0])
    q = torch.tensor([0.3, 0.1, 0.1, 0.3, 0.1, 0.1])
    lengths, counts, tables = np.full(R, 3), np.full(R, n), np.arange(R)[:, None]
    parents = np.tile([-1, 0, 0, 0], R) if kind == "tree" else None
    plan, _ = plan_of(lengths, counts, tables, np.zeros(0), 16, n * R, n, R, parents)
    probs, drafts = p.repeat(n * R, 1), q.repeat(n * R, 1)
    rs, found = np.random.RandomState(0), np.zeros(vocab)
    for _ in range(turns):
        tokens = rs.choice(vocab, n * R, p=q.double().numpy() / q.double().sum().item())
        uniforms, draws = rs.uniform(0, 1, n * R).astype(np.float32), rs.uniform(0, 1, R).astype(np.float32)
        kept, path, answers = run(plan, probs, tokens, np.minimum(uniforms, np.float32(1 - 2.0 ** -24)),
                                  np.minimum(draws, np.float32(1 - 2.0 ** -24)), drafts if kind == "drawn" else None)
        first = np.where(kept > 1, tokens[np.arange(R) * n + np.maximum(path.reshape(R, n)[:, 1], 0)], answers)
        found += np.bincount(first, minlength=vocab)
    total = R * turns
    share = p.double().numpy()
    assert (np.abs(found - total * share) <= 5 * np.sqrt(total * share * (1 - share))).all()


@pytest.mark.gpu
def test_captured_calls_follow_their_inputs(gpu_device):
    from kv_cache_repair_amd.kernels.verification import verify_drafts

    plan, expect, probs, tokens, uniforms, draws, q = step(6, 9, 6, False, 3001, fewest=1, drafts=True)
    held = [probs.cuda(), torch.from_numpy(tokens).cuda(), torch.from_numpy(uniforms).cuda(),
            torch.from_numpy(draws).cuda(), q.cuda()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        verify_drafts(held[0], held[1], plan, held[2], held[3], held[4])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        done = verify_drafts(held[0], held[1], plan, held[2], held[3], held[4])
    rs = np.random.RandomState(2)
    for _ in range(3):
        uniforms, draws = rs.uniform(0, 1, uniforms.size).astype(np.float32), rs.uniform(0, 1, 9).astype(np.float32)
        held[2].copy_(torch.from_numpy(uniforms))
        held[3].copy_(torch.from_numpy(draws))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = verify(probs.numpy(), tokens, uniforms, draws, expect["masks"], expect["row_starts"], plan.rows, q.numpy())
        assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip(done, want))
        eager = verify_drafts(held[0], held[1], plan, held[2], held[3], held[4])
        assert all(torch.equal(g, e) for g, e in zip(done, eager))


@pytest.mark.gpu
def test_checks_its_tensors(gpu_device):
    from kv_cache_repair_amd.kernels.step_plan import StepPlan
    from kv_cache_repair_amd.kernels.verification import verify_drafts

    plan = StepPlan(2, 6, page_size=16, n_slots=64, table_width=2, max_rows=3)
    ok = {"probs": torch.ones(6, 9, device="cuda"), "tokens": torch.zeros(6, dtype=torch.int64, device="cuda"), "plan": plan,
          "uniforms": torch.zeros(6, device="cuda"), "draws": torch.zeros(2, device="cuda")}
    with pytest.raises(ValueError, match="updated"):
        verify_drafts(**ok)
    plan.update(gpu([1, 1]), gpu([3, 3]), gpu([[0, 1], [2, 3]]), parents=gpu([-1, 0, 0] * 2))
    verify_drafts(**ok)
    many = StepPlan(2, 6, page_size=16, n_slots=64, table_width=20, max_rows=65)
    for name, bad in (("plan", None), ("plan", many), ("probs", ok["probs"].half()), ("probs", ok["probs"].cpu()),
                      ("probs", ok["probs"][:5]), ("probs", ok["probs"].t().contiguous().t()), ("probs", ok["probs"][0]),
                      ("probs", ok["probs"][:1].expand(6, 9)), ("probs", ok["probs"][:, :0]), ("tokens", ok["tokens"].int()),
                      ("tokens", ok["tokens"][:5]), ("uniforms", ok["uniforms"].double()), ("uniforms", None),
                      ("draws", ok["uniforms"]), ("draws", torch.zeros(4, device="cuda")[::2]),
                      ("draft_probs", ok["probs"][:, :8]), ("probs", ok["probs"].clone().requires_grad_())):
        with pytest.raises(ValueError):
            verify_drafts(**(ok | {name: bad}))
    with pytest.raises(ValueError, match="chains"):
        verify_drafts(**ok, draft_probs=ok["probs"])


@pytest.mark.parametrize("status,desc,call", [
    (-5, {}, {"probs": None}), (-5, {}, {"tokens": None}), (-5, {}, {"uniforms": None}), (-5, {}, {"draws": None}),
    (-5, {}, {"kept": None}), (-5, {}, {"path": None}), (-5, {}, {"answers": None}), (-4, {}, {"ld": 99}),
    (-4, {}, {"ldd": 99}), (-3, {}, {"vocab": 0}), (-3, {}, {"vocab": (1 << 30) + 1}), (-3, {"requests": 0}, {}),
    (-3, {"schedule": None, "masks": None, "max_rows": 65}, {})])
def test_refuses_before_any_launch(status, desc, call):
    from kv_cache_repair_amd import _native

    at = {name: call.get(name, 1 << 20) for name in ("probs", "drafts", "tokens", "uniforms", "draws", "kept", "path",
                                                     "answers")}
    assert _native.lib().kvr_verify_drafts(
        at["probs"], call.get("ld", 100), at["drafts"], call.get("ldd", 100), call.get("vocab", 100), at["tokens"],
        at["uniforms"], at["draws"], ctypes.byref(_desc(**desc)), at["kept"], at["path"], at["answers"], None, 0, None) == status


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [9, 40009])
def test_draft_entries_enter_as_they_are(gpu_device, vocab):
    """What counts as zero is an entry of the target's, and a difference, not a draft's entry by itself: an infinite
    or NaN one leaves nothing of its token, a negative one adds to it, and a product that is NaN or +inf keeps nothing."""
    odd = [math.nan, math.inf, -math.inf, -0.25]
    R = 2 * len(odd)
    plan, _ = plan_of(np.full(R, 3), np.full(R, 2), np.arange(R)[:, None], np.zeros(0), 16, 2 * R, 2, R)
    probs, q = torch.zeros(2 * R, vocab), torch.zeros(2 * R, vocab)
    probs[:, 2], probs[:, 5] = 0.25, 0.5
    tokens = np.tile([0, 5], R)
    for i, value in enumerate(odd):
        q[2 * i, 5] = value                          # of the drafted token
        q[2 * (len(odd) + i), 2] = value             # of another one, and the drafted one is refused
        q[2 * (len(odd) + i), 5] = 2.0
    uniforms, draws = np.full(2 * R, 0.5, np.float32), np.full(R, 0.125, np.float32)
    got = run(plan, probs, tokens, uniforms, draws, q)
    # NaN and inf refuse it and leave token 2 alone; below zero it is kept, and the next row is drawn from
    assert got[0][:4].tolist() == [1, 1, 2, 2] and got[2][:4].tolist() == [2, 2, 2, 2]
    # token 2's share: none (nothing left: the target's own, of which an eighth is token 2's), or 0.5
    assert got[0][4:].tolist() == [1] * 4 and got[2][4:].tolist() == [2] * 4
    draws[:] = 0.5
    got = run(plan, probs, tokens, uniforms, draws, q)
    assert got[2].tolist() == [2, 2, 5, 5, 5, 5, 5, 2]
