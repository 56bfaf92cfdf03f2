"""tree_attention (kvr_tree_attention) against attention in float64 over the
plan's own definition (test_step_plan.walk), at every row-group size, head
layout and page size, with chunks that split and trees that branch; masked keys
that hold NaN and infinities; failed requests, pages outside the pool, rows of
no request; strides; captured steps.

Tolerance: the result is rounded once, half a step eps / 2 of the value. Before
that, with scores of a few units: products are exact in fp32 and a score's sum
of 128 of them is off by at most 128 * 2^-24 of sum |q k| * scale (about 8 here),
6e-5, so a weight by 6e-5 of itself (numerator and sum: 1.2e-4 at most); the
exponential, the hi + lo pair (2^-16 in bf16) and the sums add less than 4e-5.
Together less than 2^-12 of sum p |v|."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from test_step_plan import _desc, gpu, make, plan_of, walk

pytestmark = []
BF16, FP16 = torch.bfloat16, torch.float16


def exact(q, k, v, plan, lengths, counts, page, pages, scale):
    """(result, sum of p |v|) in float64 by the plan `walk` gives: rows that see nothing are zero."""
    _, heads, rows, dim = q.shape
    group = heads // k.shape[1]
    out = torch.zeros(heads, rows, dim, dtype=torch.float64)
    size = torch.zeros_like(out)
    q, k, v = (t.double().cpu() for t in (q, k, v))
    for r in range(len(lengths)):
        if plan["status"][r]:
            continue
        length, count, start = int(lengths[r]), int(counts[r]), int(plan["row_starts"][r])
        token = np.arange(length + count)
        page_of = plan["tables"][r][token // page].astype(np.int64)
        inside = (page_of >= 0) & (page_of < pages)
        slot = torch.from_numpy(np.where(inside, page_of * page + token % page, 0))
        for t in range(count):
            bits = int(plan["masks"][start + t])
            see = inside & np.array([bits != 0] * length + [bool(bits >> u & 1) for u in range(count)], bool)
            if not see.any():
                continue
            at = slot[torch.from_numpy(see)]
            for h in range(heads):
                p = torch.softmax(k[0, h // group][at] @ q[0, h, start + t] * scale, 0)
                out[h, start + t] = p @ v[0, h // group][at]
                size[h, start + t] = p @ v[0, h // group][at].abs()
    return out[None], size[None]


def assert_close(got, expect, size):
    eps = torch.finfo(got.dtype).eps
    got = got.double().cpu()
    # the result's type may have no smaller step than its smallest subnormal's
    bound = eps / 2 * expect.abs() + 2.0 ** -12 * size * (1 + eps) + (2.0 ** -25 if eps < 2.0 ** -8 else 0.0)
    off = (got - expect).abs()
    assert torch.isfinite(got).all() and (off <= bound).all(), (off - bound).max().item()


def tensors(seed, heads, kv_heads, dim, rows, slots, dtype, token_major=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape = (1, rows, heads, dim) if token_major else (1, heads, rows, dim)
    q = torch.randn(shape, device="cuda", generator=gen).to(dtype)
    k = torch.randn(1, kv_heads, slots, dim, device="cuda", generator=gen).to(dtype)
    v = torch.randn(1, kv_heads, slots, dim, device="cuda", generator=gen).to(dtype)
    return q.transpose(1, 2) if token_major else q, k, v


def step(seed, R, low, high, most, page, tree, heads, kv_heads, dim, dtype, fewest=0, **kw):
    rs = np.random.RandomState(seed)
    lengths, counts, tables, free, pages, rows, parents = make(rs, R, low, high, most, page, tree, fewest, **kw)
    expect = walk(lengths, counts, tables, free, page, rows, most, pages, parents)
    plan, _ = plan_of(lengths, counts, tables, free, page, rows, most, pages, parents, heads=(heads, kv_heads))
    q, k, v = tensors(seed, heads, kv_heads, dim, rows, pages * page, dtype)
    return lengths, counts, pages, expect, plan, q, k, v


CASES = [  # R, low, high, most, page, tree, heads, kv_heads, dim, dtype
    (1, 0, 0, 1, 16, False, 4, 4, 128, BF16), (1, 31, 31, 1, 16, False, 8, 2, 64, FP16),
    (1, 127, 127, 1, 32, False, 8, 2, 128, BF16), (1, 128, 128, 1, 16, False, 8, 2, 128, FP16),
    (3, 0, 40, 5, 16, True, 4, 2, 128, BF16), (5, 0, 700, 1, 16, False, 8, 8, 64, BF16),
    (2, 900, 1100, 64, 64, True, 8, 2, 128, BF16), (2, 900, 1100, 64, 64, True, 8, 2, 64, FP16),
    (4, 100, 3000, 8, 32, True, 8, 2, 128, FP16), (3, 2000, 2500, 4, 256, True, 7, 1, 128, BF16),
    (3, 2000, 2500, 9, 128, True, 14, 2, 64, BF16), (2, 0, 300, 64, 16, False, 16, 1, 128, BF16),
    (2, 0, 300, 33, 16, True, 32, 1, 64, FP16), (1, 5000, 5000, 3, 16, True, 4, 1, 128, BF16),
    (40, 0, 600, 2, 16, True, 4, 2, 64, BF16), (130, 0, 90, 3, 16, True, 2, 2, 128, BF16),
    (2, 500, 700, 26, 32, True, 8, 2, 128, FP16), (1, 700, 700, 64, 16, True, 20, 2, 128, BF16),
    (2, 40, 400, 2, 16, False, 260, 130, 64, BF16), (2, 40, 300, 1, 16, False, 300, 300, 64, FP16),
    (1, 40000, 40000, 2, 16, True, 1, 1, 64, BF16), (1, 9999, 9999, 64, 16, True, 3, 3, 64, FP16), (6, 1, 200, 16, 512, True, 3, 1, 128, BF16)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_matches_float64(gpu_device, case):
    R, low, high, most, page, tree, heads, kv_heads, dim, dtype = case
    from kv_cache_repair_amd.kernels.tree_attention import tree_attention

    lengths, counts, pages, expect, plan, q, k, v = step(11, *case, fewest=1 if R == 1 else 0)
    got = tree_attention(q, k, v, plan)
    want, size = exact(q, k, v, expect, lengths, counts, page, pages, dim ** -0.5)
    assert_close(got, want, size)
    assert torch.equal(got, tree_attention(q, k, v, plan))  # no sum depends on the order of arrival


@pytest.mark.gpu
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, FP16)])
@pytest.mark.parametrize("most", [1, 13, 64])
def test_what_a_row_does_not_see_never_reaches_it(gpu_device, dim, dtype, most):
    """NaN and infinities in every slot that no row sees, and in drafted keys that
    only some rows see: rows that do not see them are exact, rows that do are not finite."""
    from kv_cache_repair_amd.kernels.tree_attention import tree_attention

    lengths, counts, pages, expect, plan, q, k, v = step(7, 5, 0, 333, most, 16, True, 8, 2, dim, dtype, fewest=1,
                                                         padded=0.15)
    used = torch.zeros(pages * 16, dtype=torch.bool)
    for r in range(5):
        token = np.arange(int(lengths[r]))
        used[torch.from_numpy(expect["tables"][r][token // 16].astype(np.int64) * 16 + token % 16)] = True
    slots = torch.from_numpy(expect["slots"])
    used[slots[slots >= 0]] = True
    bad = torch.tensor([math.nan, math.inf, -math.inf], dtype=dtype, device="cuda")
    hidden = (~used).nonzero()[:, 0].cuda()
    for t, shift in ((k, 0), (v, 1)):
        t[:, :, hidden] = bad[(torch.arange(dim, device="cuda") + shift) % 3]
    want, size = exact(q, k, v, expect, lengths, counts, 16, pages, dim ** -0.5)
    assert torch.isfinite(want).all()
    assert_close(tree_attention(q, k, v, plan), want, size)
    # a drafted value of one branch: only the rows that see it
    start = expect["row_starts"]
    r = int(np.argmax(counts))
    row = int(start[r]) + int(counts[r]) - 1
    while expect["slots"][row] < 0:
        row -= 1
    node = row - int(start[r])
    v[0, 0, slots[row].item(), 3] = math.inf
    k[0, 1, slots[row].item(), 5] = math.nan
    got = tree_attention(q, k, v, plan).cpu()
    for i in range(int(start[r]), int(start[r]) + int(counts[r])):
        sees = bool(int(expect["masks"][i]) >> node & 1)
        assert torch.isfinite(got[0, :4, i, :3]).all() and torch.isfinite(got[0, :4, i, 4:]).all()
        assert (got[0, :4, i, 3] == math.inf).all() if sees else torch.isfinite(got[0, :4, i, 3]).all()
        assert torch.isnan(got[0, 4:, i]).all() if sees else torch.isfinite(got[0, 4:, i]).all()
        if not sees:
            row_got, row_want = got[:, :, i].double(), want[:, :, i]
            assert ((row_got - row_want).abs() <= 2.0 ** -7 * size[:, :, i] + 1e-30).all()


@pytest.mark.gpu
def test_failed_requests_and_pages_outside_the_pool(gpu_device):
    from kv_cache_repair_amd.kernels.tree_attention import tree_attention

    rs = np.random.RandomState(2)
    lengths, counts, tables, free, pages, rows, _ = make(rs, 8, 300, 900, 7, 16, False, fewest=2)
    lengths[1], counts[3] = -1, 9                    # INVALID, with more rows than a request may have
    tables[4, 2:5] = [-1, pages, 1 << 30]            # 48 keys of one request, 16 of another, not to be read
    tables[6, 0] = -(1 << 31)
    free = free[:-4]
    rows = int(np.maximum(counts, 0).sum()) + 6
    expect = walk(lengths, counts, tables, free, 16, rows, 7, pages)
    assert expect["status"].tolist()[1] == 3 and expect["status"].tolist()[3] == 3 and 0 in expect["status"]
    plan, _ = plan_of(lengths, counts, tables, free, 16, rows, 7, pages, heads=(8, 2))
    q, k, v = tensors(4, 8, 2, 128, rows, pages * 16, BF16)
    want, size = exact(q, k, v, expect, lengths, counts, 16, pages, 0.07)
    assert_close(tree_attention(q, k, v, plan, scale=0.07), want, size)


@pytest.mark.gpu
def test_only_pages_outside_the_pool(gpu_device):
    """A request none of whose keys can be read: zeros, no NaN."""
    from kv_cache_repair_amd.kernels.tree_attention import tree_attention

    tables = np.full((2, 3), 99)
    tables[1] = [0, 1, 2]
    lengths, counts, free = np.array([40, 40]), np.array([3, 3]), np.arange(3, 6)
    plan, _ = plan_of(lengths, counts, tables, free, 16, 6, 3, 6, heads=(4, 2))
    q, k, v = tensors(1, 4, 2, 64, 6, 96, BF16)
    got = tree_attention(q, k, v, plan)
    expect = walk(lengths, counts, tables, free, 16, 6, 3, 6)
    want, size = exact(q, k, v, expect, lengths, counts, 16, 6, 64 ** -0.5)
    assert_close(got, want, size)
    assert (got[:, :, :3] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_scores_far_apart(gpu_device, dtype):
    """Maxima that move in every sub-tile, and weights that vanish beside them."""
    from kv_cache_repair_amd.kernels.tree_attention import tree_attention

    lengths, counts, pages, expect, plan, q, k, v = step(3, 2, 1500, 1600, 3, 16, True, 4, 2, 128, dtype, fewest=2)
    ramp = torch.ones(pages * 16, device="cuda")
    for r in range(2):
        token = np.arange(int(lengths[r]))
        ramp[torch.from_numpy(expect["tables"][r][token // 16].astype(np.int64) * 16 + token % 16)] = \
            torch.linspace(0.05, 3.0, len(token), device="cuda")
    k.mul_(ramp[None, None, :, None])
    want, size = exact(q, k, v, expect, lengths, counts, 16, pages, 128 ** -0.5)
    got = tree_attention(q, k, v, plan)
    # three times the scores of the other tests: three times their absolute error
    eps = torch.finfo(dtype).eps
    assert ((got.double().cpu() - want).abs() <= eps / 2 * want.abs() + 3 * 2.0 ** -12 * size * (1 + eps)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_layouts_give_the_same_bits(gpu_device, dim):
    """Head-major and token-major queries, pools and outputs, padded rows, sliced heads."""
    from kv_cache_repair_amd.kernels.tree_attention import tree_attention

    lengths, counts, pages, expect, plan, q, k, v = step(9, 4, 0, 500, 6, 32, True, 8, 4, dim, BF16, fewest=1)
    want = tree_attention(q, k, v, plan)
    slots, rows = pages * 32, plan.rows
    for qq in (q.contiguous(), torch.cat((q, q), 3)[..., :dim], torch.cat((q, q), 1)[:, 8:]):
        assert torch.equal(tree_attention(qq, k, v, plan), want)
    major = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]
    assert torch.equal(tree_attention(q, *major, plan), want)
    both = torch.cat((k, v), 3)
    assert torch.equal(tree_attention(q, both[..., :dim], both[..., dim:], plan), want)
    assert torch.equal(tree_attention(q, k, torch.cat((v, v), 1)[:, 4:], plan), want)
    held = torch.full((1, 8, rows + 2, dim + 4), 3.0, dtype=BF16, device="cuda")
    out = held[:, :, 1:rows + 1, 4:]
    assert tree_attention(q, k, v, plan, out=out) is out
    total = int(expect["row_starts"][-1])
    assert total < rows
    assert torch.equal(out[:, :, :total], want[:, :, :total]) and (want[:, :, total:] == 0).all()
    out[:, :, :total] = 3.0
    assert (held == 3.0).all()  # rows of no request, and everything between the rows, as they were


@pytest.mark.gpu
def test_strides_of_a_single_head_and_row_may_be_anything(gpu_device):
    from kv_cache_repair_amd.kernels.step_plan import StepPlan
    from kv_cache_repair_amd.kernels.tree_attention import tree_attention

    plan = StepPlan(1, 1, page_size=16, n_slots=64, table_width=4, heads=(1, 1))
    plan.update(gpu([37]), gpu([1]), gpu([[2, 0, 3, 1]]))
    q, k, v = tensors(4, 1, 1, 64, 1, 64, BF16)
    want = tree_attention(q, k, v, plan)
    qq = q.as_strided(q.shape, (0, 0, 1, 1))
    kk, vv = (t.as_strided(t.shape, (7, 0, 64, 1)) for t in (k, v))
    out = torch.zeros(64, dtype=BF16, device="cuda").as_strided((1, 1, 1, 64), (1, 3, 5, 1))
    assert torch.equal(tree_attention(qq, kk, vv, plan, out=out), want) and want.any()


@pytest.mark.gpu
def test_a_pool_past_32_bits(gpu_device):
    """Slots whose byte and element offsets pass 2^31 and 2^32."""
    from kv_cache_repair_amd.kernels.tree_attention import tree_attention

    page, pages, dim = 256, 160 * 1024, 128   # 40 M slots of 128: 5.4e9 elements in K
    k = torch.zeros(1, 1, pages * page, dim, dtype=BF16, device="cuda")
    tables = np.array([[pages - 1, 3, pages // 2, -1], [pages - 2, 1, pages // 4, pages - 3]])
    lengths, counts, free = np.array([730, 800]), np.array([63, 2]), np.array([pages - 5])
    expect = walk(lengths, counts, tables, free, page, 65, 64, pages)
    plan, _ = plan_of(lengths, counts, tables, free, page, 65, 64, pages, heads=(4, 1))
    gen = torch.Generator(device="cuda").manual_seed(1)
    used = torch.tensor(sorted({int(p) for p in expect["tables"].ravel() if p >= 0}), device="cuda")
    for p in used.tolist():
        k[0, 0, p * page:(p + 1) * page] = torch.randn(page, dim, device="cuda", generator=gen).to(BF16)
    q = torch.randn(1, 65, 4, dim, device="cuda", generator=gen).to(BF16).transpose(1, 2)
    got = tree_attention(q, k, k, plan)
    # the same step over a small pool of the pages that are used
    index = {p: i for i, p in enumerate(used.tolist())}
    small = torch.cat([k[:, :, p * page:(p + 1) * page] for p in used.tolist()], 2)
    near = np.vectorize(lambda p: index.get(int(p), -1))(expect["tables"])
    near_free = np.array([index[pages - 5]])
    plan_near, _ = plan_of(lengths, counts, near, near_free, page, 65, 64, len(index), heads=(4, 1))
    assert torch.equal(got, tree_attention(q, small, small, plan_near))
    expect = walk(lengths, counts, near, near_free, page, 65, 64, len(index))
    want, size = exact(q, small, small, expect, lengths, counts, page, len(index), dim ** -0.5)
    assert_close(got, want, size)


@pytest.mark.gpu
def test_another_stream_and_a_captured_step(gpu_device):
    """Update and attention on a stream of their own, then captured and replayed with
    other lengths and values, eager calls of the same plan's shapes between the replays."""
    from kv_cache_repair_amd.kernels.step_plan import StepPlan
    from kv_cache_repair_amd.kernels.tree_attention import tree_attention

    R, page, most, width, pages = 6, 16, 9, 90, 600
    held = StepPlan(R, R * most, page_size=page, n_slots=pages * page, table_width=width, max_rows=most, heads=(8, 2))
    other = StepPlan(R, R * most, page_size=page, n_slots=pages * page, table_width=width, max_rows=most, heads=(8, 2))
    ints = {n: torch.zeros(R, dtype=torch.int32, device="cuda") for n in ("lengths", "counts")}
    ints |= {"block_tables": torch.zeros(R, width, dtype=torch.int32, device="cuda"),
             "free_pages": torch.zeros(pages, dtype=torch.int32, device="cuda"),
             "parents": torch.full((R * most,), -1, dtype=torch.int32, device="cuda")}
    q, k, v = tensors(1, 8, 2, 128, R * most, pages * page, BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        held.update(**ints)
        tree_attention(q, k, v, held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held.update(**ints)
        got = tree_attention(q, k, v, held)
    rs = np.random.RandomState(8)
    for turn in range(4):
        lengths, counts = rs.randint(0, 1300, R), rs.randint(0, most + 1, R)
        order, table, at = rs.permutation(pages), np.zeros((R, width), int), 0
        for r in range(R):
            have = -(-int(lengths[r]) // page)
            table[r, :have] = order[at:at + have]
            at += have
        parents = np.array([rs.randint(-1, 2) for _ in range(R * most)])
        free = np.concatenate((order[at:], order[:at]))
        for name, value in (("lengths", lengths), ("counts", counts), ("block_tables", table), ("free_pages", free),
                            ("parents", parents)):
            ints[name].copy_(gpu(value))
        q.copy_(torch.randn(q.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(turn)).to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        eager = tree_attention(q, k, v, other.update(**ints))
        assert torch.equal(got, eager)
        expect = walk(lengths, counts, table, free, page, R * most, most, pages, parents)
        want, size = exact(q, k, v, expect, lengths, counts, page, pages, 128 ** -0.5)
        assert_close(got, want, size)


@pytest.mark.gpu
def test_two_steps_at_once(gpu_device):
    """Two plans on two streams without waiting for each other."""
    from kv_cache_repair_amd.kernels.tree_attention import tree_attention

    steps = [step(seed, 4, 2000, 9000, 5, 16, True, 16, 4, 128, BF16, fewest=1) for seed in (1, 2)]
    alone = [tree_attention(*s[5:], s[4]) for s in steps]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in steps], [[], []]
    for _ in range(5):
        for i, (s, stream) in enumerate(zip(steps, streams)):
            with torch.cuda.stream(stream):
                got[i].append(tree_attention(*s[5:], s[4]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, alone[i]) for i in range(2) for g in got[i])


@pytest.mark.gpu
def test_checks_its_tensors(gpu_device):
    from kv_cache_repair_amd.kernels.step_plan import StepPlan
    from kv_cache_repair_amd.kernels.tree_attention import tree_attention

    lengths, counts, pages, _, plan, q, k, v = step(1, 2, 5, 50, 3, 16, False, 4, 2, 64, BF16)
    tree_attention(q, k, v, plan)
    bare = StepPlan(2, plan.rows, page_size=16, n_slots=pages * 16, table_width=9, max_rows=3)
    new = StepPlan(2, plan.rows, page_size=16, n_slots=pages * 16, table_width=9, max_rows=3, heads=(4, 2))
    odd = torch.zeros(1, 2, pages * 16, 65, dtype=BF16, device="cuda")[..., 1:]
    for bad in ((q, k, v, bare), (q, k, v, new), (q, k, v, None), (q.float(), k, v, plan), (q, k.half(), v, plan),
                (q, k, v[:, :, 1:], plan), (q[:, :2], k, v, plan), (q[..., :32], k[..., :32], v[..., :32], plan),
                (q[:, :, 1:], k, v, plan), (q, k.cpu(), v, plan), (q, odd, v, plan), (q, k, odd, plan),
                (q, k[:, :1].expand(1, 2, -1, -1), v, plan), (q.clone().requires_grad_(), k, v, plan)):
        with pytest.raises(ValueError):
            tree_attention(*bad)
    for scale in (0, -1.0, math.nan, math.inf, True, "1"):
        with pytest.raises(ValueError, match="scale"):
            tree_attention(q, k, v, plan, scale=scale)
    for out in (q, torch.empty_like(q).float(), torch.empty(1, 4, plan.rows, 66, dtype=BF16, device="cuda")[..., 1:65],
                torch.empty(1, 4, 1, 64, dtype=BF16, device="cuda").expand(1, 4, plan.rows, 64)):
        with pytest.raises(ValueError):
            tree_attention(q, k, v, plan, out=out)


STRIDES = [64, 256, 1] + 2 * [65536, 64, 1] + [64, 256, 1]


@pytest.mark.parametrize("status,desc,call", [
    (-2, {}, {"dtype": 0}), (-5, {"schedule": None}, {}), (-3, {}, {"dim": 96}), (-1, {}, {"scale": 0.0}),
    (-1, {}, {"scale": -1.0}), (-1, {}, {"scale": math.nan}), (-1, {}, {"scale": math.inf}), (-5, {}, {"q": None}),
    (-5, {}, {"k": None}), (-5, {}, {"v": None}), (-5, {}, {"out": None}), (-4, {}, {"q": (1 << 30) + 8}),
    (-4, {}, {"k": (1 << 30) + 2}), (-4, {}, {"out": (1 << 30) + 4}), (-4, {}, {"strides": (2, 2)}),
    (-4, {}, {"strides": (0, 60)}), (-4, {}, {"strides": (4, (1 << 26) + 8)}), (-4, {}, {"strides": (10, 258)}),
    (-4, {}, {"strides": (6, 0)}), (-6, {}, {"workspace": None}), (-6, {}, {"workspace": (1 << 30) + 8}),
    (-6, {}, {"bytes": -1}), (-3, {"requests": 0}, {}), (-3, {"max_rows": 65}, {})])
def test_attention_refuses_before_any_launch(status, desc, call):
    from kv_cache_repair_amd import _native

    lib, d = _native.lib(), _desc(**desc)
    strides = list(STRIDES)
    if "strides" in call:
        strides[call["strides"][0]] = call["strides"][1]
    need = lib.kvr_tree_workspace_bytes(ctypes.byref(_desc()), 64)
    assert need > 0
    at = 1 << 30
    assert lib.kvr_tree_attention(
        call.get("q", at), call.get("k", at), call.get("v", at), call.get("out", at), ctypes.byref(d),
        call.get("dim", 64), call.get("scale", 0.125), _native.i64_array(strides), 0, call.get("workspace", at),
        need + call.get("bytes", 0), call.get("dtype", 2), None) == status
