"""Adapter projections (kvr_adapter_linear, kernels/adapters.py) against float64:
both projection kernels, shapes that neither takes at once, one to three weights
whose boundaries cut tiles, ranks that leave half a tile, rows of one adapter and
of many, in any order, and of none.

Tolerance: the result is rounded once, half a step. Before that the fp32 sums are
off by at most 2^-20 of the sums of their products' sizes (assert_linear_close's
bound of the projections), and the inner product enters the second one as two
16-bit values, off by at most 2^-17 of it (bf16: 2^-9 of what 2^-9 leaves), in
fp16 2^-22 of the largest of 16 ranks."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

BF16, FP16 = torch.bfloat16, torch.float16


def make(seed, m, k, widths, count, rank, dtype, std=0.05):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, device="cuda", generator=gen)  # noqa: E731
    x = rand(m, k).to(dtype)
    weights = [(rand(n, k) * 0.02).to(dtype) for n in widths]
    down = [(rand(count, rank, k) * k ** -0.5).to(dtype) for _ in widths]
    up = [(rand(count, n, rank) * std).to(dtype) for n in widths]
    scales = torch.rand(count, device="cuda", generator=gen) + 0.5
    return x, weights, down, up, scales


def exact(x, weights, down, up, scales, ids):
    """(result, error allowed before the rounding) in float64."""
    parts, allowed = [], []
    x = x.double()
    for w, a, b in zip(weights, down, up):
        y, off = x @ w.double().T, 2.0 ** -20 * (x.abs() @ w.double().abs().T)
        for ad in range(len(scales)):
            rows = (ids == ad).nonzero()[:, 0]
            if not len(rows):
                continue
            s, t = scales[ad].double(), x[rows] @ a[ad].double().T
            t_off = 2.0 ** -20 * (x[rows].abs() @ a[ad].double().abs().T) + 2.0 ** -17 * t.abs() \
                + 2.0 ** -22 * t.abs().amax(1, keepdim=True) + 2.0 ** -20 * t.abs()
            y[rows] += s * (t @ b[ad].double().T)
            off[rows] += s * (t_off @ b[ad].double().abs().T)
        parts.append(y)
        allowed.append(off)
    return torch.cat(parts, 1), torch.cat(allowed, 1)


def assert_close(got, want, off):
    info = torch.finfo(got.dtype)
    bound = info.eps / 2 * (want.abs() + off) + off + (2.0 ** -25 if got.dtype == FP16 else 0.0)
    far = (got.double() - want).abs() - bound
    assert torch.isfinite(got).all() and (far <= 0).all(), far.max().item()


CASES = [  # rows, k, widths, adapters, rank, dtype
    (1, 256, (64,), 1, 8, BF16), (1, 4096, (4096, 1024, 1024), 4, 16, BF16), (2, 8, (1,), 3, 8, FP16),
    (3, 1000, (17, 5, 130), 2, 24, BF16), (16, 520, (40,), 16, 40, FP16), (17, 512, (72, 8, 24), 30, 64, BF16),
    (37, 4096, (520,), 5, 8, FP16), (64, 14336, (256,), 64, 16, BF16), (64, 2048, (16384 + 33,), 9, 16, BF16),
    (64, 640, (200, 100), 3, 136, FP16), (65, 512, (64,), 7, 16, BF16), (80, 1024, (264, 72, 40), 80, 16, FP16),
    (129, 4096, (512,), 4, 128, BF16), (300, 640, (768, 256), 6, 72, BF16), (1000, 256, (4096,), 2, 32, FP16),
    (700, 512, (768, 256, 64), 1, 64, BF16), (600, 64, (512,), 2, 32, BF16), (1100, 1024, (1024, 128), 3, 64, FP16),
    (256, 192, (264,), 1, 32, FP16), (100, 4096, (4096,), 1, 96, BF16),
    (70, 500 * 8, (100,), 5, 16, BF16), (130, 64 * 5, (33, 7), 5, 16, FP16), (2051, 128, (136,), 11, 8, BF16),
    (81, 640, (1416,), 47, 16, FP16), (256, 1024, (264, 72), 200, 24, BF16), (255, 4096, (64, 8, 8), 5, 64, BF16),
    (257, 512, (264, 72), 90, 16, BF16), (320, 704, (528,), 1, 32, FP16)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
@pytest.mark.parametrize("order", ["mixed", "runs"])
def test_matches_float64(gpu_device, case, order):
    from kv_cache_repair_amd.kernels.adapters import AdapterProjectionPlan

    m, k, widths, count, rank, dtype = case
    x, weights, down, up, scales = make(1, m, k, widths, count, rank, dtype)
    gen = torch.Generator().manual_seed(m)
    ids = torch.randint(-1, count, (m,), generator=gen)
    if order == "runs":
        ids = ids.sort().values
    ids = ids.int().cuda()
    plan = AdapterProjectionPlan(weights, down, up, scales)
    got = plan(x, ids)
    assert_close(got, *exact(x, weights, down, up, scales, ids))
    assert torch.equal(got, plan(x, ids))


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,widths", [(5, 512, (72,)), (64, 4096, (4096, 1024)), (200, 512, (512, 64)),
                                       (300, 512, (512, 64))])
def test_no_adapter_is_the_projection_alone(gpu_device, m, k, widths):
    """Ids outside the pool, whatever they are; adapters of zeros and of zero scale."""
    from kv_cache_repair_amd.kernels.adapters import AdapterProjectionPlan

    x, weights, down, up, scales = make(2, m, k, widths, 3, 16, BF16)
    plan = AdapterProjectionPlan(weights, down, up, scales)
    ids = torch.tensor([-1, 3, -(1 << 31), (1 << 31) - 1], device="cuda").repeat(m)[:m].int()
    alone = plan(x, ids)
    assert_close(alone, *exact(x, weights, down, up, scales, ids))
    some = torch.arange(m, device="cuda").int() % 3
    for zeroed in (up, [scales]):
        for t in zeroed:
            t.zero_()
        assert torch.equal(plan(x, some), alone)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [6, 64, 130, 300])
def test_infinities_stay_with_their_rows_and_weights(gpu_device, m):
    from kv_cache_repair_amd.kernels.adapters import AdapterProjectionPlan

    x, weights, down, up, scales = make(3, m, 512, (40, 24), 3, 16, BF16)
    ids = (torch.arange(m, device="cuda") % 3).int()
    want, off = exact(x, weights, down, up, scales, ids)
    down[0][1, 3, 7] = math.inf      # adapter 1, first weight
    up[1][2, 5, 2] = math.nan        # adapter 2, one column of the second weight
    got = AdapterProjectionPlan(weights, down, up, scales)(x, ids)
    hit = torch.zeros_like(want, dtype=torch.bool)
    hit[ids == 1, :40] = True
    hit[ids == 2, 45] = True
    assert not torch.isfinite(got[hit]).any()
    assert_close(torch.where(hit, torch.zeros_like(got), got), want.masked_fill(hit, 0), off.masked_fill(hit, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** -14, 1.0, 2.0 ** 7])
def test_inner_products_of_any_size_in_fp16(gpu_device, size):
    """Inner products that fp16 itself would lose or overflow on: up to 2^7 * 2^10 and down to 2^-24."""
    from kv_cache_repair_amd.kernels.adapters import adapter_linear

    x, (w,), (a,), (b,), scales = make(4, 20, 1024, (64,), 2, 16, FP16)
    w.zero_()
    x = (x.abs() * size).to(FP16)
    a = (a.abs() * 32 * size).to(FP16)
    b = (b / size / max(size, 1) / 2 ** 5).to(FP16) if size >= 1 else b
    ids = (torch.arange(20, device="cuda") % 2).int()
    got = adapter_linear(x, w, a, b, scales, ids)
    assert_close(got, *exact(x, [w], [a], [b], scales, ids))


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** -9, 1.0, 2.0 ** 5])
def test_inner_products_of_any_size_in_fp16_over_many_rows(gpu_device, size):
    """The same over a tile's rows of one adapter: with and without a power of two of their own."""
    from kv_cache_repair_amd.kernels.adapters import adapter_linear

    x, (w,), (a,), (b,), scales = make(4, 300, 512, (128,), 2, 32, FP16)
    x = (x * size).to(FP16)
    x[:100] *= 2.0 ** -4
    a = (a * 32 * size).to(FP16)
    b = (b / size).clamp(-100, 100).to(FP16)
    ids = (torch.arange(300, device="cuda") >= 290).int()
    got = adapter_linear(x, w, a, b, scales, ids)
    assert_close(got, *exact(x, [w], [a], [b], scales, ids))


@pytest.mark.gpu
def test_infinities_in_a_tile_of_one_adapter(gpu_device):
    from kv_cache_repair_amd.kernels.adapters import AdapterProjectionPlan

    x, weights, down, up, scales = make(3, 700, 512, (512, 128), 2, 32, BF16)
    ids = torch.zeros(700, device="cuda").int()
    want, off = exact(x, weights, down, up, scales, ids)
    up[0][0, 5, 2] = math.nan
    up[0][1] = math.inf
    got = AdapterProjectionPlan(weights, down, up, scales)(x, ids)
    hit = torch.zeros_like(want, dtype=torch.bool)
    hit[:, 5] = True
    assert torch.isnan(got[hit]).all()
    assert_close(torch.where(hit, torch.zeros_like(got), got), want.masked_fill(hit, 0), off.masked_fill(hit, 0))


@pytest.mark.gpu
def test_layouts_and_shapes_of_x(gpu_device):
    from kv_cache_repair_amd.kernels.adapters import AdapterProjectionPlan

    x, weights, down, up, scales = make(5, 24, 256, (72, 24), 4, 16, BF16)
    wide = [torch.cat((w, w), 1)[:, :256] for w in weights]  # padded rows
    plan = AdapterProjectionPlan(weights, down, up, scales)
    ids = (torch.arange(24, device="cuda") % 5).int()
    want = plan(x, ids)
    assert torch.equal(AdapterProjectionPlan(wide, down, up, scales)(x, ids), want)
    assert torch.equal(plan(torch.cat((x, x), 1)[:, 256:], ids), want)
    assert torch.equal(plan(x.view(2, 3, 4, 256), ids.view(2, 12)), want.view(2, 3, 4, 96))

    assert plan(x[:0], ids[:0]).shape == (0, 96)
    assert torch.equal(plan(x[3], ids[3:4]), plan(x[3:4], ids[3:4])[0])


@pytest.mark.gpu
def test_pools_past_32_bits(gpu_device):
    """The last adapter of pools whose offsets pass 2^31 elements."""
    from kv_cache_repair_amd.kernels.adapters import AdapterProjectionPlan

    count, rank, k, n = 9000, 64, 4096, 4096  # 2.4e9 elements a pool
    gen = torch.Generator(device="cuda").manual_seed(1)
    down = torch.zeros(count, rank, k, dtype=BF16, device="cuda")
    up = torch.zeros(count, n, rank, dtype=BF16, device="cuda")
    x, (w,), _, _, _ = make(6, 3, k, (n,), 1, 8, BF16)
    scales = torch.ones(count, device="cuda")
    for ad in (0, count - 1):
        down[ad] = torch.randn(rank, k, device="cuda", generator=gen) / 64
        up[ad] = torch.randn(n, rank, device="cuda", generator=gen) / 20
    ids = torch.tensor([count - 1, 0, count], device="cuda").int()
    got = AdapterProjectionPlan([w], [down], [up], scales)(x, ids)
    small = torch.tensor([1, 0, -1], device="cuda").int()
    pick = torch.tensor([0, count - 1], device="cuda")
    want = exact(x, [w], [down[pick]], [up[pick]], scales[:2], small)
    assert_close(got, *want)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [33, 200, 300])
def test_captured_and_on_two_streams(gpu_device, m):
    from kv_cache_repair_amd.kernels.adapters import AdapterProjectionPlan

    x, weights, down, up, scales = make(7, m, 1024, (520, 264), 6, 16, BF16)
    plan = AdapterProjectionPlan(weights, down, up, scales)
    ids = torch.zeros(m, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        plan(x, ids)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs of the same plan, which share nothing that they write
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = plan(x, ids)
        graphs.append((graph, got))
    for turn in range(3):
        gen = torch.Generator().manual_seed(turn)
        x.copy_(torch.randn(x.shape, generator=gen))
        ids.copy_(torch.randint(-1, 6, (m,), generator=gen))
        torch.cuda.synchronize()
        for (graph, _), stream in zip(graphs, (side, torch.cuda.Stream())):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        eager = plan(x, ids)
        assert all(torch.equal(got, eager) for _, got in graphs)
        assert_close(eager, *exact(x, weights, down, up, scales, ids))


@pytest.mark.gpu
def test_checks_its_tensors(gpu_device):
    from kv_cache_repair_amd.kernels.adapters import AdapterProjectionPlan

    x, weights, down, up, scales = make(8, 4, 256, (72, 24), 3, 16, BF16)
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    plan = AdapterProjectionPlan(weights, down, up, scales)
    for bad in ((weights * 2, down * 2, up * 2, scales), ([], [], [], scales), (weights, down[:1], up, scales),
                (weights, down, up[::-1], scales), (weights, [d[:, :12] for d in down], [u[..., :12] for u in up], scales),
                (weights, [d[:, :, :128] for d in down], up, scales), (weights, down, up, scales.double()),
                (weights, down, up, scales[:2]), (weights, down, [u.float() for u in up], scales),
                (weights, [d.transpose(1, 2).contiguous().transpose(1, 2) for d in down], up, scales),
                ([w.float() for w in weights], down, up, scales),
                (weights, down, up, scales.clone().requires_grad_())):
        with pytest.raises(ValueError):
            AdapterProjectionPlan(*bad)
    for bad_x, bad_ids in ((x.half(), ids), (x[:, :128], ids), (x.cpu(), ids), (x, ids.long()), (x, ids[:3]),
                           (x, ids.cpu()), (x, torch.zeros(8, dtype=torch.int32, device="cuda")[::2]),
                           (torch.cat((x, x[:, :4]), 1)[:, :256], ids), (torch.cat((x, x), 1)[:, 1:257], ids),
                           (x.t().contiguous().t(), ids), (x.clone().requires_grad_(), ids)):
        with pytest.raises(ValueError):
            plan(bad_x, bad_ids)
    for t in (weights[0], down[1], up[0], scales):  # gradients asked for after the plan was made
        t.requires_grad_()
        with pytest.raises(ValueError, match="detach"):
            plan(x, ids)
        with torch.no_grad():
            plan(x, ids)
        t.requires_grad_(False)
    plan(x, ids)


def _call(**changes):
    from kv_cache_repair_amd import _native

    at = 1 << 30  # aligned, never read: every call below is refused
    c = {"x": at, "weights": 2, "w": [at, at], "rows": [64, 32], "ldw": [128, 128], "down": [at, at], "up": [at, at],
         "scales": at, "adapters": 4, "rank": 16, "ids": at, "y": at, "m": 8, "k": 128, "ldx": 128, "ldy": 96,
         "workspace": at, "bytes": 1 << 40, "dtype": 2} | changes
    lib = _native.lib()
    pointers = lambda v: None if v is None else (ctypes.c_void_p * len(v))(*v)  # noqa: E731
    return lib.kvr_adapter_linear(
        c["x"], c["weights"], pointers(c["w"]), (ctypes.c_int32 * 2)(*c["rows"]), _native.i64_array(c["ldw"]),
        pointers(c["down"]), pointers(c["up"]), c["scales"], c["adapters"], c["rank"], c["ids"], c["y"], c["m"], c["k"],
        c["ldx"], c["ldy"], c["workspace"], c["bytes"], c["dtype"], None)


@pytest.mark.parametrize("status,changes", [
    (-2, {"dtype": 0}), (-1, {"weights": 0}), (-1, {"weights": 4}), (-3, {"rows": [64, 0]}), (-3, {"m": 0}),
    (-3, {"m": (1 << 20) + 1}), (-3, {"k": 132}), (-3, {"k": 0}), (-3, {"rank": 0}), (-3, {"rank": 12}),
    (-3, {"rank": 520}), (-3, {"adapters": 0}), (-5, {"x": None}), (-5, {"w": None}), (-5, {"w": [1 << 30, None]}),
    (-5, {"down": None}), (-5, {"up": [None, 1 << 30]}), (-5, {"scales": None}), (-5, {"ids": None}), (-5, {"y": None}),
    (-4, {"ldw": [128, 120]}), (-4, {"ldw": [132, 128]}), (-4, {"w": [(1 << 30) + 8, 1 << 30]}),
    (-4, {"down": [(1 << 30) + 8, 1 << 30]}), (-4, {"up": [1 << 30, (1 << 30) + 8]}), (-4, {"ldx": 120}),
    (-4, {"ldx": 132}), (-4, {"ldy": 95}), (-4, {"x": (1 << 30) + 8}), (-4, {"y": (1 << 30) + 1}),
    (-6, {"workspace": None}), (-6, {"workspace": (1 << 30) + 8}), (-6, {"bytes": 1024}),
    (-3, {"m": 1 << 20, "rows": [1 << 23, 1 << 23]})])
def test_adapter_linear_refuses_before_any_launch(status, changes):
    assert _call(**changes) == status


def test_workspace_sizes():
    from kv_cache_repair_amd import _native

    lib, rows = _native.lib(), (ctypes.c_int32 * 2)(64, 32)
    sizes = [lib.kvr_adapter_linear_workspace_bytes(m, 2, rows, 128, 16) for m in (1, 64, 65, 4096)]
    assert all(s > 0 for s in sizes)
    assert lib.kvr_adapter_linear_workspace_bytes(0, 2, rows, 128, 16) == -3
    assert lib.kvr_adapter_linear_workspace_bytes(8, 2, rows, 128, 20) == -3
