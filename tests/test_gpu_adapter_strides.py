"""Adapter projections of any row strides, at row counts on both sides of the tiled
projections' first (65) and of where these add the adapters' part themselves (257):
strides past 2^21 elements, outputs that those projections cannot write. Tolerance:
test_gpu_adapters'."""

from __future__ import annotations

import ctypes

import pytest
import torch

from test_gpu_adapters import BF16, _call, assert_close, exact, make

LONG = (1 << 21) + 8  # elements of a row


def spread(t, ld, offset=0):
    """The values of t in rows ld elements apart."""
    held = torch.empty(offset + (t.shape[0] - 1) * ld + t.shape[1], dtype=t.dtype, device=t.device)
    out = held[offset:].as_strided(t.shape, (ld, 1))
    return out.copy_(t)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [64, 65, 200, 300])
@pytest.mark.parametrize("long", ["x", "weight"])
def test_rows_far_apart(gpu_device, m, long):
    from kv_cache_repair_amd.kernels.adapters import AdapterProjectionPlan

    x, weights, down, up, scales = make(1, m, 128, (64, 8), 3, 16, BF16)
    ids = (torch.arange(m, device="cuda") % 4).int()
    want = exact(x, weights, down, up, scales, ids)
    if long == "x":
        x = spread(x, LONG)
    else:
        weights[0] = spread(weights[0], LONG)
    assert_close(AdapterProjectionPlan(weights, down, up, scales)(x, ids), *want)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [64, 65, 300])
@pytest.mark.parametrize("ldy,offset", [(75, 0), (76, 1), (74, 2), (80, 0)])
def test_outputs_of_any_stride_and_alignment(gpu_device, m, ldy, offset):
    """The C entry: ldy no multiple of 4, y on an odd element; what lies between the rows stays."""
    from kv_cache_repair_amd import _native

    lib = _native.lib()
    x, weights, down, up, scales = make(2, m, 128, (64, 8), 3, 16, BF16)
    ids = (torch.arange(m, device="cuda") % 4).int()
    held = torch.full((offset + m * ldy,), 5.0, dtype=BF16, device="cuda")
    y = held[offset:].view(m, ldy)
    rows = (ctypes.c_int32 * 2)(64, 8)
    need = lib.kvr_adapter_linear_workspace_bytes(m, 2, rows, 128, 16)
    workspace = torch.empty(need, dtype=torch.uint8, device="cuda")
    at = lambda ts: (ctypes.c_void_p * 2)(*(t.data_ptr() for t in ts))  # noqa: E731
    status = lib.kvr_adapter_linear(
        x.data_ptr(), 2, at(weights), rows, _native.i64_array([128, 128]), at(down), at(up), scales.data_ptr(), 3, 16,
        ids.data_ptr(), y.data_ptr(), m, 128, 128, ldy, workspace.data_ptr(), need, 2,
        torch.cuda.current_stream().cuda_stream)
    assert status == 0
    assert_close(y[:, :72], *exact(x, weights, down, up, scales, ids))
    assert (y[:, 72:] == 5).all() and (held[:offset] == 5).all()


@pytest.mark.parametrize("changes", [{"ldx": LONG}, {"ldw": [LONG, 128]}, {"ldy": 97}, {"y": (1 << 30) + 2}])
@pytest.mark.parametrize("m", [64, 65, 300])
def test_strides_do_not_depend_on_the_row_count(changes, m):
    """Nothing but the workspace that is too small refuses them."""
    assert _call(m=m, bytes=1024, **changes) == -6


def test_the_workspace_holds_either_projection():
    """Of 65 rows on it has room for 64 rows at a time too."""
    from kv_cache_repair_amd import _native

    lib, rows = _native.lib(), (ctypes.c_int32 * 2)(64, 32)
    sizes = [lib.kvr_adapter_linear_workspace_bytes(m, 2, rows, 4096, 16) for m in (64, 65, 300, 4096)]
    assert all(s >= sizes[0] for s in sizes)


@pytest.mark.gpu
def test_weights_whose_rows_overlap(gpu_device):
    """Refused by the plan; a single row has no stride to look at."""
    from kv_cache_repair_amd.kernels.adapters import AdapterProjectionPlan

    x, weights, down, up, scales = make(3, 5, 128, (16, 1), 2, 8, BF16)
    for bad in (weights[0][:1].expand(16, 128), weights[0].as_strided((16, 128), (64, 1))):
        with pytest.raises(ValueError, match="rows"):
            AdapterProjectionPlan([bad, weights[1]], down, up, scales)
    ids = (torch.arange(5, device="cuda") % 3).int()
    want = AdapterProjectionPlan(weights, down, up, scales)(x, ids)
    one = weights[1].as_strided((1, 128), (0, 1))
    assert torch.equal(AdapterProjectionPlan([weights[0], one], down, up, scales)(x, ids), want)


@pytest.mark.gpu
def test_tensors_with_other_storage_are_not_read(gpu_device):
    """What a plan has bound is gone when a module is moved or cast: refused, not read."""
    from kv_cache_repair_amd.kernels.adapters import AdapterProjectionPlan

    x, weights, down, up, scales = make(4, 3, 128, (16, 8), 2, 8, BF16)
    weights = [torch.nn.Parameter(w, requires_grad=False) for w in weights]
    ids = (torch.arange(3, device="cuda") % 3).int()
    for t in (weights[1], down[0], up[1], scales):
        plan = AdapterProjectionPlan(weights, down, up, scales)
        want = plan(x, ids)
        old = t.data
        t.data = old * 2
        with pytest.raises(ValueError, match="new plan"):
            plan(x, ids)
        assert not torch.equal(AdapterProjectionPlan(weights, down, up, scales)(x, ids), want)
        t.data = old
        assert torch.equal(plan(x, ids), want)
