"""What an AdapterProjectionPlan keeps from call to call: the workspace sizes of a few row counts."""

from __future__ import annotations

import ctypes


def test_a_plan_keeps_the_sizes_of_a_few_row_counts():
    from kv_cache_repair_amd import _native
    from kv_cache_repair_amd.kernels.adapters import AdapterProjectionPlan

    plan = AdapterProjectionPlan.__new__(AdapterProjectionPlan)  # its sizes alone, which need no device
    plan._count, plan._rows, plan.k, plan.rank, plan._workspace = 1, (ctypes.c_int32 * 1)(64), 128, 16, {}
    for m in (*range(1, 400), 1, 399):
        assert plan.workspace_bytes(m) == _native.lib().kvr_adapter_linear_workspace_bytes(m, 1, plan._rows, 128, 16)
        assert len(plan._workspace) <= 64
