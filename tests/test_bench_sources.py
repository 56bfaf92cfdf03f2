"""Recorded traffic counts only for the sources that it was measured on: all of a kernel's."""

from __future__ import annotations

import re

import pytest

import bench

CSRC = bench.ROOT / "budgeted-kv-cache-repair_amd" / "csrc"


@pytest.mark.parametrize("kernel", sorted(bench.KERNEL_SOURCES))
def test_a_digest_covers_the_headers_that_hold_kernel_code(kernel):
    """All that its sources include; kvr_internal.h, which every source includes, aside."""
    names = bench.KERNEL_SOURCES[kernel].split()
    for name in names:
        included = set(re.findall(r'#include "(kvr_\w+\.h)"', (CSRC / name).read_text()))
        assert included - {"kvr_internal.h"} <= set(names)
