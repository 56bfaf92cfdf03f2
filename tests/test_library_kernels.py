"""Kernels that the library holds: none that no call can reach."""

from __future__ import annotations

import shutil
import subprocess

import pytest

from kv_cache_repair_amd import _native


def symbols() -> list:
    tool = shutil.which("nm")
    if tool is None:
        pytest.skip("no nm")
    return subprocess.run([tool, "-C", _native.lib()._name], check=True, capture_output=True, text=True).stdout.splitlines()


def test_no_streaming_tile_adds_adapters():
    """The tiled projection adds adapters' parts from 257 rows on, and streams its weights up to 192."""
    tiles = [line for line in symbols() if "tiled_gemm_kernel<" in line]
    assert any(", true, " in line for line in tiles) and any("AdapterEpilogue>" in line for line in tiles)
    assert not [line for line in tiles if ", true, " in line and "AdapterEpilogue>" in line]
