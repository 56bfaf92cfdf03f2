"""Static LDS of the library's kernels, from the metadata of the code objects that it holds."""

from __future__ import annotations

import re
import struct
from pathlib import Path

import pytest

from kv_cache_repair_amd import _native


def static_lds() -> dict:
    """Bytes of every kernel, by name: the code objects' notes."""
    msgpack = pytest.importorskip("msgpack")
    data, found, at = Path(_native.lib()._name).read_bytes(), {}, 0
    while (at := data.find(b"__CLANG_OFFLOAD_BUNDLE__", at)) >= 0:
        entry = at + 32
        for _ in range(struct.unpack_from("<Q", data, at + 24)[0]):
            offset, size, name = struct.unpack_from("<QQQ", data, entry)
            target, entry = data[entry + 24:entry + 24 + name], entry + 24 + name
            if b"gfx950" not in target or not size:
                continue
            elf = data[at + offset:at + offset + size]
            headers, = struct.unpack_from("<Q", elf, 40)
            each, count = struct.unpack_from("<HH", elf, 58)
            for header in range(headers, headers + each * count, each):
                if struct.unpack_from("<I", elf, header + 4)[0] == 7:  # notes
                    note, = struct.unpack_from("<Q", elf, header + 24)
                    owner, length, _ = struct.unpack_from("<III", elf, note)
                    text = note + 12 + (owner + 3) // 4 * 4
                    for kernel in msgpack.unpackb(elf[text:text + length])["amdhsa.kernels"]:
                        found[kernel[".name"]] = kernel[".group_segment_fixed_size"]
        at += 24
    return found


def test_chunk_stages_start_at_rows():
    """The dynamic LDS of chunk attention follows the static part: rows of K and V stay where their addresses' bits are
    changed by XOR, and the launch asks for both parts."""
    source = (Path(__file__).resolve().parents[1] / "budgeted-kv-cache-repair_amd" / "csrc" / "kvr_chunk_attention.hip").read_text()
    align, votes = (int(re.search(rf"constexpr int {name} = (\d+);", source)[1]) for name in ("kRowAlign", "kVoteLds"))
    parts = {name: size for name, size in static_lds().items() if "chunk_attention_kernel" in name}
    assert len(parts) == 4
    for name, size in parts.items():
        row = 2 * int(re.search(r"Li(64|128)E", name)[1])
        assert size <= votes and size % align == 0 and align % row == 0 and 8 * 64 * row + votes <= 160 * 1024
