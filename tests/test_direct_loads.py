"""Direct loads into LDS written as inline assembly take their LDS address from M0,
and a scalar write of M0 needs one wait state before such a load. The compiler puts it
there for its own loads and does not look into assembly, so each text has to hold it."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "budgeted-kv-cache-repair_amd" / "csrc"
SOURCES = sorted(p for p in CSRC.iterdir() if p.suffix in (".h", ".hip"))


def texts(source: str):
    """The instructions of every asm statement."""
    for found in re.finditer(r'\basm\s*(?:volatile)?\s*\(\s*((?:"(?:[^"\\]|\\.)*"\s*)+)', source):
        text = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', found[1]))
        yield [line.strip() for line in re.split(r"\\n|;", text.replace("\\t", " ")) if line.strip()]


def unwaited(lines) -> list:
    """Loads into LDS with fewer than one wait state behind a write of M0."""
    bad, states = [], 9
    for line in lines:
        name, _, rest = line.partition(" ")
        if re.search(r"_lds(_|$)", name) or re.search(r"\blds\b", rest):
            if states < 1:
                bad.append(line)
        states += int(rest, 0) + 1 if name == "s_nop" else 1
        if name.startswith("s_") and rest.split(",")[0].strip() == "m0":
            states = 0
    return bad


def test_what_it_looks_for():
    load = "global_load_lds_dwordx4 %0, %1"
    assert unwaited(["s_mov_b32 m0, %2", load]) == [load]
    assert not unwaited(["s_mov_b32 m0, %2", "s_nop 0", load]) and not unwaited([load])
    assert list(texts('asm volatile("s_mov_b32 m0, %2\\n\\t" "s_nop 0" :: "s"(m));')) == [["s_mov_b32 m0, %2", "s_nop 0"]]


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_m0_is_written_a_wait_state_before_its_load(path):
    assert [bad for lines in texts(path.read_text()) for bad in unwaited(lines)] == []


def test_some_source_has_such_loads():
    loads = [line for path in SOURCES for lines in texts(path.read_text()) for line in lines if "load_lds" in line]
    assert len(loads) >= 2


def test_the_build_hears_of_assembly():
    """No flag silences what the compiler has to say of assembly in every source."""
    import build_lib

    assert not [flag for flag in build_lib.HIP_FLAGS if "asm" in flag]
