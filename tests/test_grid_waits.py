"""Kernels that may start while the one before them in the stream still runs
(programmatic dependent launch): each of their threads waits for that kernel before
it reads or writes global memory.  Read from the sources; nothing is launched."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "twilight-cpu-gpu-offloading_b200" / "csrc"

# what reads or writes global memory in the paged kernels' own terms
GLOBAL = re.compile(r"\b(?:a|w\.a|pool|sp)\.\w+\s*\[|\ba\.cu_q\b|\ba\.kv_lens\b|\ba\.block_table\b|"
                    r"\bpaged_request\(|\bpaged_clear_padding|\bpaged_store_|\bfirst_above\(|"
                    r"\braise_error\(|\btma_load_|\b__ld\w+\(|\*\s*a\.")


def kernels():
    """(file, name, body) of every __global__ function that waits anywhere."""
    for path in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for m in re.finditer(r"__global__", text):
            brace = text.index("{", m.end())
            depth, end = 0, brace
            for end in range(brace, len(text)):
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                if depth == 0:
                    break
            head = text[m.end():brace]
            name = re.findall(r"(\w+)\s*\(", re.sub(r"__launch_bounds__\([^)]*\)", "", head))[0]
            body = text[brace + 1:end]
            if "pdl_" in body or name.startswith("paged_"):
                yield path.name, name, body


KERNELS = list(kernels())


def test_the_paged_kernels_are_among_them():
    names = {name for _, name, _ in KERNELS}
    assert {"paged_step_kernel", "paged_write_kernel", "paged_token_kernel", "paged_chunk_kernel",
            "paged_merge_kernel"} <= names


@pytest.mark.parametrize("file,name,body", KERNELS, ids=[f"{f}:{n}" for f, n, _ in KERNELS])
def test_waits_first(file, name, body):
    at = body.index("pdl_wait();")
    before = body[:at]
    # every thread gets there: not under a condition, not in a block, no way out before it
    assert before.count("{") == before.count("}"), "the wait is inside a block"
    assert before.rstrip().endswith((";", "}", "{")) or not before.strip(), "the wait is conditional"
    assert not re.search(r"\breturn\b", before), "a thread may leave before the wait"
    if name.startswith("paged_"):
        found = GLOBAL.search(before)
        assert not found, f"{found.group(0)!r} comes before the wait"
    assert "pdl_launch_dependents();" not in before
