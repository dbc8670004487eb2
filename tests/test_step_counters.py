"""The step plan's loops over counts that come from lengths, up to 2^31 - 1: their counters
must not pass what their type holds (a signed one would wrap to negative indices).  Read
from the source, since such lengths cannot be run before that is so."""

from __future__ import annotations

import re
from pathlib import Path

SOURCE = (Path(__file__).resolve().parents[1] / "twilight-cpu-gpu-offloading_b200" / "csrc"
          / "paged.cu")
# largest value + one step of all threads (148 CTAs of 512)
BITS = {"int": 31, "unsigned": 32, "uint32_t": 32, "int64_t": 63, "long long": 63}


def test_counters_hold_one_step_past_the_end():
    body = SOURCE.read_text().split("void __launch_bounds__(kStepThreads) paged_step_kernel")[1]
    body = body.split("// ---- row write")[0]
    loops = re.findall(r"for \(([a-z0-9_ ]+?) (\w) = first; [^;]*; \2 \+= step\)", body)
    assert {name for _, name in loops} == {"t", "k", "b"} and len(loops) == 4
    for kind, name in loops:
        most = 8192 if name == "b" else 2 ** 31 - 1  # requests are at most 8192
        assert most + 148 * 512 < 2 ** BITS[kind], (kind, name)
