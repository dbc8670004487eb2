"""Barriers that the tensor cores arrive at by themselves (mma_commit): the arrival of the last
commit of a block is waited for on every way out, or it could come when the shared memory is
another block's.  Read from the source; nothing is launched."""

from __future__ import annotations

import re
from pathlib import Path

SOURCE = (Path(__file__).resolve().parents[1] / "twilight-cpu-gpu-offloading_b200" / "csrc"
          / "paged_weights.cu")


def test_weights_kernel():
    text = re.sub(r"//[^\n]*", "", SOURCE.read_text())
    kernel = text.split("paged_weights_kernel(const", 1)[1].split("\n}\n", 1)[0]
    issuing = kernel.split("} else if (warp == kMmaWarp) {", 1)[1].split("\n  } else {", 1)[0]
    assert len(re.findall(r"mma_commit\(", kernel)) == len(re.findall(r"mma_commit\(", issuing))
    # behind the loop, at the branch's own level: the loop's commits come before it
    at = issuing.rindex("mma_commit(")
    assert issuing[at:].startswith("mma_commit(&sh.drain)")
    before = issuing[:at]
    assert before.count("{") == before.count("}"), "the last commit is inside a block"
    condition = before[before.rindex("\n"):].strip()
    assert condition == "if (elect_one())", "the last commit is conditional"
    after = issuing[at:]
    wait = after.index("mbar_wait(&sh.drain, 0,")
    assert after[:wait].count("{") == after[:wait].count("}") == 0, "its wait is in a block"
    assert not re.search(r"\bif\b|\breturn\b", after[:wait]), "its wait is conditional"
    assert not re.search(r"\breturn\b", issuing), "a way out before the wait"
