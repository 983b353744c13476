"""Rings in shared memory whose lanes read what other lanes' asynchronous copies
brought: cp.async.wait_group makes a lane's own copies visible to that lane, and a
warp's vote orders no memory, so a barrier of the warp comes directly behind it.
Read in the sources, since a race may well give right results."""
import re
from pathlib import Path

import pytest

KERNELS = Path(__file__).resolve().parents[1] / "tensoros_b200" / "csrc" / "kernels"


def statements_behind(text, wait):
    """The statement that follows each `wait`, comments taken off."""
    text = re.sub(r"//[^\n]*", "", text)
    return [text[m.end():].split(";")[0].strip() for m in re.finditer(r"asm volatile\(\"cp\.async\.%s[^;]*;[^;]*;" % wait, text)]


@pytest.mark.parametrize("name,rings", [("paged_decode.cu", 2), ("paged8_decode.cu", 1)])
def test_waits_for_copies_are_followed_by_a_barrier(name, rings):
    text = (KERNELS / name).read_text()
    assert statements_behind(text, "wait_group") == ["__syncwarp()"] * rings
    ends = statements_behind(text, "wait_all")
    assert len(ends) == rings and all(s == "__syncthreads()" for s in ends)
