"""What the kernels' synchronisation relies on, checked on the CPU: no run on a GPU shows a missing wait reliably."""

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "lookatmyquant_b200" / "csrc"


def test_a_warp_reconverges_before_an_aligned_cluster_barrier():
    """barrier.cluster with .aligned needs all threads of a warp at the instruction. The attention kernels' first warp comes
    to it from a branch of one lane: each such instruction has a __syncwarp() before it in its function."""
    found = 0
    for src in sorted(CSRC.glob("*.cu*")):
        text = src.read_text()
        for m in re.finditer(r"barrier\.cluster\.arrive[a-z.]*\.aligned", text):
            body = text[text.rindex("{\n", 0, m.start()):m.start()]
            assert "__syncwarp();" in body, src.name
            found += 1
    assert found
