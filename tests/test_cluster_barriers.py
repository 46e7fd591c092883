"""The cluster barriers are PTX's `.aligned` ones: all lanes of a warp have to execute them together, and nothing but a
__syncwarp() says that they do where they come from loops or branches of different lengths.  Read from the sources."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "blackwell-inference-server_b200" / "csrc"
SOURCES = sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")])


def _without_comments(text):
    return re.sub(r"//[^\n]*", "", text)


def test_aligned_cluster_barriers_follow_a_syncwarp():
    found = 0
    for path in SOURCES:
        text = _without_comments(path.read_text())
        for m in re.finditer(r"barrier\.cluster\.[\w.]*", text):
            if ".aligned" not in m.group():
                continue
            found += 1
            before = text[:m.start()]
            assert re.search(r"__syncwarp\(\);\s*asm volatile\(\"$", before), (path.name, text[m.start() - 120:m.end()])
    assert found >= 2, "the cluster barriers are written elsewhere"


@pytest.mark.parametrize("name", ["cluster_arrive", "cluster_wait", "cluster_sync_all"])
def test_kernels_use_the_helpers(name):
    assert any(re.search(r"\b" + name + r"\(\)", _without_comments(p.read_text())) for p in SOURCES)
