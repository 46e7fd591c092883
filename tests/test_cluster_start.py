"""A CTA of a cluster may touch another one's shared memory only once that one runs: before a kernel's first remote
access every CTA has to pass a cluster barrier.  Read from the sources (nothing here runs on a GPU)."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "blackwell-inference-server_b200" / "csrc"
REMOTE = r"\b(cluster_share|mapa_shared|st_shared_cluster_f32|mbar_arrive_remote)\s*\("


def _body(text, name):
    """The body of the __global__ function `name`, without comments."""
    text = re.sub(r"//[^\n]*", "", text)
    at = re.search(r"__global__[^;{]*?\b" + name + r"\s*\(", text)
    start = text.index("{", at.end())
    depth, i = 1, start + 1
    while depth:
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        i += 1
    return text[start:i]


@pytest.mark.parametrize("file,kernel", [("verify.cu", "verify_tree_kernel"), ("kv_quant.cu", "kv_quant_cluster_kernel")])
def test_cluster_runs_before_remote_access(file, kernel):
    body = _body((CSRC / file).read_text(), kernel)
    first = re.search(REMOTE, body)
    assert first, "the kernel no longer reaches another CTA's shared memory"
    passed = re.search(r"\b(cluster_sync_all|cluster_wait)\s*\(\)", body)
    assert passed and passed.start() < first.start(), "remote access before the cluster is known to run"
    arrived = re.search(r"\b(cluster_sync_all|cluster_arrive)\s*\(\)", body)
    assert arrived.start() <= passed.start()
