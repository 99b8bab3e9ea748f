"""Kernels of clusters that read or write another CTA's shared memory: that CTA has to have begun, which only a barrier of the
cluster shows.  Read from the sources: a kernel without it works as long as its CTAs begin together."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(__file__), "..", "gpt.c_b200", "csrc")
REMOTE = re.compile(r"map_shared_rank\(|\bmapa\(|\bthere\(&")
BARRIER = re.compile(r"\b(?:cluster|r)\.sync\(\);|\bcluster_sync_all\(\);|\bcluster_wait\(\);")


def kernels():
    """(name, body) of every kernel that reaches into another CTA's shared memory."""
    found = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        text = open(path).read()
        for m in re.finditer(r"__global__.*?\b(\w+_kernel)\(", text, re.S):
            body = text[m.end():text.index("\n}\n", m.end())]
            if REMOTE.search(body):
                found.append((m.group(1), body))
    return found


def test_kernels_are_found():
    assert {"few_rows_kernel", "rows_kernel", "packed_kernel", "tile_kernel", "sample_kernel", "linear_split_kernel"} <= {n for n, _ in kernels()}


@pytest.mark.parametrize("name,body", kernels(), ids=lambda v: v if len(v) < 64 else "")
def test_a_barrier_of_the_cluster_comes_first(name, body):
    barrier = BARRIER.search(body)
    assert barrier and barrier.start() < REMOTE.search(body).start(), f"{name} may reach into the memory of a CTA that has not begun"
    if "cluster_wait" in barrier.group():
        arrive = body.find("cluster_arrive();")
        assert 0 <= arrive < barrier.start(), f"{name} waits for a barrier that its threads have not arrived at"
