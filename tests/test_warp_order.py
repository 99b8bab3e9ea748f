"""One lane arriving at a barrier for its warp: what the other lanes have stored in shared memory is behind that arrival only if the
warp has met at __syncwarp since; votes and shuffles order nothing in memory.  Read from the sources: the order shows in a run
only where the hardware makes use of its freedom."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(__file__), "..", "gpt.c_b200", "csrc")
STORE = re.compile(r"\*reinterpret_cast<(?:uint[24]|float[24]) \*>\([^;]*\) = ")
FOR_THE_WARP = re.compile(r"if \([^;{]*(?:lane|& 31\)) == 0\)")
NEAR = 16  # lines


def arrivals():
    """(place, lines from the last store in shared memory in front of an arrival for the warp up to it)."""
    found = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        lines = open(path).read().split("\n")
        for n, line in enumerate(lines):
            if "mbar_arrive(" not in line or not any(FOR_THE_WARP.search(before) for before in lines[max(0, n - 3):n + 1]):
                continue
            for i in range(n - 1, max(-1, n - NEAR), -1):
                if STORE.search(lines[i]):
                    found.append((f"{os.path.basename(path)}:{n + 1}", "\n".join(lines[i:n + 1])))
                    break
    return found


def test_arrivals_are_found():
    assert sum(place.startswith("paged_tile_sm100.cu") for place, _ in arrivals()) >= 3


@pytest.mark.parametrize("place,code", arrivals(), ids=lambda v: v if len(v) < 40 else "")
def test_the_warp_has_met_before_one_lane_arrives_for_it(place, code):
    assert "__syncwarp();" in code, f"{place}: other lanes' stores need not be visible to whoever waits"
