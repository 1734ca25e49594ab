"""Bounded waits in the kernels of 8-bit integers, read from their sources as `test_warp_waits` reads the others': where a whole warp waits, its lanes
go on alike (`warp_waits`), and `lane_waits` is called by one lane only."""
import os

import pytest

from test_warp_waits import CSRC, waits

SOURCES = ["attention_int8.cu", "gemm_int8.cu"]


def read(source):
    return open(os.path.join(CSRC, source)).read().replace("warp_waits", "mbar_wait_warp").replace("lane_waits", "mbar_wait")


@pytest.mark.parametrize("source", SOURCES)
def test_whole_warps_wait_alike(source):
    found = waits(read(source))
    assert len(found) >= 7
    wrong = [(line, name) for line, name, one in found if one == (name == "mbar_wait_warp")]
    assert not wrong, f"{source}: {wrong}"


def test_no_other_source_of_theirs_waits():
    assert not [f for f in ("quantize.cu", "int8_rows.cuh") if "try_wait" in open(os.path.join(CSRC, f)).read()]
