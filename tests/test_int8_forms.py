"""Which form a product of 8-bit integers takes, where both were measured."""
import pytest

from gpt_fast_b200.ops.cuda import int8_plan


@pytest.mark.parametrize("M,N,K,mode,pairs", [
    (333, 4096, 14336, "add", False), (1000, 4096, 14336, "add", False), (2000, 4096, 14336, "add", False), (2500, 4096, 14336, "add", True), (8192, 4096, 14336, "add", True),
    (8192, 4096, 4096, "add", False), (300, 12288, 4096, "add", False), (2000, 8192, 8192, "add", False), (400, 8192, 28672, "add", False), (1000, 8192, 28672, "add", True),
    (512, 6144, 4096, "store", False), (1024, 6144, 4096, "store", True), (129, 28672, 4096, "swiglu", True), (128, 28672, 4096, "swiglu", False), (2000, 130, 14336, "add", False),
])
def test_the_faster_form(M, N, K, mode, pairs):
    assert (int8_plan(M, N, K, mode, 148)[0] == 256) == pairs
