"""Products of rows of 8-bit integers: bits that depend on nothing but the row, functions of 32-bit outputs, rows that stand for NaN."""
import pytest
import torch

from gpt_fast_b200 import ops
from test_int8_rows_gpu import draw

pytestmark = pytest.mark.gpu
F64 = torch.float64


@pytest.mark.parametrize("N", [1536, 1531, 250])
@pytest.mark.parametrize("mode,dtype", [("store", torch.float32), ("add", torch.float32), ("swiglu", torch.bfloat16), ("swiglu", torch.float32), ("gelu", torch.float32), ("gelu_tanh", torch.float32),
                                        ("silu", torch.float32), ("relu2", torch.float32)])
def test_a_rows_bits_depend_on_nothing_else(mode, dtype, N):
    """One row alone, in a decode step's batch and in a prompt, whichever kernel and tile make it; N that fill whole vectors and that do not."""
    K = 2048
    N += N % 2 if mode == "swiglu" else 0
    x, w = draw((700, K), 1, torch.bfloat16), ops.quantize_rows(draw((N, K), 2, outliers=False))
    base = draw((700, N // 2 if mode == "swiglu" else N), 3).to(dtype)
    whole = base.clone()
    ops.linear(x, w, whole, mode=mode)
    for n in (1, 2, 9, 31, 64, 100, 128, 129, 300, 513):
        part = base[:n].clone()
        ops.linear(x[:n].contiguous(), w, part, mode=mode)
        assert torch.equal(part, whole[:n]), n
