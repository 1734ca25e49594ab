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


@pytest.mark.parametrize("M", [127, 700])
@pytest.mark.parametrize("mode", ["swiglu", "silu", "gelu_tanh"])
def test_32_bit_outputs_of_gates_have_32_bits(mode, M):
    """Gates that are exact: one integer of either side, with powers of two for scales, i j 2^-6 for i up to 127 and j from -127 to 127; so the function's own error is
    all there is, far below zero too."""
    i, j = torch.arange(1, M + 1) % 127 + 1, torch.arange(-127, 128)
    a = ops.Int8Rows(torch.zeros(M, 16, dtype=torch.int8), torch.ones(M), 16)
    a.q[:, 3] = i.to(torch.int8)
    rows = torch.stack([j, torch.full_like(j, 64)], 1).flatten() if mode == "swiglu" else j
    w = ops.Int8Rows(torch.zeros(len(rows), 16, dtype=torch.int8), torch.full((len(rows),), 2.0 ** -6), 16)
    w.q[:, 3] = rows.to(torch.int8)
    a, w = (ops.Int8Rows(r.q.cuda(), r.scale.cuda(), 16) for r in (a, w))
    out = torch.empty(M, len(j), device="cuda")
    ops.linear(a, w, out, mode=mode)
    x = (i[:, None] * j[None]).to(F64).cuda() / 64
    up = i[:, None].to(F64).cuda() if mode == "swiglu" else 1.0
    # the exponent t of x / (1 + e^t): exact for SiLU; for the tanh form of GELU four roundings of numbers no larger than itself, each 2^-24 of it
    t = -x if mode != "gelu_tanh" else -2 * (2 / torch.pi) ** 0.5 * (x + 0.044715 * x ** 3)
    want = x / (1 + torch.exp(t)) * up
    # half steps: the exponential 2, the sum, the quotient and the product by `up` 1 each; the last step of 2^-24 is for their products.  Below t = 88.72 e^t leaves 32 bits and the
    # result is 0, where |x| / e^t is less than 2^-121; results below 2^-126 have steps of 2^-149
    rel = (6 + (4 * t.abs() if mode == "gelu_tanh" else 0)) * 2.0 ** -24
    tol = want.abs() * rel + torch.as_tensor(up) * (2.0 ** -149 + torch.where(t > 88.72, x.abs() * 2.0 ** -127, 0.0))
    bad = (out.to(F64) - want).abs() / tol.clamp(min=1e-60)
    assert bool(bad.le(1).all()), float(bad.max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M", [3, 40, 300])
@pytest.mark.parametrize("mode", ["store", "add", "swiglu", "gelu", "gelu_tanh", "silu", "relu2"])
def test_rows_that_stand_for_nan_stay_nan(mode, M, dtype):
    """Through every function, in activations and in weights, and nowhere else."""
    K, N = 256, 392
    x, w = draw((M, K), 1, dtype, outliers=False), ops.quantize_rows(draw((N, K), 2, outliers=False) * K ** -0.5)
    base = draw((M, N // 2 if mode == "swiglu" else N), 3).to(torch.float32 if mode == "add" else dtype)
    clean, out = base.clone(), base.clone()
    ops.linear(x, w, clean, mode=mode)
    x[M - 2, 7] = float("nan")
    w.scale[11] = float("nan")
    ops.linear(x, w, out, mode=mode)
    column = 5 if mode == "swiglu" else 11                   # row 11 of W is the up row of output 5
    assert out[M - 2].isnan().all() and out[:, column].isnan().all()
    out[M - 2], out[:, column] = clean[M - 2], clean[:, column]
    assert torch.equal(out, clean)


def test_products_beyond_two_to_the_31_numbers():
    """The last rows of 70,000 x 32,768 outputs have the bits they have by themselves; the same for rows and norms of as many numbers."""
    M, K, N = 70000, 64, 32768
    x, w = draw((M, K), 1, torch.bfloat16), ops.quantize_rows(draw((N, K), 2))
    for mode, n in (("store", N), ("swiglu", N // 2)):
        out, part = torch.empty(M, n, dtype=torch.bfloat16, device="cuda"), torch.empty(300, n, dtype=torch.bfloat16, device="cuda")
        ops.linear(x, w, out, mode=mode)
        ops.linear(x[-300:].contiguous(), w, part, mode=mode)
        assert torch.equal(out[-300:], part)
    out = torch.randn(M, N, dtype=torch.bfloat16, device="cuda")
    whole, part = ops.quantize_rows(out), ops.quantize_rows(out[-300:].contiguous())
    assert torch.equal(whole.q[-300:], part.q) and torch.equal(whole.scale[-300:], part.scale)
    del whole
    x32, weight = out.float(), torch.rand(N, device="cuda")
    del out
    whole, part = ops.int8_rows(M, N, "cuda"), ops.int8_rows(300, N, "cuda")
    ops.rmsnorm(x32, weight, 1e-5, whole)
    ops.rmsnorm(x32[-300:].contiguous(), weight, 1e-5, part)
    # (few rows have more threads each, so the sum of squares has another order: scales within 2 (N / 2 + 4) steps, integers one apart next to a tie)
    assert (whole.q[-300:].int() - part.q.int()).abs().max() <= 1 and (whole.scale[-300:] / part.scale - 1).abs().max() <= (N + 8) * 2.0 ** -24
