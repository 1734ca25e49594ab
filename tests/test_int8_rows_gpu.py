"""Rows of 8-bit integers: quantising them, the norm that quantises its output, and their products, against 64 bits."""
import pytest
import torch

from gpt_fast_b200 import ops

pytestmark = pytest.mark.gpu
F64 = torch.float64


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def quantised(x):
    """(integers, scales) by the definition, decided in 64 bits."""
    x = x.to(F64)
    most = x.abs().amax(1)
    q = torch.where(most[:, None] > 0, (x * 127 / most.clamp(min=5e-324)[:, None]).round(), 0.0)
    return q, most / 127


def draw(shape, seed, dtype=torch.float32, outliers=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda")
    if outliers and shape[-1] > 8:
        x[..., ::max(2, shape[-1] // 5)] *= 9
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,K", [(1, 1), (3, 7), (2, 16), (5, 33), (1, 4096), (17, 1000), (4, 4104), (130, 2048), (2, 14336), (1, 20001), (2, 53248)])
def test_rows(R, K, dtype):
    x = draw((R, K), R * 7 + K, dtype)
    got = ops.quantize_rows(x)
    q, scale = quantised(x)
    assert got.q.shape == (R, -(-K // 16) * 16) and got.cols == K
    assert torch.equal(got.q[:, :K].to(F64), q)
    assert (got.q[:, K:] == 0).all()
    assert (got.scale.to(F64) - scale).abs().le(scale * 2.0 ** -24).all()           # one division, rounded once


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ties_go_to_even(dtype):
    # with 127 as the largest number the quotients are the numbers themselves, and halves are ties; +-1/64 beside them is not
    v = torch.arange(-126, 126, dtype=torch.float32) + 0.5
    near = torch.cat([v[:32], v[-32:]])
    x = torch.cat([torch.tensor([127.0]), v, near * (1 + 2.0 ** -20) if dtype == torch.float32 else v[:64], torch.tensor([-127.0])])[None].cuda().to(dtype)
    got = ops.quantize_rows(x)
    assert torch.equal(got.q[0, :x.shape[1]].to(F64), x[0].to(F64).round())
    assert got.scale[0] == 1


def test_rows_next_to_ties():
    """Numbers whose quotient a 32-bit division may put on the wrong side: all multiples of 2^-12 / 127 around odd halves, for awkward maxima."""
    for most in (1.0, 0.7310585618019104, 3.0000002384185791, 1e-30, 1e30):
        m = torch.tensor(most, dtype=torch.float32)
        half = (torch.arange(0, 127, dtype=F64) + 0.5) / 127 * m.to(F64)
        x = torch.cat([m[None], half.float(), torch.nextafter(half.float(), torch.tensor(float("inf"))), torch.nextafter(half.float(), torch.tensor(0.0))])
        x = torch.cat([x, -x[1:]])[None].cuda()
        got = ops.quantize_rows(x)
        assert torch.equal(got.q[0, :x.shape[1]].to(F64), quantised(x)[0][0]), most


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_zeros_tiny_large_and_not_finite(dtype):
    x = draw((8, 96), 3, dtype, outliers=False)
    x[0] = 0
    x[1] = x[1] * 2.0 ** -120
    x[2] = x[2] * 2.0 ** 100
    x[3, 5] = float("nan")
    x[4, 95] = float("inf")
    x[5, 0] = float("-inf")
    x[6] = 0
    x[6, 50] = -torch.finfo(dtype).max
    x[7] = 0
    x[7, 1] = 2.0 ** -130                                    # a subnormal maximum
    x[7, 2] = -(2.0 ** -131)
    got = ops.quantize_rows(x)
    q, scale = quantised(x)
    live = [0, 1, 2, 6, 7]
    assert torch.equal(got.q[live].to(F64), q[live])
    assert got.scale[0] == 0
    step = torch.maximum(scale * 2.0 ** -24, torch.full_like(scale, 2.0 ** -150))        # half a step of subnormal numbers is 2^-150
    assert (got.scale.to(F64) - scale).abs()[live].le(step[live]).all()
    assert (got.q[3:6] == 0).all() and got.scale[3:6].isnan().all()


@pytest.mark.parametrize("wdtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,D,S,picked", [(1, 4096, 0, False), (3, 96, 0, False), (2, 1001, 0, False), (8, 4096, 3, False), (200, 1024, 2, False), (9, 288, 0, True),
                                          (5, 8192, 0, False), (2, 20000, 1, False)])
def test_norm_that_quantises(T, D, S, picked, wdtype):
    x = draw((T, D), T + D)
    w = (1 + 0.2 * draw((D,), 4, outliers=False)).to(wdtype)
    pending = draw((S, T, D), 5, outliers=False) if S else None
    rows = torch.tensor([T - 1, 0, T // 2], dtype=torch.int32, device="cuda") if picked else None
    total = x.to(F64) + (pending.to(F64).sum(0) if S else 0)
    x_in = x.clone()
    out = ops.int8_rows(3 if picked else T, D, "cuda")
    ops.rmsnorm(x_in, w, 1e-5, out, rows, pending)
    if S:
        # ascending 32-bit sums of S + 1 numbers
        assert (x_in.to(F64) - total).abs().le((x.abs().to(F64) + pending.abs().to(F64).sum(0)) * S * 2.0 ** -24).all()
    total = x_in.to(F64)
    if picked:
        total = total[rows.long()]
    h = total / (total.pow(2).mean(1, keepdim=True) + 1e-5).sqrt() * w.to(F64)
    q, scale = quantised(h)
    # a 32-bit sum of squares in any order is within D 2^-24 of itself, half of that behind the root; the root, two products and the quotient add 8 steps
    rel = (D / 2 + 8) * 2.0 ** -24
    assert (out.scale.to(F64) - scale).abs().le(scale * rel).all()
    far = (out.q[:, :D].to(F64) - h * 127 / h.abs().amax(1, keepdim=True)).abs()
    assert far.le(0.5 + 127 * 2 * rel).all()
    assert (out.q[:, D:] == 0).all()


def test_norm_and_rows_agree():
    """What the norm quantises is what `quantize_rows` makes of the norm's own 32-bit output, but for numbers next to a tie."""
    x, w = draw((64, 2048), 1), 1 + 0.2 * draw((2048,), 2, outliers=False)
    h = torch.empty_like(x)
    ops.rmsnorm(x, w, 1e-5, h)
    a = ops.int8_rows(64, 2048, "cuda")
    ops.rmsnorm(x, w, 1e-5, a)
    b = ops.quantize_rows(h)
    assert (a.q.int() - b.q.int()).abs().max() <= 1 and (a.q != b.q).float().mean() < 1e-3


# ---- products -----------------------------------------------------------------------------------------------

def product(a: ops.Int8Rows, w: ops.Int8Rows):
    """Exact sums times the scales, in 64 bits."""
    K = a.cols
    return (a.q[:, :K].to(F64) @ w.q[:, :K].to(F64).t()) * a.scale.to(F64)[:, None] * w.scale.to(F64)


def unary(kind, y):
    if kind == "gelu":
        return 0.5 * y * (1 + torch.erf(y / 2 ** 0.5))
    if kind == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (y + 0.044715 * y ** 3)))
    if kind == "silu":
        return y * torch.sigmoid(y)
    if kind == "relu2":
        return y.clamp(min=0) ** 2
    return y


SIZES = [(1, 64, 64), (1, 4096, 6144), (3, 257, 130), (8, 4096, 1024), (16, 1000, 520), (17, 515, 514), (33, 2048, 256), (64, 768, 2304), (65, 130, 62), (128, 4096, 514),
         (129, 512, 1030), (333, 1056, 768), (512, 96, 128), (700, 2080, 1536), (2050, 640, 1282), (2, 14336, 128), (5, 1, 6), (1, 20, 2)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("mode", ["store", "add", "swiglu"])
def test_product(M, K, N, mode, dtype):
    x = draw((M, K), M + K, dtype)
    w = ops.quantize_rows(draw((N, K), N, outliers=False) * K ** -0.5)
    a = ops.quantize_rows(x)
    y = product(a, w)
    # the sum is exact, its way into 32 bits and the two scales round: 3 steps, and a fourth for the products' product
    err = y.abs() * 4 * 2.0 ** -24
    if mode == "add":
        res = draw((M, N), 8)
        out = res.clone()
        ops.linear(x, w, out, mode="add")
        want = res.to(F64) + y
        tol = err + want.abs() * 2.0 ** -24
    elif mode == "store":
        out = torch.full((M, N), float("nan"), dtype=dtype, device="cuda")
        ops.linear(x, w, out)
        want, tol = y, err + y.abs() * half_step(dtype)
    else:
        out = torch.full((M, N // 2), float("nan"), dtype=dtype, device="cuda")
        ops.linear(x, w, out, mode="swiglu")
        g, u = y[:, 0::2], y[:, 1::2]
        want = unary("silu", g) * u
        # silu'(g) g / silu(g) is at most 1 + |g|; the exponential, the sum, the quotient and the product are worth 8 steps more
        tol = want.abs() * ((4 * (2 + g.abs()) + 8 + 2 * g.abs()) * 2.0 ** -24 + half_step(dtype)) + 1e-37
    assert (out.to(F64) - want).abs().le(tol).all(), float(((out.to(F64) - want).abs() / tol.clamp(min=1e-300)).max())
    again = torch.empty_like(out) if mode != "add" else res.clone()
    ops.linear(a, w, again, mode=mode)                       # rows that come quantised: the same bits
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M", [1, 40, 300])
@pytest.mark.parametrize("mode", ["gelu", "gelu_tanh", "silu", "relu2"])
def test_product_with_an_activation(M, mode, dtype):
    K, N = 512, 392
    x, w = draw((M, K), 1, dtype, outliers=False), ops.quantize_rows(draw((N, K), 2, outliers=False) * K ** -0.5)
    out = torch.empty(M, N, dtype=dtype, device="cuda")
    ops.linear(x, w, out, mode=mode)
    y = product(ops.quantize_rows(x), w)
    want = unary(mode, y)
    # |f(y + e) - f(y)| <= (2 + |y|) |e| for all four, e = 4 steps of y; the functions themselves cost 16 steps of |y| (erf and tanh near -1 cancel)
    tol = (2 + y.abs()) * y.abs() * 4 * 2.0 ** -24 + 16 * y.abs().clamp(min=1) * 2.0 ** -24 + want.abs() * half_step(dtype)
    assert (out.to(F64) - want).abs().le(tol).all()


def test_a_rows_result_is_the_same_in_any_batch():
    """Integer sums have no order: one row alone, in a decode step's batch and in a prompt give the same bits."""
    K, N = 2048, 1536
    x, w = draw((700, K), 1, torch.bfloat16), ops.quantize_rows(draw((N, K), 2, outliers=False))
    whole = torch.empty(700, N, dtype=torch.bfloat16, device="cuda")
    ops.linear(x, w, whole)
    for n in (1, 2, 9, 31, 64, 100, 128, 129, 300):
        part = torch.empty(n, N, dtype=torch.bfloat16, device="cuda")
        ops.linear(x[:n].contiguous(), w, part)
        assert torch.equal(part, whole[:n]), n


def test_the_largest_sum():
    """Every integer +-127 at the longest row: 127^2 * 133,144 = 2,147,479,576, just within 2^31 - 1 = 2,147,483,647 (one number more is not)."""
    K, pitch = 133144, 133152

    def rows(n):
        q = torch.zeros(n, pitch, dtype=torch.int8, device="cuda")
        q[:, :K] = 127
        return ops.Int8Rows(q, torch.ones(n, device="cuda"), K)
    w = rows(34)
    w.q[1::2] *= -1
    for M in (1, 20, 200):
        out = torch.empty(M, 34, dtype=torch.float32, device="cuda")
        ops.linear(rows(M), w, out)
        want = torch.tensor(127.0 * 127 * K, dtype=F64).float().cuda()
        assert (out[:, 0::2] == want).all() and (out[:, 1::2] == -want).all()
    with pytest.raises(ops.KernelError, match="32 bits"):
        ops.linear(torch.zeros(1, K + 1, device="cuda"), ops.Int8Rows(w.q[:2], w.scale[:2], K + 1), torch.empty(1, 2, device="cuda"))


def test_rows_that_are_not_finite_stay_apart():
    x, w = draw((40, 256), 1, torch.bfloat16), ops.quantize_rows(draw((96, 256), 2))
    clean = torch.empty(40, 96, dtype=torch.bfloat16, device="cuda")
    ops.linear(x, w, clean)
    x[7, 3], x[20, 100] = float("inf"), float("nan")
    out = torch.empty_like(clean)
    ops.linear(x, w, out)
    others = [i for i in range(40) if i not in (7, 20)]
    assert torch.equal(out[others], clean[others]) and out[[7, 20]].isnan().all()


@pytest.mark.parametrize("M", [4, 40, 200])
def test_nothing_beside_the_output_is_written(M):
    K, N = 256, 136
    x, w = draw((M, K), 1, torch.bfloat16), ops.quantize_rows(draw((N, K), 2))
    for dtype, mode, n in ((torch.bfloat16, "store", N), (torch.float32, "store", N), (torch.bfloat16, "swiglu", N // 2), (torch.float32, "add", N)):
        room = torch.full((M * n + 512,), 7.0, dtype=dtype, device="cuda")
        ops.linear(x, w, room[256:256 + M * n].view(M, n), mode=mode)
        assert (room[:256] == 7).all() and (room[256 + M * n:] == 7).all()


def test_captured_and_replayed():
    """Two graphs with the same weights, replayed in turn over new inputs."""
    K, N = 1024, 768
    w = ops.quantize_rows(draw((N, K), 2))
    sides = []
    for M in (4, 200):
        x, out = draw((M, K), M, torch.bfloat16), torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
        ops.linear(x, w, out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.linear(x, w, out)
        sides.append((x, out, g))
    for round_ in range(3):
        for x, out, g in sides:
            x.copy_(draw(tuple(x.shape), 50 + round_, torch.bfloat16))
            out.zero_()
            g.replay()
        torch.cuda.synchronize()
        for x, out, _ in sides:
            want = torch.empty_like(out)
            ops.linear(x, w, want)
            assert torch.equal(out, want)


def test_on_another_stream():
    K, N = 1024, 768
    x, w = draw((5, K), 1, torch.bfloat16), ops.quantize_rows(draw((N, K), 2))
    want, out = torch.empty(5, N, dtype=torch.bfloat16, device="cuda"), torch.empty(5, N, dtype=torch.bfloat16, device="cuda")
    ops.linear(x, w, want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.linear(x, w, out)
    s.synchronize()
    assert torch.equal(out, want)


def test_refusals():
    x, w = draw((4, 64), 1, torch.bfloat16), ops.quantize_rows(draw((32, 64), 2))
    out = torch.empty(4, 32, dtype=torch.bfloat16, device="cuda")

    def refused(match, *a, **kw):
        with pytest.raises(ops.KernelError, match=match):
            ops.linear(*a, **kw)
    refused("shape", x, w, out[:3])
    refused("8-bit rows", draw((4, 48), 1, torch.bfloat16), w, out)
    refused("contiguous", x[:, ::2], ops.quantize_rows(draw((32, 32), 2)), out)
    refused("float32 or bfloat16", x.half(), w, out)
    refused("float32 or bfloat16", x, w, out.half())
    refused("residual", x, w, out, mode="add")
    refused("unknown mode", x, w, out, mode="sigmoid")
    refused("pairs", x, ops.quantize_rows(draw((31, 64), 2)), torch.empty(4, 15, dtype=torch.bfloat16, device="cuda"), mode="swiglu")
    refused("pitch", x, ops.Int8Rows(w.q[:, :40].contiguous(), w.scale, 64), out)
    refused("pitch", draw((4, 40), 1), ops.Int8Rows(w.q[:, :40].contiguous(), w.scale, 40), out)
    refused("scales", x, ops.Int8Rows(w.q, w.scale[:8], 64), out)
    refused("int8", x, ops.Int8Rows(w.q.to(torch.uint8), w.scale, 64), out)
    refused("CUDA device", x.cpu(), w, out)
    with pytest.raises(ops.KernelError, match="CUDA device"):
        ops.quantize_rows(x.cpu())
    with pytest.raises(ops.KernelError, match=r"\[R, K\]"):
        ops.quantize_rows(x[0], ops.int8_rows(1, 64, "cuda"))
    with pytest.raises(ops.KernelError, match="8-bit rows"):
        ops.quantize_rows(x, ops.int8_rows(5, 64, "cuda"))
    with pytest.raises(ops.KernelError, match="8-bit rows"):
        ops.rmsnorm(draw((4, 64), 1), draw((64,), 1), 1e-5, ops.int8_rows(4, 48, "cuda"))


def test_no_rows():
    w = ops.quantize_rows(draw((32, 64), 2))
    ops.linear(torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"), w, torch.empty(0, 32, dtype=torch.bfloat16, device="cuda"))
    assert ops.quantize_rows(torch.empty(0, 64, device="cuda")).q.shape == (0, 64)
