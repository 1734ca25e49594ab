"""Attention over the cache of 8-bit integers where queries, keys and values leave the ordinary: zeros, numbers that are not finite, sizes far apart."""
from dataclasses import replace

import pytest
import torch

from gpt_fast_b200 import ops
from gpt_fast_b200.ops.cuda import int8_pairs, int8_shares
from test_int8_cache_gpu import BF16, check, make_batch, make_cache

pytestmark = pytest.mark.gpu

# cached and new tokens: single tokens in slices and in equal shares of all pages, prompts in whole items and in equal shares of all keys
SLICES, SHARES = ([300, 70], [1, 1]), ([60000], [1])
WHOLE, EVEN = ([200, 70], [90, 40]), ([5000], [70])
WAYS = [SLICES, SHARES, WHOLE, EVEN]
H, G = 8, 2


def set_up(cached, new, d, seed=0):
    batch = make_batch(cached, new)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    if batch.max_q_len > 1:
        assert int8_pairs(batch.n_tokens, batch.n_seqs, batch.max_q_len, batch.max_kv_len, H // G, G, sms)[1] == (max(cached) >= 5000)
    else:
        assert bool(int8_shares(-(-batch.max_kv_len // 64) * 64, 64, batch.n_tokens * G, sms)[1]) == (max(cached) >= 60000)
    kv = make_cache(batch, cached, new, G, d, seed=seed)
    q = torch.randn((batch.n_tokens, H, d), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + 5)).to(BF16)
    return batch, kv, q


def attend(q, kv, batch, d, window=None):
    out = torch.full((batch.n_tokens, H * d), 7.0, dtype=BF16, device="cuda")
    ops.attention(q, kv, batch, out, H, G, d, d ** -0.5, window)
    ops.check_status(batch.status)
    return out


def set_rows(kv, batch, seq, first, last, **fields):
    """Positions first .. last - 1 of a sequence: k_pool=, k_scale=, ... to the given values."""
    at = torch.arange(first, last, device="cuda")
    page = kv.page_table[batch.slots[seq].long(), at // 64].long()
    for name, value in fields.items():
        getattr(kv, name)[page, :, at % 64] = value


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cached,new,window", [([0], [2], None), ([0], [300], None), ([100, 0], [50, 200], 30), (*WHOLE, None), (*EVEN, None), (*EVEN, 3000), (*SLICES, None), (*SHARES, None),
                                               ([0, 0], [1, 1], None)])
def test_zero_queries_over_zero_keys(cached, new, window, d):
    """Scores of zero, seen or masked beside: the mean of the seen values."""
    batch = make_batch(cached, new)
    kv = make_cache(batch, cached, new, G, d)
    kv.k_pool.zero_(), kv.k_scale.zero_()
    q = torch.zeros(batch.n_tokens, H, d, dtype=BF16, device="cuda")
    check(attend(q, kv, batch, d, window), q, kv, batch, H, G, d, d ** -0.5, window)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [None, 40])
def test_a_prompt_that_begins_with_zeros(d, window):
    """130 rows of zeros, more than a block of keys, ahead of ordinary ones; then zero queries over ordinary keys and the other way round."""
    batch = make_batch([0, 0], [300, 200])
    kv = make_cache(batch, [0, 0], [300, 200], G, d)
    q = torch.randn(500, H, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(BF16)
    keep = kv.k_pool.clone(), kv.k_scale.clone(), q.clone()
    set_rows(kv, batch, 0, 0, 130, k_pool=0, k_scale=0.0, v_pool=0, v_scale=0.0)
    q[:130] = 0
    check(attend(q, kv, batch, d, window), q, kv, batch, H, G, d, d ** -0.5, window)
    kv.k_pool.copy_(keep[0]), kv.k_scale.copy_(keep[1])
    check(attend(q, kv, batch, d, window), q, kv, batch, H, G, d, d ** -0.5, window)
    set_rows(kv, batch, 0, 0, 130, k_pool=0, k_scale=0.0)
    check(attend(keep[2], kv, batch, d, window), keep[2], kv, batch, H, G, d, d ** -0.5, window)


@pytest.mark.parametrize("cached,new", [([60, 200], [10, 5]), ([5000], [70])])
def test_zero_queries_and_a_missing_page(cached, new):
    """Keys without a page are masked like those that a row does not see."""
    d = 128
    batch = make_batch(cached, new)
    kv = make_cache(batch, cached, new, G, d)
    kv.k_pool.zero_(), kv.k_scale.zero_(), kv.v_pool.fill_(50), kv.v_scale.fill_(0.5)
    kv.page_table[batch.slots[0].long(), 1] = -1
    out = torch.empty(batch.n_tokens, H * d, dtype=BF16, device="cuda")
    ops.attention(torch.zeros(batch.n_tokens, H, d, dtype=BF16, device="cuda"), kv, batch, out, H, G, d, d ** -0.5)
    with pytest.raises(ops.KernelError, match="no page"):
        ops.check_status(batch.status)
    assert (out == 25).all()                                  # the mean of what is there, every value being 25


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("what", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("cached,new", WAYS)
def test_queries_that_are_not_finite(cached, new, what, d):
    """A query with a NaN or an infinity is NaN whichever way its keys are cut up, and no other query notices.  One number of all keys has one sign, so that the
    infinite scores are all +infinity or all -infinity."""
    batch, kv, q = set_up(cached, new, d)
    kv.k_pool[..., 5] = kv.k_pool[..., 5].abs().clamp(min=1)
    clean = attend(q, kv, batch, d).view(-1, H, d)
    row, whole = batch.n_tokens // 2, q.clone()
    q[row, 3, 5] = float(what)
    out = attend(q, kv, batch, d).view(-1, H, d)
    assert out[row, 3].isnan().all()
    # The single-token kernels move the references of a key head's queries together, when one of them has to be moved: what is kept in float16 under another
    # reference is rounded elsewhere.  So these four queries are held to the bounds of `check`, all others to their bits.
    mates = out[row, :H // G].clone()
    mates[3] = clean[row, 3]
    out[row, :H // G] = clean[row, :H // G]
    assert torch.equal(out, clean)
    out[row, :H // G] = mates
    check(out, whole, kv, batch, H, G, d, d ** -0.5)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("field", ["k_scale", "v_scale"])
@pytest.mark.parametrize("cached,new", WAYS)
def test_many_rows_that_stand_for_nan(cached, new, field, d):
    """Parts of the keys in which every row stands for NaN: whoever sees them is NaN, a window that passes them by is not."""
    batch, kv, q = set_up(cached, new, d)
    clean = replace(kv, **{field: getattr(kv, field).clone()})
    for seq in range(len(new)):
        set_rows(kv, batch, seq, 0, cached[seq] // 2, **{field: float("nan")})
    assert attend(q, kv, batch, d).isnan().all()
    window = min(c - c // 2 for c in cached)
    check(attend(q, kv, batch, d, window), q, clean, batch, H, G, d, d ** -0.5, window)


@pytest.mark.parametrize("d", [64, 128])
def test_one_part_of_a_row_is_nan(d):
    """All keys of some parts of the shared prompt stand for NaN, other parts are clean: the rows are NaN, wherever the parts are cut."""
    batch, kv, q = set_up(*EVEN, d)
    for first, n in ((0, 128), (0, 640), (640, 512), (1152, 1024), (2000, 900), (4224, 700)):       # whole shares of four blocks of keys among them
        keep = kv.k_scale.clone()
        set_rows(kv, batch, 0, first, first + n, k_scale=float("nan"))
        assert attend(q, kv, batch, d).isnan().all()
        kv.k_scale.copy_(keep)


@pytest.mark.parametrize("size", [2.0 ** -110, 2.0 ** -60, 2.0 ** 60, 2.0 ** 102, 2.0 ** 112, 2.0 ** 120])
@pytest.mark.parametrize("cached,new", WAYS)
def test_queries_and_keys_of_any_size(cached, new, size):
    """Queries of 2^-112 to 2^122 and keys as much smaller or larger, so that their products are ordinary."""
    d = 128
    batch, kv, q = set_up(cached, new, d)
    kv.k_scale.mul_(1 / size)
    q.mul_(size)
    assert q.isfinite().all() and kv.k_scale.isfinite().all()
    check(attend(q, kv, batch, d), q, kv, batch, H, G, d, d ** -0.5)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("k,v", [(2.0 ** 4, 2.0 ** 4), (2.0 ** 12, 1.0), (2.0 ** 20, 1.0), (2.0 ** 40, 1.0), (2.0 ** 120, 1.0), (1.0, 2.0 ** 12), (1.0, 2.0 ** 20), (1.0, 2.0 ** 40), (1.0, 2.0 ** 95),
                                 (1.0, 2.0 ** 120), (2.0 ** -40, 2.0 ** -40), (2.0 ** 60, 2.0 ** 60)])
@pytest.mark.parametrize("cached,new", [([10, 0], [100, 300]), EVEN])
def test_a_row_unlike_its_neighbours_reaches_who_sees_it(cached, new, k, v, d):
    """Keys and values far larger (or smaller) than those beside them: queries ahead of them, and queries whose window is past them, have the result they have without."""
    batch, kv, q = set_up(cached, new, d)
    last, n = cached[0] + new[0] - 1, int(batch.cu_seqlens[1]) - 1
    at = [last, cached[0] - 3] if cached[0] >= 5000 else [last]
    clean = attend(q, kv, batch, d, 3)
    for i in at:
        page = kv.page_table[batch.slots[0].long(), i // 64].long()
        kv.k_scale[page, :, i % 64] *= k
        kv.v_scale[page, :, i % 64] *= v
    out = attend(q, kv, batch, d, 3)
    # rows 3 .. n - 1 of the first sequence see neither of them: exact sums aside, whose order is the same, the references of a block may differ by a power of two and
    # a weight's float16 rounding with them, so these are held to the bounds of `check`
    plain = replace(kv, k_scale=kv.k_scale.clone(), v_scale=kv.v_scale.clone())
    for i in at:
        page = kv.page_table[batch.slots[0].long(), i // 64].long()
        plain.k_scale[page, :, i % 64] /= k
        plain.v_scale[page, :, i % 64] /= v
    out[:3], out[n] = clean[:3], clean[n]
    check(out, q, plain, batch, H, G, d, d ** -0.5, 3)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("span", [2, 9, 14, 30, 80])
@pytest.mark.parametrize("cached,new", WAYS)
def test_scales_that_span_many_powers_of_two(cached, new, span, d):
    """Keys and values whose scales lie anywhere in a range of 2^span, zeros among them, all seen and two at a time."""
    batch, kv, q = set_up(cached, new, d)
    g = torch.Generator(device="cuda").manual_seed(span)
    for scale in (kv.k_scale, kv.v_scale):
        scale.mul_(torch.exp2(torch.rand(scale.shape, generator=g, device="cuda") * span - span))
        scale.masked_fill_(torch.rand(scale.shape, generator=g, device="cuda") < 0.05, 0.0)
    kv.k_pool.masked_fill_(kv.k_scale[..., None] == 0, 0)
    kv.v_pool.masked_fill_(kv.v_scale[..., None] == 0, 0)
    check(attend(q, kv, batch, d), q, kv, batch, H, G, d, d ** -0.5)
    check(attend(q, kv, batch, d, 2), q, kv, batch, H, G, d, d ** -0.5, 2)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("d", [128, 24, 20])
def test_a_cache_without_pages(d, dtype):
    """Nothing is written, zeros are read, and the status says so."""
    batch = make_batch([3], [2])
    pool, scale = torch.empty((0, G, 64, d), dtype=torch.int8, device="cuda"), torch.empty((0, G, 64), device="cuda")
    kv = ops.Int8KV(pool, pool.clone(), torch.zeros((1, 1), dtype=torch.int32, device="cuda"), 64, k_scale=scale, v_scale=scale.clone())
    qkv, q = torch.randn(2, (H + 2 * G) * d, device="cuda").to(dtype), torch.empty(2, H, d, dtype=dtype, device="cuda")
    ops.rope_append(qkv, q, kv, batch, torch.ones(8, d // 2, 2, device="cuda"), H, G, d)
    with pytest.raises(ops.KernelError, match="position beyond"):
        ops.check_status(batch.status)
    k, v = (torch.full((2, G, d), 3.0, dtype=dtype, device="cuda") for _ in range(2))
    ops.read_cache(kv, batch, k, v)
    with pytest.raises(ops.KernelError, match="position beyond"):
        ops.check_status(batch.status)
    assert (k == 0).all() and (v == 0).all() and (q == 0).all()
    out = torch.full((2, H * d), 3.0, dtype=dtype, device="cuda")
    ops.attention(q, kv, batch, out, H, G, d, d ** -0.5)
    with pytest.raises(ops.KernelError, match="no page"):
        ops.check_status(batch.status)
    assert (out == 0).all()


MANY = [([i * 37 % 300 for i in range(40)], [30 + i % 5 for i in range(40)]), ([i * 7 % 150 for i in range(1100)], [1 + i % 3 for i in range(1100)]), ([32000, 5], [300, 40])]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cached,new", MANY)
def test_scales_far_apart_in_many_items(cached, new, d):
    """Blocks of threads that go through several items twice, among them such as have no scale of the kind; more pairs of tiles than are sorted; shares.  The same bits each time."""
    batch = make_batch(cached, new)
    kv = make_cache(batch, cached, new, G, d)
    g = torch.Generator(device="cuda").manual_seed(4)
    for scale in (kv.k_scale, kv.v_scale):
        scale[torch.rand(scale.shape, generator=g, device="cuda") < 0.002] *= 2.0 ** -30
    kv.v_scale[torch.rand(kv.v_scale.shape, generator=g, device="cuda") < 0.002] *= 2.0 ** 14
    q = torch.randn((batch.n_tokens, H, d), generator=g, device="cuda").to(BF16)
    out = attend(q, kv, batch, d)
    check(out, q, kv, batch, H, G, d, d ** -0.5)
    assert torch.equal(out, attend(q, kv, batch, d))


@pytest.mark.parametrize("cached,new", [([200, 70], [90, 40]), ([5000], [70])])
def test_scales_far_apart_beside_nan_and_missing_pages(cached, new):
    d = 128
    batch, kv, q = set_up(cached, new, d)
    end = cached[0] + new[0]
    set_rows(kv, batch, 0, 70, 71, v_scale=1e9, k_scale=1e-12)
    set_rows(kv, batch, 0, end - 20, end - 19, k_scale=float("nan"))        # seen by the first sequence's last 20 queries
    n = new[0] - 20
    clean = replace(kv, k_scale=kv.k_scale.clone())
    clean.k_scale[kv.page_table[batch.slots[0].long(), (end - 20) // 64].long(), :, (end - 20) % 64] = 0.01
    out = attend(q, kv, batch, d)
    assert out[n:new[0]].isnan().all()
    sound = attend(q, clean, batch, d)
    out[n:new[0]] = sound[n:new[0]]
    check(out, q, clean, batch, H, G, d, d ** -0.5)
    kv.page_table[batch.slots[0].long(), 0] = -1
    out = torch.empty(batch.n_tokens, H * d, dtype=BF16, device="cuda")
    ops.attention(q, kv, batch, out, H, G, d, d ** -0.5)
    with pytest.raises(ops.KernelError, match="no page"):
        ops.check_status(batch.status)
    assert out[n:new[0]].isnan().all() and not out[:n].isnan().any()
