"""Attention over the cache of 8-bit integers, whichever way a call is cut up: equal shares over several sequences, pages that are missing, many or empty sequences, many heads per
key head, caches beyond 2^31 numbers; against 64 bits, within what the kernels' own roundings add up to."""
from dataclasses import replace

import pytest
import torch

from gpt_fast_b200 import ops
from gpt_fast_b200.ops import Int8KV
from gpt_fast_b200.ops.cuda import int8_pairs
from test_int8_cache_gpu import BF16, F64, make_batch, make_cache, reference, rope

pytestmark = pytest.mark.gpu


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def even(batch, H, G, window=None):
    reach = batch.max_kv_len if window is None else min(batch.max_kv_len, window + 256)
    return int8_pairs(batch.n_tokens, batch.n_seqs, batch.max_q_len, reach, H // G, G, sms())[1]


def random_queries(batch, H, d, factor=1.0, seed=1):
    return (factor * torch.randn(batch.n_tokens, H, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))).to(BF16)


def attend(q, kv, batch, H, G, d, window=None):
    out = torch.full((batch.n_tokens, H * d), float("nan"), dtype=q.dtype, device="cuda")
    ops.attention(q, kv, batch, out, H, G, d, d ** -0.5, window)
    return out


def bounds(q, kv, batch, H, G, d, window=None):
    """(result in 64 bits, how far a bfloat16 output may be off) [T, H, d], for the kernels of pages of 64 and heads of 64 and 128."""
    o, mag, most, top = reference(q, kv, batch, H, G, d, d ** -0.5, window)
    L, prompt = batch.max_kv_len, batch.max_q_len > 1 or H // G > 8
    # A score: d products summed in 32 bits and three products more; in prompts the number that key and scale stand for is rounded to float16, half a step being 2^-11.  A weight
    # is off by twice that (its own and the largest's), 8 steps of the exponential and its argument, the sum of weights by 2 L steps, and the weight
    # itself is rounded to float16, 2^-11; in prompts so is the value.
    score = (d + 4) * 2.0 ** -24 + (2.0 ** -11 if prompt else 0.0)
    rel = 2 * score * most + (8 + 2 * L) * 2.0 ** -24 + (2 if prompt else 1) * 2.0 ** -11
    # Small weights: off by 2^-25 where the row's largest is 2^12 at least, each meeting an integer of at most 127; four times as much where a block's largest scale stands for all
    # (make_cache's scales are within a factor of four: rows of a normal distribution times 0.5 to 1.5).
    return o, mag * rel * 1.01 + o.abs() * 2.0 ** -8 + L * 127 * 2.0 ** -37 * (4 if prompt else 1) * top + 1e-30


def check(out, q, kv, batch, H, G, d, window=None):
    o, tol = bounds(q, kv, batch, H, G, d, window)
    bad = (out.view(-1, H, d).to(F64) - o).abs() / tol
    assert bool(bad.le(1).all()), float(bad.nan_to_num(1e9).max())


# ---- the precision that the kernels keep -----------------------------------------------------------------------

@pytest.mark.parametrize("H,G,d", [(32, 8, 128), (6, 2, 64)])
@pytest.mark.parametrize("new", [1, 2])
def test_weights_keep_eleven_bits(new, H, G, d):
    """Few keys and flat scores, so that a weight's rounding is most of what a result is off by: that of bfloat16 weights would not pass."""
    cached = [i % 6 + 1 for i in range(60)]
    batch = make_batch(cached, [new] * 60)
    kv = make_cache(batch, cached, [new] * 60, G, d)
    q = random_queries(batch, H, d, 0.5 if new == 1 else 0.02)
    check(attend(q, kv, batch, H, G, d), q, kv, batch, H, G, d)
    ops.check_status(batch.status)
    # the oracle with weights of eight bits (a rounding of their common factor aside, which both sums have)
    o, tol = bounds(q, kv, batch, H, G, d)
    far = torch.zeros_like(o)
    for s in range(60):
        slot, n = int(batch.slots[s]), cached[s] + new
        page = kv.page_table[slot, :1].long()
        k, v = ((pool[page].to(F64) * scale[page].to(F64)[..., None])[0, :, :n].repeat_interleave(H // G, 0) for pool, scale in ((kv.k_pool, kv.k_scale), (kv.v_pool, kv.v_scale)))
        for i in range(new):
            t = s * new + i
            w = torch.einsum("hd,hjd->hj", q[t].to(F64), k[:, :cached[s] + i + 1]).mul(d ** -0.5)
            w = (w - w.amax(-1, keepdim=True)).exp()
            far[t] = torch.einsum("hj,hjd->hd", w.to(BF16).to(F64), v[:, :cached[s] + i + 1]) / w.sum(-1, keepdim=True) - o[t]
    assert bool((far.abs() > tol).any())


# ---- equal shares over several sequences --------------------------------------------------------------------------

SHARED = [([32001, 0, 500, 1000, 1500, 2000, 2500, 3000, 3500], [512, 1, 1, 1, 1, 1, 1, 1, 1], None), ([3000, 9000, 100, 20000, 5000, 7000], [64, 64, 64, 64, 64, 64], None),
          ([4000, 3800, 4100], [100, 90, 80], None), ([9000, 0, 9100], [40, 3, 41], 4000), ([30000, 12, 30], [2, 1, 70], None), ([15000, 14000], [33, 300], 12000)]


@pytest.mark.parametrize("H,G,d", [(32, 8, 128), (6, 2, 64), (7, 1, 128)])
@pytest.mark.parametrize("cached,new,window", SHARED)
def test_shares_of_several_sequences(cached, new, window, H, G, d):
    """Blocks that end one sequence's keys and begin another's, sequences far apart in length, a chunk beside single tokens."""
    batch = make_batch(cached, new, n_slots=len(new) + 1)
    if not even(batch, H, G, window):
        assert (H, G) != (32, 8)
        pytest.skip("whole items at this layout")
    kv = make_cache(batch, cached, new, G, d, seed=len(cached))
    q = random_queries(batch, H, d)
    out = attend(q, kv, batch, H, G, d, window)
    ops.check_status(batch.status)
    check(out, q, kv, batch, H, G, d, window)
    assert torch.equal(out, attend(q, kv, batch, H, G, d, window))


# ---- missing pages ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("d,page", [(128, 64), (64, 64), (48, 64), (128, 16)])
@pytest.mark.parametrize("cached,new,gone,window", [([300, 0, 70], [1, 1, 1], (0, 2), None), ([60000], [1], (0, 300, 937), None), ([300], [1], (0, 1, 2, 3, 4), None), ([200, 0], [100, 40], (0, 3), None),
                                                    ([200, 0], [100, 40], (0, 1, 2, 3, 4), None), ([5000], [70], (0, 1, 40, 78), None), ([5000], [70], (70, 78), 200), ([0], [130], (0,), None)])
def test_what_is_read_beside_missing_pages(cached, new, gone, window, d, page):
    """The keys of a missing page are left out, in the first page, in the last, in all of a block and in all that a row sees (which then gets zeros)."""
    H, G = 8, 2
    if max(cached) > 10000 and (d, page) != (128, 64):
        pytest.skip("the long cache at one layout")
    batch = make_batch(cached, new)
    kv = make_cache(batch, cached, new, G, d, page)
    q = random_queries(batch, H, d)
    slot, end = int(batch.slots[0]), cached[0] + new[0]
    holes = kv.page_table.clone()
    hidden = torch.zeros(end, dtype=torch.bool, device="cuda")
    for i in gone:
        for p in range(i * 64 // page, min((i + 1) * 64, end + page - 1) // page):
            holes[slot, p] = -1 if p % 2 == 0 else kv.k_pool.shape[0] + 5            # neither is a page
            hidden[p * page:(p + 1) * page] = True
    out = attend(q, replace(kv, page_table=holes), batch, H, G, d, window).view(-1, H, d).to(F64)
    with pytest.raises(ops.KernelError, match="no page"):
        ops.check_status(batch.status)
    # the first sequence's rows by hand; all others as `reference` has them
    n0 = new[0]
    if batch.n_tokens > n0:
        o, tol = bounds(q, kv, batch, H, G, d, window)
        assert bool(((out - o).abs() <= tol)[n0:].all())
    p = kv.page_table[slot, :-(-end // page)].long()
    k, v = ((pool[p].to(F64) * scale[p].to(F64)[..., None]).transpose(1, 2).reshape(-1, G, d)[:end].repeat_interleave(H // G, 1) for pool, scale in ((kv.k_pool, kv.k_scale), (kv.v_pool, kv.v_scale)))
    far = torch.arange(cached[0], end, device="cuda")[:, None] - torch.arange(end, device="cuda")
    mask = (far < 0) | (far >= (window or end + 1)) | hidden
    s = torch.einsum("thd,jhd->htj", q[:n0].to(F64), k) * d ** -0.5
    a = (torch.einsum("thd,jhd->htj", q[:n0].to(F64).abs(), k.abs()) * d ** -0.5).masked_fill(mask, 0).amax(-1).t()[..., None]
    w = torch.softmax(s.masked_fill(mask, -torch.inf), -1).nan_to_num(0.0)           # (a row of nothing but -infinity)
    o, mag = torch.einsum("htj,jhd->thd", w, v), torch.einsum("htj,jhd->thd", w, v.abs())
    # as in `bounds`, the prompt kernel's terms for all; a value is at most 127 times its scale, and a weight times a scale at most the largest
    tol = mag * (2 * ((d + 4) * 2.0 ** -24 + 2.0 ** -11) * a + (8 + 2 * end) * 2.0 ** -24 + 2 * 2.0 ** -11) * 1.01 + o.abs() * 2.0 ** -8 + end * 127 * 2.0 ** -35 * float(kv.v_scale.max())
    got = out[:n0]
    empty = mask.all(1)
    assert (got[empty] == 0).all()
    bad = ((got - o).abs() / tol)[~empty]
    assert bool(bad.le(1).all()), float(bad.nan_to_num(1e9).max())


# ---- sequences and heads ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("H,G,d", [(8, 2, 128), (8, 2, 64), (8, 2, 48)])
@pytest.mark.parametrize("cached,new", [([50, 100, 7], [1, 0, 1]), ([50, 100, 7, 20], [40, 0, 200, 0]), ([5000, 100, 30], [70, 0, 2]), ([0, 0], [0, 3])])
def test_sequences_without_new_tokens(cached, new, H, G, d):
    """A sequence of the batch that has nothing new neither writes nor is in another's way."""
    batch = make_batch(cached, new)
    kv = make_cache(batch, cached, [max(n, 1) for n in new], G, d)
    q = random_queries(batch, H, d)
    out = attend(q, kv, batch, H, G, d)
    ops.check_status(batch.status)
    keep = [i for i, n in enumerate(new) if n]
    some = make_batch([cached[i] for i in keep], [new[i] for i in keep], slots=[int(batch.slots[i]) for i in keep], n_slots=len(new))
    if d == 48:
        o, mag, _, _ = reference(q, kv, some, H, G, d, d ** -0.5, None)
        assert bool(((out.view(-1, H, d).to(F64) - o).abs() <= mag * 2.0 ** -8 + 1e-30).all())         # (32-bit sums: the output's rounding, and a little of the value)
    else:
        check(out, q, kv, some, H, G, d)


@pytest.mark.parametrize("H,G,d", [(40, 1, 128), (128, 1, 64), (100, 2, 128), (33, 3, 128)])
@pytest.mark.parametrize("cached,new", [([300, 5], [1, 1]), ([100, 0], [3, 40]), ([6000], [5])])
def test_many_heads_per_key_head(cached, new, H, G, d):
    """Tiles of one to eleven tokens, rows of a tile that no token has; and single tokens of more heads than their own kernel takes."""
    batch = make_batch(cached, new)
    kv = make_cache(batch, cached, new, G, d)
    q = random_queries(batch, H, d)
    out = attend(q, kv, batch, H, G, d)
    ops.check_status(batch.status)
    check(out, q, kv, batch, H, G, d)


@pytest.mark.parametrize("n", [4096, 4097])
def test_thousands_of_single_tokens(n):
    """As many as the kernel of equal shares counts, and one more."""
    H, G, d = 4, 2, 64
    cached = [(37 * i) % 200 for i in range(n)]
    batch = make_batch(cached, [1] * n)
    kv = make_cache(batch, cached, [1] * n, G, d)
    q = random_queries(batch, H, d)
    out = attend(q, kv, batch, H, G, d)
    ops.check_status(batch.status)
    check(out, q, kv, batch, H, G, d)


@pytest.mark.parametrize("size", [2.0 ** -80, 2.0 ** -40, 2.0 ** 40, 2.0 ** 100])
@pytest.mark.parametrize("cached,new", [([300, 70], [1, 1]), ([60000], [1]), ([200, 70], [90, 40]), ([5000], [70])])
def test_values_of_any_size(cached, new, size):
    H, G, d = 8, 2, 128
    batch = make_batch(cached, new)
    kv = make_cache(batch, cached, new, G, d)
    kv.v_scale.mul_(size)
    q = random_queries(batch, H, d)
    check(attend(q, kv, batch, H, G, d), q, kv, batch, H, G, d)


# ---- offsets beyond 32 bits ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("cached,new", [([500, 70], [1, 1]), ([60000], [1]), ([200, 70], [90, 40]), ([5000], [70])])
def test_a_cache_beyond_two_to_the_31(cached, new):
    """Pools of 2.7e9 numbers each, the sequences in their last pages: written, read back and attended to."""
    H, G, d, pages = 8, 8, 128, 41000
    batch = make_batch(cached, new)
    small = make_cache(batch, cached, new, G, d)
    P = small.k_pool.shape[0]
    far = pages - P
    pools = [torch.zeros((pages, G, 64, d), dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros((pages, G, 64), device="cuda") for _ in range(2)]
    for big, little in zip(pools + scales, (small.k_pool, small.v_pool, small.k_scale, small.v_scale)):
        big[far:] = little
    kv = Int8KV(*pools, torch.where(small.page_table >= 0, small.page_table + far, -1), 64, k_scale=scales[0], v_scale=scales[1])
    T = batch.n_tokens
    qkv = random_queries(batch, H + 2 * G, d).view(T, -1)
    q, want = (torch.empty(T, H, d, dtype=BF16, device="cuda") for _ in range(2))
    table = rope(batch.max_kv_len, d)
    ops.rope_append(qkv, q, kv, batch, table, H, G, d)
    ops.rope_append(qkv, want, small, batch, table, H, G, d)
    assert torch.equal(q, want)
    for big, little in zip(pools + scales, (small.k_pool, small.v_pool, small.k_scale, small.v_scale)):
        assert torch.equal(big[far:], little) and not big[:64].any()
    k, v = (torch.empty(T, G, d, dtype=BF16, device="cuda") for _ in range(2))
    k2, v2 = torch.empty_like(k), torch.empty_like(v)
    ops.read_cache(kv, batch, k, v)
    ops.read_cache(small, batch, k2, v2)
    assert torch.equal(k, k2) and torch.equal(v, v2)
    assert torch.equal(attend(q, kv, batch, H, G, d), attend(q, small, batch, H, G, d))
    ops.check_status(batch.status)


# ---- what the cache is given ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("pairing", ["interleaved", "half"])
@pytest.mark.parametrize("d", [128, 64, 48])
def test_rows_that_are_not_finite_on_their_way_into_the_cache(d, pairing, dtype):
    """A key or value row with a NaN or an infinity is kept as NaN, its neighbours as they are."""
    H, G = 4, 3
    cached, new = [60, 0], [7, 20]
    batch = make_batch(cached, new)
    kv, kv2 = (make_cache(batch, cached, new, G, d, fill=False) for _ in range(2))
    T = batch.n_tokens
    qkv = torch.randn(T, H + 2 * G, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(dtype)
    bad = qkv.clone()
    bad[2, H + 1, 5], bad[9, H + G + 2, d - 1], bad[20, H, 0], bad[11, 1, 3] = float("nan"), float("inf"), float("-inf"), float("nan")
    table, q, q2 = rope(128, d), *(torch.empty(T, H, d, dtype=dtype, device="cuda") for _ in range(2))
    ops.rope_append(qkv.view(T, -1), q, kv, batch, table, H, G, d, pairing)
    ops.rope_append(bad.view(T, -1), q2, kv2, batch, table, H, G, d, pairing)
    ops.check_status(batch.status)
    k, v, k2, v2 = (torch.empty(T, G, d, device="cuda") for _ in range(4))
    ops.read_cache(kv, batch, k, v)
    ops.read_cache(kv2, batch, k2, v2)
    assert k2[2, 1].isnan().all() and v2[9, 2].isnan().all() and k2[20, 0].isnan().all()
    k2[2, 1], v2[9, 2], k2[20, 0], q2[11, 1] = k[2, 1], v[9, 2], k[20, 0], q[11, 1]
    assert torch.equal(k, k2) and torch.equal(v, v2) and torch.equal(q, q2)
