"""A paged cache of 8-bit integers: writing it, reading it back, and attention over it, against 64 bits."""
import pytest
import torch

from gpt_fast_b200 import ops
from gpt_fast_b200.ops import BatchMeta, Int8KV

pytestmark = pytest.mark.gpu
F64 = torch.float64
BF16 = torch.bfloat16


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make_batch(cached, new, slots=None, n_slots=None):
    """Sequences with `cached` tokens before the step and `new` in it; slots: which slot each is in (default: in reverse order)."""
    n = len(new)
    slots = list(reversed(range(n))) if slots is None else slots
    lengths = [0] * (n_slots or max(slots) + 1)
    for s, c in zip(slots, cached):
        lengths[s] = c
    cu = [0]
    for q in new:
        cu.append(cu[-1] + q)
    return BatchMeta(i32(cu), i32([i for i, q in enumerate(new) for _ in range(q)]), i32(slots), i32(lengths), n, cu[-1], max(new),
                     max(a + b for a, b in zip(cached, new)), ops.new_status("cuda"))


def make_cache(batch, cached, new, G, d, page=64, seed=0, spare=3, fill=True):
    """A cache with room for the batch, its pages shuffled, filled with rows of a normal distribution; `spare` pages belong to nobody."""
    need = [-(-(a + b) // page) for a, b in zip(cached, new)]
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(sum(need) + spare, generator=g).tolist()
    table = torch.full((batch.lengths.shape[0], max(need) + 1), -1, dtype=torch.int32)
    for s, k in zip(batch.slots.tolist(), need):
        for i in range(k):
            table[s, i] = order.pop()
    P = sum(need) + spare
    gg = torch.Generator(device="cuda").manual_seed(seed + 1)

    def pool():
        x = torch.randn((P, G, page, d), generator=gg, device="cuda") * (0.5 + torch.rand((P, G, page, 1), generator=gg, device="cuda"))
        most = x.abs().amax(-1)
        return (x / most[..., None] * 127).round().to(torch.int8), most / 127
    (k, ks), (v, vs) = pool(), pool()
    if not fill:
        k.zero_(), v.zero_(), ks.zero_(), vs.zero_()
    return Int8KV(k, v, table.cuda(), page, k_scale=ks, v_scale=vs)


def rows_of(kv, slot, n, pool, scale):
    """The first n rows of a slot as 64-bit numbers [n, G, d]."""
    page = kv.page_size
    p = kv.page_table[slot, :-(-n // page)].long()
    x = pool[p].to(F64) * scale[p].to(F64)[..., None]
    return x.transpose(1, 2).reshape(-1, pool.shape[1], pool.shape[3])[:n]


def places(batch):
    seq = batch.tok_seq.long()
    slot = batch.slots.long()[seq]
    return slot, batch.lengths.long()[slot] + torch.arange(batch.n_tokens, device="cuda") - batch.cu_seqlens.long()[seq]


def rope(P, d, seed=0):
    f = 10000.0 ** (-torch.arange(0, d, 2, dtype=F64, device="cuda") / d)
    a = torch.arange(P, dtype=F64, device="cuda")[:, None] * f
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def turned(x, table, pos, pairing):
    """32-bit rotation, every product and sum rounded by itself."""
    cs = table[pos][:, None]
    c, s = cs[..., 0], cs[..., 1]
    d = x.shape[-1]
    a, b = (x[..., :d // 2], x[..., d // 2:]) if pairing == "half" else (x[..., 0::2], x[..., 1::2])
    p, q = a * c, b * s
    r, t = b * c, a * s
    y = [p - q, r + t]
    return torch.cat(y, -1) if pairing == "half" else torch.stack(y, -1).flatten(-2)


def quantised(x):
    most = x.abs().amax(-1)
    q = torch.where(most[..., None] > 0, (x.to(F64) * 127 / most.to(F64).clamp(min=5e-324)[..., None]).round(), 0.0)
    return q.to(torch.int8), (most.to(F64) / 127).float()      # the quotient, rounded once (a 32-bit tensor over a number is a product with its reciprocal)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("pairing", ["interleaved", "half"])
@pytest.mark.parametrize("H,G,d,page", [(32, 8, 128, 64), (4, 4, 64, 64), (12, 3, 128, 64), (6, 2, 48, 64), (5, 1, 256, 16), (2, 2, 2, 64), (40, 40, 128, 64), (3, 3, 66, 32)])
@pytest.mark.parametrize("cached,new", [([0], [1]), ([63, 64, 5], [1, 1, 1]), ([0, 7, 130], [65, 1, 40]), ([100] * 70, [1] * 70), ([0, 3], [200, 130])])
def test_append_and_read(H, G, d, page, cached, new, pairing, dtype):
    batch = make_batch(cached, new, n_slots=len(new) + 2)
    kv = make_cache(batch, cached, new, G, d, page, seed=d)
    before = [t.clone() for t in (kv.k_pool, kv.v_pool, kv.k_scale, kv.v_scale)]
    T = batch.n_tokens
    g = torch.Generator(device="cuda").manual_seed(7)
    qkv = torch.randn((T, (H + 2 * G) * d), generator=g, device="cuda").to(dtype)
    table = rope(batch.max_kv_len, d)
    q = torch.empty(T, H, d, dtype=dtype, device="cuda")
    ops.rope_append(qkv, q, kv, batch, table, H, G, d, pairing)
    ops.check_status(batch.status)
    x = qkv.float().view(T, H + 2 * G, d)
    slot, pos = places(batch)
    y = turned(x[:, :H + G], table, pos, pairing)
    assert torch.equal(q, y[:, :H].to(dtype))
    (kq, ks), (vq, vs) = quantised(y[:, H:]), quantised(x[:, H + G:])
    page_of = kv.page_table[slot, pos // page].long()
    where = (page_of, slice(None), pos % page)
    for i, want in enumerate((kq, vq, ks, vs)):
        pool = (kv.k_pool, kv.v_pool, kv.k_scale, kv.v_scale)[i]
        assert torch.equal(pool[where], want)
        expect = before[i]
        expect[where] = want                                 # everything else is as it was
        assert torch.equal(pool, expect)
    for out in (BF16, torch.float32):
        k, v = (torch.empty(T, G, d, dtype=out, device="cuda") for _ in range(2))
        ops.read_cache(kv, batch, k, v)
        ops.check_status(batch.status)
        assert torch.equal(k, (kq.float() * ks[..., None]).to(out)) and torch.equal(v, (vq.float() * vs[..., None]).to(out))


def test_append_without_storing():
    """append=False: only the queries are made; the cache another layer wrote stays as it is."""
    batch = make_batch([10, 3], [1, 5])
    kv = make_cache(batch, [10, 3], [1, 5], 2, 64)
    before = kv.k_pool.clone()
    qkv = torch.randn(6, (4 + 4) * 64, device="cuda").to(BF16)
    q = torch.empty(6, 4, 64, dtype=BF16, device="cuda")
    table = rope(64, 64)
    ops.rope_append(qkv, q, kv, batch, table, 4, 2, 64, "interleaved", append=False)
    assert torch.equal(kv.k_pool, before)
    assert torch.equal(q, turned(qkv.float().view(6, 8, 64)[:, :4], table, places(batch)[1], "interleaved").to(BF16))


def test_an_empty_rotary_table_is_refused():
    batch = make_batch([0], [2])
    kv = make_cache(batch, [0], [2], 2, 64)
    qkv, q = torch.zeros(2, 8 * 64, device="cuda"), torch.empty(2, 4, 64, device="cuda")
    with pytest.raises(ops.KernelError, match="empty rotary table"):
        ops.rope_append(qkv, q, kv, batch, rope(4, 64)[:0], 4, 2, 64)


def test_missing_pages_are_reported():
    batch = make_batch([60, 0], [10, 3])
    kv = make_cache(batch, [60, 0], [10, 3], 2, 64)
    kv.page_table[batch.slots[0].long(), 1] = -1              # positions 64 .. 69 of the first sequence have no page
    before = kv.k_pool.clone()
    qkv = torch.randn(13, 8 * 64, device="cuda").to(BF16)
    q = torch.empty(13, 4, 64, dtype=BF16, device="cuda")
    ops.rope_append(qkv, q, kv, batch, rope(128, 64), 4, 2, 64)
    with pytest.raises(ops.KernelError, match="position beyond"):
        ops.check_status(batch.status)
    slot, pos = places(batch)
    good = ~((batch.tok_seq == 0) & (pos >= 64))
    assert (q[~good] == 0).all()
    page_of = kv.page_table[slot[good], pos[good] // 64].long()
    before[page_of, :, pos[good] % 64] = kv.k_pool[page_of, :, pos[good] % 64]
    assert torch.equal(kv.k_pool, before)
    k, v = (torch.empty(13, 2, 64, dtype=BF16, device="cuda") for _ in range(2))
    ops.read_cache(kv, batch, k, v)
    with pytest.raises(ops.KernelError, match="position beyond"):
        ops.check_status(batch.status)
    assert (k[~good] == 0).all() and (v[~good] == 0).all()
    for new in (1, 10):                                        # attention: the missing page's keys are left out, the rest is read
        b = make_batch([70 - new, 0], [new, 3])
        out = torch.empty(b.n_tokens, 4 * 64, dtype=BF16, device="cuda")
        ops.attention(torch.randn(b.n_tokens, 4, 64, device="cuda").to(BF16), kv, b, out, 4, 2, 64, 0.125)
        with pytest.raises(ops.KernelError, match="no page"):
            ops.check_status(b.status)


# ---- attention ----------------------------------------------------------------------------------------------

def reference(q, kv, batch, H, G, d, scale, window):
    """(output, mean of |value| under the weights, largest score sum of absolute products, largest weight times its value's scale) per row, in 64 bits."""
    outs, mags, sums, tops = [], [], [], []
    cu = batch.cu_seqlens.tolist()
    lengths = batch.lengths.tolist()
    for i, slot in enumerate(batch.slots.tolist()):
        n = lengths[slot] + cu[i + 1] - cu[i]
        k = rows_of(kv, slot, n, kv.k_pool, kv.k_scale).repeat_interleave(H // G, 1)
        v = rows_of(kv, slot, n, kv.v_pool, kv.v_scale).repeat_interleave(H // G, 1)
        x = q[cu[i]:cu[i + 1]].to(F64)
        far = torch.arange(lengths[slot], n, device="cuda")[:, None] - torch.arange(n, device="cuda")
        hidden = (far < 0) | (far >= (window or n + 1))
        s = torch.einsum("thd,jhd->htj", x, k) * scale
        a = torch.einsum("thd,jhd->htj", x.abs(), k.abs()) * scale
        s = s.masked_fill(hidden, -torch.inf)
        p = torch.softmax(s, -1)
        hidden_p = p.masked_fill(hidden, 0)
        v0 = torch.nan_to_num(v, 0.0) if bool(v.isnan().any()) else v
        o = torch.einsum("htj,jhd->thd", hidden_p, v0)
        if v0 is not v:
            o = o + torch.einsum("htj,jh->th", (~hidden).to(F64).expand_as(p), v.isnan().any(-1).to(F64)).bool()[..., None] * torch.nan
        outs.append(o)
        mags.append(torch.einsum("htj,jhd->thd", hidden_p, v0.abs()))
        sums.append(a.masked_fill(hidden, 0).amax(-1).t()[..., None].expand(-1, -1, d))
        page = kv.page_size
        vs = kv.v_scale[kv.page_table[slot, :-(-n // page)].long()].transpose(1, 2).reshape(-1, G)[:n].repeat_interleave(H // G, 1).to(F64).nan_to_num(0.0)
        tops.append((hidden_p * vs.t()[:, None]).amax(-1).t()[..., None].expand(-1, -1, d))
    return torch.cat(outs), torch.cat(mags), torch.cat(sums), torch.cat(tops)


def check(got, q, kv, batch, H, G, d, scale, window=None):
    o, mag, most, top = reference(q, kv, batch, H, G, d, scale, window)
    got = got.view(-1, H, d).to(F64)
    # a score is a 32-bit sum of d products (each half a step, any order) and three products more: e = (d + 4) 2^-24 of its sum of absolute products.  A weight is off by
    # e and the maximum's e, by 4 steps of the exponential (and the lag of a reference maximum), and, in 16-bit kernels, by half a bfloat16 step; a
    # sum over L keys by L steps
    L = batch.max_kv_len
    rel = 2 * (d + 4) * 2.0 ** -24 * most + (8 + 2 * L) * 2.0 ** -24
    half = torch.finfo(q.dtype).eps / 2
    if q.dtype == BF16:
        rel = rel + 2.0 ** -8
        if batch.max_q_len > 1:
            # The prompt kernel rounds the numbers that integers and scales stand for to float16, half a step being 2^-11 of each: a score is off by up to 2^-11 of
            # its sum of absolute products (the weight by twice that, its own and the maximum's), and a value by 2^-11 of itself.
            rel = rel + 2 * 2.0 ** -11 * most + 2.0 ** -11
    tol = mag * rel * 1.01 + o.abs() * half + 1e-30
    if q.dtype == BF16:
        # Weights times scales that are kept in float16 stand in units in which the row's largest lies between 2^12 and 2^15 (LIFT, and what it may pass its
        # reference by); float16's smallest step is 2^-24, so one that is small is off by up to 2^-25, that is 2^-37 of the largest, and
        # meets an integer of at most 127, for each of L keys.
        tol = tol + L * 127 * 2.0 ** -37 * top
    bad = (got - o).abs() / tol
    assert bool(bad.le(1).all()), float(bad.nan_to_num(1e9).max())


DECODE = [([0], 0), ([1], 0), ([63], 0), ([64], 0), ([911], 0), ([5, 700, 64, 0, 129], 0), ([2000, 3], 100), ([4095], 0), ([9000, 8999, 20], 0), ([300, 17], 1), ([130] * 40, 0),
          ([20000], 0), ([33000, 70000], 0), ([700, 1500], 64), ([640, 128], 65)]
HEADS = [(32, 8, 128), (8, 8, 128), (12, 3, 128), (6, 2, 64), (7, 1, 128), (16, 2, 64), (16, 1, 128), (4, 2, 48), (3, 3, 256), (4, 4, 20)]


@pytest.mark.parametrize("H,G,d", HEADS)
@pytest.mark.parametrize("cached,window", DECODE)
def test_attention_of_single_tokens(cached, window, H, G, d):
    new = [1] * len(cached)
    if max(cached) > 10000 and (H, G, d) not in ((32, 8, 128), (6, 2, 64), (7, 1, 128)):
        pytest.skip("long caches at three head layouts")
    batch = make_batch(cached, new, n_slots=len(new) + 1)
    kv = make_cache(batch, cached, new, G, d, seed=len(cached))
    q = (2 * torch.randn(len(new), H, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))).to(BF16)
    out = torch.full((len(new), H * d), float("nan"), dtype=BF16, device="cuda")
    ops.attention(q, kv, batch, out, H, G, d, d ** -0.5, window or None)
    ops.check_status(batch.status)
    check(out, q, kv, batch, H, G, d, d ** -0.5, window)


PROMPTS = [([0], [2], 0), ([0], [128], 0), ([0, 0], [65, 3], 0), ([100], [33], 0), ([1000], [70], 0), ([0, 30, 200, 1], [300, 1, 129, 64], 0), ([500, 0], [40, 257], 50), ([64], [64], 1),
           ([127, 128, 129], [1, 2, 3], 0), ([3000], [150], 1000), ([5000], [2], 0), ([0], [1000], 128)]


@pytest.mark.parametrize("H,G,d", HEADS)
@pytest.mark.parametrize("cached,new,window", PROMPTS)
def test_attention_of_prompts(cached, new, window, H, G, d):
    batch = make_batch(cached, new, n_slots=len(new) + 1)
    kv = make_cache(batch, cached, new, G, d, seed=len(cached))
    T = batch.n_tokens
    q = (2 * torch.randn(T, H, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))).to(BF16)
    out = torch.full((T, H * d), float("nan"), dtype=BF16, device="cuda")
    ops.attention(q, kv, batch, out, H, G, d, d ** -0.5, window or None)
    ops.check_status(batch.status)
    check(out, q, kv, batch, H, G, d, d ** -0.5, window)


@pytest.mark.parametrize("n", [1000, 1100])
def test_attention_of_a_thousand_short_prompts(n):
    """More pairs of tiles than a block sorts, and as many as it does."""
    g = torch.Generator().manual_seed(n)
    cached, new = torch.randint(0, 150, (n,), generator=g).tolist(), torch.randint(1, 4, (n,), generator=g).tolist()
    new[7] = 300
    batch = make_batch(cached, new)
    kv = make_cache(batch, cached, new, 2, 64, seed=3)
    q = torch.randn((batch.n_tokens, 4, 64), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(BF16)
    out = torch.empty(batch.n_tokens, 4 * 64, dtype=BF16, device="cuda")
    ops.attention(q, kv, batch, out, 4, 2, 64, 0.125)
    ops.check_status(batch.status)
    check(out, q, kv, batch, 4, 2, 64, 0.125)


@pytest.mark.parametrize("H,G,d,page", [(4, 2, 64, 64), (6, 2, 48, 16), (2, 2, 130, 64), (8, 2, 128, 64)])
@pytest.mark.parametrize("cached,new,window", [([0], [1], 0), ([700, 40], [1, 1], 0), ([0, 130], [90, 33], 0), ([300], [20], 70)])
def test_attention_in_32_bits(cached, new, window, H, G, d, page):
    batch = make_batch(cached, new)
    kv = make_cache(batch, cached, new, G, d, page)
    q = 2 * torch.randn(batch.n_tokens, H, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    out = torch.empty(batch.n_tokens, H * d, device="cuda")
    ops.attention(q, kv, batch, out, H, G, d, d ** -0.5, window or None)
    ops.check_status(batch.status)
    check(out, q, kv, batch, H, G, d, d ** -0.5, window)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cached,new", [([200, 70], [1, 1]), ([200, 70], [90, 40])])
def test_rows_that_are_not_finite(cached, new, d):
    """A key or value row that stands for NaN reaches the queries that see it and no others; what lies behind a sequence's end reaches nobody."""
    H, G = 8, 2
    batch = make_batch(cached, new)
    kv = make_cache(batch, cached, new, G, d)
    q = torch.randn(batch.n_tokens, H, d, device="cuda").to(BF16)
    clean = torch.empty(batch.n_tokens, H * d, dtype=BF16, device="cuda")
    for s, c, n in zip(batch.slots.tolist(), cached, new):      # behind the end of each sequence, in its last page
        last = kv.page_table[s, (c + n - 1) // 64].long()
        for scale in (kv.k_scale, kv.v_scale):
            scale[last, :, (c + n - 1) % 64 + 1:] = float("nan")
    ops.attention(q, kv, batch, clean, H, G, d, d ** -0.5)
    check(clean, q, kv, batch, H, G, d, d ** -0.5)
    out = torch.empty_like(clean)
    at = cached[0] + new[0] - 1                               # the first sequence's last position: its last query alone sees it
    page = kv.page_table[batch.slots[0].long(), at // 64].long()
    for scale in (kv.k_scale, kv.v_scale):
        keep = scale[page, 0, at % 64].clone()
        scale[page, 0, at % 64] = float("nan")
        ops.attention(q, kv, batch, out, H, G, d, d ** -0.5)
        scale[page, 0, at % 64] = keep
        row, hit = int(batch.cu_seqlens[1]) - 1, H // G * d   # heads of key head 0
        assert out[row, :hit].isnan().all()
        assert torch.equal(out[row, hit:], clean[row, hit:])
        rest = [i for i in range(batch.n_tokens) if i != row]
        assert torch.equal(out[rest], clean[rest])


@pytest.mark.parametrize("new", [1, 130])
def test_large_and_tiny_scores(new):
    """Queries of any size: scores far beyond the exponential's range give one key all the weight, tiny ones give the mean."""
    H, G, d = 8, 2, 128
    cached = [400]
    batch = make_batch(cached, [new])
    kv = make_cache(batch, cached, [new], G, d)
    base = torch.randn(new, H, d, device="cuda").to(BF16)
    for factor in (2.0 ** -30, 2.0 ** 7):
        q = base * factor
        out = torch.empty(new, H * d, dtype=BF16, device="cuda")
        ops.attention(q, kv, batch, out, H, G, d, d ** -0.5)
        check(out, q, kv, batch, H, G, d, d ** -0.5)


@pytest.mark.parametrize("new", [1, 90])
def test_values_of_very_different_sizes(new):
    """A value's scale joins its weight, whatever its size; a flat softmax over rows whose scales span 2^40."""
    H, G, d = 8, 2, 128
    cached = [600]
    batch = make_batch(cached, [new])
    kv = make_cache(batch, cached, [new], G, d)
    kv.v_scale.copy_(torch.exp2(torch.rand(kv.v_scale.shape, device="cuda") * 40 - 30))
    q = torch.randn(new, H, d, device="cuda").to(BF16) * 0.05
    out = torch.empty(new, H * d, dtype=BF16, device="cuda")
    ops.attention(q, kv, batch, out, H, G, d, d ** -0.5)
    check(out, q, kv, batch, H, G, d, d ** -0.5)


def test_captured_steps_share_nothing():
    """Decode steps of two caches captured in two graphs, replayed in turn with advancing lengths."""
    H, G, d = 32, 8, 128
    sides = []
    for seed, cached in ((1, [900, 40]), (2, [70, 3000, 5])):
        new = [1] * len(cached)
        room = [c + 20 for c in cached]
        batch = make_batch(cached, new)
        kv = make_cache(batch, room, new, G, d, seed=seed)
        batch.max_kv_len = max(room)
        q = torch.randn(len(new), H, d, device="cuda").to(BF16)
        out = torch.empty(len(new), H * d, dtype=BF16, device="cuda")
        ops.attention(q, kv, batch, out, H, G, d, d ** -0.5)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.attention(q, kv, batch, out, H, G, d, d ** -0.5)
        sides.append((batch, kv, q, out, g))
    for _ in range(3):
        for batch, kv, q, out, g in sides:
            batch.lengths += 5
            q.copy_(torch.randn_like(q.float()))
            out.fill_(float("nan"))
            g.replay()
        torch.cuda.synchronize()
        for batch, kv, q, out, g in sides:
            check(out, q, kv, batch, H, G, d, d ** -0.5)


def test_the_whole_step_together():
    """Rotate and append, then attend, as a layer does: prompts first, then single tokens, in one call each and in two."""
    H, G, d = 8, 2, 128
    table = rope(512, d)
    sizes = [200, 5, 66]
    end = [s + 3 for s in sizes]
    batch = make_batch([0] * 3, sizes)
    kv = make_cache(make_batch([0] * 3, end), [0] * 3, end, G, d, fill=False)
    for step in range(4):
        T = batch.n_tokens
        qkv = torch.randn(T, (H + 2 * G) * d, device="cuda").to(BF16)
        out = torch.empty(T, H * d, dtype=BF16, device="cuda")
        ops.rope_append_attention(qkv, None, kv, batch, table, out, H, G, d, "interleaved", True, d ** -0.5)
        q = torch.empty(T, H, d, dtype=BF16, device="cuda")
        ops.rope_append(qkv, q, kv, batch, table, H, G, d)
        ops.check_status(batch.status)
        check(out, q, kv, batch, H, G, d, d ** -0.5)
        ops.advance_lengths(batch)
        batch = make_batch([s + step for s in sizes], [1, 1, 1])


def test_rows_behind_the_last_sequence_stay():
    """Outputs beyond the step's tokens are not touched."""
    H, G, d = 8, 2, 128
    for cached, new in (([100, 20], [1, 1]), ([100, 0], [30, 70])):
        batch = make_batch(cached, new)
        kv = make_cache(batch, cached, new, G, d)
        T = batch.n_tokens
        room = torch.full(((T + 6) * H * d,), 5.0, dtype=BF16, device="cuda")
        ops.attention(torch.randn(T, H, d, device="cuda").to(BF16), kv, batch, room[3 * H * d:(T + 3) * H * d].view(T, H * d), H, G, d, d ** -0.5)
        assert (room[:3 * H * d] == 5).all() and (room[(T + 3) * H * d:] == 5).all()


def test_refusals():
    H, G, d = 4, 2, 64
    batch = make_batch([10], [1])
    kv = make_cache(batch, [10], [1], G, d)
    q, out = torch.randn(1, H, d, device="cuda").to(BF16), torch.empty(1, H * d, dtype=BF16, device="cuda")

    def refused(match, **kw):
        a = dict(q=q, kv=kv, batch=batch, out=out, n_head=H, n_kv=G, head_dim=d, scale=0.125)
        a.update(kw)
        with pytest.raises(ops.KernelError, match=match):
            ops.attention(**a)
    refused("sink", sink=torch.zeros(H, device="cuda"))
    refused("block mask", chunk=64)
    refused("soft cap", softcap=30.0)
    refused("divide", n_kv=3)
    refused("window", window=0)
    refused("attention output", out=out.float())
    refused("shape", q=q[:, :2])
    refused("scales", kv=Int8KV(kv.k_pool, kv.v_pool, kv.page_table, 64))
    refused("scales", kv=Int8KV(kv.k_pool, kv.v_pool, kv.page_table, 64, k_scale=kv.k_scale.double(), v_scale=kv.v_scale))
    refused("pool", kv=Int8KV(kv.k_pool.float(), kv.v_pool, kv.page_table, 64, k_scale=kv.k_scale, v_scale=kv.v_scale))
    refused("pool", kv=Int8KV(kv.k_pool, kv.v_pool, kv.page_table, 32, k_scale=kv.k_scale, v_scale=kv.v_scale))
    refused("page table", kv=Int8KV(kv.k_pool, kv.v_pool, kv.page_table.long(), 64, k_scale=kv.k_scale, v_scale=kv.v_scale))
    refused("float32 or bfloat16", q=q.half(), out=out.half())
    qkv = torch.randn(1, (H + 2 * G) * d, device="cuda").to(BF16)
    for a, kw in (((qkv[:, :-2].contiguous(), q), {}), ((qkv, q.float()), {}), ((qkv, q), dict(partials=torch.zeros(1, 1, qkv.shape[1], device="cuda")))):
        with pytest.raises(ops.KernelError):
            ops.rope_append(a[0], a[1], kv, batch, rope(64, d), H, G, d, **kw)
    with pytest.raises(ops.KernelError, match="rotary table"):
        ops.rope_append(qkv, q, kv, batch, rope(64, 32), H, G, d)
    with pytest.raises(ops.KernelError, match="pairing"):
        ops.rope_append(qkv, q, kv, batch, rope(64, d), H, G, d, pairing="neox")
    from gpt_fast_b200.ops import PagedKV
    with pytest.raises(ops.KernelError, match="8-bit"):
        ops.read_cache(PagedKV(kv.k_pool, kv.v_pool, kv.page_table, 64), batch, q, q)
