"""The operators of 8-bit serving: products of 8-bit integers with a scale per token and per channel, a cache of 8-bit integers, and attention over it.

A case names an `op`:

    linear   y = x W^T with W held as 8-bit integers and a scale per row, x quantised per row on the way; `norm`: x is the 32-bit residual
             stream and a root-mean-square norm precedes; `mode` store, add (into the 32-bit residual) or swiglu (rows of W alternate gate, up)
    append   rotate queries and keys of new tokens, quantise keys and values per (token, head) into the paged cache, and read them back
    attend   causal attention of new tokens over such a cache: one token per sequence (a decode step) or runs of them (prompts, and chunks
             behind a cached context), with or without a window

Quantising a row x: scale = max |x| / 127, integers nearest to 127 x / max |x|, ties to even.
"""
import math

import torch

own = False

PAGE = 64
EPS = 1e-5
F32, F64 = torch.float32, torch.float64


def listed():
    return [
        # one token of one chat at the 8B size, norm and q/k/v projection: the smallest product of a decode step, launches and 25 MB of weights
        dict(name="linear-qkv-decode-1", op="linear", rows=1, k=4096, n=6144, mode="store", norm=True, dtype="bfloat16"),
        # gate/up of eight chats: the largest product of a decode step, one pass over 117 MB of weights
        dict(name="linear-gate-up-decode-8", op="linear", rows=8, k=4096, n=28672, mode="swiglu", norm=True, dtype="bfloat16"),
        # the down projection of a few packed short prompts, an odd number of rows, added to the residual
        dict(name="linear-down-packed-333", op="linear", rows=333, k=14336, n=4096, mode="add", norm=False, dtype="bfloat16"),
        # gate/up of a long prompt: the tensor cores' case
        dict(name="linear-gate-up-prefill-8192", op="linear", rows=8192, k=4096, n=28672, mode="swiglu", norm=False, dtype="bfloat16"),
        # 32-bit activations at sizes that fill no tile
        dict(name="linear-float32-ragged", op="linear", rows=61, k=1001, n=515, mode="store", norm=False, dtype="float32"),
        # a decode step of a served batch: one token for each of 64 sequences
        dict(name="append-decode-64", op="append", seqs=64, new_lo=1, new_hi=1, ctx_lo=100, ctx_hi=4000, heads=32, kv_heads=8, dim=128, pairing="interleaved", dtype="bfloat16"),
        # sixteen packed prompts of unequal length
        dict(name="append-packed-16", op="append", seqs=16, new_lo=31, new_hi=1025, ctx_lo=0, ctx_hi=0, heads=32, kv_heads=8, dim=128, pairing="half", dtype="bfloat16"),
        # one chat, one token: latency
        dict(name="attend-decode-1", op="attend", seqs=1, new_lo=1, new_hi=1, ctx_lo=911, ctx_hi=911, heads=32, kv_heads=8, dim=128, window=0, dtype="bfloat16"),
        # a served batch of unequal chats: the cache is what a step reads
        dict(name="attend-decode-64", op="attend", seqs=64, new_lo=1, new_hi=1, ctx_lo=501, ctx_hi=8190, heads=32, kv_heads=8, dim=128, window=0, dtype="bfloat16"),
        # two very long documents: few rows, long axis
        dict(name="attend-decode-long-2", op="attend", seqs=2, new_lo=1, new_hi=1, ctx_lo=99001, ctx_hi=100003, heads=24, kv_heads=8, dim=128, window=0, dtype="bfloat16"),
        # the next chunk of a long prompt behind its cached part
        dict(name="attend-chunk-512", op="attend", seqs=1, new_lo=512, new_hi=512, ctx_lo=32001, ctx_hi=32001, heads=32, kv_heads=8, dim=128, window=0, dtype="bfloat16"),
        # packed prompts of unequal length at a size with a key head per query head, some of them continued
        dict(name="attend-packed-12", op="attend", seqs=12, new_lo=17, new_hi=901, ctx_lo=0, ctx_hi=130, heads=32, kv_heads=32, dim=128, window=0, dtype="bfloat16"),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "append", "attend", "attend", "attend"])
    dtype = "float32" if rng.random() < 0.15 else "bfloat16"
    if op == "linear":
        wide = dtype == "float32"
        c = dict(op=op, rows=_between(rng, 1, 300 if wide else 8192), k=_between(rng, 64, 2048 if wide else 14336), n=_between(rng, 64, 2048 if wide else 28672),
                 mode=rng.choice(["store", "store", "add", "swiglu"]), norm=not wide and rng.random() < 0.4, dtype=dtype)
        if rng.random() < 0.7:                      # most models' sizes are multiples of 64; any other is allowed
            c["k"], c["n"] = -(-c["k"] // 64) * 64, -(-c["n"] // 64) * 64
        if c["mode"] == "swiglu":
            c["n"] += c["n"] % 2
        if c["mode"] == "add":
            c["norm"] = False                       # a norm is ahead of the products that store
        while c["rows"] * c["k"] * c["n"] > 8192 * 4096 * 28672:
            c["rows"] = c["rows"] * 2 // 3
        return c
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (24, 8), (32, 32), (40, 40), (8, 4), (12, 3)])
    c = dict(op=op, heads=heads, kv_heads=kv_heads, dim=rng.choice([128, 128, 128, 64]), dtype=dtype)
    if dtype == "float32":
        c["dim"] = rng.choice([128, 64, 48, 36])
    new = rng.random() < 0.5
    c["seqs"] = _between(rng, 1, 64) if not new else _between(rng, 1, 16)
    c["new_hi"] = 1 if not new else _between(rng, 2, (512 if dtype == "float32" else 4096) // c["seqs"] + 2)
    c["new_lo"] = _between(rng, 1, c["new_hi"])
    most = (1 << 15 if dtype == "float32" else 1 << 18) // c["seqs"]
    c["ctx_hi"] = _between(rng, 1, most if not new else min(most, 40000))
    c["ctx_lo"] = 0 if rng.random() < 0.3 else _between(rng, 1, c["ctx_hi"])
    if op == "append":
        c["pairing"] = rng.choice(["interleaved", "half"])
        return c
    c["window"] = rng.choice([0, 0, 0, 100, 1000])
    while c["seqs"] * heads * c["new_hi"] * (c["ctx_hi"] + c["new_hi"]) > 560e6:     # scores of the plain form: 2.3 GB
        c["ctx_hi"] = c["ctx_hi"] * 3 // 4
        c["new_hi"] = max(1, c["new_hi"] * 9 // 10)
        c["ctx_lo"], c["new_lo"] = min(c["ctx_lo"], c["ctx_hi"]), min(c["new_lo"], c["new_hi"])
    return c


# ---- the numbers of a case -------------------------------------------------------------------------------

def _spread(lo, hi, n):
    """n lengths from lo to hi, unsorted."""
    v = [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]
    return v[1::2] + v[0::2]


def lengths(case):
    """(cached tokens, new tokens) per sequence."""
    return _spread(case["ctx_lo"], case["ctx_hi"], case["seqs"]), _spread(case["new_lo"], case["new_hi"], case["seqs"])


def _dtype(case):
    return F32 if case["dtype"] == "float32" else torch.bfloat16


def _normal(g, shape, std=1.0, dtype=F32):
    t = torch.empty(shape, dtype=F32, device="cuda").normal_(generator=g)
    return (t if std == 1.0 else t.mul_(std)).to(dtype)


def _int8(x):
    """(integers, scales) of the rows of x: weights and cached rows as a program holds them."""
    most = x.abs().amax(-1)
    return (x * (127.0 / most).unsqueeze(-1)).round_().to(torch.int8), most / 127.0


def _i32(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) + 1)
    dt = _dtype(case)
    if case["op"] == "linear":
        M, K, N = case["rows"], case["k"], case["n"]
        x = _normal(g, (M, K))
        # a few columns of a language model's activations are far larger than the rest
        x[:, torch.randint(0, K, (max(1, K // 500),), device="cuda", generator=g)] *= 12.0
        wq, ws = _int8(_normal(g, (N, K), K ** -0.5))
        if K % 16:
            wq = torch.nn.functional.pad(wq, (0, -K % 16))          # rows of whole 16 bytes
        s = dict(case=case, x=x if case["norm"] else x.to(dt), wq=wq.contiguous(), ws=ws)
        if case["norm"]:
            s["norm"] = (1.0 + _normal(g, (K,), 0.1)).to(dt)
        if case["mode"] == "add":
            s["residual"] = _normal(g, (M, N))
        return s
    H, G, d = case["heads"], case["kv_heads"], case["dim"]
    ctx, new = lengths(case)
    n, T = len(new), sum(new)
    need = [-(-(a + b) // PAGE) for a, b in zip(ctx, new)]
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(int(seed)))
    seq = torch.repeat_interleave(torch.arange(n), torch.tensor(need))
    first = torch.tensor([0] + need[:-1]).cumsum(0)
    table = torch.full((n, max(need)), -1, dtype=torch.int32)
    table[seq, torch.arange(sum(need)) - first[seq]] = order.to(torch.int32)
    cu = [0]
    for q in new:
        cu.append(cu[-1] + q)
    tok_seq = torch.repeat_interleave(torch.arange(n), torch.tensor(new)).to(torch.int32).cuda()
    s = dict(case=case, table=table.cuda(), cu=_i32(cu), tok_seq=tok_seq, slots=_i32(list(range(n))), ctx=_i32(ctx), n=n, tokens=T, longest_new=max(new),
             longest=max(a + b for a, b in zip(ctx, new)), status=torch.zeros(4, dtype=torch.int32, device="cuda"))
    pool = (sum(need), G, PAGE, d)
    if case["op"] == "append":
        s["qkv"] = _normal(g, (T, (H + 2 * G) * d), dtype=dt)
        freq = 500000.0 ** (-torch.arange(0, d, 2, dtype=F64, device="cuda") / d)
        angle = torch.arange(s["longest"], dtype=F64, device="cuda")[:, None] * freq
        s["rope"] = torch.stack([angle.cos(), angle.sin()], -1).to(F32).contiguous()
        s["k_pool"], s["v_pool"] = (torch.zeros(pool, dtype=torch.int8, device="cuda") for _ in range(2))
        s["k_scale"], s["v_scale"] = (torch.zeros(pool[:3], device="cuda") for _ in range(2))
        return s
    s["q"] = _normal(g, (T, H, d), 2.0, dt)
    s["k_pool"], s["k_scale"] = _int8(_normal(g, pool))
    s["v_pool"], s["v_scale"] = _int8(_normal(g, pool))
    return s


# ---- one pass ------------------------------------------------------------------------------------------------

def run(s):
    return (_own if own else _plain)(s)


def _own(s):
    from gpt_fast_b200 import ops

    c = s["case"]
    dt = _dtype(c)
    if c["op"] == "linear":
        x, M = s["x"], c["rows"]
        w = ops.Int8Rows(s["wq"], s["ws"], c["k"])
        if c["norm"]:
            h = ops.int8_rows(M, c["k"], x.device)
            ops.rmsnorm(x, s["norm"], EPS, h)
            x = h
        if c["mode"] == "add":
            out = s["residual"].clone()
        else:
            out = torch.empty(M, c["n"] // 2 if c["mode"] == "swiglu" else c["n"], dtype=dt, device="cuda")
        ops.linear(x, w, out, mode=c["mode"])
        return out
    H, G, d = c["heads"], c["kv_heads"], c["dim"]
    batch = ops.BatchMeta(s["cu"], s["tok_seq"], s["slots"], s["ctx"], s["n"], s["tokens"], s["longest_new"], s["longest"], s["status"])
    kv = ops.Int8KV(s["k_pool"], s["v_pool"], s["table"], PAGE, k_scale=s["k_scale"], v_scale=s["v_scale"])
    if c["op"] == "append":
        q = torch.empty(s["tokens"], H, d, dtype=dt, device="cuda")
        ops.rope_append(s["qkv"], q, kv, batch, s["rope"], H, G, d, c["pairing"])
        k, v = (torch.empty(s["tokens"], G, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        ops.read_cache(kv, batch, k, v)
        return {"q": q, "k": k, "v": v}
    out = torch.empty(s["tokens"], H * d, dtype=dt, device="cuda")
    ops.attention(s["q"], kv, batch, out, H, G, d, d ** -0.5, c["window"] or None)
    return out


def _quantised(x):
    """(integers as 32-bit numbers, scales) of the rows of x; the integers are decided in 64 bits."""
    most = x.abs().amax(-1, keepdim=True)
    q = torch.where(most > 0, (x.to(F64) * 127.0 / most.to(F64)).round(), 0.0)
    return q.to(F32), most / 127.0


def _plain(s):
    c = s["case"]
    dt = _dtype(c)
    if c["op"] == "linear":
        x = s["x"].to(F32)
        if c["norm"]:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["norm"].to(F32)
        q, scale = _quantised(x)
        y = (q @ s["wq"][:, :c["k"]].to(F32).t()) * scale * s["ws"]
        if c["mode"] == "add":
            return s["residual"] + y
        if c["mode"] == "swiglu":
            y = y[:, 0::2] / (1.0 + torch.exp(-y[:, 0::2])) * y[:, 1::2]
        return y.to(dt)
    H, G, d = c["heads"], c["kv_heads"], c["dim"]
    T, seq = s["tokens"], s["tok_seq"].long()
    pos = s["ctx"][seq].long() + torch.arange(T, device="cuda") - s["cu"][seq].long()
    if c["op"] == "append":
        x = s["qkv"].to(F32).view(T, H + 2 * G, d)
        cos, sin = s["rope"][pos].unbind(-1)
        cos, sin = cos[:, None], sin[:, None]
        half = c["pairing"] == "half"
        qk = x[:, :H + G]
        a, b = (qk[..., :d // 2], qk[..., d // 2:]) if half else (qk[..., 0::2], qk[..., 1::2])
        a, b = a * cos - b * sin, b * cos + a * sin
        qk = torch.cat([a, b], -1) if half else torch.stack([a, b], -1).flatten(-2)
        kq, ks = _quantised(qk[:, H:])
        vq, vs = _quantised(x[:, H + G:])
        return {"q": qk[:, :H].to(dt), "k": (kq * ks).to(torch.bfloat16), "v": (vq * vs).to(torch.bfloat16)}
    # every sequence's keys and values side by side, padded to the longest; every sequence's queries likewise
    page = s["table"].clamp(min=0).long()
    n, L, R = s["n"], page.shape[1] * PAGE, H // G
    k = (s["k_pool"][page].to(F32) * s["k_scale"][page].unsqueeze(-1)).transpose(1, 2).reshape(n, G, L, d)
    v = (s["v_pool"][page].to(F32) * s["v_scale"][page].unsqueeze(-1)).transpose(1, 2).reshape(n, G, L, d)
    Q = s["longest_new"]
    at = torch.arange(Q, device="cuda")
    rows = (s["cu"][:-1, None].long() + at).clamp(max=T - 1)                            # [n, Q]
    q = s["q"].to(F32)[rows].view(n, Q, G, R, d).permute(0, 2, 3, 1, 4).reshape(n, G, R * Q, d)
    scores = (q @ k.transpose(-1, -2)).mul_(d ** -0.5).view(n, G, R, Q, L)
    key, mine = torch.arange(L, device="cuda"), (s["ctx"][:, None].long() + at)[..., None]  # [L], [n, Q, 1]
    hidden = key > mine
    if c["window"]:
        hidden |= key <= mine - c["window"]
    scores.masked_fill_(hidden[:, None, None], float("-inf"))
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.view(n, G, R * Q, L) @ v).view(n, G, R, Q, d) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(n, Q, H * d)
    return out[seq, torch.arange(T, device="cuda") - s["cu"][seq].long()].to(dt)


# ---- what a pass cannot do without ---------------------------------------------------------------------------

def work(case):
    es = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "linear":
        M, K, N = case["rows"], case["k"], case["n"]
        out = M * (N // 2) * es if case["mode"] == "swiglu" else 8 * M * N if case["mode"] == "add" else M * N * es
        return {"bytes": M * K * (4 if case["norm"] else es) + N * (K + 4) + (K * es if case["norm"] else 0) + out, "flops": 2.0 * M * N * K}
    H, G, d = case["heads"], case["kv_heads"], case["dim"]
    ctx, new = lengths(case)
    T = sum(new)
    if case["op"] == "append":
        # in; queries out; cached rows written; rows read back written
        return {"bytes": T * (H + 2 * G) * d * es + T * H * d * es + T * 2 * G * (d + 4) + T * 2 * G * d * 2 + 4 * T * d, "flops": 6.0 * T * (H + G) * d}
    w = case["window"] or (1 << 60)
    seen = sum(b + a if a + b <= w else min(a + b, w + b - 1) for a, b in zip(ctx, new))
    # keys that the i-th of b new tokens behind a cached ones sees: min(a + i + 1, w)
    full = [min(b, max(0, w - a)) for a, b in zip(ctx, new)]           # how many of them see everything ahead of them
    pairs = sum(f * a + f * (f + 1) // 2 + (b - f) * min(w, a + b) for a, b, f in zip(ctx, new, full))
    return {"bytes": 2 * T * H * d * es + seen * 2 * G * (d + 4), "flops": 4.0 * H * d * pairs}


# ---- the definition, in 64 bits ----------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        x = s["x"].double()
        if case["norm"]:
            x = x / (x.pow(2).sum(1, keepdim=True) / case["k"] + EPS).sqrt() * s["norm"].double()
        top = x.abs().max(1).values
        step = top / 127
        units = torch.zeros_like(x)
        live = top > 0
        units[live] = torch.round(x[live] * 127 / top[live, None])
        w = s["wq"].double()[:, :case["k"]] * s["ws"].double()[:, None]
        y = torch.mm(units * step[:, None], w.t())
        if case["mode"] == "swiglu":
            gate, up = y[:, ::2], y[:, 1::2]
            return gate * torch.sigmoid(gate) * up
        return y + s["residual"].double() if case["mode"] == "add" else y
    H, G, d = case["heads"], case["kv_heads"], case["dim"]
    ctx, new = lengths(case)
    cu = s["cu"].tolist()
    if case["op"] == "append":
        where = torch.cat([torch.arange(a, a + b) for a, b in zip(ctx, new)]).cuda()
        turn = torch.view_as_complex(s["rope"].double())[where][:, None]
        row = s["qkv"].double().view(-1, H + 2 * G, d)
        turned = row[:, :H + G]
        if case["pairing"] == "half":
            z = torch.complex(turned[..., :d // 2], turned[..., d // 2:]) * turn
            turned = torch.cat([z.real, z.imag], 2)
        else:
            z = torch.view_as_complex(turned.reshape(len(where), H + G, d // 2, 2).contiguous()) * turn
            turned = torch.view_as_real(z).flatten(2)
        held = []
        for part in (turned[:, H:], row[:, H + G:]):
            step = part.abs().max(2, keepdim=True).values / 127
            held.append(torch.round(part / step.clamp(min=1e-300)) * step)
        return {"q": turned[:, :H], "k": held[0], "v": held[1]}
    out = torch.empty(s["tokens"], H, d, dtype=F64, device="cuda")
    for i, (a, b) in enumerate(zip(ctx, new)):
        own_pages = s["table"][i, :-(-(a + b) // PAGE)].long()
        lo = max(0, a - case["window"] + 1) if case["window"] else 0
        far = torch.arange(a, a + b, device="cuda")[:, None] - torch.arange(lo, a + b, device="cuda")
        blind = (far < 0) | (far >= case["window"]) if case["window"] else far < 0
        for g in range(G):
            key = (s["k_pool"][own_pages, g].double() * s["k_scale"][own_pages, g, :, None].double()).reshape(-1, d)[lo:a + b]
            val = (s["v_pool"][own_pages, g].double() * s["v_scale"][own_pages, g, :, None].double()).reshape(-1, d)[lo:a + b]
            heads = s["q"][cu[i]:cu[i + 1], g * (H // G):(g + 1) * (H // G)].double()
            weight = torch.einsum("thd,jd->htj", heads, key) / math.sqrt(d)
            weight = torch.softmax(weight.masked_fill(blind, -math.inf), 2)
            out[cu[i]:cu[i + 1], g * (H // G):(g + 1) * (H // G)] = torch.einsum("htj,jd->thd", weight, val)
    return out.flatten(1)
