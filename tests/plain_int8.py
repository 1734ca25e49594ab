"""The operations on 8-bit integers, stated plainly in 64 bits: the stand-in `plain_ops` with them, and the dense decoder with 8-bit weights
and an 8-bit cache for whole sequences (no cache, no packing)."""
import torch

import plain_llama
from plain_llama import rounded
from plain_ops import PlainOps, token_positions

F64 = torch.float64


def quantised(x):
    """(integers, scales) of rows: scale = max |x| / 127 in 32 bits, integers nearest to 127 x / max |x|, ties to even."""
    x = x.to(F64)
    most = x.abs().amax(-1)
    q = torch.where(most[..., None] > 0, (x * 127 / most.clamp(min=5e-324)[..., None]).round(), 0.0)
    return q, (most / 127).float()


def back(x):
    q, s = quantised(x)
    return q * s.to(F64)[..., None]


def numbers(r):
    return r.q[:, :r.cols].to(F64) * r.scale.to(F64)[:, None]


class PlainInt8(PlainOps):
    def quantize_rows(self, x, out):
        q, s = quantised(x)
        out.q.zero_()
        out.q[:, :out.cols] = q.to(torch.int8)
        out.scale.copy_(s)

    def rmsnorm_int8(self, x, weight, eps, out, rows=None, pending=None):
        h = torch.empty(out.q.shape[0], out.cols, dtype=F64, device=x.device)
        self.rmsnorm(x, weight, eps, h, rows, pending)
        self.quantize_rows(h.float(), out)

    def linear_int8(self, a, w, out, mode="store"):
        self.linear(numbers(a) if hasattr(a, "q") else back(a), numbers(w), out, mode)

    def rope_append_int8(self, qkv, q_out, kv, batch, table, n_head, n_kv, head_dim, pairing, append):
        class Whole:
            page_table, page_size = kv.page_table, kv.page_size
            k_pool = kv.k_pool.to(F64) * kv.k_scale.to(F64)[..., None]
            v_pool = kv.v_pool.to(F64) * kv.v_scale.to(F64)[..., None]
        self.rope_append(qkv, q_out, Whole, batch, table, n_head, n_kv, head_dim, pairing, append)
        if append:
            pos, slots = token_positions(batch)
            where = (kv.page_table.long()[slots, pos // kv.page_size], slice(None), pos % kv.page_size)
            for pool, ints, scales in ((Whole.k_pool, kv.k_pool, kv.k_scale), (Whole.v_pool, kv.v_pool, kv.v_scale)):
                q, s = quantised(pool[where].float())
                ints[where], scales[where] = q.to(torch.int8), s

    def attention_int8(self, q, kv, batch, out, n_head, n_kv, head_dim, scale, window=None):
        class Whole:
            page_table, page_size = kv.page_table, kv.page_size
            k_pool = kv.k_pool.to(F64) * kv.k_scale.to(F64)[..., None]
            v_pool = kv.v_pool.to(F64) * kv.v_scale.to(F64)[..., None]
        self.attention(q, Whole, batch, out, n_head, n_kv, head_dim, scale, window)


def forward(tokens, p, cfg, act=None, weights=True, cache=True, windows=None):
    """Token ids [S] -> logits [S, V].  `act`: the type in which the library stores activations (None: 64 bits); weights, cache: whether these are
    8-bit; windows: per layer how many latest positions are seen (None: all)."""
    def product(a, w):
        return back(a) @ back(w).T if weights else a @ w.T

    def norm(x, w):
        n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + cfg["norm_eps"]) * w
        return n if weights else rounded(n, act)              # (8-bit rows are made of the norm's 32-bit numbers)

    p = {k: v.to(F64) for k, v in p.items()}
    H, G, d = cfg["n_head"], cfg["n_local_heads"], cfg["head_dim"]
    tokens = torch.as_tensor(tokens, dtype=torch.long)
    S = tokens.shape[0]
    cos, sin = (t.to(F64) for t in plain_llama.rope_angles(torch.arange(S), plain_llama.rope_frequencies(d, cfg["rope_base"], cfg.get("rope_scaling"))))

    def turn(x):
        a, b = x[..., 0::2], x[..., 1::2]
        c, s = cos[:, None], sin[:, None]
        return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)

    x = p["tok_embeddings.weight"][tokens]
    for i in range(cfg["n_layer"]):
        t = f"layers.{i}."
        qkv = rounded(product(norm(x, p[t + "attention_norm.weight"]), p[t + "attention.wqkv.weight"]), act).view(S, H + 2 * G, d)
        q, k, v = rounded(turn(qkv[:, :H]), act), turn(qkv[:, H:H + G]), qkv[:, H + G:]
        k, v = (back(k), back(v)) if cache else (rounded(k, act), v)
        scores = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(H // G, 1)) / d ** 0.5
        n = torch.arange(S)[:, None] - torch.arange(S)[None]
        hidden = n < 0 if not windows or not windows[i] else (n < 0) | (n >= windows[i])
        y = torch.einsum("hqk,khd->qhd", torch.softmax(scores.masked_fill(hidden, float("-inf")), -1), v.repeat_interleave(H // G, 1))
        x = x + product(rounded(y.reshape(S, H * d), act), p[t + "attention.wo.weight"])
        h = norm(x, p[t + "ffn_norm.weight"])
        f = torch.nn.functional.silu(product(h, p[t + "feed_forward.w1.weight"])) * product(h, p[t + "feed_forward.w3.weight"])
        x = x + product(rounded(f, act), p[t + "feed_forward.w2.weight"])
    n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + cfg["norm_eps"]) * p["norm.weight"]
    return (rounded(n, act) @ p["output.weight"].T).float()
