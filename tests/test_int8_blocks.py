"""8-bit weights (and, where attention is plain, an 8-bit cache) in every arrangement of a layer, with every norm and both kinds of feed-forward: against the same model
whose products quantise both of their sides."""
import pytest
import torch

import gpt_fast_b200 as gf
from gpt_fast_b200 import ops
from gpt_fast_b200.config.spec import LayerSpec, ModelSpec, PartSpec, ScheduleEntry
from gpt_fast_b200.engine.model import Transformer
import plain_int8
import plain_ops
from conftest import assert_within_bf16_noise

DIM, H, G, D, VOCAB = 128, 4, 2, 64, 97
BACKENDS = [
    pytest.param(("cpu", torch.float32), id="cpu-standin-f32"),
    pytest.param(("cuda", torch.float32), id="cuda-f32", marks=pytest.mark.gpu),
    pytest.param(("cuda", torch.bfloat16), id="cuda-bf16", marks=pytest.mark.gpu),
]


class Quantised(plain_ops.PlainOps):
    """The plain statement with both sides of a layer's products quantised where they are used (and keys and values as they are stored)."""
    def __init__(self, cache):
        super().__init__()
        self.cache = cache

    def linear(self, a, w, out, mode="store", defer=False):
        if w.shape[0] != VOCAB:
            a, w = plain_int8.back(a), plain_int8.back(w)
        return super().linear(a, w, out, mode, defer)

    def rope_append(self, qkv, q_out, kv, batch, table, n_head, n_kv, head_dim, pairing="interleaved", append=True, partials=None):
        super().rope_append(qkv, q_out, kv, batch, table, n_head, n_kv, head_dim, pairing, append, partials)
        if self.cache and append:
            pos, slots = plain_ops.token_positions(batch)
            where = (kv.page_table.long()[slots, pos // kv.page_size], slice(None), pos % kv.page_size)
            for pool in (kv.k_pool, kv.v_pool):
                pool[where] = plain_int8.back(pool[where]).to(pool.dtype)


def norm(kind="rmsnorm", **kw):
    return PartSpec(kind, dict(dict(dim=DIM, eps=1e-5), **kw) if kind != "none" else dict(dim=DIM))


def attention(**kw):
    return PartSpec("attention", dict(dim=DIM, n_head=H, n_kv=G, head_dim=D, **kw))


SWIGLU = PartSpec("swiglu", dict(dim=DIM, hidden=168))


def dense(activation):
    return PartSpec("dense", dict(dim=DIM, hidden=200, activation=activation))


# name: (block, its parts, its constants, residual streams, whether keys and values may be 8-bit integers)
LAYERS = {
    "sandwich": ("sandwich", dict(mixer=attention(), feed_forward=SWIGLU, mixer_norm=norm(), mixer_post_norm=norm(), ffn_norm=norm(), ffn_post_norm=norm()), dict(residual_mult=0.7), 0, True),
    "sandwich without norms ahead": ("sandwich", dict(mixer=attention(window=9), feed_forward=dense("silu"), mixer_norm=norm("none"), mixer_post_norm=norm(one_plus=True), ffn_norm=norm("none"),
                                                      ffn_post_norm=norm(one_plus=True)), {}, 0, True),
    "sandwich of layer norms": ("sandwich", dict(mixer=attention(), feed_forward=dense("gelu"), mixer_norm=norm("layernorm"), mixer_post_norm=norm("layernorm"), ffn_norm=norm("layernorm"),
                                                 ffn_post_norm=norm("layernorm")), {}, 0, True),
    "parallel": ("parallel", dict(mixer=attention(), feed_forward=dense("relu2"), mixer_norm=norm("layernorm", bias=False), ffn_norm=norm("layernorm", bias=False)), dict(layer_scale=True), 0, True),
    "parallel with one norm": ("parallel", dict(mixer=attention(), feed_forward=SWIGLU, mixer_norm=norm()), {}, 0, True),
    "streams": ("streams", dict(mixer=attention(), feed_forward=dense("gelu_tanh"), mixer_norm=norm(), ffn_norm=norm()), dict(streams=3), 3, True),
    "pre-norm, layer norms": ("prenorm", dict(mixer=attention(), feed_forward=dense("relu2"), mixer_norm=norm("layernorm"), ffn_norm=norm("layernorm")), {}, 0, True),
    "pre-norm, 1 + w, layer scale": ("prenorm", dict(mixer=attention(), feed_forward=SWIGLU, mixer_norm=norm(one_plus=True), ffn_norm=norm(one_plus=True)), dict(layer_scale=True), 0, True),
    "pre-norm, gated heads with normed queries": ("prenorm", dict(mixer=attention(gate="head", qk_norm_eps=1e-5), feed_forward=SWIGLU, mixer_norm=norm(), ffn_norm=norm()), {}, 0, False),
    "pre-norm, biases and a convolution": ("prenorm", dict(mixer=attention(conv_taps=3), feed_forward=dense("gelu"), mixer_norm=norm(), ffn_norm=norm()), {}, 0, False),
}


def logits(model, seqs):
    """Whole prompts, then two more tokens of each one by one."""
    with torch.no_grad():
        cache = model.new_cache(max_tokens=len(seqs) * 64)
        st = gf.Stepper(model, cache)
        slots = cache.begin(len(seqs))
        out = [st.step(slots, [s[:-2] for s in seqs], "all").float().cpu()]
        for k in (-2, -1):
            out.append(st.step(slots, [[s[k]] for s in seqs], "all").float().cpu())
        st.check()
    return torch.cat(out)


@pytest.mark.parametrize("cache", [None, "int8"])
@pytest.mark.parametrize("name", list(LAYERS))
@pytest.mark.parametrize("backend", BACKENDS)
def test_every_arrangement(backend, name, cache):
    device, dtype = backend
    block, parts, constants, streams, may_cache = LAYERS[name]
    rope = PartSpec("rope", dict(head_dim=D, base=10000.0))
    layer = LayerSpec(block, parts, rope, constants)
    spec = ModelSpec("toy", DIM, VOCAB, [layer, layer], [ScheduleEntry(0, 0), ScheduleEntry(1, 1)], norm(), max_position=64, streams=streams)
    if cache and not may_cache:
        with pytest.raises(gf.ConfigError, match="8-bit integers"):
            Transformer(spec, dtype, "cpu", "int8", cache)
        return
    g = torch.Generator().manual_seed(3)
    seqs = [torch.randint(0, VOCAB, (n,), generator=g).tolist() for n in (21, 3, 12)]
    P = {}

    def made(dtype, device, *options):
        model = Transformer(spec, dtype, device, *options)
        for i, (key, ps) in enumerate(sorted(model.param_specs().items())):
            if key not in P:
                t = torch.randn(ps.shape, generator=torch.Generator().manual_seed(100 + i)) * 0.05
                P[key] = (1 + t if ps.role == "vector" else t).bfloat16().float()
        model.load_params({k: v.to(dtype if model.param_specs()[k].role == "matrix" else torch.float32).to(device) for k, v in P.items()})
        return model
    prev = ops.use_kernels(plain_ops.PlainOps())
    try:
        want = logits(made(torch.float32, "cpu"), seqs)
        ops.use_kernels(Quantised(cache))
        emu = logits(made(torch.float32, "cpu"), seqs)
        ops.use_kernels(plain_int8.PlainInt8() if device == "cpu" else None)
        got = logits(made(dtype, device, "int8", cache), seqs)
    finally:
        ops.use_kernels(prev)
    assert_within_bf16_noise(got, want, emu, name)
    if device == "cpu":                                      # the same numbers but for the last bits of sums in another order, which move an integer next to a tie
        assert (got - emu).pow(2).mean().sqrt() <= 0.3 * (emu - want).pow(2).mean().sqrt()
