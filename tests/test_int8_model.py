"""Models with 8-bit weights and an 8-bit cache, whole requests, chunks and decode steps, against the dense decoder stated in 64 bits.

Every run is made on the CPU with the plain statement of the kernels standing in (the host-side logic) and, marked gpu, with the kernels."""
import pytest
import torch

import gpt_fast_b200 as gf
from gpt_fast_b200 import ops
from gpt_fast_b200.cache import Cache
from gpt_fast_b200.cache.needs import CacheNeeds, KVNeed
from gpt_fast_b200.engine.step import Stepper
import plain_int8
import plain_llama
from conftest import assert_within_bf16_noise, rms

BASE = dict(model_type="llama", num_hidden_layers=2, vocab_size=193, max_position_embeddings=512, rope_theta=10000.0, rms_norm_eps=1e-5,
            rope_scaling=None, tie_word_embeddings=False, hidden_act="silu")
CONFIGS = {
    "heads of 64": dict(BASE, hidden_size=256, num_attention_heads=4, num_key_value_heads=2, intermediate_size=416),
    "heads of 128": dict(BASE, hidden_size=512, num_attention_heads=4, num_key_value_heads=1, intermediate_size=1000),
    "heads of 36": dict(BASE, hidden_size=108, num_attention_heads=3, num_key_value_heads=3, intermediate_size=200),
}
BACKENDS = [
    pytest.param(("cpu", "float32"), id="cpu-standin-f32"),
    pytest.param(("cuda", "float32"), id="cuda-f32", marks=pytest.mark.gpu),
    pytest.param(("cuda", "bfloat16"), id="cuda-bf16", marks=pytest.mark.gpu),
]


@pytest.fixture(params=BACKENDS)
def backend(request):
    device, dtype = request.param
    prev = ops.use_kernels(plain_int8.PlainInt8()) if device == "cpu" else None
    yield device, dtype
    if device == "cpu":
        ops.use_kernels(prev)


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    out = {}
    for i, (name, cfg) in enumerate(CONFIGS.items()):
        out[name] = str(tmp_path_factory.mktemp(f"int8_{i}"))
        gf.write_model_folder(out[name], cfg, 31 + i, std=0.05)
    return out


def judge(got, want, emu, dtype, where, weights):
    """`want`: the logits without any 8-bit number, `emu`: with them; their difference is the noise of the format on this model, and the run has to be
    as near to `want` as `emu` is (`assert_within_bf16_noise`).  Nearer to `emu` than that it need not be where activations are quantised: a step is
    3 sigma / 127 = 0.024 sigma of a row of size sigma; one integer that a rounding elsewhere moved across a tie changes every output of a product
    over K numbers by 0.024 / sqrt(K) of its size, 0.0015 for K = 256; so 0.0015 / 0.024 = 6 % of the next row's integers move by a step each, an error
    of sqrt(0.06) steps beside the rounding's own 1 / sqrt(12): 0.85 of the noise, drawn anew.  With 2,400 integers per token and 10^-5 of them that
    near to a tie for 32-bit sums, that happens in every request of some tokens.  Behind quantised keys and values no integer is made of a moved one
    in the same layer, and a moved one is one of all the positions seen: a 32-bit run stays within a quarter of the noise."""
    assert_within_bf16_noise(got, want, emu, where)
    if dtype == "float32" and not weights:
        assert rms(got - emu) <= 0.25 * rms(emu - want), f"{where}: {rms(got - emu):.6f} beside a noise of {rms(emu - want):.6f}"


@pytest.mark.parametrize("weights,cache", [("int8", "int8"), ("int8", None), (None, "int8")])
@pytest.mark.parametrize("name", list(CONFIGS))
def test_prompts_chunks_and_decode_steps(backend, folders, name, weights, cache):
    device, dtype = backend
    model = gf.load(folders[name], dtype=dtype, device=device, weight_dtype=weights, cache_dtype=cache)
    p, cfg = plain_llama.load_folder(folders[name])
    windows = [None, 40]
    model.blocks[1].mixer.window = 40                       # the second layer sees the latest 40 positions only
    g = torch.Generator().manual_seed(9)
    reqs = [torch.randint(0, cfg["vocab_size"], (n,), generator=g).tolist() for n in ((70, 3, 12) if device == "cpu" else (230, 3, 131))]
    parts = [(len(r) - 2) * 3 // 5 or 1 for r in reqs]       # a first step, a second one with the rest but two tokens, two decode steps
    kv = model.new_cache(1024, max_seqs=5, max_seq_len=256)
    st = Stepper(model, kv)
    slots = kv.begin(4)[1:]
    for s, r in zip(slots, reqs):
        kv.reserve(s, len(r))
    rows = [[] for _ in reqs]

    def take(logits, counts):
        for i, x in enumerate(logits.float().cpu().split(counts)):
            rows[i].append(x.clone())
    take(st.step(slots, [r[:n] for r, n in zip(reqs, parts)], want="all"), parts)
    rest = [len(r) - 2 - n for r, n in zip(reqs, parts)]
    some = [i for i, n in enumerate(rest) if n]
    out = st.step([slots[i] for i in some], [reqs[i][parts[i]:-2] for i in some], want="all").float().cpu().split([rest[i] for i in some])
    for i, x in zip(some, out):
        rows[i].append(x)
    batch = st.decode_batch(slots)
    for step in (-2, -1):
        batch.tokens.copy_(torch.tensor([r[step] for r in reqs], dtype=torch.int32))
        take(batch.run(), [1] * len(reqs))
    st.check()
    act = torch.bfloat16 if dtype == "bfloat16" else None
    for i, r in enumerate(reqs):
        got = torch.cat(rows[i])
        want = plain_int8.forward(r, p, cfg, weights=False, cache=False, windows=windows)
        emu = plain_int8.forward(r, p, cfg, act=act, weights=bool(weights), cache=bool(cache), windows=windows)
        judge(got, want, emu, dtype, f"{name}, request {i}", weights)


@pytest.mark.gpu
@pytest.mark.parametrize("weights,cache", [(None, "int8"), ("int8", None), ("int8", "int8")])
def test_products_that_are_split_over_their_sums(tmp_path, weights, cache):
    """A layer as wide as an 8B model's: in bfloat16 the products of a few tokens leave partial sums, which the quantising append does not take."""
    cfg = dict(BASE, hidden_size=4096, num_attention_heads=32, num_key_value_heads=8, intermediate_size=2048, num_hidden_layers=1)
    folder = str(tmp_path / "wide")
    gf.write_model_folder(folder, cfg, 5)
    model = gf.load(folder, weight_dtype=weights, cache_dtype=cache)
    p, c = plain_llama.load_folder(folder)
    toks = torch.randint(0, c["vocab_size"], (12,), generator=torch.Generator().manual_seed(4)).tolist()
    kv = model.new_cache(128, max_seqs=2)
    st = Stepper(model, kv)
    slot = kv.begin(1)
    got = [st.step(slot, [toks[:9]], want="all").cpu()]
    kv.reserve(slot[0], 64)
    batch = st.decode_batch(slot)
    for t in toks[9:]:
        batch.tokens.fill_(t)
        got.append(batch.run().cpu().clone())
    st.check()
    emu = plain_int8.forward(toks, p, c, act=torch.bfloat16, weights=bool(weights), cache=bool(cache))
    judge(torch.cat(got), plain_int8.forward(toks, p, c, weights=False, cache=False), emu, "bfloat16", f"{weights} {cache}", weights)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["heads of 64", "heads of 128"])
def test_generation_with_and_without_graphs_and_reading_the_cache(folders, name):
    model = gf.load(folders[name], weight_dtype="int8", cache_dtype="int8")
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 193, (n,), generator=g).tolist() for n in (100, 1, 65, 40, 7)]
    one, _ = gf.generate(model, prompts, 40, batch_size=3, temperature=0.0, use_graph=False)
    two, _ = gf.generate(model, prompts, 40, batch_size=3, temperature=0.0, use_graph=True)
    again, _ = gf.generate(model, prompts, 40, batch_size=3, temperature=0.0, use_graph=True)      # the kept cache and its captured steps
    assert one == two == again
    # the cache holds what a product and a rotation made: read back, its rows are the keys and values that attention takes
    cache = model.new_cache(256, max_seqs=2, max_seq_len=128)
    st = Stepper(model, cache)
    slot = cache.begin(2)[1]
    st.step([slot], [prompts[0]], want="none")
    cfg = CONFIGS[name]
    d, G, T = cfg["hidden_size"] // cfg["num_attention_heads"], cfg["num_key_value_heads"], len(prompts[0])
    dev = model.device
    meta = ops.BatchMeta(torch.tensor([0, T], dtype=torch.int32, device=dev), torch.zeros(T, dtype=torch.int32, device=dev),
                         torch.tensor([slot], dtype=torch.int32, device=dev), torch.zeros_like(cache.lengths), 1, T, T, T, st.status)
    k, v = (torch.empty(T, G, d, dtype=torch.float32, device=dev) for _ in range(2))
    kv = cache.view(0).kv
    ops.read_cache(kv, meta, k, v)
    st.check()
    at = torch.arange(T, device=dev)
    page = kv.page_table.long()[slot, at // 64]
    for got, pool, scale in ((k, kv.k_pool, kv.k_scale), (v, kv.v_pool, kv.v_scale)):
        assert torch.equal(got, pool[page, :, at % 64].float() * scale[page, :, at % 64][..., None])
        assert (got.abs().amax(-1) > 0).all()


def test_bytes(plain_kernels):
    ops.use_kernels(plain_int8.PlainInt8())
    cfg = CONFIGS["heads of 36"]
    plain = gf.load(cfg, dtype="bfloat16", device="cpu", random_weights=True)
    small = gf.load(cfg, dtype="bfloat16", device="cpu", random_weights=True, weight_dtype="int8", cache_dtype="int8")
    D, F, V = 108, 200, 193
    outputs, vectors = 3 * D + D + 2 * F + D, 2 * D
    pitch = lambda n: -(-n // 16) * 16
    assert plain.weight_bytes() == 2 * (V * D + D + 2 * (4 * D * D + 3 * D * F + vectors))
    assert small.weight_bytes() == 2 * (V * D + D + 2 * vectors) + 2 * ((4 * D + 2 * F) * pitch(D) + D * pitch(F) + 4 * outputs)
    assert small.weight_count() == plain.weight_count() == plain.weight_bytes() // 2
    a, b = plain.new_cache(640), small.new_cache(640)
    assert a.kv_bytes_per_token() == 2 * 3 * 2 * 36 * 2 and b.kv_bytes_per_token() == 2 * 3 * 2 * (36 + 4)
    assert a.bytes() == 640 * a.kv_bytes_per_token() and b.bytes() == 640 * b.kv_bytes_per_token()


def test_refusals(plain_kernels, tmp_path):
    ops.use_kernels(plain_int8.PlainInt8())
    cfg = CONFIGS["heads of 36"]
    with pytest.raises(ValueError, match="weight_dtype 'int4'"):
        gf.load(cfg, device="cpu", random_weights=True, weight_dtype="int4")
    with pytest.raises(ValueError, match="cache_dtype 'fp8'"):
        gf.load(cfg, device="cpu", random_weights=True, cache_dtype="fp8")
    with pytest.raises(gf.ConfigError, match="layer 0: the mixer .*8-bit"):
        gf.load("lasezen-tiny-a", device="cpu", random_weights=True, cache_dtype="int8")
    with pytest.raises(gf.ConfigError, match="has no form with 8-bit weights"):
        gf.load("dufizen-tiny-a", device="cpu", random_weights=True, weight_dtype="int8")
    model = gf.load(cfg, device="cpu", random_weights=True, weight_dtype="int8")
    with pytest.raises(ValueError, match="quantised"):
        gf.save_folder(model, tmp_path / "out")
    assert not (tmp_path / "out").exists()
    gf.save_folder(gf.load(cfg, device="cpu", random_weights=True, cache_dtype="int8"), tmp_path / "out")     # (a cache's type is no part of it)
    needs = {0: CacheNeeds(kv=KVNeed(2, 16, None, 8))}
    with pytest.raises(ValueError, match="values of the keys' size"):
        Cache(needs, torch.bfloat16, "cpu", max_tokens=64, kv_dtype="int8")
    with pytest.raises(ValueError, match="'int4'"):
        Cache({}, torch.bfloat16, "cpu", max_tokens=64, kv_dtype="int4")


@pytest.mark.parametrize("owes", ["partial sums", "a scaled branch", "a normed branch"])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_a_norm_writes_8_bit_rows_of_a_stream_that_is_owed_something(owes, device):
    from gpt_fast_b200.parts.norm import RMSNorm
    from gpt_fast_b200.parts.residual import Branch, Residual
    prev = ops.use_kernels(plain_int8.PlainInt8()) if device == "cpu" else None
    try:
        g = torch.Generator().manual_seed(1)
        T, D = 5, 96
        x0, add, w = (torch.randn(s, generator=g).to(device) for s in ((T, D), (T, D), (D,)))
        x = Residual(x0.clone())
        norm = RMSNorm(D, 1e-5, torch.bfloat16)
        norm.load({"weight": w})
        if owes == "partial sums":
            x.pending = torch.stack([add, add]).contiguous()
            total = x0.double() + 2 * add.double()
        else:
            b = Branch(T, D, device)
            b.add(add)
            if owes == "a scaled branch":
                x.add_scaled(b, w)
                total = x0.double() + w.double() * add.double()
            else:
                x.add_normed(b, norm, 0.5)
                a = add.double()
                total = x0.double() + 0.5 * a * torch.rsqrt((a * a).mean(-1, keepdim=True) + 1e-5) * w.double()
        out = norm.forward(x, ops.int8_rows(T, D, device))
        want = total * torch.rsqrt((total * total).mean(-1, keepdim=True) + 1e-5) * w.double()
        step = want.abs().amax(-1, keepdim=True) / 127
        # half a step of the integers, and the 32-bit roundings of the stream and of the norm (a few 2^-24 of the largest number, far below 1/100 step)
        assert ((plain_int8.numbers(out) - want).abs() <= 0.51 * step).all()
    finally:
        if device == "cpu":
            ops.use_kernels(prev)


@pytest.mark.gpu
def test_the_command_line(folders, tmp_path):
    from test_cli_gpu import read_lines, run_cli
    out = tmp_path / "tokens.jsonl"
    args = ["--checkpoint_path", folders["heads of 64"], "--prompt", "5,70", "--max_new_tokens", "9", "--temperature", "0", "--num_samples", "1", "--output", str(out)]
    r = run_cli(*args, "--weight_dtype", "int8", "--cache_dtype", "int8")
    assert r.returncode == 0, r.stderr[-2000:]
    rows = read_lines(out)
    model = gf.load(folders["heads of 64"], weight_dtype="int8", cache_dtype="int8")
    seqs, _ = gf.generate(model, [x["prompt"] for x in rows], 9, temperature=0.0)
    assert [x["prompt"] + x["tokens"] for x in rows] == seqs
    r = run_cli("--random_weights", "--model_name", "dufizen-tiny-a", "--prompt", "5", "--weight_dtype", "int8")
    assert r.returncode == 2 and "8-bit weights" in r.stderr
