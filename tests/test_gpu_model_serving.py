"""The models with what a serving program asks for: the LLaMA model over a cache in 8 bits, and sampled tokens in every family."""
import numpy as np
import pytest
import torch

import duponex_cases
import kv8_cases as K
import soluzen_cases

pytestmark = pytest.mark.gpu


def llama(seed=0, kv_cache="bf16", layers=2):
    from baranet_bdml_b200.layers import LLaMAConfig
    from baranet_bdml_b200.model import LLaMAModelBF16
    np.random.seed(seed)
    return LLaMAModelBF16(LLaMAConfig(vocab_size=1000, hidden_size=256, intermediate_size=512, num_hidden_layers=layers, num_attention_heads=4,
                                      num_key_value_heads=2, max_position_embeddings=256), kv_cache=kv_cache)


def family(name):
    if name == "llama":
        return llama(3), 1000
    from baranet_bdml_b200 import registry
    from baranet_bdml_b200.checkpoint import Weights
    cases = {"soluzen": soluzen_cases, "duponex": duponex_cases}[name]
    return registry.build_model(cases.CASES["even"], Weights(cases.weights(cases.CASES["even"], 1)), torch.bfloat16), cases.CASES["even"]["vocab"]


def ids_of(rng, *shape, vocab=1000):
    return torch.from_numpy(rng.integers(3, vocab, shape).astype(np.int32)).cuda()


@pytest.mark.parametrize("values", ["e4m3", "int8"])
@pytest.mark.parametrize("B", [1, 3, 20])
def test_cache_holds_what_the_bf16_cache_holds(lib, values, B):
    """After a prompt and a step the 8-bit cache gives back the bf16 cache's keys and values, each off by its rounding: 2^-4 of the number (or
    half a step of the smallest) and, for what the bf16 cache rounded too, 2^-8; the queries' and keys' own path is the same until
    the first layer's attention reads the cache, so it is the first layer that is compared."""
    rng = np.random.default_rng(B)
    S = 37
    ids, tok = ids_of(rng, B, S), ids_of(rng, B)
    plain, eight = llama(5, layers=1), llama(5, values, layers=1)
    for m in (plain, eight):
        m.prefill(ids, S + 4)
        m.decode_step(tok)
        m.status()
    assert eight.caches[0].values == values and torch.equal(eight.seq_lens, plain.seq_lens) and int(eight.seq_lens[0]) == S + 1
    rows, zero = torch.arange(B, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    got = eight.caches[0].gather(rows, zero, S + 1, dtype=torch.float32)
    pool, table = plain.caches[0].pool, plain.caches[0].page_table.long()
    for i, g in enumerate(got):
        want = pool[table][:, :, :, i].permute(0, 1, 3, 2, 4).reshape(B, -1, 2, 64)[:, :S + 1].double()
        # keys of the step are rotated from bf16 products by angles of another precision: 2^-8 of the pair
        most = want.abs().amax(-1, keepdim=True)
        step = want.abs() * 2.0 ** -4 + most / 448 * 2 * 2.0 ** -10 if values == "e4m3" else most / 127 * 0.5 * (1 + 2.0 ** -7)
        assert ((g.double() - want).abs() <= step + most * 2.0 ** -7).all()


@pytest.mark.parametrize("values", ["e4m3", "int8"])
@pytest.mark.parametrize("B", [2, 20])
def test_steps_over_eight_bits_follow_the_model(lib, values, B):
    """Teacher-forced logits of every position against whole-sequence recomputation.  A score is a sum of 64 products whose keys are off by
    2^-4 (e4m3; 1 / 254 of the largest for int8) at most, at random signs, and values likewise: within 0.1 of the logits' range where
    the bf16 cache's own test allows 0.03."""
    rng = np.random.default_rng(2)
    S, new = 30, 5
    ids = ids_of(rng, B, S + new)
    model = llama(1, values)
    logits = model.prefill(ids[:, :S].contiguous(), S + new)
    for t in range(new + 1):
        full = model(ids[:, :S + t].contiguous())[:, -1]
        assert float((logits - full).abs().max()) <= 0.1 * float(full.abs().max())
        if t < new:
            logits = model.decode_step(ids[:, S + t].contiguous())
    model.status()


@pytest.mark.parametrize("values", ["bf16", "e4m3", "int8"])
def test_captured_steps_equal_eager_ones(lib, values):
    """Bit for bit, sampled tokens included: the warm-up's token in the cache leaves no trace."""
    rng = np.random.default_rng(6)
    ids, toks = ids_of(rng, 3, 30), ids_of(rng, 20, 3)
    u = torch.rand((20, 3), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    how = dict(temperature=0.9, top_k=40, top_p=0.95, min_p=0.01)
    eager, graphed = llama(5, values), llama(5, values)
    eager.prefill(ids, 64)
    want = []
    for t, w in zip(toks, u):
        logits = eager.decode_step(t)
        want.append((logits.clone(), eager.choose(logits, w, **how)))
    graphed.prefill(ids, 64)
    step = graphed.capture_decode_step(**how)
    for t, w, (logits, nxt) in zip(toks, u, want):
        got = step(t, w)
        torch.cuda.synchronize()
        assert torch.equal(got[0], logits) and torch.equal(got[1], nxt)
    with pytest.raises(RuntimeError):
        step(toks[0])
    with pytest.raises(RuntimeError):
        graphed.capture_decode_step()(toks[0], u[0])


def test_knobs_of_a_captured_step_are_read_at_the_replay(lib):
    rng = np.random.default_rng(8)
    model = llama(2)
    model.prefill(ids_of(rng, 4, 20), 64)
    temperature = torch.full((4,), 1.0, device="cuda")
    step = model.capture_decode_step(temperature=temperature)
    tok, u = ids_of(rng, 4), torch.tensor([0.1, 0.4, 0.6, 0.9], device="cuda")
    logits, nxt = step(tok, u)
    assert nxt.tolist() == [K.choose(x, float(w)) for x, w in zip(logits.cpu().numpy(), u)]
    temperature.fill_(0.0)
    logits, nxt = step(tok, u)
    assert torch.equal(nxt, model.argmax(logits))


@pytest.mark.parametrize("name", ["llama", "soluzen", "duponex"])
def test_generate_samples_in_every_family(lib, name):
    """Every generated id is the one that the definition takes from the logits at hand and the seed's random numbers; the same seed, the same
    ids; temperature 0 is the greedy call."""
    model, vocab = family(name)
    rng = np.random.default_rng(4)
    prompt = rng.integers(3, vocab, (2, 12)).astype(np.int32)
    how = dict(temperature=1.3, top_k=50, top_p=0.9, min_p=0.005)
    seen, choose = [], model.choose
    model.choose = lambda logits, uniform=None, **kw: seen.append((logits.clone(), uniform, kw, choose(logits, uniform, **kw))) or seen[-1][-1]
    out = model.generate(prompt, 6, seed=11, **how)
    model.choose = choose
    model.status()
    u = torch.rand((6, 2), generator=torch.Generator(device="cuda").manual_seed(11), device="cuda")
    assert len(seen) == 6
    for n, (logits, uniform, kw, ids) in enumerate(seen):
        assert kw == how and torch.equal(uniform, u[n])
        assert ids.tolist() == [K.choose(x, float(w), **how) for x, w in zip(logits.cpu().numpy(), uniform)]
        for b in range(2):
            if len(out[b]) > 12 + n:
                assert out[b][12 + n] == int(ids[b])
    assert model.generate(prompt, 6, seed=11, **how) == out
    assert model.generate(prompt, 6, temperature=0.0) == model.generate(prompt, 6)
    with pytest.raises(RuntimeError):
        model.generate(prompt, 2, temperature=-1.0)


def test_rows_of_attend_by_itself(lib):
    """The attention layer with an 8-bit cache, its rows worked out by itself, from a position on"""
    from baranet_bdml_b200.kv_cache import QuantizedKVCache
    model = llama(7, layers=1)
    at = model.layers[0].self_attn
    cache = QuantizedKVCache(12, 2, 6, 2, values="int8")
    cache.page_table.copy_(torch.arange(12).view(2, 6))
    cache.seq_lens.fill_(40)
    x = torch.randn((2 * 20, 256), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    out = at.attend(x, 2, 20, 20, True, cache=cache)
    assert torch.equal(out, at.attend(x, 2, 20, 20, True))
    k, v = cache.gather(torch.arange(2, dtype=torch.int32, device="cuda"), torch.full((2,), 20, dtype=torch.int32, device="cuda"), 20, dtype=torch.float32)
    want = (x.double() @ at.v_proj.double().T).view(2, 20, 2, 64)
    assert ((v.double() - want).abs() <= want.abs().amax(-1, keepdim=True) * (0.5 / 127 * (1 + 2.0 ** -7) + 2.0 ** -8)).all()
    want = K.rotated((x.double() @ at.k_proj.double().T).view(40, 2, 64).cpu(), list(range(20, 40)) * 2).view(2, 20, 2, 64)
    assert ((k.double().cpu() - want).abs() <= want.abs().amax(-1, keepdim=True) * (0.5 / 127 * (1 + 2.0 ** -7) + 2.0 ** -7)).all()


def test_refusals(lib):
    model = llama(0, "fp8")
    with pytest.raises(RuntimeError, match="kv_cache"):
        model.prefill(ids_of(np.random.default_rng(0), 1, 5), 8)
    model.kv_cache = "bf16"
    model.prefill(ids_of(np.random.default_rng(0), 1, 5), 8)
    with pytest.raises(RuntimeError, match="random numbers"):
        model.choose(torch.zeros((1, 10), device="cuda"), top_k=3)
