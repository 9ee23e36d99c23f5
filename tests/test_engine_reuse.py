"""One engine over calls that differ: what a captured step has baked in is that of the present call. CPU here, the captured steps with -m gpu."""
import pytest
import torch

from jax_llama_amd import GenerationConfig, LLaMAConfig, LLaMAForCausalLM
from jax_llama_amd.runtime.engine import DecodeEngine

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]
V = 96


def sizes():
    return LLaMAConfig(vocab_size=V, hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=2,
                       num_key_value_heads=1, max_sequence_length=128, rms_norm_eps=1e-5)


def model_of(device):
    return LLaMAForCausalLM(sizes(), device=device, _do_init=False).init_random(seed=3, std=0.12)


def prompts(b, s, seed=0):
    return torch.randint(3, V, (b, s), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


def config(**kw):
    return GenerationConfig(**{**dict(max_length=26, do_sample=True, temperature=1.5, top_k=20, top_p=0.95, seed=1, pad_token_id=0, eos_token_id=-1), **kw})


@pytest.mark.parametrize("device", DEVICES)
def test_sampling_settings_of_the_present_call(device):
    model, ids = model_of(device), prompts(3, 8)
    kept = DecodeEngine(model, 3, 26)
    seen = []
    for kw in (dict(), dict(seed=2), dict(temperature=0.8), dict(top_p=0.7), dict(top_k=5), dict(top_k=0), dict(top_k=0, temperature=0.9), dict(),
               dict(seed=2 ** 40 + 1), dict(do_sample=False), dict(do_sample=False, seed=7)):
        got = kept.run(ids, None, config(**kw)).cpu().clone()
        assert torch.equal(got, DecodeEngine(model, 3, 26).run(ids, None, config(**kw)).cpu()), kw
        seen.append(tuple(got.reshape(-1).tolist()))
    assert len(set(seen)) == 9  # (the first twice, greedy twice)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("sampled", [False, True])
def test_end_and_pad_tokens_of_the_present_call(device, sampled):
    model, ids = model_of(device), prompts(3, 8)
    kept = DecodeEngine(model, 3, 26)
    free = kept.run(ids, None, config(do_sample=sampled)).cpu().clone()
    for at, pad in ((14, 0), (17, 1), (14, 2)):  # the end tokens: what the first row says late
        gc = config(do_sample=sampled, eos_token_id=int(free[0, at]), pad_token_id=pad)
        got = kept.run(ids, None, gc).cpu().clone()
        first = free[0].tolist().index(gc.eos_token_id, 8)
        assert got[0].tolist() == free[0, :first + 1].tolist() + [pad] * (25 - first)
        assert torch.equal(got, DecodeEngine(model, 3, 26).run(ids, None, gc).cpu())


def test_state_of_a_captured_step():
    """A greedy step does not depend on what is for sampling: it is not captured again."""
    model = model_of("cpu")
    eng = DecodeEngine(model, 2, 20)
    ids = prompts(2, 8)

    def state(**kw):
        eng.prefill_only(ids, None, config(max_length=20, **kw))
        return eng._graph_state()

    base = state()
    for kw in (dict(seed=2), dict(temperature=0.5), dict(top_p=0.5), dict(top_k=4), dict(eos_token_id=5), dict(pad_token_id=3), dict(do_sample=False)):
        assert state(**kw) != base
    assert state() == base
    greedy = state(do_sample=False)
    assert state(do_sample=False, seed=9, temperature=0.1, top_k=1, top_p=0.2) == greedy
    assert state(do_sample=False, eos_token_id=4) != greedy


def holes(b, s, seed):
    mask = (torch.rand(b, s, generator=torch.Generator().manual_seed(seed)) < 0.6).to(torch.int32)
    mask[:, 0] = mask[:, -1] = 1
    mask[:, s // 2] = 0
    return mask


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("penalty", [1.0, 1.4])
def test_masks_with_holes_of_the_present_call(device, penalty):
    model, ids = model_of(device), prompts(4, 12)
    kept = DecodeEngine(model, 4, 40)
    gc = config(max_length=40, do_sample=False, repetition_penalty=penalty)
    seen, places = set(), set()
    for seed in (0, 1, 2, 1):
        got = kept.run(ids, holes(4, 12, seed), gc).cpu().clone()
        places.add(kept.key_mask.data_ptr())
        torch.full((4, 40), 0, dtype=torch.uint8, device=device)  # (memory that an earlier call has given back is used again)
        assert torch.equal(got, DecodeEngine(model, 4, 40).run(ids, holes(4, 12, seed), gc).cpu())
        seen.add(tuple(got.reshape(-1).tolist()))
        assert torch.equal(kept.run(ids, None, gc), DecodeEngine(model, 4, 40).run(ids, None, gc))
    assert len(seen) == 3 and len(places) == 1  # (a captured step holds the mask's address)


@pytest.mark.parametrize("device", DEVICES)
def test_weights_of_the_present_call(device):
    """``generate(params=...)`` and loading again: the engine kept for these sizes runs the weights that the model holds now."""
    from helpers import build
    cfg = sizes()
    trees = [build(cfg, seed=s)[3] for s in (1, 2)]
    ids = torch.randint(3, cfg.vocab_size, (2, 6), generator=torch.Generator().manual_seed(0), dtype=torch.int32)
    gc = GenerationConfig(max_length=24, pad_token_id=0, eos_token_id=-1)
    model = LLaMAForCausalLM(cfg, device=device, _do_init=False)
    kept, seen, states = DecodeEngine(model, 2, 24), [], []
    for i in (0, 1, 0):
        model.load_params(trees[i])
        got = kept.run(ids, None, gc).cpu().clone()
        fresh = LLaMAForCausalLM(cfg, device=device, _do_init=False).load_params(trees[i])
        assert torch.equal(got, DecodeEngine(fresh, 2, 24).run(ids, None, gc).cpu())
        seen.append(tuple(got.reshape(-1).tolist()))
        states.append(kept._graph_state())
    assert len(set(seen)) == 2 and states[0] != states[1] != states[2]


@pytest.mark.parametrize("device", DEVICES)
def test_weights_of_layer_list_models(device):
    import test_besulix
    model, sd = test_besulix.build(test_besulix.cfg_full(), device)
    other = {k: t.flip(0) if k == "embed" else t for k, t in sd.items()}
    ids = torch.randint(3, 37, (2, 6), generator=torch.Generator().manual_seed(0), dtype=torch.int32)
    gc = GenerationConfig(max_length=20, pad_token_id=0, eos_token_id=-1)
    kept, seen = DecodeEngine(model, 2, 20), []
    for weights in (sd, other, sd):
        model.load_state_dict(weights)
        got = kept.run(ids, None, gc).cpu().clone()
        assert torch.equal(got, DecodeEngine(model, 2, 20).run(ids, None, gc).cpu())
        seen.append((tuple(got.reshape(-1).tolist()), kept._graph_state()))
    assert seen[0][0] == seen[2][0] != seen[1][0] and seen[0][1] != seen[1][1] != seen[2][1]


def test_bytes_of_engines_behind_one_prefix(monkeypatch):
    """A prefix counts once, however many engines keep it alive, and as long as one of them does."""
    from jax_llama_amd.runtime import engine
    model = model_of("cpu")
    big, other = model.encode_prefix(prompts(1, 60)), model.encode_prefix(prompts(1, 60, seed=1))

    def call(prefix, b):
        model.generate(prompts(b, 4), None, config(max_length=8), prefix=prefix)

    def kept():
        return [(e.prefix, e.b) for e in engine._ENGINES.values()]

    engine._ENGINES.clear()
    own = model.init_cache(1, 8).nbytes()
    monkeypatch.setattr(engine, "_engine_budget", lambda m: big.nbytes() + 6 * own)
    for b in (1, 2, 3):  # 6 rows of own keys and one prefix
        call(big, b)
    engines = list(engine._ENGINES.values())
    assert kept() == [(big, 1), (big, 2), (big, 3)] and engine._held_bytes(engines) == big.nbytes() + 6 * own
    for b in (1, 2, 3):  # the same engines again
        call(big, b)
    assert list(engine._ENGINES.values()) == engines
    call(big, 4)  # 3 + 4 rows are too many, the prefix stays
    assert kept() == [(big, 4)]
    call(other, 1)  # another prefix does not fit beside it
    assert kept() == [(other, 1)] and engine._held_bytes(engine._ENGINES.values()) == big.nbytes() + own
    engine._ENGINES.clear()
