"""Samples without top-k, or with more than the device sampler's 64, follow the distribution they are drawn from."""
import types

import pytest
import torch

from jax_llama_amd import GenerationConfig, LLaMAConfig, LLaMAForCausalLM
from jax_llama_amd.parallel.comm import NO_COMM
from jax_llama_amd.runtime import engine

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("top_k,top_p,temperature", [(0, 1.0, 1.0), (0, 0.8, 1.0), (70, 1.0, 0.5), (70, 0.9, 2.0)])
def test_frequencies(device, top_k, top_p, temperature):
    """40000 rows of one distribution: a token's count is off by five standard deviations at most."""
    rows, v = 40000, 90
    x = torch.full((v,), -3.0)
    x[torch.tensor([5, 17, 40, 71, 88])] = torch.tensor([1.0, 3.0, 2.0, 2.5, 0.0])
    model = types.SimpleNamespace(comm=NO_COMM, gather_logits=lambda t: t)
    gc = GenerationConfig(do_sample=True, top_k=top_k, top_p=top_p, temperature=temperature)
    gen = torch.Generator(device=device).manual_seed(1)
    got = engine._sample(model, x.to(device).expand(rows, v), gc, gen).cpu().long()
    p, order = torch.softmax(x.double() / temperature, 0).sort(descending=True, stable=True)
    p = p[:top_k or v] / p[:top_k or v].sum()
    p = torch.where(p.cumsum(0) - p < top_p, p, 0.0)
    want = torch.zeros(v, dtype=torch.float64)
    want[order[:len(p)]] = p / p.sum()
    count = torch.bincount(got, minlength=v).double()
    ties = [t for t in range(v) if x[t] == -3.0]  # (which of them top-k and top-p keep is the sort's choice)
    lone = [t for t in range(v) if x[t] > -3.0]
    for c, w in [*((count[t], want[t]) for t in lone), (count[ties].sum(), want[ties].sum())]:
        assert abs(float(c) - rows * float(w)) <= 5 * (rows * float(w) * (1 - float(w))) ** 0.5 + 1e-9, (float(c), rows * float(w))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("top_k", [0, 80])
def test_samples_of_one_prompt_differ(device, top_k):
    cfg = LLaMAConfig(vocab_size=96, hidden_size=256, intermediate_size=256, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=1,
                      max_sequence_length=64, rms_norm_eps=1e-5)
    model = LLaMAForCausalLM(cfg, device=device, _do_init=False).init_random(seed=3, std=0.05)
    gc = GenerationConfig(max_length=20, do_sample=True, top_k=top_k, pad_token_id=0, eos_token_id=-1)
    rows = model.generate(torch.tensor([[5, 6, 7]], dtype=torch.int32), None, gc, num_return_sequences=6).sequences.tolist()
    assert len({tuple(r) for r in rows}) == 6
    engine._ENGINES.clear()
