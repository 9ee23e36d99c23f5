"""generate(num_return_sequences=), generate(prefix=) and share_prefix with a model whose choices hang on attention: against whole calls of the
model over prefix, prompt and continuation. CPU here, the kernels with -m gpu."""
import pytest
import torch

from jax_llama_amd import GenerationConfig, LLaMAConfig, LLaMAForCausalLM
from jax_llama_amd.runtime import engine

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]
V = 96
# Two ways through the same model differ by roundings to bf16: some 8 a layer (normed input, q, k, v, weights, result, gate, down), each of
# 2^-9 / sqrt(3) of its number in the mean, so sqrt(16) times that for two layers, twice as much behind the norms that scale what is left of a
# sum up, and sqrt(2) for two ways: 1.3 % of the logits' root mean square. Allowed: 2^-4 of it.
OFF = 2.0 ** -4


@pytest.fixture(autouse=True)
def _no_engines():
    yield
    engine._ENGINES.clear()


def model_of(device):
    """Ordinary random weights, small embeddings: without attention, or with another row's, hardly a token is the same."""
    cfg = LLaMAConfig(vocab_size=V, hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=2,
                      num_key_value_heads=1, max_sequence_length=128, rms_norm_eps=1e-5)
    model = LLaMAForCausalLM(cfg, device=device, _do_init=False).init_random(seed=3, std=0.12)
    model.wte.mul_(0.3)
    return model


def prompts(b, s, seed=0):
    return torch.randint(3, V, (b, s), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


def padded(*pads, s):
    mask = torch.ones(len(pads), s, dtype=torch.int32)
    for i, n in enumerate(pads):
        mask[i, :n] = 0
    return mask


def holes(b, s):
    mask = (torch.rand(b, s, generator=torch.Generator().manual_seed(5)) < 0.6).to(torch.int32)
    mask[:, 0] = mask[:, -1] = 1
    mask[:, s // 2] = 0
    return mask


def config(n_new, s, **kw):
    return GenerationConfig(max_length=s + n_new, pad_token_id=0, eos_token_id=-1, **kw)


def rms(x):
    return float(x.float().square().mean().sqrt())


def likeliest(model, seq, mask, n_new):
    """The last ``n_new`` tokens of ``seq`` are what a whole call finds likeliest, up to what roundings move: two logits are off by 1.3 % of the
    root mean square in the mean, so that a gap of twice that can turn round (the CPU has one of 0.6 % in 500 tokens); allowed: 4 OFF."""
    mask = torch.ones_like(seq) if mask is None else torch.cat([mask, torch.ones(seq.shape[0], seq.shape[1] - mask.shape[1], dtype=mask.dtype)], 1)
    x = model(seq, attention_mask=mask, position_ids=mask.cumsum(-1) - 1).logits[:, -n_new - 1:-1].float().cpu()
    said = seq[:, -n_new:].long()
    short = x.amax(-1) - x.gather(2, said[:, :, None])[:, :, 0]
    assert float(short.max()) <= 4 * OFF * rms(x), short


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["whole", "padded", "holes"])
def test_samples_attend_over_their_prompts(device, kind):
    model, ids = model_of(device), prompts(3, 11)
    mask = dict(whole=None, padded=padded(0, 4, 7, s=11), holes=holes(3, 11))[kind]
    gc = config(14, 11, do_sample=True, top_k=1)
    for _ in range(2):
        got = model.generate(ids, mask, gc, num_return_sequences=2).sequences.cpu()
        assert torch.equal(got[::2], got[1::2]) and torch.equal(got[::2, :11], ids)
        likeliest(model, got, None if mask is None else mask.repeat_interleave(2, 0), 14)
    if device == "cpu":
        gc = config(14, 11, do_sample=True, top_k=8, temperature=0.8, seed=4)
        got = model.generate(ids, mask, gc, num_return_sequences=3).sequences
        assert torch.equal(got, model.generate(ids.repeat_interleave(3, 0), None if mask is None else mask.repeat_interleave(3, 0), gc).sequences)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("g,b,pads", [(1, 4, None), (2, 4, (6, 0)), (3, 3, (0, 5, 2)), (1, 1, None)])
def test_prompts_attend_over_their_prefixes(device, g, b, pads):
    model, head, ids = model_of(device), prompts(g, 13), prompts(b, 6, seed=2)
    hm = None if pads is None else padded(*pads, s=13)
    im = None if pads is None else padded(*[(2 * i) % 5 for i in range(b)], s=6)
    prefix, each = model.encode_prefix(head, hm), b // g
    whole = head.repeat_interleave(each, 0)
    mask = None if pads is None else torch.cat([hm.repeat_interleave(each, 0), im], 1)  # (padding between prefix and prompt)
    for _ in range(2):
        got = model.generate(ids, im, config(14, 6), prefix=prefix).sequences.cpu()
        assert torch.equal(got[:, :6], ids)
        likeliest(model, torch.cat([whole, got], 1), mask, 14)
    sampled = model.generate(ids, im, config(14, 6, do_sample=True, top_k=1), prefix=prefix, num_return_sequences=2).sequences.cpu()
    assert torch.equal(sampled[::2], sampled[1::2])
    likeliest(model, torch.cat([whole, sampled[::2]], 1), mask, 14)


@pytest.mark.parametrize("device", DEVICES)
def test_logits_behind_prefixes_in_portions(device):
    model, head, ids, hm = model_of(device), prompts(2, 20), prompts(4, 10, seed=4), padded(7, 0, s=20)
    shared = model.share_prefix(model.encode_prefix(head, hm), 4, 10)
    first = torch.tensor([13, 13, 20, 20], dtype=torch.int32)[:, None]
    got = torch.cat([model(ids[:, a:z], past_key_values=shared, position_ids=first + torch.arange(a, z, dtype=torch.int32)).logits
                     for a, z in ((0, 7), (7, 8), (8, 10))], 1)
    mask = torch.cat([hm.repeat_interleave(2, 0), torch.ones(4, 10, dtype=torch.int32)], 1)
    want = model(torch.cat([head.repeat_interleave(2, 0), ids], 1), attention_mask=mask, position_ids=mask.cumsum(-1) - 1).logits[:, 20:]
    assert rms(got - want) <= OFF * rms(want)
    # the same with another prefix before them is something else
    other = model.share_prefix(model.encode_prefix(head.flip(0), hm), 4, 10)
    far = model(ids, past_key_values=other, position_ids=first + torch.arange(10, dtype=torch.int32)).logits
    assert rms(far - want) > 4 * OFF * rms(want)
