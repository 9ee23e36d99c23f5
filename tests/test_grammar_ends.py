"""Generations whose settings leave a row no token: refused where the settings say so, ended where the logits do."""
import pytest
import torch

from jax_llama_amd import GenerationConfig, LLaMAConfig, LLaMAForCausalLM, TokenGrammar
from jax_llama_amd.runtime import engine

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]
V = 96


@pytest.fixture(autouse=True)
def _no_engines():
    yield
    engine._ENGINES.clear()


def model_of(device):
    cfg = LLaMAConfig(vocab_size=V, hidden_size=256, intermediate_size=256, num_hidden_layers=1, num_attention_heads=2,
                      num_key_value_heads=1, max_sequence_length=64, rms_norm_eps=1e-5)
    return LLaMAForCausalLM(cfg, device=device, _do_init=False).init_random(seed=3, std=0.12)


def table(*rules, states):
    t = torch.full((states, V), -1, dtype=torch.int32)
    for state, token, to in rules:
        t[state, token] = to
    return t


def config(**kw):
    return GenerationConfig(**{**dict(max_length=13, pad_token_id=4, eos_token_id=-1), **kw})


IDS = torch.tensor([[5, 6, 7, 8, 9], [9, 8, 7, 6, 5]], dtype=torch.int32)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("sampled", [False, True])
def test_settings_that_leave_no_token(device, sampled):
    model, kw = model_of(device), dict(do_sample=True, top_k=5) if sampled else {}
    turn = TokenGrammar(table((0, 10, 1), (0, 11, 1), (1, 12, 0), states=2))
    fine = model.generate(IDS, None, config(grammar=turn, **kw)).sequences[:, 5:].tolist()
    for bad in (dict(suppress_tokens=[12]), dict(suppress_tokens=[10, 11]), dict(logit_bias={12: float("-inf")}), dict(suppress_tokens=[0, 12, 13])):
        with pytest.raises(ValueError):
            model.generate(IDS, None, config(grammar=turn, **bad, **kw))
    with pytest.raises(ValueError):
        model.generate(IDS, None, config(suppress_tokens=list(range(V)), **kw))
    # a state that the suppressed tokens keep out of reach may be without one
    rows = model.generate(IDS, None, config(grammar=TokenGrammar(table((0, 10, 1), (0, 11, 2), (1, 12, 0), (2, 13, 0), states=3)), suppress_tokens=[11, 13], **kw)).sequences
    assert rows[:, 5:].tolist() == [[10, 12] * 4] * 2
    rows = model.generate(IDS, None, config(grammar=turn, suppress_tokens=[11, 50], **kw)).sequences
    assert rows[:, 5:].tolist() == [[10, 12] * 4] * 2
    assert model.generate(IDS, None, config(grammar=turn, **kw)).sequences[:, 5:].tolist() == fine
    assert all(t in ((10, 11), (12,))[i % 2] for row in fine for i, t in enumerate(row))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("sampled", [False, True])
def test_rows_that_come_to_a_dead_end_are_padded(device, sampled):
    """In state 1 token 12 alone is allowed, in state 2 token 13. A bias of -3.3e38 on 12 is a number, with 3e38 off for having been said
    it is -inf: the row has no token left and ends; rows in state 2 go on."""
    model, kw = model_of(device), dict(do_sample=True, top_k=5, num_return_sequences=4) if sampled else {}
    rules = table((0, 10, 1), (0, 11, 2), (1, 12, 1), (2, 13, 2), states=3)
    gc = dict(logit_bias={12: -3.3e38}, presence_penalty=3e38, **kw)

    def rows(start):
        return model.generate(IDS, None, config(grammar=TokenGrammar(rules, start), **gc)).sequences[:, 5:].tolist()

    for _ in range(2):
        assert all(r == [12] + [4] * 7 for r in rows(1))
        assert all(r == [13] * 8 for r in rows(2))
        both = rows(0)
        assert all(r in ([10, 12] + [4] * 6, [11] + [13] * 7) for r in both) and (not sampled or len({r[0] for r in both}) == 2)
    # ended rows end the call where there are no others
    assert all(r == [12] + [4] * 7 for r in model.generate(IDS, None, config(grammar=TokenGrammar(rules, 1), eos_token_id=2, **gc)).sequences[:, 5:].tolist())


def test_states_of_a_grammar_with_its_end():
    g = TokenGrammar(table((0, 3, 1), (1, 4, 0), states=2))
    nxt, allowed = g.on("cpu")
    assert nxt.shape == (3, V) and allowed.shape == (2, V // 32)
    assert nxt[0, 3] == 1 and nxt[1, 4] == 0 and int((nxt != 2).sum()) == 2 and bool((g.next_state >= -1).all())


class _Largest(torch.utils._python_dispatch.TorchDispatchMode):
    """The largest tensor that the operations within give back, in bytes."""

    def __init__(self):
        super().__init__()
        self.bytes = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        for t in out if isinstance(out, (tuple, list)) else (out,):
            if torch.is_tensor(t):
                self.bytes = max(self.bytes, t.untyped_storage().nbytes())
        return out


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n,v", [(1, 1), (3, 32), (5, 33), (7, 100), (1200, 32001), (2, 2 ** 21 + 5)])
def test_packed_masks(device, n, v):
    """Against the definition; what it takes on the way stays within 64 MiB or a few times the truth values."""
    from jax_llama_amd import ops
    mask = (torch.rand(n, v, generator=torch.Generator().manual_seed(1)) < 0.3).to(device)
    with _Largest() as most:
        words = ops.pack_allowed(mask)
    assert words.dtype == torch.int32 and words.shape == (n, -(-v // 32))
    assert most.bytes <= max(2 ** 26, 16 * (v + 31))
    at = torch.arange(v, device=device)
    for a in range(0, n, 200):
        assert torch.equal((words[a:a + 200][:, at // 32] >> (at % 32).to(torch.int32)) & 1 == 1, mask[a:a + 200])
    if v % 32:
        assert not bool((words[:, -1] >> (v % 32) & ((1 << (32 - v % 32)) - 1)).any())  # (bits past V)


def test_packed_masks_of_other_types():
    from jax_llama_amd import ops
    mask = torch.tensor([[0, 2, 0, -1], [1, 0, 0, 0]])
    for t in (mask, mask.float(), mask.to(torch.uint8), mask.t().contiguous().t()):
        assert ops.pack_allowed(t).tolist() == [[10], [1]]
    assert ops.pack_allowed(torch.zeros(0, 40)).shape == (0, 2)
    assert ops.pack_allowed(torch.ones(1, 32)).tolist() == [[-1]]
    with pytest.raises(ValueError):
        ops.pack_allowed(torch.zeros(4))
