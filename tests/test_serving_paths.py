"""Several samples per prompt, shared prefixes, penalties, grammars and forked requests through the public calls: equal to the same work
done row by row without sharing. CPU here, the GPU's kernels with -m gpu."""
import pytest
import torch

from jax_llama_amd import GenerationConfig, LLaMA, LLaMAConfig, LLaMAForCausalLM, SequenceStepper, TokenGrammar
from jax_llama_amd.runtime import engine

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]
V = 96


@pytest.fixture(autouse=True)
def _no_engines():
    yield
    engine._ENGINES.clear()


def llama(device, **kw):
    cfg = LLaMAConfig(vocab_size=V, hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=2,
                      num_key_value_heads=1, max_sequence_length=128, rms_norm_eps=1e-5)
    model = LLaMAForCausalLM(cfg, device=device, seed=3, **kw)
    # sharp choices: rows of the head follow the embedding of the token before (equal work in another order must choose equally)
    from jax_llama_amd.models.weights import PackedLinear
    model.lm_head = PackedLinear.from_dense(model.wte.float().roll(1, 0) * 0.2, model.device, fold=model.ln_f)
    return model


def prompts(b, s, seed=0):
    return torch.randint(3, V, (b, s), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


def left_padded(b, s):
    mask = torch.ones(b, s, dtype=torch.int32)
    for i in range(b):
        mask[i, :i % s] = 0
    return mask


def config(n_new, s, **kw):
    return GenerationConfig(max_length=s + n_new, pad_token_id=0, eos_token_id=-1, **kw)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("n", [2, 5])
def test_samples_equal_repeated_prompts(device, padded, n):
    model, ids = llama(device), prompts(3, 11)
    mask = left_padded(3, 11) if padded else None
    gc = config(9, 11, do_sample=True, top_k=8, temperature=0.7, seed=5)
    got = model.generate(ids, mask, gc, num_return_sequences=n).sequences
    want = model.generate(ids.repeat_interleave(n, 0), None if mask is None else mask.repeat_interleave(n, 0), gc).sequences
    assert got.shape == (3 * n, 20) and torch.equal(got, want)
    assert torch.equal(got, model.generate(ids, mask, gc, num_return_sequences=n).sequences)  # (the captured step again)
    other = prompts(3, 11, seed=1)
    got = model.generate(other, None, gc, num_return_sequences=n).sequences
    assert torch.equal(got, model.generate(other.repeat_interleave(n, 0), None, gc).sequences)


@pytest.mark.parametrize("device", DEVICES)
def test_samples_with_holes_in_the_mask(device):
    model, ids = llama(device), prompts(2, 9)
    mask = torch.ones(2, 9, dtype=torch.int32)
    mask[0, 4] = mask[1, 2:5] = 0
    gc = config(7, 9, do_sample=True, top_k=4, temperature=0.5, repetition_penalty=1.3)
    got = model.generate(ids, mask, gc, num_return_sequences=3).sequences
    engine._ENGINES.clear()
    assert torch.equal(got, model.generate(ids.repeat_interleave(3, 0), mask.repeat_interleave(3, 0), gc).sequences)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("g,b,padded", [(1, 4, False), (2, 4, True), (1, 1, False)])
def test_prefix_equals_whole_prompts(device, g, b, padded):
    model, head, ids = llama(device), prompts(g, 13), prompts(b, 6, seed=2)
    hm, im = (left_padded(g, 13).flip(0), left_padded(b, 6)) if padded else (None, None)
    prefix = model.encode_prefix(head, hm)
    each = b // g
    got = model.generate(ids, im, config(8, 6), prefix=prefix).sequences
    whole = torch.cat([head.repeat_interleave(each, 0), ids], 1)
    mask = torch.cat([hm.repeat_interleave(each, 0), im], 1) if padded else None  # (pads in the middle)
    assert torch.equal(got, model.generate(whole, mask, config(8, 19)).sequences[:, 13:])
    gc = config(8, 6, do_sample=True, top_k=5)
    sampled = model.generate(ids, im, gc, prefix=prefix, num_return_sequences=3).sequences
    again = model.generate(ids.repeat_interleave(3, 0), im.repeat_interleave(3, 0) if padded else None, gc, prefix=prefix).sequences
    assert torch.equal(sampled, again)


@pytest.mark.parametrize("device", DEVICES)
def test_prefix_in_model_calls(device):
    """Logits of prompts behind a shared prefix, portion by portion, against whole calls; bf16 keys and values are the same in both."""
    model, head, ids = llama(device), prompts(1, 20), prompts(3, 10, seed=4)
    shared = model.share_prefix(model.encode_prefix(head), 3, 10)
    outs = []
    for a, z in ((0, 7), (7, 8), (8, 10)):
        pos = torch.arange(20 + a, 20 + z, dtype=torch.int32).expand(3, z - a)
        outs.append(model(ids[:, a:z], past_key_values=shared, position_ids=pos).logits)
    want = model(torch.cat([head.expand(3, 20), ids], 1)).logits[:, 20:]
    got = torch.cat(outs, 1)
    # two layers of attention whose bf16 results differ by a step (2^-7 of them) here and there, and what follows from it
    assert float((got - want).abs().max()) <= 2.0 ** -5 * float(want.abs().max())
    assert torch.equal(got.argmax(-1), want.argmax(-1))


@pytest.mark.parametrize("device", DEVICES)
def test_penalties_and_bias(device):
    model, ids = llama(device), prompts(2, 8)
    free = model.generate(ids, None, config(12, 8)).sequences.cpu()
    ban = sorted({int(t) for t in free[:, 8:].reshape(-1)})[:5]
    for kw in (dict(suppress_tokens=ban), dict(logit_bias={t: -1e4 for t in ban})):
        out = model.generate(ids, None, config(12, 8, **kw)).sequences[:, 8:]
        assert not set(out.reshape(-1).tolist()) & set(ban)
    # every token at most once: a penalty larger than all logits
    for kw in (dict(presence_penalty=1e4), dict(frequency_penalty=1e4)):
        out = model.generate(ids, None, config(30, 8, **kw)).sequences[:, 8:]
        assert all(len(set(row)) == 30 for row in out.tolist())
    assert torch.equal(model.generate(ids, None, config(12, 8)).sequences.cpu(), free)
    # against the definition, step by step on whole calls
    gc = config(6, 8, repetition_penalty=1.7, frequency_penalty=0.3)
    got = model.generate(ids, None, gc).sequences.cpu()
    seq = ids.clone()
    for _ in range(6):
        x = model(seq).logits[:, -1].float().cpu()
        for i in range(2):
            for t in set(seq[i].tolist()):
                x[i, t] = x[i, t] * 1.7 if x[i, t] < 0 else x[i, t] / 1.7
                x[i, t] -= 0.3 * seq[i, 8:].tolist().count(t)
        seq = torch.cat([seq, x.argmax(-1, keepdim=True).to(torch.int32)], 1)
    assert torch.equal(got, seq)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("sampled", [False, True])
def test_grammar(device, sampled):
    """Digits, then a separator after two to four of them, twice, then the end token."""
    digits, sep, end = list(range(10, 20)), 30, 2
    n = 12
    table = torch.full((n, V), -1, dtype=torch.int32)
    for part in (0, 5):
        for k in range(4):
            table[part + k, digits] = part + k + 1
            if k >= 2:
                table[part + k, sep] = part + 5
        table[part + 4, sep] = part + 5
    table[10, end] = 11
    table[11, end] = 11
    grammar = TokenGrammar(table)
    model = llama(device)
    kw = dict(do_sample=True, top_k=20, num_return_sequences=3) if sampled else {}
    gc = GenerationConfig(max_length=20, pad_token_id=0, eos_token_id=end, grammar=grammar, **kw)
    for seed in (0, 1):
        for row in model.generate(prompts(4, 5, seed), None, gc).sequences[:, 5:].tolist():
            assert row.count(end) == 1 and set(row[row.index(end) + 1:]) <= {0}
            words = "".join(chr(48 + t - 10) if t in digits else "," for t in row[:row.index(end)]).split(",")
            assert len(words) == 3 and words[2] == "" and all(2 <= len(w) <= 4 and w.isdigit() for w in words[:2])


def test_generation_refusals():
    model, ids = llama("cpu"), prompts(2, 5)
    for kw in (dict(num_return_sequences=2), dict(num_return_sequences=0), dict(suppress_tokens=[V]), dict(logit_bias={-1: 1.0}),
               dict(logit_bias=torch.zeros(V - 1)), dict(grammar=TokenGrammar(torch.zeros(1, V - 1, dtype=torch.int32))), dict(repetition_penalty=0.0)):
        with pytest.raises(ValueError):
            model.generate(ids, None, config(4, 5, **kw))
    for table, start in ((torch.full((1, 4), -1), 0), (torch.full((1, 4), 1), 0), (torch.zeros(1, 4), 0), (torch.zeros(4, dtype=torch.int32), 0),
                         (torch.zeros(1, 4, dtype=torch.int32), 1)):
        with pytest.raises(ValueError):
            TokenGrammar(table, start)
    prefix = model.encode_prefix(prompts(3, 4))
    with pytest.raises(ValueError):
        model.generate(ids, None, config(4, 5), prefix=prefix)
    holes = torch.tensor([[1, 0, 1, 1, 1], [1, 1, 1, 1, 1]])
    with pytest.raises(ValueError):
        model.generate(ids, holes, config(4, 5), prefix=model.encode_prefix(prompts(1, 4)))
    with pytest.raises(ValueError):
        model.encode_prefix(ids, holes)
    with pytest.raises(ValueError):
        model.share_prefix(prefix, 4, 8)
    with pytest.raises(ValueError):
        model.share_prefix(prefix, 3, 256)
    shared = model.share_prefix(prefix, 6, 8)
    with pytest.raises(ValueError):
        shared.copy_rows([0], [2], tokens=1)
    with pytest.raises(ValueError):
        shared.rows(1, 5)


@pytest.mark.parametrize("device", DEVICES)
def test_prefix_prefill_in_chunks(device, monkeypatch):
    model, prefix_ids, ids = llama(device), prompts(2, 9), prompts(6, 5, seed=2)
    prefix = model.encode_prefix(prefix_ids)
    gc = config(6, 5)
    want = model.generate(ids, None, gc, prefix=prefix).sequences
    for tokens in (10, 15, 20, 30):  # rows per chunk: some of one prefix's, all of one's
        engine._ENGINES.clear()
        monkeypatch.setattr(engine, "PREFILL_TOKENS", tokens)
        assert torch.equal(model.generate(ids, None, gc, prefix=prefix).sequences, want)


class _Tokenizer:
    bos_id, eos_id = 1, 2

    def encode(self, x, bos, eos):
        return [1] + [3 + ord(c) % (V - 3) for c in x]

    def decode(self, ids):
        return " ".join(map(str, ids))


def test_prefixes_in_chunks_and_the_bytes_of_engines(monkeypatch):
    """Many prefixes run through the model some rows at a time; a prefix that an engine keeps alive counts towards the engines' bytes."""
    model, head, ids = llama("cpu"), prompts(5, 13), prompts(5, 4, seed=6)
    whole = model.encode_prefix(head, left_padded(5, 13))
    monkeypatch.setattr(engine, "PREFILL_TOKENS", 30)  # 2 rows, 2, 1
    cut = model.encode_prefix(head, left_padded(5, 13))
    assert torch.equal(whole.k, cut.k) and torch.equal(whole.v, cut.v) and torch.equal(whole.start, cut.start) and cut.index == 13
    model.generate(ids, None, config(3, 4), prefix=cut)
    eng, = engine._ENGINES.values()
    assert eng.nbytes() == eng.cache.own.nbytes() + cut.nbytes()
    monkeypatch.setattr(engine, "_engine_budget", lambda m: 3 * eng.nbytes())
    kept = [model.encode_prefix(head) for _ in range(6)]
    for prefix in kept:
        model.generate(ids, None, config(3, 4), prefix=prefix)
    assert [e.prefix for e in engine._ENGINES.values()] == kept[3:]


def test_generator_strings():
    gen = LLaMA(None, llama("cpu"), _Tokenizer())
    out = gen.generate_from_str(["ab", "cde"], 5, num_return_sequences=2, repetition_penalty=1.2)
    assert len(out) == 4
    for i, text in enumerate(out):
        want = _Tokenizer().encode(["ab", "cde"][i // 2], True, False)
        assert [int(t) for t in text.split()][:len(want)] == want and len(text.split()) <= len(want) + 5


# ---------------------------------------------------------------------------------- layer-list families
def family(name, device):
    import test_besulix
    import test_zavevik
    mod = {"besulix": test_besulix, "zavevik": test_zavevik}[name]
    return mod.build(mod.cfg_full(), device)[0]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", ["besulix", "zavevik"])
def test_samples_of_layer_list_models(device, name):
    model = family(name, device)
    ids = torch.randint(3, 37, (2, 9), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    gc = config(10, 9, do_sample=True, top_k=6, temperature=0.2, repetition_penalty=1.1)
    got = model.generate(ids, None, gc, num_return_sequences=4).sequences
    again = model.generate(ids, None, gc, num_return_sequences=4).sequences
    assert torch.equal(got, again)
    assert torch.equal(got, model.generate(ids.repeat_interleave(4, 0), None, gc).sequences)
    with pytest.raises(NotImplementedError):
        from jax_llama_amd.models.kv_cache import KVCache
        model.generate(ids, None, gc, prefix=KVCache(1, 1, 1, 4, 16, "cpu"))


@pytest.mark.parametrize("name", ["besulix", "zavevik"])
def test_samples_of_layer_list_models_refuse_holes(name):
    """As one sample of a prompt with holes in its mask does."""
    model, ids, mask = family(name, "cpu"), torch.randint(3, 37, (2, 9), dtype=torch.int32), torch.ones(2, 9, dtype=torch.int32)
    mask[1, 4] = 0
    for n in (1, 3):
        with pytest.raises(NotImplementedError):
            model.generate(ids, mask, config(4, 9, do_sample=True), num_return_sequences=n)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", ["besulix", "zavevik"])
def test_forked_requests(device, name):
    """A forked request goes on as one that was fed the same tokens, and neither touches the other."""
    model = family(name, device)
    tok = torch.randint(3, 37, (20,), generator=torch.Generator().manual_seed(2)).tolist()
    other = [(t + 7) % 37 for t in tok]
    st = SequenceStepper(model, 24)
    st.feed("a", tok[:9])
    st.fork("a", "b")
    assert st.held("b") == 9
    got_b = st.step([{"id": "b", "tokens": other[9:14], "want": [0, 4]}, {"id": "a", "tokens": tok[9:12], "want": [2]}], fork=[("a", "c")])
    got_c = st.feed("c", tok[9:12], [2])
    st.end("c")
    st.feed("d", other[:5])
    got_a = st.feed("a", tok[12:20], [7])
    want = SequenceStepper(model, 24)
    want.feed("x", tok[:9])
    wb = want.feed("x", other[9:14], [0, 4])
    want.feed("y", tok[:9])
    wc = want.feed("y", tok[9:12], [2])
    wa = want.feed("y", tok[12:20], [7])
    assert torch.equal(got_b[:2], wb) and torch.equal(got_b[2:], wc) and torch.equal(got_c, wc) and torch.equal(got_a, wa)
    for bad in (("z", "q"), ("a", "b")):
        with pytest.raises(ValueError):
            st.fork(*bad)


def test_trace_with_a_fork(tmp_path):
    import json
    import os
    import subprocess
    import sys

    import numpy as np
    import test_zavevik
    model, sd = test_zavevik.build(test_zavevik.cfg_full(), "cpu")
    model.save_pretrained(str(tmp_path / "m"), sd)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    steps = [{"step": 0, "entries": [{"id": "a", "tokens": [5, 17, 3], "want": []}], "end": []},
             {"step": 1, "fork": [["a", "b"]], "entries": [{"id": "a", "tokens": [7], "want": [0]}, {"id": "b", "tokens": [7], "want": [0]}], "end": ["a", "b"]}]
    p = subprocess.run([sys.executable, os.path.join(root, "bin", "trace_run"), "--model", str(tmp_path / "m"), "--dtype", "float32", "--device", "cpu",
                        "--out", str(tmp_path / "o")], input="".join(json.dumps(s) + "\n" for s in steps), capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and p.stdout.splitlines()[-1] == "done 1", p.stderr
    a, b = np.fromfile(tmp_path / "o" / "1.f32", dtype="<f4").reshape(2, -1)
    assert np.array_equal(a, b) and np.isfinite(a).all()
