"""The serving operators' CPU paths against 64-bit oracles, the plans of row copies, and what is refused."""
import random

import pytest
import torch

import oracle_serving as oracle
from jax_llama_amd import ops
from jax_llama_amd.models.kv_cache import HybridCache, KVCache
from jax_llama_amd.ops import serving

BF16, I32 = torch.bfloat16, torch.int32
SPECS = [("kv", 2, 16, 8), ("delta", 3, 2, 8, 8, 4), None, ("latent", 5), ("kv_from", 0), ("mlstm", 3, 4, 5),
         ("multi", ("kv", 1, 8, 8), ("linear", 2, 4, 4)), ("timemix", 2, 4, 4, 7), ("delta", 1, 1, 4, 4, 1)]


def attention_inputs(b, g, s, h, hkv, p, t, d=16):
    return (torch.randn(b, s, h, d).to(BF16) * 2, torch.randn(g, hkv, p, d).to(BF16), torch.randn(g, hkv, p, d).to(BF16),
            torch.randn(b, hkv, t, d).to(BF16), torch.randn(b, hkv, t, d).to(BF16))


@pytest.mark.parametrize("b,g,s,h,hkv,p,t,slot", [(1, 1, 1, 1, 1, 1, 1, 0), (6, 2, 1, 4, 2, 9, 5, 2), (4, 1, 3, 6, 2, 17, 8, 4), (3, 3, 2, 2, 2, 5, 4, 0)])
def test_prefix_attention_cpu(b, g, s, h, hkv, p, t, slot):
    args = attention_inputs(b, g, s, h, hkv, p, t)
    kw = dict(prefix_len=torch.randint(0, p + 1, (g,), dtype=I32), prefix_start=torch.randint(0, 2, (g,), dtype=I32),
              prefix_mask=(torch.rand(g, p) < 0.8).to(torch.uint8), kv_start=torch.randint(0, t, (b,), dtype=I32))
    for given in ({}, kw, {k: kw[k] for k in ("prefix_start", "kv_start")}):
        want, bound = oracle.prefix_attention(*args, slot, **given)
        got = ops.prefix_attention(*args, slot, **given)
        assert got.dtype == BF16 and bool(((got.double() - want).abs() <= bound).all())
        assert torch.equal(got, ops.prefix_attention(*args, torch.tensor([slot], dtype=I32), **given))


def test_prefix_attention_ignores_what_nobody_attends():
    args = attention_inputs(2, 1, 1, 2, 1, 6, 4)
    kw = dict(prefix_len=torch.tensor([4], dtype=I32), prefix_start=torch.tensor([1], dtype=I32))
    clean = ops.prefix_attention(*args, 1, **kw)
    for x, unused in ((args[1], (0, 4, 5)), (args[2], (0, 4, 5)), (args[3], (2, 3)), (args[4], (2, 3))):
        x[:, :, list(unused)] = float("nan")
    assert torch.equal(clean, ops.prefix_attention(*args, 1, **kw))
    none = ops.prefix_attention(*args, 1, prefix_len=torch.zeros(1, dtype=I32), kv_start=torch.tensor([2, 0], dtype=I32))
    assert bool((none[0] == 0).all()) and bool(torch.isfinite(none).all())


def test_prefix_attention_refusals():
    q, kp, vp, ko, vo = attention_inputs(4, 2, 1, 4, 2, 6, 3)
    bad = [dict(q=q[:3]), dict(q=q[:, :, :3]), dict(kp=kp[:, :1]), dict(vp=vp[:, :, :5]), dict(ko=ko[:3]), dict(vo=vo[:, :, :2]), dict(q=q[0]),
           dict(slot=3), dict(slot=-1), dict(kp=kp[:0], vp=vp[:0]), dict(ko=ko[:, :, :0], vo=vo[:, :, :0]), dict(prefix_len=torch.ones(1, dtype=I32)),
           dict(prefix_start=torch.ones(2)), dict(kv_start=torch.ones(2, dtype=I32)), dict(prefix_mask=torch.ones(2, 6)),
           dict(prefix_mask=torch.ones(2, 5, dtype=torch.uint8)), dict(prefix_len=torch.ones(2, 2, dtype=I32)[:, 0])]
    for change in bad:
        a = dict(q=q, kp=kp, vp=vp, ko=ko, vo=vo, slot=0)
        a.update(change)
        kw = {k: a[k] for k in a if k not in ("q", "kp", "vp", "ko", "vo", "slot")}
        with pytest.raises(ValueError):
            ops.prefix_attention(a["q"], a["kp"], a["vp"], a["ko"], a["vo"], a["slot"], **kw)


def logits_inputs(b, v, n, masks):
    tok = torch.randint(0, v + 3, (b, n + 4), dtype=I32) - 1  # (some outside the vocabulary)
    tok[:, ::2] = tok[:, :1]
    return dict(history=tok, length=n, start=torch.randint(0, max(1, n // 3), (b,), dtype=I32), prompt_len=n // 2,
                history_mask=(torch.rand(b, n + 4) < 0.7).to(torch.uint8), repetition_penalty=1 + torch.rand(b), presence_penalty=0.25,
                frequency_penalty=torch.rand(b) * 0.3, bias=torch.randn(v), allowed=torch.rand(masks, v) < 0.4,
                allowed_rows=torch.randint(-1, masks + 1, (b,), dtype=I32))


@pytest.mark.parametrize("b,v,n", [(1, 1, 1), (3, 33, 9), (2, 100, 60), (5, 64, 0)])
def test_process_logits_cpu(b, v, n):
    x, kw = torch.randn(b, v) * 3, logits_inputs(b, v, n, 4)
    want, bound = oracle.process_logits(x, **kw)
    kw["allowed"] = ops.pack_allowed(kw["allowed"])
    got = ops.process_logits(x, **kw)
    assert torch.equal(got == float("-inf"), want == float("-inf"))
    live = want > float("-inf")
    assert bool(((got.double() - want).abs() <= bound)[live].all())
    again = x.clone()
    assert ops.process_logits(again, out=again, **kw) is again and torch.equal(again, got)


def test_process_logits_shard_and_neutral():
    x, kw = torch.randn(3, 40), logits_inputs(3, 40, 12, 1)
    kw.update(allowed=ops.pack_allowed(kw["allowed"]), allowed_rows=None)
    whole = ops.process_logits(x, **kw)
    parts = [ops.process_logits(x[:, a:a + 20], vocab_start=a, **{**kw, "bias": kw["bias"][a:a + 20]}) for a in (0, 20)]
    assert torch.equal(whole, torch.cat(parts, 1))
    assert torch.equal(ops.process_logits(x), x)
    nan = x.clone()
    nan[0, 3] = float("nan")
    mask = torch.ones(1, 40, dtype=torch.bool)
    mask[0, 3] = False
    assert ops.process_logits(nan, allowed=ops.pack_allowed(mask))[0, 3] == float("-inf")


def test_process_logits_refusals():
    x, h = torch.randn(2, 40), torch.zeros(2, 5, dtype=I32)
    words = torch.zeros(3, 2, dtype=I32)
    bad = [dict(repetition_penalty=1.2), dict(repetition_penalty=0.0, history=h, length=1), dict(presence_penalty=float("inf"), history=h, length=1),
           dict(presence_penalty=0.1, history=h), dict(presence_penalty=0.1, history=h, length=6), dict(presence_penalty=0.1, history=h[:1], length=1),
           dict(presence_penalty=0.1, history=h.long(), length=1), dict(frequency_penalty=torch.zeros(3), history=h, length=1),
           dict(presence_penalty=0.1, history=h, length=1, start=torch.zeros(3, dtype=I32)), dict(bias=torch.zeros(39)), dict(bias=torch.zeros(1, 40)),
           dict(bias=torch.zeros(40, dtype=torch.float64)), dict(allowed=words[:, :1]), dict(allowed=words), dict(allowed=words.long()),
           dict(allowed_rows=torch.zeros(2, dtype=I32)), dict(allowed=words[:1], vocab_start=30), dict(vocab_start=-1), dict(out=torch.zeros(2, 41)),
           dict(presence_penalty=0.1, history=h, length=1, history_mask=torch.ones(2, 4, dtype=torch.uint8)), dict(out=torch.zeros(1, 40).expand(2, 40))]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.process_logits(x, **kw)
    with pytest.raises(ValueError):
        ops.process_logits(x.to(BF16))
    both = torch.zeros(81)
    with pytest.raises(ValueError):
        ops.process_logits(both[:80].view(2, 40), out=both[1:].view(2, 40))


# ---------------------------------------------------------------------------------- rows
def walk(rows, steps, chains, in_place):
    """What the kernel's threads do, the chains in any order."""
    old, new = rows, list(rows) if in_place else {}
    order = list(range(len(chains) - 1))
    random.shuffle(order)
    for c in order:
        saved = None
        for k in range(chains[c], chains[c + 1]):
            a, b = steps[2 * k], steps[2 * k + 1]
            source = new if in_place else old
            if b == -2:
                saved = source[a]
            else:
                new[b] = saved if a == -2 else "zero" if a == -1 else source[a]
    return new


@pytest.mark.parametrize("seed", range(60))
def test_row_plans(seed):
    if not serving.ext_available():
        pytest.skip("the extension is not built")
    rng = random.Random(seed)
    n = rng.choice([1, 2, 3, 5, 9, 40])
    kind = seed % 4
    dst = rng.sample(range(n), rng.randint(1, n))
    src = [rng.randint(-1, n - 1) for _ in dst]
    if kind == 1:  # a permutation
        dst, src = list(range(n)), rng.sample(range(n), n)
    if kind == 2:  # every row several times, in place
        dst, src = list(range(n)), [i // 3 for i in range(n)]
    for in_place in (True, False):
        steps, chains = serving.ext().plan_rows(src, dst, in_place)
        got = walk(list(range(n)), steps, chains, in_place)
        for a, b in zip(src, dst):
            assert got[b] == ("zero" if a == -1 else a), (src, dst, steps, chains)
        if in_place:  # the others stay; no chain touches what another one writes
            assert all(got[r] == r for r in range(n) if r not in dst)
            wrote, touched = [], []
            for c in range(len(chains) - 1):
                part = [(steps[2 * k], steps[2 * k + 1]) for k in range(chains[c], chains[c + 1])]
                wrote.append({b for _, b in part if b >= 0})
                touched.append(wrote[-1] | {a for a, _ in part if a >= 0})
            for i, w in enumerate(wrote):
                assert all(not w & t for j, t in enumerate(touched) if j != i)


def cache_tensors(cache):
    if isinstance(cache, KVCache):
        return [(cache.k, 1, 3), (cache.v, 1, 3)]
    return [(t, 0, 2 if has else None) for t, has in cache.row_layout().tensors]


def fill(cache):
    for t, _, _ in cache_tensors(cache):
        t.copy_(torch.randn(t.shape))
    return cache


@pytest.mark.parametrize("make", [lambda n, t: KVCache(3, n, 2, t, 16, "cpu"), lambda n, t: HybridCache(SPECS, n, t, "cpu"),
                                  lambda n, t: HybridCache(SPECS, n, t, "cpu", torch.float32)])
def test_copy_rows_cpu(make):
    for src, dst, tokens in (([0], [1], 3), ([0, 0, 1, 1], [0, 1, 2, 3], 5), ([3, 2, 1, 0], [0, 1, 2, 3], 4), ([-1, 2], [2, 0], 0), ([], [], 2)):
        cache = fill(make(4, 6))
        want = oracle.copied(cache_tensors(cache), src, dst, tokens)
        cache.copy_rows(src, dst, tokens=tokens)
        assert all(torch.equal(t, w) for (t, _, _), w in zip(cache_tensors(cache), want))
    a, b = fill(make(2, 5)), fill(make(3, 7))
    a.index = 4
    want = oracle.copied(cache_tensors(a), [1, 1, 0], [2, 0, 1], 4, cache_tensors(b))
    a.copy_rows([1, 1, 0], [2, 0, 1], to=b)
    assert all(torch.equal(t, w) for (t, _, _), w in zip(cache_tensors(b), want)) and b.index == 0


def test_copy_rows_refusals():
    kv, hy = KVCache(2, 4, 2, 6, 16, "cpu"), HybridCache(SPECS, 4, 6, "cpu")
    for cache in (kv, hy):
        for src, dst, kw in (([0], [4], {}), ([4], [0], {}), ([-2], [0], {}), ([0], [-1], {}), ([0, 1], [2, 2], {}), ([0, 1], [2], {}),
                             ([0], [1], dict(tokens=7)), ([0], [1], dict(tokens=-1))):
            with pytest.raises(ValueError):
                cache.copy_rows(src, dst, **kw)
    with pytest.raises(ValueError):
        kv.copy_rows([0], [1], to=hy)
    with pytest.raises(ValueError):
        kv.copy_rows([0], [1], tokens=1, to=KVCache(2, 4, 3, 6, 16, "cpu"))
    with pytest.raises(ValueError):
        hy.copy_rows([0], [1], tokens=1, to=HybridCache(SPECS[:3], 4, 6, "cpu"))
    with pytest.raises(ValueError):
        kv.copy_rows([0], [1], tokens=5, to=KVCache(2, 4, 2, 4, 16, "cpu"))
    with pytest.raises(ValueError):  # as many bytes, other numbers
        kv.copy_rows([0], [1], tokens=1, to=KVCache(2, 4, 2, 6, 8, "cpu", torch.float32))
