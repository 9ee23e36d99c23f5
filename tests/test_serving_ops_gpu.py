"""The serving kernels against 64-bit oracles (tests/oracle_serving.py), at the sizes and masks where they can go wrong, captured into
graphs, on other streams and strides, and together as a batch of samples uses them."""
import pytest
import torch

import oracle_serving as oracle
from jax_llama_amd import ops
from jax_llama_amd.models.kv_cache import HybridCache, KVCache
from jax_llama_amd.ops import serving
from test_serving_ops import SPECS, cache_tensors

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, I32 = torch.bfloat16, torch.int32


def dev(kw):
    return {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in kw.items()}


def inputs(b, g, s, h, hkv, p, t, unused=float("nan"), slot=0):
    """Places past the queries' own slots hold ``unused``."""
    d = 128
    q, kp, vp, ko, vo = (torch.randn(*n).to(BF16) for n in ((b, s, h, d), (g, hkv, p, d), (g, hkv, p, d), (b, hkv, t, d), (b, hkv, t, d)))
    ko[:, :, slot + s:] = unused
    vo[:, :, slot + s:] = unused
    return q * 2, kp, vp, ko, vo


def close(got, want, bound):
    err = (got.double().cpu() - want).abs()
    assert bool((err <= bound).all()), f"largest excess {float((err - bound).max()):.3e}, largest error {float(err.max()):.3e}"


SHAPES = [  # and the way they go (csrc/serving/prefix_attn.hip prefix_attn_plan)
    (1, 1, 1, 1, 1, 1, 1, 0, "short"),              # one key each
    (2, 1, 1, 8, 2, 63, 5, 3, "short"),
    (3, 3, 1, 4, 4, 64, 40, 31, "short"),           # every row its own prefix
    (6, 2, 1, 10, 2, 65, 70, 63, "short"),          # five query heads per kv head
    (40, 1, 1, 8, 1, 130, 33, 32, "short"),
    (33, 1, 1, 16, 1, 300, 3, 1, "short"),          # 16 query heads per kv head
    (5, 1, 7, 9, 3, 129, 20, 9, "short"),           # 21 columns
    (2, 2, 33, 8, 2, 70, 40, 4, "short"),
    (40, 1, 1, 8, 1, 2000, 33, 32, "group+join"),   # 320 columns
    (4, 2, 2, 6, 2, 2200, 130, 100, "group+join"),  # two queries a row
    (9, 3, 1, 6, 2, 1025, 300, 290, "group+join"),
    (2, 1, 1, 4, 1, 4100, 1200, 1111, "row+join"), 
    (70, 7, 3, 20, 4, 700, 40, 8, "short"),         # 5 query heads, 280 workgroups
    (70, 7, 3, 20, 4, 1100, 40, 8, "group+join"),   # 150 columns a prefix, 15 of own keys
    (3, 1, 130, 4, 2, 1257, 200, 66, "row+join"),   # tiles of one row over both
    (1, 1, 96, 1, 1, 1000, 96, 0, "row+join"),
    (64, 2, 60, 8, 4, 500, 80, 20, "row"),          # 120 columns a row, one part
    (13, 1, 97, 12, 4, 640, 130, 33, "row"),        # 291
]


@pytest.mark.parametrize("b,g,s,h,hkv,p,t,slot,way", SHAPES)
def test_prefix_attention(b, g, s, h, hkv, p, t, slot, way):
    assert serving.ext().prefix_plan(b, s, h, hkv, g, p, t) == way
    args = inputs(b, g, s, h, hkv, p, t, slot=slot)
    want, bound = oracle.prefix_attention(*args, slot)
    gpu = [x.to(DEV) for x in args]
    got = ops.prefix_attention(*gpu, slot)
    close(got, want, bound)
    assert torch.equal(got, ops.prefix_attention(*gpu, torch.tensor([slot], dtype=I32, device=DEV)))


@pytest.mark.parametrize("b,g,s,h,hkv,p,t,slot,way", [
    (8, 4, 1, 4, 2, 150, 70, 60, "short"), (6, 3, 3, 4, 1, 70, 40, 33, "short"), (6, 3, 40, 3, 1, 200, 90, 20, "short"),
    (8, 4, 1, 8, 2, 1900, 70, 60, "group+join"), (6, 3, 5, 4, 2, 1500, 40, 33, "group+join"), (6, 3, 50, 4, 1, 1100, 190, 20, "row+join"),
    (60, 3, 50, 8, 4, 600, 90, 20, "row")])
def test_prefix_attention_masks(b, g, s, h, hkv, p, t, slot, way):
    assert serving.ext().prefix_plan(b, s, h, hkv, g, p, t) == way
    args = inputs(b, g, s, h, hkv, p, t, slot=slot)
    kw = dict(prefix_len=torch.randint(p // 2, p + 1, (g,), dtype=I32), prefix_start=torch.randint(0, p // 3, (g,), dtype=I32),
              prefix_mask=(torch.rand(g, p) < 0.6).to(torch.uint8), kv_start=torch.randint(0, slot + 1, (b,), dtype=I32))
    kw["prefix_len"][0] = 0                      # nothing of its prefix
    kw["prefix_start"][1] = p + 5                # nor here: it starts behind the end
    kw["prefix_mask"][2, :] = 0
    kw["kv_start"][:3] = slot + s // 2 + 1       # some queries have nothing at all
    kw["kv_start"][3] = -4
    for keys in (("prefix_len",), ("prefix_start", "kv_start"), ("prefix_mask",), ("prefix_len", "prefix_start", "prefix_mask", "kv_start")):
        given = {k: kw[k] for k in keys}
        q, kp, vp, ko, vo = (x.clone() for x in args)
        for i in range(g):  # whatever nobody attends
            ok = torch.ones(p, dtype=torch.bool)
            at = torch.arange(p)
            if "prefix_len" in given:
                ok &= at < given["prefix_len"][i]
            if "prefix_start" in given:
                ok &= at >= given["prefix_start"][i]
            if "prefix_mask" in given:
                ok &= given["prefix_mask"][i] != 0
            kp[i][:, ~ok] = float("nan")
            vp[i][:, ~ok] = float("inf")
        if "kv_start" in given:
            for i in range(b):
                ko[i][:, :max(0, int(given["kv_start"][i]))] = float("nan")
                vo[i][:, :max(0, int(given["kv_start"][i]))] = float("nan")
        want, bound = oracle.prefix_attention(q, kp, vp, ko, vo, slot, **given)
        close(ops.prefix_attention(*(x.to(DEV) for x in (q, kp, vp, ko, vo)), slot, **dev(given)), want, bound)


@pytest.mark.parametrize("p", [700, 5000])
def test_prefix_attention_large_scores(p):
    """Scores of some hundreds, ascending along the keys (the maximum moves all the time)."""
    q, kp, vp, ko, vo = inputs(3, 1, 1, 4, 2, p, 8, slot=2)
    kp = (kp.float() * torch.linspace(0.1, 12, p)[None, None, :, None]).to(BF16)
    want, bound = oracle.prefix_attention(q, kp, vp, ko, vo, 2)
    close(ops.prefix_attention(*(x.to(DEV) for x in (q, kp, vp, ko, vo)), 2), want, bound)


@pytest.mark.parametrize("p", [100, 2500])
def test_prefix_attention_views_streams_and_packed(p):
    q, kp, vp, ko, vo = inputs(12, 2, 1, 8, 2, p, 30, unused=0.0, slot=20)
    want, bound = oracle.prefix_attention(q, kp, vp, ko, vo, 20)
    wide = [torch.full((x.shape[0] + 1, x.shape[1] + 2, x.shape[2] + 5, 128), float("nan"), dtype=BF16, device=DEV) for x in (kp, vp, ko, vo)]
    views = []
    for w, x in zip(wide, (kp, vp, ko, vo)):
        v = w[1:, 1:-1, :x.shape[2]]
        v.copy_(x)
        views.append(v)
    qd = q.to(DEV)
    packed = ops.packed_empty(12, 8 * 128, DEV)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = ops.prefix_attention(qd, *views, 20, out_packed=packed)
    torch.cuda.current_stream().wait_stream(other)
    close(got, want, bound)
    p = packed.view(torch.int16).view(1, 8 * 128 // 32, 4, 16, 8)  # [m tile][k step][k / 8 % 4][row][k % 8]
    rows = p.permute(0, 3, 1, 2, 4).reshape(16, 8 * 128)[:12]
    assert torch.equal(rows, got.view(torch.int16))


@pytest.mark.parametrize("p", [100, 2500])
def test_prefix_attention_rows_past_32_bits(p):
    """The second prefix lies 2^31 elements behind the first."""
    q, kp, vp, ko, vo = inputs(6, 2, 1, 8, 2, p, 30, slot=20)
    want, bound = oracle.prefix_attention(q, kp, vp, ko, vo, 20)
    n = 2 * p * 128
    far = torch.empty(2 ** 31 + 2 * n, dtype=BF16, device=DEV)
    views = [far.as_strided((2, 2, p, 128), (2 ** 31, p * 128, 128, 1), at) for at in (0, n)]
    for view, x in zip(views, (kp, vp)):
        view.copy_(x)
    close(ops.prefix_attention(q.to(DEV), *views, ko.to(DEV), vo.to(DEV), 20), want, bound)


@pytest.mark.parametrize("s,h", [(1, 2), (60, 2)])
def test_prefix_attention_tokens_past_32_bits(s, h):
    """The last keys of a prefix of 2^24 tokens (2^31 elements) and of own keys as far in; the others are unset and not attended."""
    far, live = 2 ** 24 + 77, 500
    q, kp, vp, ko, vo = inputs(2, 1, s, h, 1, live, live, slot=live - s)
    want, bound = oracle.prefix_attention(q, kp, vp, ko, vo, live - s)
    k, v = (torch.empty(2, 1, far, 128, dtype=BF16, device=DEV) for _ in range(2))
    for x, a, b in ((k, kp, ko), (v, vp, vo)):
        x[:1, :, far - live:] = a.to(DEV)
    start = torch.full((1,), far - live, dtype=I32, device=DEV)
    close(ops.prefix_attention(q.to(DEV), k[:1], v[:1], ko.to(DEV), vo.to(DEV), live - s, prefix_start=start), want, bound)
    for x, b in ((k, ko), (v, vo)):
        x[:, :, far - live:] = b.to(DEV)
    close(ops.prefix_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, far - s, kv_start=start.expand(2).contiguous()), want, bound)


@pytest.mark.parametrize("p", [100, 2500])
def test_prefix_attention_two_streams(p):
    """Calls under way at once on two streams have parts of their own."""
    sets = [[x.to(DEV) for x in inputs(12, 2, 1, 8, 2, p, 30, slot=20)] for _ in range(2)]
    want = [ops.prefix_attention(*s, 20) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.prefix_attention(*sets[i], 20))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


@pytest.mark.parametrize("p", [190, 2500])
def test_prefix_attention_graph(p):
    """A captured call sees the slot, the masks and the keys of each replay; two graphs and eager calls between them do not meet."""
    b, g, h, hkv, t = 10, 2, 8, 2, 50
    args = inputs(b, g, 1, h, hkv, p, t, unused=0.5)
    gpu = [x.to(DEV) for x in args]
    slot, start = torch.zeros(1, dtype=I32, device=DEV), torch.zeros(g, dtype=I32, device=DEV)
    graphs = []
    for _ in range(2):
        ops.prefix_attention(*gpu, slot, prefix_start=start)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.prefix_attention(*gpu, slot, prefix_start=start)
        graphs.append((graph, out))
    for step in range(4):
        slot.fill_(7 * step)
        start.copy_(torch.tensor([step, 40 * step], dtype=I32))
        gpu[0].copy_(torch.randn(gpu[0].shape))
        eager = ops.prefix_attention(*gpu, slot, prefix_start=start)
        for graph, out in graphs:
            out.zero_()
            graph.replay()
        again = ops.prefix_attention(*gpu, slot, prefix_start=start)
        torch.cuda.synchronize()
        assert torch.equal(eager, again) and all(torch.equal(out, eager) for _, out in graphs)


def test_prefix_attention_refusals_gpu():
    q, kp, vp, ko, vo = (x.to(DEV) for x in inputs(2, 1, 1, 4, 2, 16, 8, unused=0.0))
    for bad in ((q[..., :64].contiguous(), kp[..., :64].contiguous(), vp[..., :64].contiguous(), ko[..., :64].contiguous(), vo[..., :64].contiguous()),
                (q, kp.cpu(), vp, ko, vo), (q.float(), kp, vp, ko, vo), (q, kp.float(), vp, ko, vo), (q.repeat(1, 1, 1, 2)[..., :128], kp, vp, ko, vo)):
        with pytest.raises(ValueError):
            ops.prefix_attention(*bad, 0)
    for kw in (dict(prefix_len=torch.ones(2, dtype=I32, device=DEV)), dict(prefix_start=torch.ones(1, device=DEV)), dict(kv_start=torch.ones(1, dtype=I32, device=DEV)),
               dict(prefix_mask=torch.ones(1, 15, dtype=torch.uint8, device=DEV)), dict(prefix_len=torch.ones(1, dtype=I32))):
        with pytest.raises(ValueError):
            ops.prefix_attention(q, kp, vp, ko, vo, 0, **kw)
    for slot in (8, -1):
        with pytest.raises(ValueError):
            ops.prefix_attention(q, kp, vp, ko, vo, slot)
    odd = torch.zeros(1, 2, 16 * 128 + 8, dtype=BF16, device=DEV)
    with pytest.raises(ValueError):  # tokens that do not follow one another
        ops.prefix_attention(q, kp.transpose(1, 2).contiguous().transpose(1, 2), vp, ko, vo, 0)
    with pytest.raises(ValueError):  # not at a multiple of 16 bytes
        ops.prefix_attention(q, odd[:, :, 1:16 * 128 + 1].unflatten(2, (16, 128)), vp, ko, vo, 0)


# ---------------------------------------------------------------------------------- logits
def logits_inputs(b, v, n, masks):
    tok = torch.randint(0, v + 3, (b, n + 4), dtype=I32) - 1  # (some outside the vocabulary)
    tok[:, ::3] = tok[:, :1]
    return dict(history=tok, length=n, start=torch.randint(0, max(1, n // 3), (b,), dtype=I32), prompt_len=n // 2,
                history_mask=(torch.rand(b, n + 4) < 0.7).to(torch.uint8), repetition_penalty=1 + torch.rand(b), presence_penalty=0.25,
                frequency_penalty=torch.rand(b) * 0.3, bias=torch.randn(v), allowed=torch.rand(masks, v) < 0.4,
                allowed_rows=torch.randint(-1, masks + 1, (b,), dtype=I32))


def packed(kw):
    return dev({**kw, "allowed": ops.pack_allowed(kw["allowed"]) if kw.get("allowed") is not None else None})


@pytest.mark.parametrize("b,v,n", [(1, 1, 1), (1, 2, 0), (3, 33, 9), (2, 8191, 300), (2, 8192, 40), (3, 8193, 700), (2, 32001, 2500), (5, 128256, 90), (17, 128256, 50),
                                   (150, 14001, 600)])
def test_process_logits(b, v, n):
    x, kw = torch.randn(b, v) * 3, logits_inputs(b, v, n, 4)
    for drop in ((), ("bias",), ("allowed", "allowed_rows"), ("bias", "allowed", "allowed_rows"), ("start", "history_mask"),
                 ("history", "repetition_penalty", "presence_penalty", "frequency_penalty", "start", "history_mask")):
        given = {k: w for k, w in kw.items() if k not in drop}
        want, bound = oracle.process_logits(x, **given)
        g, xd = packed(given), x.to(DEV)
        got = ops.process_logits(xd, **g)
        live = want > float("-inf")
        assert torch.equal(got.cpu() == float("-inf"), ~live)
        close(torch.where(live.to(DEV), got, 0.0), torch.where(live, want, 0.0), torch.where(live, bound, 0.0))
        assert torch.equal(xd.cpu(), x)
        if g.get("history") is not None:
            assert torch.equal(got, ops.process_logits(xd, **{**g, "length": torch.tensor([n], dtype=I32, device=DEV)}))
        assert ops.process_logits(xd, out=xd, **g) is xd and torch.equal(xd, got)


def test_process_logits_strides_rows_and_shards():
    b, v = 4, 1001
    x, kw = torch.randn(b, v), logits_inputs(b, v, 200, 1)
    kw.update(allowed_rows=None, bias=torch.randn(b, v))
    want = ops.process_logits(x.to(DEV), **packed(kw))
    wide = torch.full((b, v + 7), float("nan"), device=DEV)
    wide[:, 3:v + 3] = x.to(DEV)
    bias = torch.zeros(b, v + 2, device=DEV)
    bias[:, 1:v + 1] = kw["bias"].to(DEV)
    got = ops.process_logits(wide[:, 3:v + 3], out=wide[:, 3:v + 3], **{**packed(kw), "bias": bias[:, 1:v + 1]})
    assert torch.equal(got, want) and bool(wide[:, :3].isnan().all()) and bool(wide[:, v + 3:].isnan().all())
    for cut in (1, 31, 32, 500, 1000):
        parts = [ops.process_logits(x[:, a:z].to(DEV), vocab_start=a, **{**packed(kw), "bias": kw["bias"][:, a:z].to(DEV)}) for a, z in ((0, cut), (cut, v))]
        assert torch.equal(torch.cat(parts, 1), want)


def test_process_logits_past_32_bits():
    """Rows behind 2^31 elements, out of place and in place."""
    v = 32000
    b = 2 ** 31 // v + 5
    x = torch.empty(b, v, device=DEV)
    x[-4:] = torch.randn(4, v)
    kw = packed({k: t for k, t in logits_inputs(b, v, 40, 3).items() if k != "bias"})
    last = {k: t[-4:].contiguous() if torch.is_tensor(t) and t.shape[0] == b else t for k, t in kw.items()}
    want = ops.process_logits(x[-4:].clone(), **last)
    assert torch.equal(ops.process_logits(x, **kw)[-4:], want)
    for k in ("allowed", "allowed_rows"):
        kw.pop(k), last.pop(k)
    want = ops.process_logits(x[-4:].clone(), **last)
    ops.process_logits(x, out=x, **kw)
    assert torch.equal(x[-4:], want)


def test_process_logits_masked_nan_and_dead_ends():
    v = 70
    x = torch.randn(2, v, device=DEV)
    x[0, 5], x[1, 6] = float("nan"), float("inf")
    mask = torch.ones(2, v, dtype=torch.bool, device=DEV)
    mask[0, 5] = mask[1, 6] = False
    got = ops.process_logits(x, allowed=ops.pack_allowed(mask))
    assert got[0, 5] == float("-inf") and got[1, 6] == float("-inf") and torch.equal(got[mask], x[mask])
    none = ops.process_logits(x, allowed=torch.zeros(1, 3, dtype=I32, device=DEV))
    step = torch.zeros(1, dtype=I32, device=DEV)
    assert bool((none == float("-inf")).all()) and ops.argmax(none)[0].tolist() == [0, 0]
    assert ops.topk_sample(none, 5, 1.0, 1.0, 0, step).tolist() == [0, 0]


def test_process_logits_graph():
    b, v, n = 5, 20000, 60
    x, kw = torch.randn(b, v, device=DEV), packed(logits_inputs(b, v, n, 3))
    length = torch.zeros(1, dtype=I32, device=DEV)
    kw.update(length=length)
    for drop in ((), ("bias", "allowed", "allowed_rows")):
        given = {k: w for k, w in kw.items() if k not in drop}
        buf = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.process_logits(buf, out=buf, **given)
        for step in (0, 7, 33, 60):
            length.fill_(step)
            buf.copy_(x)
            kw["history"].copy_(torch.randint(0, v, kw["history"].shape))
            eager = ops.process_logits(x, **given)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(buf, eager)


# ---------------------------------------------------------------------------------- rows
def fill(cache):
    for t, _, _ in cache_tensors(cache):
        t.copy_(torch.randn(t.shape))
    return cache


@pytest.mark.parametrize("make", [lambda n, t: KVCache(3, n, 2, t, 128, DEV), lambda n, t: KVCache(2, n, 1, t, 3, DEV),
                                  lambda n, t: HybridCache(SPECS, n, t, DEV), lambda n, t: HybridCache(SPECS, n, t, DEV, torch.float32)])
def test_copy_rows(make):
    perm = torch.randperm(50).tolist()
    for n, src, dst, tokens in ((2, [0], [1], 3), (4, [0, 0, 1, 1], [0, 1, 2, 3], 5), (4, [3, 2, 1, 0], [0, 1, 2, 3], 6), (3, [-1, 2], [2, 0], 0),
                                (50, perm, list(range(50)), 4), (50, [i // 7 for i in range(50)], list(range(50)), 1), (6, [5, 4], [0, 1], 6),
                                (450, [(i * 7 + 3) % 450 for i in range(450)], list(range(450)), 2), (3, [], [], 1)):
        cache = fill(make(n, 6))
        want = oracle.copied(cache_tensors(cache), src, dst, tokens)
        cache.copy_rows(src, dst, tokens=tokens)
        assert all(torch.equal(t, w) for (t, _, _), w in zip(cache_tensors(cache), want)), (n, src, dst, tokens)
    a, b = fill(make(2, 5)), fill(make(30, 7))
    want = oracle.copied(cache_tensors(a), [i % 2 for i in range(29)], list(range(1, 30)), 4, cache_tensors(b))
    a.copy_rows([i % 2 for i in range(29)], range(1, 30), tokens=4, to=b)
    assert all(torch.equal(t, w) for (t, _, _), w in zip(cache_tensors(b), want))


def test_copy_rows_large_cache_and_moved_tensors():
    """Rows past 2^32 bytes; a cache whose tensors were replaced."""
    cache = KVCache(1, 40, 1, 1 << 19, 128, DEV)  # rows of 128 MiB, 5 GiB each of keys and values
    cache.k[0, 38, :, :3] = torch.randn(1, 3, 128, device=DEV).to(BF16)
    cache.v[0, 38, :, -2:] = 2.0
    cache.copy_rows([38], [36], tokens=1 << 19)
    assert torch.equal(cache.k[0, 36], cache.k[0, 38]) and torch.equal(cache.v[0, 36], cache.v[0, 38])
    assert not bool(cache.k[0, 37].any()) and not bool(cache.v[0, 35].any())
    small = fill(KVCache(2, 3, 1, 4, 128, DEV))
    small.copy_rows([0], [1], tokens=2)
    small.k = small.k.clone()
    want = oracle.copied(cache_tensors(small), [2], [0], 4)
    small.copy_rows([2], [0], tokens=4)
    assert torch.equal(small.k, want[0]) and torch.equal(small.v, want[1])


def test_copy_rows_graph():
    cache = fill(HybridCache(SPECS, 4, 6, DEV))
    cache.copy_rows([1], [3], tokens=1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.copy_rows([1, 0, 3], [0, 1, 2], tokens=5)
    for _ in range(3):
        fill(cache)
        want = oracle.copied(cache_tensors(cache), [1, 0, 3], [0, 1, 2], 5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t, w) for (t, _, _), w in zip(cache_tensors(cache), want))
    fresh = HybridCache(SPECS, 4, 6, DEV)
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fresh.copy_rows([0], [1], tokens=1)


def test_copy_rows_refusals_gpu():
    kv, hy = KVCache(2, 4, 2, 6, 128, DEV), HybridCache(SPECS, 4, 6, DEV)
    for cache in (kv, hy):
        for src, dst, kw in (([0], [4], {}), ([4], [0], {}), ([-2], [0], {}), ([0], [-1], {}), ([0, 1], [2, 2], {}), ([0, 1], [2], {}),
                             ([0], [1], dict(tokens=7)), ([0], [1], dict(tokens=-1))):
            with pytest.raises(ValueError):
                cache.copy_rows(src, dst, **kw)
    cpu = KVCache(2, 4, 2, 6, 128, "cpu")
    for a, b in ((kv, cpu), (cpu, kv)):
        with pytest.raises(ValueError):
            a.copy_rows([0], [1], tokens=1, to=b)
    for other in (hy, KVCache(2, 4, 3, 6, 128, DEV), KVCache(3, 4, 2, 6, 128, DEV), KVCache(2, 4, 2, 6, 64, DEV, torch.float32)):
        with pytest.raises(ValueError):
            kv.copy_rows([0], [1], tokens=1, to=other)


def test_process_logits_refusals_gpu():
    x, h = torch.randn(2, 40, device=DEV), torch.zeros(2, 5, dtype=I32, device=DEV)
    words = torch.zeros(3, 2, dtype=I32, device=DEV)
    ok = dict(presence_penalty=0.1, history=h, length=1)
    bad = [dict(repetition_penalty=1.2), {**ok, "repetition_penalty": 0.0}, {**ok, "presence_penalty": float("inf")}, dict(presence_penalty=0.1, history=h),
           {**ok, "length": 6}, {**ok, "length": -1}, {**ok, "history": h[:1]}, {**ok, "history": h.long()}, {**ok, "history": h.cpu()},
           {**ok, "frequency_penalty": torch.zeros(3, device=DEV)}, {**ok, "start": torch.zeros(3, dtype=I32, device=DEV)}, {**ok, "prompt_len": -1},
           {**ok, "history_mask": torch.ones(2, 4, dtype=torch.uint8, device=DEV)}, dict(bias=torch.zeros(39, device=DEV)), dict(bias=torch.zeros(40)),
           dict(bias=torch.zeros(1, 40, device=DEV)), dict(bias=torch.zeros(40, dtype=torch.float64, device=DEV)), dict(allowed=words[:, :1]),
           dict(allowed=words), dict(allowed=words.long()), dict(allowed_rows=torch.zeros(2, dtype=I32, device=DEV)),
           dict(allowed=words[:1], vocab_start=30), dict(vocab_start=-1), dict(out=torch.zeros(2, 41, device=DEV)), dict(out=torch.zeros(2, 40)),
           dict(out=torch.zeros(1, 40, device=DEV).expand(2, 40))]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.process_logits(x, **kw)
    for other in (x.to(BF16), x[0], x.t()):
        with pytest.raises(ValueError):
            ops.process_logits(other)
    both = torch.zeros(81, device=DEV)
    with pytest.raises(ValueError):
        ops.process_logits(both[:80].view(2, 40), out=both[1:].view(2, 40))


# ---------------------------------------------------------------------------------- together
def test_together():
    """A prompt's cache forked and reordered, its prefix attended by samples, their logits penalised and masked, all in one captured step."""
    b, h, hkv, p, t, v = 6, 8, 2, 77, 16, 500
    prompts, own = fill(KVCache(1, 2, hkv, p, 128, DEV)), fill(KVCache(1, b, hkv, t, 128, DEV))
    q = (torch.randn(b, 1, h, 128) * 2).to(BF16).to(DEV)
    head = torch.randn(h * 128, v, device=DEV) * 0.1
    kw = packed(logits_inputs(b, v, 20, 2))
    slot = torch.full((1,), 3, dtype=I32, device=DEV)

    def step():
        own.copy_rows([0, 0, 0, 3, 3, 3], range(6), tokens=4)
        att = ops.prefix_attention(q, *prompts.layer(0), *own.layer(0), slot)
        return att, ops.process_logits(att.float() @ head, **kw)

    step()
    fill(own)
    before = [x.clone() for x in (own.k, own.v)]
    att, out = step()
    k, w = (oracle.copied([(x, 1, 3)], [0, 0, 0, 3, 3, 3], range(6), 4)[0][0].cpu() for x in before)
    want, bound = oracle.prefix_attention(q.cpu(), prompts.k[0].cpu(), prompts.v[0].cpu(), k, w, 3)
    close(att, want, bound)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        att2, out2 = step()
    for _ in range(3):
        own.k.copy_(before[0])
        own.v.copy_(before[1])
        att2.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(att, att2) and torch.equal(out, out2)
