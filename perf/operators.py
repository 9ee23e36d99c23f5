"""Operators of serving many continuations of shared prompts, and what they are measured on.

* attention of a batch whose rows share prefixes (``ops.prefix_attention``): several continuations of one prompt decoded
  side by side, or prompts behind a common system prompt; row ``b`` of ``B`` reads prefix ``b // (B / G)`` and its own keys;
* penalties for repeated tokens, biases and grammar masks on logits (``ops.process_logits``);
* copying, forking and compacting rows of a cache (``copy_rows`` of the cache objects).

``run`` makes these calls where ``own`` is true, and otherwise computes the same from elementary torch operations in 32 bits.
The framework runs models, it does not train them: the operators have no gradients.
"""
import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # two samples of a short prompt, a few tokens in: the smallest step, where latency counts (8B heads)
        dict(name="prefix-2-samples", op="attention", groups=1, each=2, queries=1, heads=32, kv_heads=8, prefix=130, held=3,
             room=64, pad=False),
        # one token of 32 samples of a 2k prompt (8B heads)
        dict(name="prefix-32-samples-2k", op="attention", groups=1, each=32, queries=1, heads=32, kv_heads=8, prefix=2048,
             held=100, room=256, pad=False),
        # one token of 16 samples of each of four left-padded prompts of odd length (70B heads: 8 query heads per kv head)
        dict(name="prefix-4x16-8k-padded", op="attention", groups=4, each=16, queries=1, heads=64, kv_heads=8, prefix=8011,
             held=333, room=512, pad=True),
        # one token of 64 requests behind a 64k document: the prefix alone bounds it
        dict(name="prefix-64-samples-64k", op="attention", groups=1, each=64, queries=1, heads=32, kv_heads=8, prefix=65536,
             held=64, room=128, pad=False),
        # the prompts of 16 requests, left-padded to 200 tokens, behind a system prompt of 4k (time to first token)
        dict(name="prefix-16-prompts-4k", op="attention", groups=1, each=16, queries=200, heads=32, kv_heads=8, prefix=4097,
             held=0, room=256, pad=True),
        # one user with a repetition penalty, the smallest vocabulary of the presets: latency
        dict(name="logits-1x32000", op="logits", rows=1, vocab=32000, history=200, penalties=True, bias="none", masks=0),
        # a serving batch with every penalty, a bias shared by the rows and a grammar state per row
        dict(name="logits-64x128256-grammar", op="logits", rows=64, vocab=128256, history=2048, penalties=True, bias="shared",
             masks=40),
        # a throughput batch
        dict(name="logits-1024x128256", op="logits", rows=1024, vocab=128256, history=384, penalties=True, bias="shared", masks=0),
        # one request of a few tokens branched into a second one (8B cache rows, four layers): latency
        dict(name="fork-one-request", op="fork", layers=4, kind="kv", kv_heads=8, dim=128, sources=1, each=1, room=128, tokens=37),
        # two prompts forked into eight samples each (8B cache rows)
        dict(name="fork-2x8-samples", op="fork", layers=16, kind="kv", kv_heads=8, dim=128, sources=2, each=8, room=640, tokens=517),
        # the same for a stack that mixes attention with recurrent layers (odd widths of carried state)
        dict(name="fork-mixed-state", op="fork", layers=12, kind="mixed", kv_heads=4, dim=128, sources=3, each=4, room=512, tokens=300),
        # 24 live rows of a batch of 64 moved to its front
        dict(name="compact-24-of-64", op="compact", layers=8, kind="kv", kv_heads=8, dim=128, rows=64, live=24, room=384, tokens=301),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "prompts", "logits", "logits", "fork", "compact"])
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (64, 8), (32, 32), (8, 1), (40, 40), (12, 4)])
    if kind == "attention":
        groups, each = rng.choice([1, 1, 2, 5]), _log(rng, 1, 64)
        prefix = _log(rng, 1, min(40000, 520000 // (kv_heads * groups)))
        held = _log(rng, 1, 400) - 1
        return dict(op="attention", groups=groups, each=each, queries=1, heads=heads, kv_heads=kv_heads, prefix=prefix,
                    held=held, room=held + 1 + rng.choice([0, 1, 63]), pad=rng.random() < 0.5)
    if kind == "prompts":
        groups, each, queries = rng.choice([1, 1, 2]), _log(rng, 1, 16), _log(rng, 2, 250)
        held = rng.choice([0, 0, rng.randint(1, 90)])
        return dict(op="attention", groups=groups, each=each, queries=queries, heads=heads, kv_heads=kv_heads,
                    prefix=_log(rng, 3, min(4000, 3000000 // (each * groups * queries))), held=held,
                    room=held + queries + rng.choice([0, 5, 64]), pad=rng.random() < 0.5)
    if kind == "logits":
        vocab = rng.choice([32000, 32001, 128256, 50257])
        rows = _log(rng, 1, 500)
        return dict(op="logits", rows=rows, vocab=vocab, history=_log(rng, 1, 8000), penalties=rng.random() < 0.8,
                    bias=rng.choice(["none", "shared", "rows"]), masks=rng.choice([0, 1, 17]))
    if kind == "fork":
        mixed = rng.random() < 0.5
        sources, each = rng.randint(1, 4), _log(rng, 1, 10)
        tokens = _log(rng, 1, 500)
        return dict(op="fork", layers=rng.randint(1, 10), kind="mixed" if mixed else "kv", kv_heads=rng.choice([1, 4, 8]), dim=128,
                    sources=sources, each=each, room=tokens + rng.randint(0, 100), tokens=tokens)
    rows = rng.randint(2, 60)
    tokens = _log(rng, 1, 300)
    return dict(op="compact", layers=rng.randint(1, 8), kind="kv", kv_heads=rng.choice([1, 4, 8]), dim=128, rows=rows,
                live=rng.randint(1, max(1, rows // 2)), room=tokens + rng.randint(0, 100), tokens=tokens)


# ------------------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, gen, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _attention_inputs(c, seed):
    """Queries and keys with scores of a standard deviation of about two (some keys far ahead, as behind a trained model); rows left-padded
    to the longest where ``pad``: in the prefix (token steps) or in their own part (prompts)."""
    gen = _generator(seed)
    b, s, h, g, d = c["groups"] * c["each"], c["queries"], c["heads"], c["kv_heads"], 128
    st = dict(q=_normal((b, s, h, d), gen, BF16, 2.0), kp=_normal((c["groups"], g, c["prefix"], d), gen, BF16),
              vp=_normal((c["groups"], g, c["prefix"], d), gen, BF16))
    for name in ("ko", "vo"):
        st[name] = torch.zeros(b, g, c["room"], d, dtype=BF16, device="cuda")
        st[name][:, :, :c["held"] + s] = _normal((b, g, c["held"] + s, d), gen, BF16)
    st["slot"] = torch.full((1,), c["held"], dtype=torch.int32, device="cuda")
    ints = dict(generator=gen, device="cuda", dtype=torch.int32)
    in_prefix = c["pad"] and s == 1
    st["start"] = torch.randint(0, max(1, c["prefix"] // 2), (c["groups"],), **ints) if in_prefix else None
    st["own_start"] = torch.randint(0, max(1, s // 2), (b,), **ints) if c["pad"] and s > 1 else None
    return st


def _logits_inputs(c, seed):
    """Logits of a trained model's spread; the row's tokens repeat (a skewed distribution); masks that leave about one token in eight."""
    gen = _generator(seed)
    b, v, n = c["rows"], c["vocab"], c["history"]
    st = dict(logits=_normal((b, v), gen, F32, 3.0))
    u = torch.rand(b, n + 5, generator=gen, device="cuda")
    st["history"] = ((u ** 4) * v).to(torch.int32).clamp_(max=v - 1)
    st["length"] = torch.full((1,), n, dtype=torch.int32, device="cuda")
    st["start"] = torch.randint(0, max(1, n // 4), (b,), generator=gen, device="cuda", dtype=torch.int32)
    st["prompt"] = n // 2
    st["repetition"] = 1.0 + 0.5 * torch.rand(b, generator=gen, device="cuda")
    st["presence"] = 0.5 * torch.rand(b, generator=gen, device="cuda")
    st["frequency"] = 0.2 * torch.rand(b, generator=gen, device="cuda")
    if not c["penalties"]:
        st["history"] = None
    st["bias"] = None if c["bias"] == "none" else _normal((v,) if c["bias"] == "shared" else (b, v), gen)
    st["allowed"] = st["rows"] = None
    if c["masks"]:
        words = (v + 31) // 32
        st["allowed"] = torch.full((c["masks"], words), -1, dtype=torch.int32, device="cuda")
        for _ in range(3):
            st["allowed"] &= torch.randint(-2 ** 31, 2 ** 31, (c["masks"], words), generator=gen, device="cuda").to(torch.int32)
        st["rows"] = torch.randint(0, c["masks"], (b,), generator=gen, device="cuda", dtype=torch.int32)
    return st


def _specs(c):
    """Layers of the cache: keys and values; or these, a latent, and the recurrences' states in turn."""
    g, d = c["kv_heads"], c["dim"]
    if c["kind"] == "kv":
        return [("kv", g, d, d)] * c["layers"]
    turn = [("kv", g, d, d), ("delta", 8, g, d, d, 4), ("latent", 96), ("mlstm", 3, 64, 65), ("timemix", 5, 64, 64, 1001)]
    return [turn[i % len(turn)] for i in range(c["layers"])]


def _layer_shapes(spec, rows, room):
    """(shape, element type, whether its third axis is the tokens) of a layer's tensors."""
    kind = spec[0]
    if kind == "kv":
        return [((rows, spec[1], room, spec[2]), BF16, True), ((rows, spec[1], room, spec[3]), BF16, True)]
    if kind == "latent":
        return [((rows, 1, room, spec[1]), BF16, True)]
    if kind == "delta":
        _, h, g, d, e, taps = spec
        return [((rows, h, d, e), F32, False), ((rows, 2 * g * d + h * e, taps - 1), F32, False)]
    if kind == "mlstm":
        return [((rows, spec[1], spec[2], spec[3] + 1), F32, False), ((rows, spec[1]), F32, False)]
    return [((rows, spec[1], spec[2], spec[3]), F32, False), ((rows, spec[4]), F32, False)]


def _cache(c, rows, gen, filled):
    """A cache's tensors (and, for the framework's calls, the cache itself): KVCache ``[layers, rows, kv heads, room, dim]`` twice, or one
    layer's after the other. ``filled``: rows with contents; the others hold zeros."""
    specs = _specs(c)
    cache = None
    if c["kind"] == "kv":
        shape = (c["layers"], rows, c["kv_heads"], c["room"], c["dim"])
        if own:
            from jax_llama_amd.models.kv_cache import KVCache
            cache = KVCache(c["layers"], rows, c["kv_heads"], c["room"], c["dim"], "cuda")
            tensors = [cache.k, cache.v]
        else:
            tensors = [torch.zeros(shape, dtype=BF16, device="cuda") for _ in range(2)]
        for t in tensors:
            t[:, filled, :, :c["tokens"]] = _normal((c["layers"], len(filled), c["kv_heads"], c["tokens"], c["dim"]), gen, BF16)
        return cache, tensors
    if own:
        from jax_llama_amd.models.kv_cache import HybridCache
        cache = HybridCache(specs, rows, c["room"], "cuda")
    tensors = []
    for i, spec in enumerate(specs):
        shapes = _layer_shapes(spec, rows, c["room"])
        if own:
            held = cache.layer(i)[:len(shapes)] if spec[0] in ("kv", "latent") else cache.recurrent(i)
        else:
            held = [torch.zeros(sh, dtype=dt, device="cuda") for sh, dt, _ in shapes]
        for t, (sh, dt, per_token) in zip(held, shapes):
            n = c["tokens"] if per_token else None
            part = t[filled, :, :n] if per_token else t[filled]
            new = _normal(tuple(part.shape), gen, dt)
            if per_token:
                t[filled, :, :n] = new
            else:
                t[filled] = new
            tensors.append(t)
    return cache, tensors


def _cache_inputs(c, seed):
    gen = _generator(seed)
    if c["op"] == "compact":
        picked = torch.randperm(c["rows"] - c["live"], generator=torch.Generator().manual_seed(seed))[:c["live"]]
        src = sorted(int(i) + c["live"] for i in picked)  # live rows behind the front (rows // 2 at most are live)
        cache, tensors = _cache(c, c["rows"], gen, src)
        return dict(src=src, dst=list(range(len(src))), source=cache, target=None, read=tensors, written=tensors)
    n = c["sources"] * c["each"]
    source, read = _cache(c, c["sources"], gen, list(range(c["sources"])))
    target, written = _cache(c, n, gen, [])
    return dict(src=[i // c["each"] for i in range(n)], dst=list(range(n)), source=source, target=target, read=read, written=written)


def prepare(case, seed):
    if case["op"] == "attention":
        st = _attention_inputs(case, seed)
    elif case["op"] == "logits":
        st = _logits_inputs(case, seed)
    else:
        st = _cache_inputs(case, seed)
    st["case"] = case
    return st


# ------------------------------------------------------------------------------------------------------------ passes
def _plain_attention(st, dtype=F32):
    """Group by group: the scores of all of a group's rows against the prefix in one product, those against their own keys row by row."""
    c = st["case"]
    n, s, h, g, d = c["each"], c["queries"], c["heads"], c["kv_heads"], 128
    rep, t = h // g, c["held"] + c["queries"]
    scale = 1.0 / math.sqrt(d)
    place = torch.arange(t, device="cuda")
    causal = place[None, :] <= c["held"] + torch.arange(s, device="cuda")[:, None]  # [S, T]
    outs = []
    for i in range(c["groups"]):
        rows = slice(i * n, (i + 1) * n)
        q = st["q"][rows].to(dtype).reshape(n, s, g, rep, d).permute(2, 0, 1, 3, 4).contiguous()  # [g, n, s, rep, d]
        ko, vo = (st[x][rows, :, :t].to(dtype).transpose(0, 1).contiguous() for x in ("ko", "vo"))  # [g, n, t, d]
        kp, vp = (st[x][i].to(dtype) for x in ("kp", "vp"))  # [g, p, d]
        ok = causal.expand(n, s, t)
        if st["own_start"] is not None:
            ok = ok & (place[None, None, :] >= st["own_start"][rows, None, None])
        a = torch.matmul(q.reshape(g, n * s * rep, d), kp.transpose(1, 2).contiguous()) * scale  # [g, n s rep, p]
        if st["start"] is not None:
            a = a.masked_fill_(torch.arange(c["prefix"], device="cuda") < st["start"][i], float("-inf"))
        b = torch.matmul(q.reshape(g, n, s * rep, d), ko.transpose(2, 3).contiguous()) * scale  # [g, n, s rep, t]
        b = b.reshape(g, n, s, rep, t).masked_fill(~ok[None, :, :, None, :], float("-inf")).reshape(g, n * s * rep, t)
        top = torch.maximum(a.amax(-1, keepdim=True), b.amax(-1, keepdim=True))
        a, b = torch.exp(a - top), torch.exp(b - top)
        total = a.sum(-1, keepdim=True) + b.sum(-1, keepdim=True)
        o = torch.matmul(a, vp) + torch.matmul(b.reshape(g, n, s * rep, t), vo).reshape(g, n * s * rep, d)
        outs.append((o / total).reshape(g, n, s, rep, d).permute(1, 2, 0, 3, 4).reshape(n * s, h * d))
    return torch.cat(outs)


def _plain_logits(st):
    x = st["logits"]
    b, v = x.shape
    if st["history"] is not None:
        n = st["case"]["history"]
        tok = st["history"][:, :n].long()
        place = torch.arange(n, device=x.device)[None, :]
        real = (place >= st["start"][:, None]).float()
        new = real * (place >= st["prompt"])
        seen = torch.zeros(b, v, device=x.device).scatter_add_(1, tok, real) > 0
        count = torch.zeros(b, v, device=x.device).scatter_add_(1, tok, new)
        r = st["repetition"][:, None]
        x = torch.where(seen, torch.where(x < 0, x * r, x / r), x)
        x = x - st["frequency"][:, None] * count - st["presence"][:, None] * (count > 0).float()
    if st["bias"] is not None:
        x = x + st["bias"]
    if st["allowed"] is not None:
        words = st["allowed"][st["rows"].long()]
        bits = (words[:, :, None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = x.masked_fill(bits.reshape(b, -1)[:, :v] == 0, float("-inf"))
    return x if x is not st["logits"] else x.clone()


def _plain_copy(st):
    c = st["case"]
    src, dst, n = torch.tensor(st["src"], device="cuda"), torch.tensor(st["dst"], device="cuda"), c["tokens"]
    if c["kind"] == "kv":
        for a, b in zip(st["read"], st["written"]):
            b[:, dst, :, :n] = a[:, src, :, :n]
        return st["written"]
    at = 0
    for spec in _specs(c):
        for _, _, per_token in _layer_shapes(spec, 1, c["room"]):
            a, b = st["read"][at], st["written"][at]
            at += 1
            if per_token:
                b[dst, :, :n] = a[src, :, :n]
            else:
                b[dst] = a[src]
    return st["written"]


def _own(st):
    c = st["case"]
    if c["op"] == "attention":
        from jax_llama_amd import ops
        return ops.prefix_attention(st["q"], st["kp"], st["vp"], st["ko"], st["vo"], st["slot"], prefix_start=st["start"],
                                    kv_start=st["own_start"])
    if c["op"] == "logits":
        from jax_llama_amd import ops
        kw = dict(bias=st["bias"], allowed=st["allowed"], allowed_rows=st["rows"])
        if st["history"] is not None:
            kw.update(history=st["history"], length=st["length"], start=st["start"], prompt_len=st["prompt"],
                      repetition_penalty=st["repetition"], presence_penalty=st["presence"], frequency_penalty=st["frequency"])
        return ops.process_logits(st["logits"], **kw)
    st["source"].copy_rows(st["src"], st["dst"], tokens=c["tokens"], to=st["target"])
    return st["written"]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "attention":
        return _plain_attention(state).to(BF16)
    if op == "logits":
        return _plain_logits(state)
    return _plain_copy(state)


# ------------------------------------------------------------------------------------------------------------ references
def _exact_attention(st):
    """One softmax over all of a row's keys in 64 bits, kv head by kv head."""
    c = st["case"]
    t, s, rep = c["held"] + c["queries"], c["queries"], c["heads"] // c["kv_heads"]
    out = torch.empty(c["groups"] * c["each"], s, c["heads"], 128, dtype=F64, device="cuda")
    place = torch.arange(t, device="cuda")
    for b in range(out.shape[0]):
        i = b // c["each"]
        p0 = 0 if st["start"] is None else int(st["start"][i])
        o0 = 0 if st["own_start"] is None else int(st["own_start"][b])
        shut = (place[None, :] > c["held"] + torch.arange(s, device="cuda")[:, None]) | (place[None, :] < o0)
        for h in range(c["kv_heads"]):
            k = torch.cat([st["kp"][i, h, p0:], st["ko"][b, h, :t]]).to(F64)
            v = torch.cat([st["vp"][i, h, p0:], st["vo"][b, h, :t]]).to(F64)
            x = st["q"][b, :, h * rep:(h + 1) * rep].to(F64).reshape(s * rep, 128) @ k.t() / 128 ** 0.5
            x = x.reshape(s, rep, -1)
            x[:, :, -t:].masked_fill_(shut[:, None, :], float("-inf"))
            out[b, :, h * rep:(h + 1) * rep] = (torch.softmax(x, -1).reshape(s * rep, -1) @ v).reshape(s, rep, 128)
    return out.reshape(-1, c["heads"] * 128)


def _exact_logits(st):
    """Row by row in 64 bits, the seen tokens one list, the counts a histogram."""
    out = st["logits"].to(F64)
    for b in range(out.shape[0]):
        if st["history"] is not None:
            tok = st["history"][b, int(st["start"][b]):st["case"]["history"]].long()
            first_new = max(0, st["prompt"] - int(st["start"][b]))
            ids = torch.unique(tok)
            r = st["repetition"][b].to(F64)
            x = out[b, ids]
            out[b, ids] = torch.where(x < 0, x * r, x / r)
            count = torch.bincount(tok[first_new:], minlength=out.shape[1]).to(F64)
            out[b] -= st["frequency"][b].to(F64) * count + st["presence"][b].to(F64) * (count > 0)
        if st["bias"] is not None:
            out[b] += (st["bias"] if st["bias"].dim() == 1 else st["bias"][b]).to(F64)
        if st["allowed"] is not None:
            v = torch.arange(out.shape[1], device="cuda")
            words = st["allowed"][st["rows"][b].long()]
            out[b][(words[v // 32] >> (v % 32).to(torch.int32)) & 1 == 0] = float("-inf")
    return out


def exact(case, seed):
    if case["op"] in ("fork", "compact"):  # bits are moved: a row's 64-bit copies say the same
        st = prepare(case, seed)
        kv = case["kind"] == "kv"
        per_token = [p for spec in _specs(case) for _, _, p in _layer_shapes(spec, 1, case["room"])]
        outs = []
        for i, (a, b) in enumerate(zip(st["read"], st["written"])):
            a, b = a.to(F64), b.to(F64)
            for x, y in zip(st["src"], st["dst"]):
                if kv:
                    b[:, y, :, :case["tokens"]] = a[:, x, :, :case["tokens"]]
                elif per_token[i]:
                    b[y, :, :case["tokens"]] = a[x, :, :case["tokens"]]
                else:
                    b[y] = a[x]
            outs.append(b)
        return outs
    st = prepare(case, seed)
    if case["op"] == "logits":
        return _exact_logits(st)
    if case["groups"] * case["each"] * case["kv_heads"] * (case["prefix"] + 2000) > 60000000:
        return None
    return _exact_attention(st)


def work(case):
    c = case
    if c["op"] == "attention":
        b, t = c["groups"] * c["each"], c["held"] + c["queries"]
        nq = b * c["queries"] * c["heads"] * 128
        kv = c["kv_heads"] * 128 * (c["groups"] * c["prefix"] + b * t)
        own_keys = c["held"] + (c["queries"] + 1) / 2
        return {"bytes": 4 * nq + 4 * kv, "flops": int(4 * nq * (c["prefix"] + own_keys))}
    if c["op"] == "logits":
        b, v = c["rows"], c["vocab"]
        n = 8 * b * v + (4 * b * c["history"] if c["penalties"] else 0)
        n += {"none": 0, "shared": 4 * v, "rows": 4 * b * v}[c["bias"]] + min(c["masks"], b) * ((v + 31) // 32) * 4
        return {"bytes": n, "flops": 6 * b * v}
    rows = 0
    for spec in _specs(c):
        for shape, dtype, per_token in _layer_shapes(spec, 1, c["tokens"]):
            rows += math.prod(shape) * (2 if dtype == BF16 else 4)
    moved = 2 * c["live"] if c["op"] == "compact" else c["sources"] * (1 + c["each"])
    return {"bytes": rows * moved, "flops": 0}
