"""The serving operators from their definitions in 64 bits, with bounds on what rounding may do to them."""
import torch

F64 = torch.float64


def prefix_attention(q, kp, vp, ko, vo, slot, prefix_len=None, prefix_start=None, prefix_mask=None, kv_start=None):
    """(result, bound) ``[B * S, H * D]`` in 64 bits, query by query over the keys it attends alone. Bound: bf16 rounds the result and, on the
    matrix cores, each weight p by half a step (2^-8) at most, p's sum stays unrounded; 32-bit sums of D products put each score off by
    at most (D + 2) 2^-24 sum |q k|, and p by e times that, twice (the sum's); exponentials, sums and joins add 2^-16 of p at most."""
    b, s, h, d = q.shape
    g, hkv, p, _ = kp.shape
    rep, n = h // hkv, b // g
    out, bound = torch.zeros(b, s, h, d, dtype=F64), torch.zeros(b, s, h, d, dtype=F64)
    for i in range(b):
        j = i // n
        pre = torch.ones(p, dtype=torch.bool)
        at = torch.arange(p)
        if prefix_start is not None:
            pre &= at >= int(prefix_start[j])
        if prefix_len is not None:
            pre &= at < int(prefix_len[j])
        if prefix_mask is not None:
            pre &= prefix_mask[j] != 0
        first = max(0, int(kv_start[i])) if kv_start is not None else 0
        for t in range(s):
            upto = min(slot + t + 1, ko.shape[2])
            for e in range(h):
                k = torch.cat([kp[j, e // rep][pre], ko[i, e // rep, first:upto]]).to(F64)
                v = torch.cat([vp[j, e // rep][pre], vo[i, e // rep, first:upto]]).to(F64)
                if not len(k):
                    continue
                x = q[i, t, e].to(F64)
                w = torch.softmax(k @ x / d ** 0.5, 0)
                spread = float((k.abs() @ x.abs()).max()) / d ** 0.5 * (d + 2) * 2.0 ** -24
                out[i, t, e] = w @ v
                bound[i, t, e] = 2.0 ** -8 * out[i, t, e].abs() + (2.0 ** -8 + 2.0 ** -16 + 2 * 2.72 * spread) * (w @ v.abs()) * 1.01
    return out.reshape(b * s, h * d), bound.reshape(b * s, h * d)


def process_logits(x, history=None, length=0, start=None, history_mask=None, prompt_len=0, vocab_start=0, repetition_penalty=1.0,
                   presence_penalty=0.0, frequency_penalty=0.0, bias=None, allowed=None, allowed_rows=None):
    """(result, bound): token by token. ``allowed``: truth values [masks, all ids]. Bound: five operations in 32 bits, each off by 2^-24 of
    what it gives or takes."""
    b, v = x.shape
    out, size = x.to(F64).clone(), x.to(F64).abs()

    def of(val, i):
        return float(val[i]) if torch.is_tensor(val) else val

    for i in range(b):
        seen, count = set(), {}
        if history is not None:
            for p in range(max(0, 0 if start is None else int(start[i])), min(length, history.shape[1])):
                t = int(history[i, p]) - vocab_start
                if 0 <= t < v and (history_mask is None or history_mask[i, p]):
                    seen.add(t)
                    if p >= prompt_len:
                        count[t] = count.get(t, 0) + 1
        for t in seen:
            r = of(repetition_penalty, i)
            out[i, t] = out[i, t] * r if out[i, t] < 0 else out[i, t] / r
            size[i, t] = torch.maximum(size[i, t], out[i, t].abs())
            if t in count:
                less = of(frequency_penalty, i) * count[t] + of(presence_penalty, i)
                out[i, t] -= less
                size[i, t] += abs(of(frequency_penalty, i) * count[t]) + abs(of(presence_penalty, i))
        if bias is not None:
            add = (bias[i] if bias.dim() == 2 else bias).to(F64)
            out[i] += add
            size[i] += add.abs()
        if allowed is not None:
            r = int(allowed_rows[i]) if allowed_rows is not None else (i if allowed.shape[0] == b else 0)
            if 0 <= r < allowed.shape[0]:
                out[i][~allowed[r, vocab_start:vocab_start + v]] = float("-inf")
    return out, 5 * 2.0 ** -24 * size


def copied(tensors, src, dst, tokens, to=None):
    """Rows copied: ``tensors`` [(tensor, row axis, token axis or None)], ``to`` the tensors written (else the same)."""
    outs = []
    for i, (t, row, tok) in enumerate(tensors):
        o = (t if to is None else to[i][0]).clone()
        for a, b in zip(src, dst):
            part = o.select(row, b)
            new = torch.zeros_like(part) if a < 0 else t.select(row, a)
            if tok is not None:
                axis = tok - (tok > row)
                n = tokens
                part.narrow(axis, 0, n).copy_(new.narrow(axis, 0, n))
            else:
                part.copy_(new)
        outs.append(o)
    return outs
