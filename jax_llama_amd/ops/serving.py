"""Ops of serving many continuations of shared prompts (``csrc/serving`` -> ``jax_llama_amd._C_serving``).

Same dispatch rule as the rest of ``ops``: GPU tensors run the hand-written gfx950 kernels (a missing extension raises), CPU
tensors the PyTorch implementation below. Shapes, types and ranges that the host can see are checked on both (for the GPU in
``csrc/serving/bindings.cpp``) and refused with a ValueError.

  * ``prefix_attention``: attention of a batch whose rows share prefixes -- continuations of one prompt, or prompts behind a
    common one -- whose keys and values are held and read once;
  * ``process_logits``: penalties for repeated tokens, biases, and masks (grammars, forbidden tokens) on logits;
  * copies of cache rows: ``copy_rows`` of the cache objects (``models/kv_cache.py``), planned in ``ops/cache_rows.py``.
"""
from __future__ import annotations

import importlib
import math
from typing import Optional, Union

import torch

BF16 = torch.bfloat16
F32 = torch.float32
HEAD_DIM = 128  # of the GPU kernels

_EXT = None
_ERR: Optional[BaseException] = None


def ext():
    """The native module, or a loud error saying how to build it."""
    global _EXT, _ERR
    if _EXT is None and _ERR is None:
        try:
            _EXT = importlib.import_module("jax_llama_amd._C_serving")
        except BaseException as e:  # ImportError, OSError (undefined symbol), ...
            _ERR = e
    if _EXT is None:
        raise RuntimeError("jax_llama_amd serving HIP extension is not available "
                           f"({type(_ERR).__name__}: {_ERR}). Build it with `python build.py --only serving` "
                           "(requires hipcc, targets gfx950). GPU tensors are never run on a fallback path.")
    return _EXT


def ext_available() -> bool:
    try:
        ext()
        return True
    except RuntimeError:
        return False


def _need(ok: bool, msg: str) -> None:
    if not ok:
        raise ValueError(msg)


def _ints(t, like: torch.Tensor, numel: int, name: str) -> None:
    if t is not None:
        _need(t.dtype == torch.int32 and t.numel() == numel and t.device == like.device and t.is_contiguous(),
              f"{name} must be a contiguous int32 tensor of {numel} elements on {like.device}")


# ---------------------------------------------------------------------------------- attention over shared prefixes
def prefix_attention(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor, k_cache: torch.Tensor,
                     v_cache: torch.Tensor, slot0, prefix_len: Optional[torch.Tensor] = None,
                     prefix_start: Optional[torch.Tensor] = None, prefix_mask: Optional[torch.Tensor] = None,
                     kv_start: Optional[torch.Tensor] = None, out_packed: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of ``q [B, S, H, D]`` over its rows' shared prefixes ``[G, Hkv, P, D]`` (row ``b`` reads prefix
    ``b // (B // G)``) and own keys ``[B, Hkv, T, D]``; returns ``[B * S, H * D]`` bf16. Query ``(b, s)`` attends

      * the prefix's keys ``prefix_start[g] <= j < prefix_len[g]`` with ``prefix_mask[g, j] != 0`` (int32 ``[G]``, uint8
        ``[G, P]`` on the device; left out: all ``P`` keys);
      * its row's own keys ``kv_start[b] <= j <= slot0 + s`` (``slot0``: an int or a device int32[1], ``kv_start`` int32 ``[B]``).

    A query with no key gives zeros. Maxima and sums are in 32 bits; on the GPU each weight is rounded to bf16 for the product with
    the values. What lies at places that no query of the call attends may be anything, NaN included; a value
    that some query attends has to be finite for the queries of its row before it. Keys and values may be views whose heads and rows
    are strided (the tokens of a head follow one another). ``out_packed``: see ``attention``, up to 64 rows."""
    if q.device.type == "cuda":
        return ext().prefix_attn(q, k_prefix, v_prefix, k_cache, v_cache, slot0, prefix_len, prefix_start, prefix_mask, kv_start, out_packed)
    return _prefix_attention_cpu(q, k_prefix, v_prefix, k_cache, v_cache, slot0, prefix_len, prefix_start, prefix_mask, kv_start)


def _prefix_attention_cpu(q, kp, vp, ko, vo, slot0, prefix_len, prefix_start, prefix_mask, kv_start) -> torch.Tensor:
    _need(q.dim() == 4 and kp.dim() == 4 and ko.dim() == 4, "prefix_attention takes q [B, S, H, D] and keys [rows, Hkv, tokens, D]")
    b, s, h, d = q.shape
    g, hkv, p, _ = kp.shape
    t = ko.shape[2]
    _need(min(b, s, h, g, hkv, p, t) > 0, "prefix_attention: an axis is empty")
    _need(b % g == 0, f"{b} rows are not a multiple of {g} prefixes")
    _need(h % hkv == 0, f"{h} heads are not a multiple of {hkv} key / value heads")
    _need(tuple(kp.shape) == tuple(vp.shape) == (g, hkv, p, d) and tuple(ko.shape) == tuple(vo.shape) == (b, hkv, t, d),
          f"prefix_attention: keys and values are [{g}, {hkv}, {p}, {d}] of the prefixes and [{b}, {hkv}, {t}, {d}] of the rows")
    _ints(prefix_len, q, g, "prefix_len")
    _ints(prefix_start, q, g, "prefix_start")
    _ints(kv_start, q, b, "kv_start")
    if prefix_mask is not None:
        _need(prefix_mask.dtype == torch.uint8 and tuple(prefix_mask.shape) == (g, p) and prefix_mask.is_contiguous()
              and prefix_mask.device == q.device, f"prefix_mask must be a contiguous uint8 [{g}, {p}] on {q.device}")
    if not torch.is_tensor(slot0):
        _need(0 <= int(slot0) and int(slot0) + s <= t, f"own slots {int(slot0)} .. {int(slot0) + s - 1} lie outside the cache's {t}")
    n, rep = b // g, h // hkv
    slot = int(slot0.reshape(-1)[0]) if torch.is_tensor(slot0) else int(slot0)
    place = torch.arange(p)[None, :]
    ok_p = torch.ones(g, p, dtype=torch.bool)
    if prefix_start is not None:
        ok_p &= place >= prefix_start[:, None]
    if prefix_len is not None:
        ok_p &= place < prefix_len[:, None]
    if prefix_mask is not None:
        ok_p &= prefix_mask != 0
    own = torch.arange(t)
    ok_o = (own[None, None, :] <= slot + torch.arange(s)[None, :, None]).expand(b, s, t)
    if kv_start is not None:
        ok_o = ok_o & (own[None, None, :] >= kv_start[:, None, None])

    def rows(x, ok):  # values nobody attends count as nothing, whatever they are
        return torch.where(ok[:, None, :, None], x.float(), torch.zeros(()))

    def heads(x):  # [B, Hkv, keys, D] -> [B, H, keys, D]
        return x.repeat_interleave(rep, 1)

    of = torch.arange(b) // n
    qf = q.float().transpose(1, 2)  # [B, H, S, D]
    kk = torch.cat([heads(rows(kp, ok_p)[of]), heads(rows(ko, ok_o.any(1)))], 2)
    vv = torch.cat([heads(rows(vp, ok_p)[of]), heads(rows(vo, ok_o.any(1)))], 2)
    ok = torch.cat([ok_p[of][:, None, :].expand(b, s, p), ok_o], 2)[:, None]
    x = (qf @ kk.transpose(-1, -2) / math.sqrt(d)).masked_fill(~ok, float("-inf"))
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == float("-inf"), torch.zeros(()), m))
    total = e.sum(-1, keepdim=True)
    o = (e @ vv) / torch.where(total == 0, torch.ones(()), total)
    return o.transpose(1, 2).reshape(b * s, h * d).to(BF16)


# ---------------------------------------------------------------------------------- logits
Number = Union[float, torch.Tensor]


def pack_allowed(allowed: torch.Tensor) -> torch.Tensor:
    """Truth values ``[masks, V]`` as the bits ``process_logits`` reads: int32 ``[masks, ceil(V / 32)]``, token ``v`` in bit ``v % 32`` of
    word ``v // 32``; bits past ``V`` are 0."""
    _need(allowed.dim() == 2, "pack_allowed takes [masks, V]")
    n, v = allowed.shape
    words = torch.empty(n, -(-v // 32), dtype=torch.int32, device=allowed.device)
    place = torch.arange(32, device=allowed.device)
    some = max(1, (1 << 22) // max(v, 1))  # masks at a time: 64 bits a token on the way
    for a in range(0, n, some):
        bits = torch.zeros(min(some, n - a), words.shape[1] * 32, dtype=torch.int64, device=allowed.device)
        bits[:, :v] = allowed[a:a + some] != 0
        packed = (bits.view(len(bits), -1, 32) << place).sum(-1)
        words[a:a + some] = torch.where(packed >= 1 << 31, packed - (1 << 32), packed)
    return words


def _neutral(v: Number, one: float) -> bool:
    return not torch.is_tensor(v) and float(v) == one


def process_logits(logits: torch.Tensor, history: Optional[torch.Tensor] = None, length=None, *, start: Optional[torch.Tensor] = None,
                   history_mask: Optional[torch.Tensor] = None, prompt_len: int = 0, vocab_start: int = 0,
                   repetition_penalty: Number = 1.0, presence_penalty: Number = 0.0, frequency_penalty: Number = 0.0,
                   bias: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None,
                   allowed_rows: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Penalties, biases and masks on fp32 ``logits [B, V]``, in this order:

      * ``repetition_penalty`` ``r`` on the tokens of a row's history: ``x < 0 ? x r : x / r``;
      * ``frequency_penalty`` times a token's occurrences from place ``prompt_len`` of the history on, and ``presence_penalty`` once if it
        has any, are subtracted;
      * ``bias`` (fp32 ``[V]`` or ``[B, V]``) is added;
      * tokens that are not ``allowed`` become -inf, whatever stood there.

    ``history`` int32 ``[B, L]`` holds the tokens; row ``b``'s are the places ``start[b] <= i < length`` (``start`` int32 ``[B]``, else 0;
    any numbers: a row that starts behind the end has no history; ``length`` an int or a device int32[1], so that a captured step sees the
    present one) with ``history_mask[b, i] != 0`` (uint8). Ids
    outside the columns are passed over. A penalty is a number or fp32 ``[B]``. ``allowed``: int32 bits ``[masks, words]``
    (``pack_allowed``), one mask for all, one per row, or row ``allowed_rows[b]`` of them (int32 ``[B]``; an index outside the masks allows
    everything). ``vocab_start``: token id of column 0 (a vocabulary shard); ``bias`` has the shard's columns, ``allowed`` all ids.
    ``out``: ``logits`` itself (in place) or another tensor."""
    if logits.device.type == "cuda":
        return ext().process_logits(logits, out, history, length, start, history_mask, prompt_len, vocab_start, repetition_penalty,
                                    presence_penalty, frequency_penalty, bias, allowed, allowed_rows)
    return _process_logits_cpu(logits, history, length, start, history_mask, prompt_len, vocab_start, repetition_penalty, presence_penalty,
                               frequency_penalty, bias, allowed, allowed_rows, out)


def _same(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and a.stride() == b.stride()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    def ends(t):
        return t.data_ptr(), t.data_ptr() + (sum((n - 1) * st for n, st in zip(t.shape, t.stride())) + 1) * t.element_size()
    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = ends(a), ends(b)
    return a0 < b1 and b0 < a1


def _process_logits_cpu(logits, history, length, start, history_mask, prompt_len, vocab_start, repetition_penalty, presence_penalty,
                        frequency_penalty, bias, allowed, allowed_rows, out) -> torch.Tensor:
    _need(logits.dim() == 2 and logits.dtype == F32, "process_logits takes fp32 logits [B, V]")
    b, v = logits.shape
    _need(v <= 1 or logits.stride(1) == 1, "logits must have unit inner stride")
    for name, val, lowest in (("repetition_penalty", repetition_penalty, 0.0), ("presence_penalty", presence_penalty, None),
                              ("frequency_penalty", frequency_penalty, None)):
        if torch.is_tensor(val):
            _need(val.dtype == F32 and tuple(val.shape) == (b,) and val.device == logits.device and val.is_contiguous(),
                  f"{name} must be a number or a contiguous fp32 [{b}] on {logits.device}")
        else:
            _need(math.isfinite(val) and (lowest is None or val > lowest), f"{name} = {val}")
    _need(vocab_start >= 0 and prompt_len >= 0, "vocab_start and prompt_len are not negative")
    if _neutral(repetition_penalty, 1.0) and _neutral(presence_penalty, 0.0) and _neutral(frequency_penalty, 0.0):
        history = None
    else:
        _need(history is not None and length is not None, "penalties need the history and its length")
    if history is not None:
        _need(history.dtype == torch.int32 and history.dim() == 2 and history.shape[0] == b and history.device == logits.device
              and (history.shape[1] <= 1 or history.stride(1) == 1), f"history must be int32 [{b}, L] on {logits.device} with unit inner stride")
        _ints(start, logits, b, "start")
        if history_mask is not None:
            _need(history_mask.dtype == torch.uint8 and history_mask.shape == history.shape and history_mask.device == logits.device
                  and (history.shape[1] <= 1 or history_mask.stride(1) == 1), "history_mask must be uint8 of the history's shape")
        if torch.is_tensor(length):
            _ints(length, logits, 1, "length")
        else:
            _need(0 <= int(length) <= history.shape[1], f"length {int(length)} of a history of {history.shape[1]}")
    if bias is not None:
        _need(bias.dtype == F32 and tuple(bias.shape) in ((v,), (b, v)) and bias.device == logits.device and (v <= 1 or bias.stride(-1) == 1),
              f"bias must be fp32 [{v}] or [{b}, {v}] on {logits.device}")
    if allowed is not None:
        _need(allowed.dtype == torch.int32 and allowed.dim() == 2 and allowed.shape[0] > 0 and allowed.shape[1] * 32 >= vocab_start + v
              and allowed.device == logits.device and allowed.stride(1) == 1,
              f"allowed must be int32 [masks, words] with bits for {vocab_start + v} tokens on {logits.device}")
        _ints(allowed_rows, logits, b, "allowed_rows")
        _need(allowed_rows is not None or allowed.shape[0] in (1, b), f"{allowed.shape[0]} masks for {b} rows: allowed_rows says which")
    else:
        _need(allowed_rows is None, "allowed_rows without allowed")
    if out is None:
        out = torch.empty(b, v, dtype=F32, device=logits.device)
    elif out is not logits:
        _need(out.dtype == F32 and out.shape == logits.shape and out.device == logits.device and (v <= 1 or out.stride(1) == 1),
              "out must be like the logits")
        _need(_same(out, logits) or not _overlap(out, logits), "out is the logits or shares nothing with them")
    if b > 1:  # rows of one output apart
        _need(out.stride(0) >= v, "rows of out overlap")
    x, rep, pres, freq = logits, repetition_penalty, presence_penalty, frequency_penalty
    y = x.clone()

    def col(val):
        return val[:, None] if torch.is_tensor(val) else val

    if history is not None:
        n = max(0, min(int(length.reshape(-1)[0]) if torch.is_tensor(length) else int(length), history.shape[1]))
        tok = history[:, :n].long() - vocab_start
        place = torch.arange(n)[None, :]
        real = (tok >= 0) & (tok < v)
        if start is not None:
            real &= place >= start[:, None]
        if history_mask is not None:
            real &= history_mask[:, :n] != 0
        at = tok.clamp(0, max(v - 1, 0))
        seen = torch.zeros(b, v, dtype=torch.int64).scatter_add_(1, at, real.long()) > 0
        count = torch.zeros(b, v, dtype=torch.int64).scatter_add_(1, at, (real & (place >= prompt_len)).long()).float()
        y = torch.where(seen, torch.where(y < 0, y * col(rep), y / col(rep)), y)
        y = torch.where(count > 0, y - col(freq) * count - col(pres), y)
    if bias is not None:
        y = y + bias
    if allowed is not None:
        r = allowed_rows.long() if allowed_rows is not None else (torch.arange(b) if allowed.shape[0] == b else torch.zeros(b, dtype=torch.long))
        known = (r >= 0) & (r < allowed.shape[0])
        t = vocab_start + torch.arange(v)
        bits = allowed[r.clamp(0, allowed.shape[0] - 1)][:, t // 32] >> (t % 32).to(torch.int32) & 1
        y = torch.where((bits == 1) | ~known[:, None], y, torch.full((), float("-inf")))
    out.copy_(y)
    return out
