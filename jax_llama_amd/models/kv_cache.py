"""Static, pre-allocated KV cache.

Reference: Flax ``"cache"`` collection created by ``init_cache`` (``model.py:459-476``) and
updated by ``_concatenate_to_cache`` (``model.py:169-199``): per layer ``cached_key`` /
``cached_value`` of shape ``(B, T_max, Hkv, Dh)`` holding post-RoPE keys, plus a scalar
``cache_index`` advanced by the number of tokens written.

Here: two tensors ``[L, B, Hkv_local, T_max, Dh]`` (bf16) so that one (b, kv-head)'s keys
are a single contiguous ``T x 256 B`` run — the decode attention kernel streams it with
1 KiB-per-wave-instruction loads — and the slot index is mirrored in a device int32 so
hipGraph-captured decode steps read/advance it without host round trips. No forward pass
is run to create it (unlike the reference's ``module.init`` trick).
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from ..ops import cache_rows


def _copy_rows(cache, src, dst, tokens, to) -> None:
    target = cache if to is None else to
    if type(target) is not type(cache):
        raise ValueError(f"rows of a {type(cache).__name__} go to a {type(cache).__name__}, not to a {type(target).__name__}")
    tokens = cache.index if tokens is None else int(tokens)
    if not 0 <= tokens <= min(cache.max_length, target.max_length):
        raise ValueError(f"{tokens} tokens of rows of {cache.max_length} and {target.max_length}")
    cache.row_layout().copy(target.row_layout(), src, dst, tokens)


class KVCache:
    def __init__(self, num_layers: int, batch_size: int, num_kv_heads: int, max_length: int,
                 head_dim: int, device, dtype=torch.bfloat16):
        device = torch.device(device)
        shape = (num_layers, batch_size, num_kv_heads, max_length, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.batch_size = batch_size
        self.max_length = max_length
        self.index = 0  # host mirror of the number of filled slots
        self.index_t = torch.zeros(1, dtype=torch.int32, device=device)
        self._start: Optional[torch.Tensor] = None  # keeps its place once there (captured copies write it); zeros where nothing is padded
        self._padded = False
        self._row_layout = None

    @property
    def device(self):
        return self.k.device

    @property
    def start(self) -> Optional[torch.Tensor]:
        """int32 ``[B]``: a left-padded prefix's first real slot of each row (``encode_prefix``); None: every row begins at slot 0."""
        return self._start if self._padded else None

    @start.setter
    def start(self, start: Optional[torch.Tensor]) -> None:
        self._padded = start is not None
        if self._start is None and start is not None:
            self._start = torch.zeros(self.batch_size, dtype=torch.int32, device=self.device)
        if self._start is not None:
            self._start.zero_() if start is None else self._start.copy_(start)

    def row_layout(self) -> cache_rows.RowLayout:
        starts = () if self._start is None else (self._start,)
        at = tuple(t.data_ptr() for t in (self.k, self.v, *starts))
        if self._row_layout is None or self._row_layout[0] != at:
            self._row_layout = at, cache_rows.RowLayout(self.batch_size, layers=(self.k, self.v), state=starts)
        return self._row_layout[1]

    def copy_rows(self, src: Sequence[int], dst: Sequence[int], tokens: Optional[int] = None, to: Optional["KVCache"] = None) -> None:
        """Row ``dst[i]`` becomes row ``src[i]`` (-1: zeros) in every layer, its first ``tokens`` tokens (default: as many as the cache
        holds by its host counter): forks, reordering, moving live rows to the front. Every source is read as it was before the call; a row is
        written once at most. A padded row's ``start`` goes with it. ``to``: the rows written are those of another cache with the same layers
        (whose slot counter stays as it is). One launch; up to some 300 rows also while a stream is captured, once the caches have copied
        rows before."""
        if isinstance(to, KVCache):
            for cache, other in ((self, to), (to, self)):
                if cache._start is None and other._start is not None:
                    if cache.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("the first copy between a padded prefix and a cache without padding cannot be captured: make one before")
                    cache._start = torch.zeros(cache.batch_size, dtype=torch.int32, device=cache.device)
        _copy_rows(self, src, dst, tokens, to)
        if isinstance(to, KVCache):
            to._padded = to._padded or self._padded

    def layer(self, i: int):
        return self.k[i], self.v[i]

    def advance(self, n: int) -> None:
        self.index += n
        self.index_t.add_(n)

    def reset(self) -> None:
        self.index = 0
        self.index_t.zero_()
        self.start = None

    def clear(self) -> None:
        """``reset`` and zero the keys and values (after a failed step may have left non-finite rows)."""
        self.reset()
        self.k.zero_()
        self.v.zero_()

    def rows(self, b0: int, b1: int) -> "KVCacheRows":
        """The cache of batch rows ``[b0, b1)`` (every layer): a view whose per-layer K / V are contiguous slices, for a
        prefill run in row chunks (runtime/engine.py)."""
        return KVCacheRows(self, b0, b1)

    def nbytes(self) -> int:
        return 2 * self.k.numel() * self.k.element_size()

    # Flax-cache-like view for API parity / debugging (per-layer dict, (B, T, Hkv, Dh)).
    def as_dict(self):
        return {
            str(i): {
                "cached_key": self.k[i].permute(0, 2, 1, 3),
                "cached_value": self.v[i].permute(0, 2, 1, 3),
                "cache_index": self.index,
            }
            for i in range(self.k.shape[0])
        }


class KVCacheRows:
    """Rows ``[b0, b1)`` of a KVCache: ``layer(i)`` gives contiguous ``[b1 - b0, Hkv, T, Dh]`` views; the slot index is
    the parent's (one position for every row)."""

    def __init__(self, parent: KVCache, b0: int, b1: int):
        self.parent = parent
        self.b0, self.b1 = b0, b1
        self.batch_size = b1 - b0
        self.max_length = parent.max_length

    @property
    def device(self):
        return self.parent.device

    @property
    def index(self):
        return self.parent.index

    @property
    def index_t(self):
        return self.parent.index_t

    @property
    def start(self):
        return None if self.parent.start is None else self.parent.start[self.b0:self.b1]

    def layer(self, i: int):
        return self.parent.k[i, self.b0:self.b1], self.parent.v[i, self.b0:self.b1]

    def rows(self, b0: int, b1: int) -> "KVCacheRows":
        return KVCacheRows(self.parent, self.b0 + b0, self.b0 + b1)


class SharedPrefixCache:
    """A batch's own cache behind prefixes that its rows share: row ``b`` of ``B`` continues row ``b // (B / G)`` of ``prefix`` (a KVCache of
    ``G`` rows holding the prefixes' keys and values, read once for all of a prefix's rows: ``ops.prefix_attention``). Slots, ``index`` and
    ``layer(i)`` are those of ``own``; positions go on where the prefix ends. ``start`` / ``mask``: the prefixes' first keys (int32
    ``[G]``; left out: the prefix's own ``start``, as it is at each call) and the keys that count (uint8 ``[G, capacity]``). Anything that
    writes here writes to ``own`` alone."""

    def __init__(self, prefix: KVCache, own, start: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None):
        if own.batch_size % prefix.batch_size:
            raise ValueError(f"{own.batch_size} rows are not a multiple of {prefix.batch_size} prefixes")
        if prefix.device != own.device:
            raise ValueError(f"the prefixes lie on {prefix.device}, the rows on {own.device}")
        self.prefix, self.own, self._start, self.mask = prefix, own, start, mask
        self.prefix_len = torch.full((prefix.batch_size,), prefix.index, dtype=torch.int32, device=prefix.device)
        self.batch_size, self.max_length = own.batch_size, own.max_length

    @property
    def device(self):
        return self.own.device

    @property
    def start(self) -> Optional[torch.Tensor]:
        return self._start if self._start is not None else self.prefix.start

    @property
    def index(self):
        return self.own.index

    @index.setter
    def index(self, n):
        self.own.index = n

    @property
    def index_t(self):
        return self.own.index_t

    def layer(self, i: int):
        return self.own.layer(i)

    def prefix_layer(self, i: int):
        return self.prefix.layer(i)

    def advance(self, n: int) -> None:
        self.own.advance(n)

    def reset(self) -> None:
        self.own.reset()

    def clear(self) -> None:
        self.own.clear()

    def copy_rows(self, src: Sequence[int], dst: Sequence[int], tokens: Optional[int] = None) -> None:
        """``KVCache.copy_rows`` of the own rows; a row only goes to rows of its own prefix."""
        n = self.batch_size // self.prefix.batch_size
        if any(a >= 0 and a // n != b // n for a, b in zip(src, dst)):
            raise ValueError("a row would continue another prefix")
        self.own.copy_rows(src, dst, tokens)

    def rows(self, b0: int, b1: int) -> "SharedPrefixCache":
        """Rows ``[b0, b1)``: whole prefixes' rows, or some of one prefix's."""
        n = self.batch_size // self.prefix.batch_size
        g0, g1 = b0 // n, -(-b1 // n)
        if g1 - g0 > 1 and (b0 % n or b1 % n):
            raise ValueError(f"rows {b0} .. {b1 - 1} hold some of one prefix's rows and others")
        part = SharedPrefixCache.__new__(SharedPrefixCache)
        part.prefix, part.own = self.prefix.rows(g0, g1), self.own.rows(b0, b1)
        part._start, part.mask = (t[g0:g1] if t is not None else None for t in (self._start, self.mask))
        part.prefix_len, part.batch_size, part.max_length = self.prefix_len[g0:g1], b1 - b0, self.max_length
        return part

    def nbytes(self) -> int:
        return self.own.nbytes()


TICKET_INTS = 64 * 32  # tickets of a cache row that has some: 64, each on a line of its own (csrc: AS_TICKET)


class HybridCache:
    """Per-layer sequence state of a stack that mixes attention and recurrent layers, pre-allocated.

    ``specs[i]`` describes layer ``i``:
      * ``("kv", kv_heads, dim, vdim)``: keys ``[B, G, T, dim]`` and values ``[B, G, T, vdim]`` (head sizes are per
        layer, keys and values may differ in width);
      * ``("latent", rank)``: one vector of ``rank`` numbers per token, ``[B, 1, T, rank]``; ``layer(i)`` returns it as
        both keys and values (every head's keys and values are linear maps of it, applied outside the cache);
      * ``("kv_from", j)``: no storage, ``layer(i)`` is layer ``j``'s keys and values (cross-layer KV sharing);
      * ``("delta", heads, kv_heads, dim, vdim, taps)``: a recurrent state ``[B, H, dim, vdim]`` (always fp32) and
        the short convolutions' input tail ``[B, 2 G dim + H vdim, taps - 1]`` (fp32);
      * ``("mlstm", heads, dim, vdim)``: a matrix memory with its normaliser as one more value column
        ``[B, H, dim, vdim + 1]`` and the running maximum of its gates ``[B, H]`` (fp32);
      * ``("timemix", heads, dim, vdim, width)``: a matrix memory ``[B, H, dim, vdim]`` and the previous token's
        mixer input ``[B, width]`` (fp32);
      * ``("linear", heads, dim, vdim)``: a matrix state alone ``[B, H, dim, vdim]`` (fp32);
      * ``("multi", spec, spec, ...)``: a layer whose mixers run side by side, each with its own entry (at most one
        that holds keys and one that is recurrent);
      * ``None``: nothing.
    The slot index (tokens held, the same for every row) is mirrored on the device like ``KVCache``'s, so captured
    decode steps advance it without the host. ``dtype`` is the key / value element type (bf16, or fp32 for exact runs).
    Recurrent state has no slot: ``reset`` zeroes it, since a new sequence starts from a zero state."""

    def __init__(self, specs, batch_size: int, max_length: int, device, dtype=torch.bfloat16):
        device = torch.device(device)
        self.specs = list(specs)
        self.batch_size = batch_size
        self.max_length = max_length
        self.dtype = dtype
        self._k, self._v, self._state, self._conv = {}, {}, {}, {}
        for i, sp in enumerate(self.specs):
            for part in self.parts(sp):
                self._alloc(i, part, batch_size, max_length, dtype, device)
        self._device = device
        self._row_layout = None
        self.index = 0
        self.index_t = torch.zeros(1, dtype=torch.int32, device=device)
        # counters of the one-launch decode steps (ops.hybrid.attn_step, delta_step), which leave them at zero: part of the cache because
        # two steps on one cache are never in flight at once. None where no layer takes those steps
        self._row_tickets = self.tickets_per_row(self.specs)
        self.tickets = torch.zeros(batch_size * self._row_tickets, dtype=torch.int32, device=device) if self._row_tickets else None

    @staticmethod
    def tickets_per_row(specs) -> int:
        """Counters (int32) of a cache row: for key / value heads of 64 or 128 numbers and delta rules of four taps, else none."""
        sizes = (64, 128)
        some = any(sp[0] == "kv" and sp[2] in sizes and sp[3] in sizes or sp[0] == "delta" and sp[5] == 4
                   for layer in specs for sp in HybridCache.parts(layer))
        return TICKET_INTS if some else 0

    @staticmethod
    def parts(sp) -> list:
        """The primitive entries of a layer's spec."""
        if sp is None:
            return []
        if sp[0] == "multi":
            kinds = [p[0] for p in sp[1:]]
            if sum(k in ("kv", "latent", "kv_from") for k in kinds) > 1 or \
                    sum(k in ("delta", "mlstm", "timemix", "linear") for k in kinds) > 1:
                raise ValueError(f"a layer holds at most one key / value entry and one recurrent entry: {sp!r}")
            return list(sp[1:])
        return [sp]

    def _alloc(self, i: int, sp, batch_size: int, max_length: int, dtype, device) -> None:
        f32 = dict(dtype=torch.float32, device=device)
        if sp[0] == "kv":
            _, g, dim, vdim = sp
            self._k[i] = torch.zeros(batch_size, g, max_length, dim, dtype=dtype, device=device)
            self._v[i] = torch.zeros(batch_size, g, max_length, vdim, dtype=dtype, device=device)
        elif sp[0] == "latent":
            self._k[i] = self._v[i] = torch.zeros(batch_size, 1, max_length, sp[1], dtype=dtype, device=device)
        elif sp[0] == "kv_from":
            j = sp[1]
            if not (0 <= j < i) or self.specs[j] is None or self.specs[j][0] != "kv":
                raise ValueError(f"layer {i} shares the keys / values of layer {j}, which holds none before it")
        elif sp[0] == "delta":
            _, h, g, dim, vdim, taps = sp
            self._state[i] = torch.zeros(batch_size, h, dim, vdim, **f32)
            self._conv[i] = torch.zeros(batch_size, 2 * g * dim + h * vdim, max(taps - 1, 0), **f32)
        elif sp[0] == "mlstm":
            _, h, dim, vdim = sp
            self._state[i] = torch.zeros(batch_size, h, dim, vdim + 1, **f32)
            self._conv[i] = torch.zeros(batch_size, h, **f32)
        elif sp[0] == "timemix":
            _, h, dim, vdim, width = sp
            self._state[i] = torch.zeros(batch_size, h, dim, vdim, **f32)
            self._conv[i] = torch.zeros(batch_size, width, **f32)
        elif sp[0] == "linear":
            self._state[i] = torch.zeros(batch_size, *sp[1:], **f32)
        else:
            raise ValueError(f"unknown cache spec {sp!r}")

    @property
    def device(self):
        return self._device

    def row_layout(self) -> cache_rows.RowLayout:
        if self._row_layout is None:
            held = {id(t): t for d in (self._k, self._v) for t in d.values()}.values()
            self._row_layout = cache_rows.RowLayout(self.batch_size, tokens=held, state=[t for d in (self._state, self._conv) for t in d.values()])
        return self._row_layout

    def copy_rows(self, src: Sequence[int], dst: Sequence[int], tokens: Optional[int] = None, to: Optional["HybridCache"] = None) -> None:
        """``KVCache.copy_rows``, with the rows' whole recurrent state."""
        _copy_rows(self, src, dst, tokens, to)

    def layer(self, i: int):
        """Keys and values layer ``i`` attends over (its own, or the layer's it shares them with)."""
        j = i
        for part in self.parts(self.specs[i]):
            if part[0] == "kv_from":
                j = part[1]
        return self._k[j], self._v[j]

    def owns_kv(self, i: int) -> bool:
        return any(part[0] == "kv" for part in self.parts(self.specs[i]))

    def recurrent(self, i: int):
        """The two carried tensors of a recurrent layer: ``(state, convolution tail)`` (delta), ``(state with the
        normaliser column, running maximum)`` (mlstm), ``(state, previous token's input)`` (timemix) or ``(state, None)``
        (linear)."""
        return self._state[i], self._conv.get(i)

    def advance(self, n: int) -> None:
        self.index += n
        self.index_t.add_(n)

    def reset(self) -> None:
        """Empty: slot 0, zero recurrent state (keys and values past the slot are never read)."""
        self.index = 0
        self.index_t.zero_()
        for t in list(self._state.values()) + list(self._conv.values()):
            t.zero_()

    def clear(self) -> None:
        """``reset`` and zero the keys and values too (after a failed step may have left non-finite rows)."""
        self.reset()
        if self.tickets is not None:
            self.tickets.zero_()
        for t in {id(t): t for t in list(self._k.values()) + list(self._v.values())}.values():
            t.zero_()

    def rows(self, b0: int, b1: int) -> "HybridCacheRows":
        return HybridCacheRows(self, b0, b1)

    def nbytes(self) -> int:
        seen = {id(t): t for d in (self._k, self._v, self._state, self._conv) for t in d.values()}
        return sum(t.numel() * t.element_size() for t in seen.values()) + 4 * self.batch_size * self._row_tickets

    @staticmethod
    def bytes_per(specs, batch_size: int, max_length: int, dtype=torch.bfloat16) -> int:
        """Bytes a cache of this geometry takes (without allocating it)."""
        es = torch.empty(0, dtype=dtype).element_size()
        n = 4 * batch_size * HybridCache.tickets_per_row(specs)
        for layer in specs:
            for sp in HybridCache.parts(layer):
                if sp[0] == "kv":
                    n += batch_size * sp[1] * max_length * (sp[2] + sp[3]) * es
                elif sp[0] == "latent":
                    n += batch_size * max_length * sp[1] * es
                elif sp[0] == "delta":
                    _, h, g, dim, vdim, taps = sp
                    n += 4 * batch_size * (h * dim * vdim + (2 * g * dim + h * vdim) * max(taps - 1, 0))
                elif sp[0] == "mlstm":
                    n += 4 * batch_size * sp[1] * (sp[2] * (sp[3] + 1) + 1)
                elif sp[0] == "timemix":
                    n += 4 * batch_size * (sp[1] * sp[2] * sp[3] + sp[4])
                elif sp[0] == "linear":
                    n += 4 * batch_size * sp[1] * sp[2] * sp[3]
        return n


class HybridCacheRows:
    """Rows ``[b0, b1)`` of a HybridCache (contiguous slices of every tensor; the slot index is the parent's)."""

    def __init__(self, parent: HybridCache, b0: int, b1: int):
        self.parent = parent
        self.b0, self.b1 = b0, b1
        self.batch_size = b1 - b0
        self.max_length = parent.max_length
        self.specs = parent.specs

    @property
    def device(self):
        return self.parent.device

    @property
    def index(self):
        return self.parent.index

    @property
    def index_t(self):
        return self.parent.index_t

    @property
    def tickets(self):
        per = self.parent._row_tickets
        return self.parent.tickets[self.b0 * per:self.b1 * per] if per else None

    def layer(self, i: int):
        k, v = self.parent.layer(i)
        return k[self.b0:self.b1], v[self.b0:self.b1]

    def rows(self, b0: int, b1: int) -> "HybridCacheRows":
        return HybridCacheRows(self.parent, self.b0 + b0, self.b0 + b1)

    def owns_kv(self, i: int) -> bool:
        return self.parent.owns_kv(i)

    def recurrent(self, i: int):
        s, c = self.parent.recurrent(i)
        return s[self.b0:self.b1], c[self.b0:self.b1] if c is not None else None
