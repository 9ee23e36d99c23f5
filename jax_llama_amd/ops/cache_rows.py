"""Copies of whole cache rows (``csrc/serving/cache_rows.hip``): forks of a request or a prompt, reordering, moving live rows to the
front, emptying rows. ``copy_rows`` of the cache objects (``models/kv_cache.py``) checks what it is asked for and comes here."""
from __future__ import annotations

from typing import List, Sequence, Tuple

import torch

from . import serving

NOTHING = -1  # as a source: zeros


class RowLayout:
    """What the rows of a cache of ``rows`` rows are made of. ``layers``: tensors ``[layers, rows, heads, tokens, width]``, ``tokens``:
    ``[rows, heads, tokens, width]`` (of both a row's first tokens go), ``state``: ``[rows, ...]`` (goes whole)."""

    def __init__(self, rows: int, layers: Sequence[torch.Tensor] = (), tokens: Sequence[torch.Tensor] = (), state: Sequence[torch.Tensor] = ()):
        self.rows = rows
        self.layers, self.tensors = list(layers), [(t, True) for t in tokens] + [(t, False) for t in state if t.numel()]
        self.parts: List[Tuple[int, ...]] = []
        self.types: List[torch.dtype] = []
        self.words: List[int] = []  # eight numbers a span: csrc/serving/serving.h RowSpan
        for t in self.layers:
            self._add(t, t.shape[1:], t.stride()[1:], True, t.shape[0], t.stride(0))
        for t, has in self.tensors:
            self._add(t, t.shape, t.stride(), has, 1, 0)
        held = self.layers + [t for t, _ in self.tensors]
        self.on = held[0] if held and held[0].device.type == "cuda" else None
        self._native = None

    def _add(self, t: torch.Tensor, shape, stride, has_tokens: bool, layers: int, layer_stride: int) -> None:
        es = t.element_size()
        if has_tokens:
            ok, part = stride[3] == 1 and stride[2] == shape[3], (layers, shape[1], shape[3] * es, 0)
        else:
            ok, n = True, 1
            for size, step in zip(reversed(shape[1:]), reversed(stride[1:])):
                ok, n = ok and (size == 1 or step == n), n * size
            part = (layers, 1, 0, n * es)
        if not ok:
            raise ValueError("a cache row must be one piece of each of its tensors")
        self.types.append(t.dtype)
        self.words += [t.data_ptr(), stride[0] * es, layer_stride * es, stride[1] * es if has_tokens else 0, *part]
        self.parts.append(part)

    def copy(self, to: "RowLayout", src: Sequence[int], dst: Sequence[int], tokens: int) -> None:
        """Row ``dst[i]`` of ``to`` becomes row ``src[i]`` (``NOTHING``: zeros). ``to is self``: every source is read as it was before."""
        if self.types != to.types:
            raise ValueError("the caches are laid out differently")
        if (self.on is None) != (to.on is None):
            raise ValueError("the caches lie on different devices")
        if self.on is None:
            self._copy_cpu(to, [int(r) for r in src], [int(r) for r in dst], tokens)
            return
        for a in (self, to):
            if a._native is None:
                a._native = serving.ext().RowLayout(a.words, a.rows, a.on)
        self._native.copy(to._native, src, dst, tokens)

    def _copy_cpu(self, to: "RowLayout", src: List[int], dst: List[int], tokens: int) -> None:
        if self.parts != to.parts:
            raise ValueError("the caches are laid out differently")
        if len(src) != len(dst):
            raise ValueError(f"{len(src)} sources for {len(dst)} rows")
        if any(not NOTHING <= r < self.rows for r in src):
            raise ValueError(f"source rows {src} of a cache of {self.rows}")
        if any(not 0 <= r < to.rows for r in dst):
            raise ValueError(f"rows {dst} of a cache of {to.rows}")
        if len(set(dst)) != len(dst):
            raise ValueError(f"a row is written twice: {dst}")
        def each(a):
            return [(x, True) for t in a.layers for x in t] + a.tensors
        for (t, has), (o, _) in zip(each(self), each(to)):
            def part(x, row):
                return x[row, :, :tokens] if has else x[row]
            held = [torch.zeros_like(part(o, d)) if s == NOTHING else part(t, s).clone() for s, d in zip(src, dst)]
            for d, h in zip(dst, held):
                part(o, d).copy_(h)
