"""Copies of whole cache rows (``csrc/serving/cache_rows.hip``): forks of a request or a prompt, reordering, moving live rows to the
front, emptying rows. ``copy_rows`` of the cache objects (``models/kv_cache.py``) checks what it is asked for and comes here."""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch

from . import serving
from .slots import device_numbers

NOTHING = -1  # as a source: zeros


class RowLayout:
    """What a cache's rows are made of: tensors ``[rows, heads, tokens, width]`` (of which a row's first tokens go), and ``[rows, ...]``
    (recurrent state, which goes whole). ``parts``: of each tensor (runs, bytes of a run per token, bytes of a run without tokens)."""

    def __init__(self, tensors: Sequence[Tuple[torch.Tensor, bool]]):
        self.tensors = [(t, has) for t, has in tensors if t.numel()]
        self.parts: List[Tuple[int, int, int]] = []
        words: List[int] = []
        for t, has in self.tensors:
            es = t.element_size()
            part = (t.shape[1], t.shape[3] * es, 0) if has else (1, 0, t[0].numel() * es)
            if not t[0].is_contiguous():
                raise ValueError("a cache row must be one piece of each of its tensors")
            words += [t.data_ptr(), t.stride(0) * es, t.stride(1) * es if has else 0, *part]
            self.parts.append(part)
        self._words, self._table = words, None
        self._token_bytes = max((runs * per for runs, per, _ in self.parts), default=0)
        self._state_bytes = max((fixed for _, _, fixed in self.parts), default=0)

    def table(self) -> torch.Tensor:
        """The tensors' addresses and strides on the device."""
        if self._table is None:
            dev = self.tensors[0][0].device
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the first copy of a cache's rows cannot be captured: make one before")
            self._table = torch.tensor(self._words, dtype=torch.int64).reshape(-1, 6).to(dev)
        return self._table

    def widest(self, tokens: int) -> int:
        return max(self._token_bytes * tokens, self._state_bytes)


def check_pairs(src: Sequence[int], dst: Sequence[int], src_rows: int, dst_rows: int) -> None:
    if len(src) != len(dst):
        raise ValueError(f"{len(src)} sources for {len(dst)} rows")
    if any(not NOTHING <= r < src_rows for r in src):
        raise ValueError(f"source rows {list(src)} of a cache of {src_rows}")
    if any(not 0 <= r < dst_rows for r in dst):
        raise ValueError(f"rows {list(dst)} of a cache of {dst_rows}")
    if len(set(dst)) != len(dst):
        raise ValueError(f"a row is written twice: {list(dst)}")


def copy_rows(a: RowLayout, b: RowLayout, src: Sequence[int], dst: Sequence[int], tokens: int) -> None:
    """Row ``dst[i]`` of ``b`` becomes row ``src[i]`` of ``a`` (``NOTHING``: zeros). ``a is b``: every source is read as it was before."""
    if a.parts != b.parts:
        raise ValueError("the caches' rows are laid out differently")
    if not a.tensors or not len(dst):
        return
    if a.tensors[0][0].device != b.tensors[0][0].device:
        raise ValueError("the caches lie on different devices")
    if a.tensors[0][0].device.type != "cuda":
        _copy_cpu(a, b, src, dst, tokens)
        return
    e = serving.ext()
    steps, chains = e.plan_rows(src, dst, a is b)
    if not steps:
        return
    program: Optional[torch.Tensor] = None
    if len(steps) > 2 * e.ROW_STEPS:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"copies to more than some {e.ROW_STEPS} rows cannot be captured")
        program = device_numbers(steps + chains, torch.int32, a.tensors[0][0].device)
    e.copy_rows(a.table(), b.table(), steps, chains, program, tokens, a.widest(tokens))


def _copy_cpu(a: RowLayout, b: RowLayout, src, dst, tokens) -> None:
    for (t, has), (o, _) in zip(a.tensors, b.tensors):
        def part(x, row):
            return x[row, :, :tokens] if has else x[row]
        held = [torch.zeros_like(part(o, d)) if s == NOTHING else part(t, s).clone() for s, d in zip(src, dst)]
        for d, h in zip(dst, held):
            part(o, d).copy_(h)
