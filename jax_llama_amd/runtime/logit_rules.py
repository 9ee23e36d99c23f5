"""What a generation does to its logits before a token is chosen: the settings of ``GenerationConfig`` on the device, and grammars."""
from __future__ import annotations

from typing import Dict, Optional, Sequence, Union

import torch

from .. import ops


class TokenGrammar:
    """A finite automaton over token ids: ``next_state [states, V]`` (integers) holds the state after a token, -1 where a state forbids it. A
    row starts in state ``start``; every state must allow a token (end tokens that may come are allowed like others)."""

    def __init__(self, next_state: torch.Tensor, start: int = 0):
        t = torch.as_tensor(next_state)
        if t.dim() != 2 or t.dtype.is_floating_point or not t.numel():
            raise ValueError("next_state is integers [states, V]")
        n = t.shape[0]
        if not 0 <= start < n or int(t.min()) < -1 or int(t.max()) >= n:
            raise ValueError(f"states lie in 0 .. {n - 1}, -1 forbids")
        if not bool((t >= 0).any(1).all()):
            raise ValueError("a state allows no token")
        self.next_state, self.start = t.to(torch.int32).contiguous(), int(start)
        self._on: Dict[torch.device, tuple] = {}

    def on(self, device) -> tuple:
        """(next_state, allowed bits) on ``device``."""
        device = torch.device(device)
        if device not in self._on:
            t = self.next_state.to(device)
            self._on[device] = t, ops.pack_allowed(t >= 0)
        return self._on[device]


def as_bias(bias: Union[Dict[int, float], torch.Tensor, None], suppress: Optional[Sequence[int]], vocab: int) -> Optional[torch.Tensor]:
    """``logit_bias`` and ``suppress_tokens`` as one fp32 ``[vocab]`` on the host, -inf for suppressed tokens; None without either."""
    if not torch.is_tensor(bias) and not bias and not suppress:
        return None
    if torch.is_tensor(bias):
        if tuple(bias.shape) != (vocab,):
            raise ValueError(f"logit_bias of shape {tuple(bias.shape)} for {vocab} tokens")
        out = bias.detach().to("cpu", torch.float32).clone()
    else:
        out = torch.zeros(vocab)
        for t, b in (bias or {}).items():
            if not 0 <= int(t) < vocab:
                raise ValueError(f"logit_bias: token {t} of {vocab}")
            out[int(t)] = float(b)
    for t in suppress or ():
        if not 0 <= int(t) < vocab:
            raise ValueError(f"suppress_tokens: token {t} of {vocab}")
        out[int(t)] = float("-inf")
    return out


class LogitRules:
    """One engine's rules: buffers that keep their place over calls (a captured step holds their addresses), filled by ``begin``."""

    def __init__(self, model, rows: int, max_length: int):
        dev = model.device
        self.model, self.rows = model, rows
        self.start = torch.zeros(rows, dtype=torch.int32, device=dev)
        self.state = torch.zeros(rows, dtype=torch.int32, device=dev)
        self.mask: Optional[torch.Tensor] = None
        self._mask_buf: Optional[torch.Tensor] = None
        self._bias_buf: Optional[torch.Tensor] = None
        self.max_length = max_length
        self.bias = self.grammar = self.config = None
        self.prompt_len = 0

    @property
    def vocab0(self) -> int:
        return self.model.comm.rank * self.model.vocab_local

    def begin(self, gc, prompt_len: int, start: torch.Tensor, mask: Optional[torch.Tensor]) -> None:
        """A new call's settings. ``start`` int32 ``[rows]``: the rows' first real tokens; ``mask`` uint8 ``[rows, max_length]`` or None."""
        v, dev = self.model.vocab_local, self.model.device
        vocab = v * self.model.comm.size
        bias = as_bias(gc.logit_bias, gc.suppress_tokens, vocab)
        self.bias = None
        if bias is not None:
            if self._bias_buf is None:
                self._bias_buf = torch.empty(v, dtype=torch.float32, device=dev)
            self.bias = self._bias_buf.copy_(bias[self.vocab0:self.vocab0 + v])
        self.grammar = gc.grammar
        if self.grammar is not None:
            if self.grammar.next_state.shape[1] != vocab:
                raise ValueError(f"the grammar is over {self.grammar.next_state.shape[1]} tokens, the model over {vocab}")
            self.grammar.on(dev)
            self.state.fill_(self.grammar.start)
        self.penalties = dict(repetition_penalty=float(gc.repetition_penalty), presence_penalty=float(gc.presence_penalty),
                              frequency_penalty=float(gc.frequency_penalty))
        self.penalised = self.penalties != dict(repetition_penalty=1.0, presence_penalty=0.0, frequency_penalty=0.0)
        self.prompt_len = prompt_len
        self.start.copy_(start)
        self.mask = None
        if mask is not None and self.penalised:
            if self._mask_buf is None:
                self._mask_buf = torch.empty(self.rows, self.max_length, dtype=torch.uint8, device=dev)
            self.mask = self._mask_buf.copy_(mask)

    @property
    def any(self) -> bool:
        return self.penalised or self.bias is not None or self.grammar is not None

    def key(self):
        """What a captured step has baked in."""
        if not self.any:
            return None
        return (tuple(self.penalties.values()), self.prompt_len if self.penalised else None, self.mask is not None, self.bias is not None, self.grammar)

    def apply(self, logits: torch.Tensor, sequences: torch.Tensor, cur_len: torch.Tensor) -> torch.Tensor:
        """The logits of the next token, in place."""
        kw = dict(self.penalties, history=sequences, length=cur_len, start=self.start, history_mask=self.mask,
                  prompt_len=self.prompt_len) if self.penalised else {}
        if self.grammar is not None:
            kw.update(allowed=self.grammar.on(logits.device)[1], allowed_rows=self.state)
        return ops.process_logits(logits, vocab_start=self.vocab0, bias=self.bias, out=logits, **kw)

    def chosen(self, tokens: torch.Tensor) -> None:
        """The rows' next tokens move their grammar states on (a finished row's are not looked at any more)."""
        if self.grammar is None:
            return
        table = self.grammar.on(tokens.device)[0]
        at = self.state.clamp(min=0).long() * table.shape[1] + tokens.long()
        self.state.copy_(table.reshape(-1).index_select(0, at))
