"""What a generation does to its logits before a token is chosen: the settings of ``GenerationConfig`` on the device, and grammars."""
from __future__ import annotations

from typing import Dict, Optional, Sequence, Union

import torch

from .. import ops


class TokenGrammar:
    """A finite automaton over token ids: ``next_state [states, V]`` (integers) holds the state after a token, -1 where a state forbids it. A
    row starts in state ``start``; every state must allow a token (end tokens that may come are allowed like others). Where suppressed
    tokens leave a state that a row can come to without one, the generation is refused; a row whose logits leave it none (all -inf)
    ends there, as behind an end token. A device that it is used on keeps its tables: 4 (states + 1) V bytes of states and states V / 8 of
    masks (2000 states over 128256 tokens: 1.06 GB)."""

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
        """On ``device``: the states after each token, int32 ``[states + 1, V]`` with ``states`` (which stays itself) for forbidden ones, and
        the allowed tokens' bits."""
        device = torch.device(device)
        if device not in self._on:
            n, v = self.next_state.shape
            t = torch.empty(n + 1, v, dtype=torch.int32, device=device)
            t[:n] = self.next_state
            t[n] = n
            allowed = ops.pack_allowed(t[:n] >= 0)
            self._on[device] = t.masked_fill_(t < 0, n), allowed
        return self._on[device]

    def check_open(self, closed: torch.Tensor, device) -> None:
        """A ValueError if a row can come to a state that allows ``closed`` tokens (truth values ``[V]``) alone."""
        table, n, opened = self.on(device)[0], self.next_state.shape[0], ~closed.to(device)
        some = max(1, (1 << 26) // table.shape[1])  # states at a time
        live = torch.cat([((table[a:min(n, a + some)] < n) & opened).any(1) for a in range(0, n, some)]).cpu()
        seen = todo = set() if bool(live.all()) else {self.start}
        while todo:
            if not bool(live[sorted(todo)].all()):
                raise ValueError(f"states {[s for s in sorted(todo) if not live[s]][:8]} of the grammar allow suppressed tokens alone")
            at, todo = sorted(todo), set()
            for a in range(0, len(at), some):
                t = table[at[a:a + some]]
                todo |= set(torch.unique(t[(t < n) & opened]).tolist())
            todo -= seen
            seen = seen | todo


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
        self.bias = self.grammar = self.table = self.allowed = None
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
        closed = None if bias is None else bias == float("-inf")
        if closed is not None and bool(closed.all()):
            raise ValueError("every token is suppressed")
        if bias is not None:
            if self._bias_buf is None:
                self._bias_buf = torch.empty(v, dtype=torch.float32, device=dev)
            self.bias = self._bias_buf.copy_(bias[self.vocab0:self.vocab0 + v])
        self.grammar = gc.grammar
        if self.grammar is not None:
            if self.grammar.next_state.shape[1] != vocab:
                raise ValueError(f"the grammar is over {self.grammar.next_state.shape[1]} tokens, the model over {vocab}")
            if closed is not None and bool(closed.any()):
                self.grammar.check_open(closed, dev)
            self.table, self.allowed = self.grammar.on(dev)
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
            kw.update(allowed=self.allowed, allowed_rows=self.state)
        return ops.process_logits(logits, vocab_start=self.vocab0, bias=self.bias, out=logits, **kw)

    def chosen(self, tokens: torch.Tensor, finished: torch.Tensor) -> None:
        """The rows' next tokens move their grammar states on (a finished row's are not looked at any more). A token that the grammar
        forbids is the choice among -inf alone: the row is ``finished`` before it is said."""
        if self.grammar is None:
            return
        states, vocab = self.table.shape
        at = self.state.long().mul_(vocab).add_(tokens.clamp(0, vocab - 1))
        torch.index_select(self.table.reshape(-1), 0, at, out=self.state)
        finished.bitwise_or_(self.state == states - 1)
