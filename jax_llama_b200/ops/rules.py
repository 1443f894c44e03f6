"""What a request asks of its tokens beyond sampling: penalties for tokens that occurred, biases, a set of allowed tokens.

`LogitRules` is what a caller writes down; `bind` turns it into the tensors that `kernels.constrain_logits` reads, once per request batch, so that a captured decode
step finds them where they were and a later batch of the same form only copies new numbers into them.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from numbers import Integral
from typing import Any, Dict, Iterable, List, Optional, Sequence, Tuple, Union

import torch

from . import kernels as K

PerRow = Union[float, Sequence[float]]


def allowed_mask(ids: Iterable[int], vocab_size: int) -> torch.Tensor:
    """int32 [words] with bit v % 32 of word v // 32 set for every v in `ids`."""
    bits = torch.zeros((vocab_size + 31) // 32 * 32, dtype=torch.int64)
    idx = torch.as_tensor(list(ids), dtype=torch.long)
    if idx.numel() and (int(idx.min()) < 0 or int(idx.max()) >= vocab_size):
        raise ValueError(f"allowed tokens outside 0..{vocab_size - 1}")
    bits[idx] = 1
    words = (bits.view(-1, 32) << torch.arange(32)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


@dataclass
class LogitRules:
    """repetition_penalty r > 0: logits of tokens that occurred, prompt included, become x / r (x > 0) or x · r.  frequency_penalty f, presence_penalty p: with n
    occurrences in the answer, n > 0, x - f · n - p.  Each a number, or one per row of the batch.  logit_bias: {token: bias}, or one such dict per row.
    allowed_tokens: token ids (None: all), one such list per row, or the masks themselves (int32 [words] or [rows, words], see `allowed_mask`).  With several
    answers per prompt, rows are prompts."""

    repetition_penalty: PerRow = 1.0
    frequency_penalty: PerRow = 0.0
    presence_penalty: PerRow = 0.0
    logit_bias: Union[Dict[int, float], Sequence[Dict[int, float]], None] = None
    allowed_tokens: Any = None

    @property
    def active(self) -> bool:
        def differs(v: PerRow, off: float) -> bool:
            return any(float(x) != off for x in v) if isinstance(v, (list, tuple)) or torch.is_tensor(v) else float(v) != off
        return differs(self.repetition_penalty, 1.0) or differs(self.frequency_penalty, 0.0) or differs(self.presence_penalty, 0.0) \
            or bool(self.logit_bias) or self.allowed_tokens is not None

    def bind(self, rows: int, vocab_size: int, device: Any, repeat: int = 1) -> "BoundRules":
        """The tensors for `rows` prompts with `repeat` answers each."""
        B = rows * repeat

        def per_row(v: PerRow, name: str) -> torch.Tensor:
            t = torch.as_tensor([float(x) for x in v] if isinstance(v, (list, tuple)) or torch.is_tensor(v) else [float(v)] * rows, dtype=torch.float32)
            if t.shape != (rows,) or not bool(torch.isfinite(t).all()):
                raise ValueError(f"{name}: a finite number, or one per row ({rows}), got {v}")
            return t.repeat_interleave(repeat)

        rep = per_row(self.repetition_penalty, "repetition_penalty")
        if bool((rep <= 0).any()):
            raise ValueError(f"repetition_penalty {self.repetition_penalty} is not above zero")
        freq, pres = per_row(self.frequency_penalty, "frequency_penalty"), per_row(self.presence_penalty, "presence_penalty")
        said = bool((rep != 1).any() or (freq != 0).any() or (pres != 0).any())
        ids = vals = None
        if self.logit_bias:
            lists: List[Dict[int, float]] = [self.logit_bias] if isinstance(self.logit_bias, dict) else list(self.logit_bias)
            if len(lists) not in (1, rows) or (not isinstance(self.logit_bias, dict) and len(lists) != rows):
                raise ValueError(f"logit_bias: one dict, or one per row ({rows}), got {len(lists)}")
            n = max(len(d) for d in lists)
            n = 1 << max(n - 1, 0).bit_length()              # few different sizes: captured steps are kept per size
            ids, vals = torch.full((len(lists), n), -1, dtype=torch.int32), torch.zeros((len(lists), n), dtype=torch.float32)
            for i, d in enumerate(lists):
                for j, (t, v) in enumerate(sorted((int(t), float(v)) for t, v in d.items())):
                    if not 0 <= t < vocab_size or math.isnan(v):
                        raise ValueError(f"logit_bias: token {t} with {v} (tokens are 0..{vocab_size - 1})")
                    ids[i, j], vals[i, j] = t, v
            if len(lists) > 1:
                ids, vals = ids.repeat_interleave(repeat, 0), vals.repeat_interleave(repeat, 0)
        mask = None
        if self.allowed_tokens is not None:
            mask = self._mask(rows, vocab_size, repeat)
        put = lambda t: None if t is None else t.contiguous().to(device)      # noqa: E731
        return BoundRules(*((put(rep), put(freq), put(pres)) if said else (None, None, None)), put(ids), put(vals), put(mask))

    def _mask(self, rows: int, vocab_size: int, repeat: int) -> torch.Tensor:
        a, words = self.allowed_tokens, (vocab_size + 31) // 32
        if torch.is_tensor(a):
            if a.dtype != torch.int32 or a.dim() not in (1, 2) or a.shape[-1] != words or (a.dim() == 2 and a.shape[0] not in (1, rows)):
                raise ValueError(f"allowed_tokens: masks are int32 [{words}] or [{rows}, {words}] (got {a.dtype}, {tuple(a.shape)})")
            m = a.reshape(-1, words).clone()                 # the caller's stays the caller's: later batches and steps write into what is bound
        else:
            a = list(a)
            nested = len(a) > 0 and not isinstance(a[0], Integral)
            if nested and len(a) != rows:
                raise ValueError(f"allowed_tokens: token ids, or one list of them per row ({rows}), got {len(a)} lists")
            m = torch.stack([allowed_mask(r if r is not None else range(vocab_size), vocab_size) for r in (a if nested else [a])])
        return m.repeat_interleave(repeat, 0) if m.shape[0] > 1 else m


@dataclass
class BoundRules:
    """The rules of a request batch on its device (None: that rule is off)."""

    repetition: Optional[torch.Tensor]
    frequency: Optional[torch.Tensor]
    presence: Optional[torch.Tensor]
    bias_ids: Optional[torch.Tensor]
    bias_values: Optional[torch.Tensor]
    allowed: Optional[torch.Tensor]

    def _all(self) -> Tuple[Optional[torch.Tensor], ...]:
        return self.repetition, self.frequency, self.presence, self.bias_ids, self.bias_values, self.allowed

    def structure(self) -> Tuple:
        """Equal for rules whose tensors a captured step may share."""
        return tuple(None if t is None else tuple(t.shape) for t in self._all())

    def copy_(self, other: "BoundRules") -> "BoundRules":
        for t, o in zip(self._all(), other._all()):
            if t is not None:
                t.copy_(o)
        return self

    def apply(self, logits: torch.Tensor, tokens: torch.Tensor, lengths: torch.Tensor, prompt_lengths: torch.Tensor, starts: Optional[torch.Tensor],
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
        said = dict(tokens=tokens, lengths=lengths, prompt_lengths=prompt_lengths, starts=starts) if self.repetition is not None else {}
        return K.constrain_logits(logits, repetition=self.repetition, frequency=self.frequency, presence=self.presence, bias_ids=self.bias_ids,
                                  bias_values=self.bias_values, allowed=self.allowed, out=out, **said)
