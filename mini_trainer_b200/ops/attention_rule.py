"""What attention does to its scores between ``q.k`` and the softmax, beyond the causal mask of the packed samples.

``AttentionRule`` is handed to ``attention`` and ``attention_bwd`` of either backend. In the order in which they apply:

* ``cap``     ``s -> cap * tanh(s / cap)`` of the scaled scores
* ``slopes``  ``s -> s - slopes[head] * |i - j|``, a bias that falls with the distance of query and key (fp32, one slope per query head; constants of
              the model: they get no gradient)
* ``window``  query ``i`` sees the keys ``j <= i`` with ``i - j < window`` (itself among them)
* ``prefix``  one length per sample: all tokens of the sample see its first ``prefix`` keys, whatever the window and on either side of them

so that ``i`` sees ``j`` of its own sample iff ``(j <= i and i - j < window) or j < prefix``. The diagonal is always seen: no row is empty, whatever the rule.
What is not finite in one sample stays there, in outputs and gradients.
A window without keys, negative prefixes and ones longer than their sample are refused.
"""
from __future__ import annotations

import operator
from dataclasses import dataclass
from typing import Optional, Sequence

import torch

_NO_WINDOW = 1 << 30


def _whole(x, what: str) -> int:
    try:
        return int(x) if isinstance(x, float) and x.is_integer() else operator.index(x)
    except TypeError:
        raise ValueError(f"{what} counts tokens, {x!r} does not") from None


@dataclass(frozen=True)
class AttentionRule:
    cap: Optional[float] = None
    window: Optional[int] = None
    prefix: Optional[Sequence[int]] = None   # host integers, one per sample, like the host's list of sequence starts
    slopes: Optional[torch.Tensor] = None    # [query heads] fp32, on the device of the activations

    def __post_init__(self):
        if self.cap is not None and not 0.0 < float(self.cap) < float("inf"):
            raise ValueError(f"a score cap is a positive number, not {self.cap}")
        own = object.__setattr__
        own(self, "window", None if self.window is None else _whole(self.window, "a window"))
        if self.window is not None and self.window < 1:
            raise ValueError(f"a window has at least the query itself, one key, not {self.window}")
        own(self, "prefix", None if self.prefix is None else tuple(_whole(x, "a prefix") for x in self.prefix))
        own(self, "keys", _NO_WINDOW if self.window is None else min(self.window, _NO_WINDOW))   # of the window; beyond any sample where there is none
        own(self, "key", (0.0 if self.cap is None else float(self.cap), 0 if self.window is None else self.keys, self.prefix))   # what a plan depends on

    def prefixes(self, cu_host) -> list:
        """The prefix of every sample, checked against its length."""
        lens = [b - a for a, b in zip(cu_host[:-1], cu_host[1:])]
        if self.prefix is None:
            return [0] * len(lens)
        p = list(self.prefix)
        if len(p) != len(lens):
            raise ValueError(f"{len(p)} prefixes for {len(lens)} samples")
        for x, n in zip(p, lens):
            if not 0 <= x <= n:
                raise ValueError(f"a prefix of {x} tokens in a sample of {n}")
        return p

    def check_slopes(self, hq: int, like) -> None:
        s = self.slopes
        if s is not None and (s.dtype is not torch.float32 or s.shape != (hq,) or not s.is_contiguous() or s.get_device() != like.get_device()):
            raise ValueError(f"slopes are {hq} contiguous fp32 numbers on {like.device}, not {tuple(s.shape)} {s.dtype} on {s.device}")

    @staticmethod
    def check_starts(cu_host, T: int) -> None:
        """``cu_host``: the samples' starts and the last one's end, at most ``T``."""
        if len(cu_host) < 1 or cu_host[0] != 0 or cu_host[-1] > T or any(b < a for a, b in zip(cu_host[:-1], cu_host[1:])):
            raise ValueError(f"sequence starts go from 0 to at most {T} without falling")

    # -- plain form, one sample at a time -------------------------------------------------
    def seen(self, n: int, prefix: int, device):
        """``[n, n]``: whether a query (row) sees a key."""
        i, j = torch.arange(n, device=device)[:, None], torch.arange(n, device=device)[None, :]
        return ((j <= i) & (i - j < self.keys)) | (j < prefix)

    def scores(self, s, seen):
        """``(scores, derivative of the cap)`` of scaled products ``[heads, n, n]``; the derivative is ``None`` without a cap."""
        n, d = s.shape[-1], None
        if self.cap is not None:
            t = torch.tanh(s / float(self.cap))
            s, d = float(self.cap) * t, 1.0 - t * t
        if self.slopes is not None:
            i = torch.arange(n, device=s.device)
            s = s - self.slopes.to(s.dtype).view(-1, 1, 1) * (i[:, None] - i[None, :]).abs()
        return s.masked_fill(~seen, float("-inf")), d
