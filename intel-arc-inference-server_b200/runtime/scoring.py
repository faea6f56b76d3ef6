"""Log probabilities on their way from the device: of the rows of a step, and of a prompt's tokens, portion by portion."""
from __future__ import annotations

from typing import List, NamedTuple, Sequence, Tuple

import torch

from ..ops import logprob as LP


class TokenScore(NamedTuple):
    """A token's log probability, the entropy of the distribution it was drawn from, and that distribution's top alternatives."""
    logprob: float
    entropy: float
    top: List[Tuple[int, float]]


def _check_top(top: int):
    if not 0 <= top <= LP.MAX_TOP:
        raise ValueError(f"log probabilities of at most {LP.MAX_TOP} alternatives, not {top}")


class ScoreBuffer:
    """Results of ``rows`` rows in one piece of memory, so that one copy reads them."""

    def __init__(self, rows: int, top: int, device):
        _check_top(top)
        self.rows, self.top = rows, top
        self.flat = torch.empty(rows * (2 + 2 * top), dtype=torch.float32, device=device)
        cut = lambda i, width: self.flat[i * rows: (i + width) * rows]                        # noqa: E731
        self.out = LP.Logprobs(cut(0, 1), cut(1, 1), cut(2, top).view(torch.int32).view(rows, top), cut(2 + top, top).view(rows, top))

    def read(self) -> List[TokenScore]:
        host = self.flat.cpu()
        n, t = self.rows, self.top
        ids, lps = host[2 * n: (2 + t) * n].view(torch.int32).view(n, t).tolist(), host[(2 + t) * n:].view(n, t).tolist()
        return [TokenScore(lp, h, [(i, v) for i, v in zip(a, b) if i >= 0]) for lp, h, a, b in zip(host[:n].tolist(), host[n: 2 * n].tolist(), ids, lps)]


class PromptScores:
    """Collects the log probabilities of a prompt's tokens while the prompt is ingested, in order, in portions of any size: row i predicts
    token i + 1.  Nothing is on the device before the first portion comes: prompts that wait for their turn hold none of its memory."""

    def __init__(self, ids: Sequence[int], top: int, device):
        _check_top(top)
        self.ids = [int(t) for t in ids]
        self.done, self.top, self.device = 0, top, device
        self.host_next = torch.tensor(self.ids[1:] + [-1], dtype=torch.int32)
        self.buf = self.next = None

    def expect(self, ids: Sequence[int]):
        """The portion about to be ingested has to be the prompt's next one."""
        if [int(t) for t in ids] != self.ids[self.done: self.done + len(ids)]:
            raise ValueError(f"these {len(ids)} tokens are not the prompt's from place {self.done} on")
        if self.buf is None:
            self.buf, self.next = ScoreBuffer(len(self.ids), self.top, self.device), self.host_next.to(self.device)

    def take(self, n: int) -> Tuple[torch.Tensor, LP.Logprobs]:
        """(tokens that the next ``n`` rows predict, their results)."""
        a, self.done = self.done, self.done + n
        return self.next[a: a + n], self.buf.out.rows(a, a + n)

    def read(self) -> List[TokenScore]:
        """A score per token; the first one has none."""
        if self.done != len(self.ids):
            raise ValueError(f"{self.done} of the prompt's {len(self.ids)} tokens were ingested")
        return [TokenScore(float("nan"), float("nan"), [])] + self.buf.read()[:-1] if self.ids else []
