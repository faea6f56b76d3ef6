"""Log probabilities in the responses: the forms of the chat and the completions endpoint, and the host's own sums where an engine has
logits but no kernel over them (sharded vocabularies, stand-ins)."""
from __future__ import annotations

import math
from typing import List, NamedTuple, Optional, Sequence, Tuple

import numpy as np

LOWEST = -9999.0        # what minus infinity is in a response: JSON has none


class Score(NamedTuple):
    logprob: float
    top: List[Tuple[int, float]]


def host_logprob(logits: np.ndarray, token: int, top: int) -> Score:
    """One row in 64 bits; ties to the lower id."""
    z = np.asarray(logits, dtype=np.float64)
    best = z.max()
    if not math.isfinite(best):
        lp = np.full_like(z, -math.inf if best == -math.inf else math.nan)
    else:
        d = z - best
        lp = d - math.log(np.exp(d).sum())
    order = np.argsort(-z, kind="stable")[:top]
    return Score(float(lp[token]) if 0 <= token < len(z) else math.nan, [(int(i), float(lp[i])) for i in order])


class Entry(NamedTuple):
    """A token of a response with its score (None: the first token of an echoed prompt, which nothing predicts)."""
    token: int
    score: Optional[Score]


def number(x: float):
    return None if math.isnan(x) else max(float(x), LOWEST)


def _text(raw: bytes) -> str:
    return raw.decode("utf-8", "replace")


def chat_block(tok, entries: Sequence[Entry]) -> dict:
    """``choices[0].logprobs`` of chat completions."""
    def one(token, lp):
        raw = tok.token_bytes(token)
        return {"token": _text(raw), "logprob": number(lp), "bytes": list(raw)}
    return {"content": [{**one(e.token, e.score.logprob), "top_logprobs": [one(i, lp) for i, lp in e.score.top]} for e in entries]}


def text_block(tok, entries: Sequence[Entry], top: int, offset: int) -> Tuple[dict, int]:
    """``choices[0].logprobs`` of completions for tokens whose text begins at ``offset``, and the offset behind them.  Alternatives whose texts are
    the same keep the likelier one's number; the token itself is always among them."""
    out = {"tokens": [], "token_logprobs": [], "top_logprobs": [] if top else None, "text_offset": []}
    for e in entries:
        text = _text(tok.token_bytes(e.token))
        out["tokens"].append(text)
        out["text_offset"].append(offset)
        out["token_logprobs"].append(None if e.score is None else number(e.score.logprob))
        if top:
            best = None
            if e.score is not None:
                best = {}
                for i, lp in e.score.top:
                    best.setdefault(_text(tok.token_bytes(i)), number(lp))
                best.setdefault(text, number(e.score.logprob))
            out["top_logprobs"].append(best)
        offset += len(text)
    return out, offset
