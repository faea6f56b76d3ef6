"""Log probabilities in the responses: the forms of the chat and the completions endpoint, and the host's own sums where an engine has
logits but no kernel over them (sharded vocabularies, stand-ins)."""
from __future__ import annotations

import codecs
import math
from typing import List, NamedTuple, Optional, Sequence, Tuple

import numpy as np

LOWEST = -9999.0        # what minus infinity is in a response: JSON has none


class Score(NamedTuple):
    logprob: float
    top: List[Tuple[int, float]]


def host_logprob(logits: np.ndarray, token: int, top: int) -> Score:
    """One row in 64 bits; ties to the lower id, NaN behind every number.  The serving thread pays for it at every token, so no more of the
    vocabulary is put in order than can be among the alternatives: one row of 151,936 takes 2 ms instead of 19."""
    z = np.asarray(logits, dtype=np.float64)
    best = z.max()
    if math.isfinite(best):
        lse = math.log(np.exp(z - best).sum())
        lp = lambda i: float(z[i] - best - lse)                                # noqa: E731
    else:
        lp = lambda i: -math.inf if best == -math.inf else math.nan            # noqa: E731
    order = ()
    if top:
        key = np.where(np.isnan(z), math.inf, -z)
        n = min(top, len(z))
        # those that reach the n-th smallest, in order of their ids; a stable sort keeps it where they are equal
        near = np.flatnonzero(key <= np.partition(key, n - 1)[n - 1])
        order = near[np.lexsort((np.isnan(z[near]), key[near]))][:n]
    return Score(lp(token) if 0 <= token < len(z) else math.nan, [(int(i), lp(i)) for i in order])


class Entry(NamedTuple):
    """A token of a response with its score (None: the first token of an echoed prompt, which nothing predicts), and where its text begins
    in the response's (None: behind the entries before it)."""
    token: int
    score: Optional[Score]
    at: Optional[int] = None


class Place:
    """Counts the characters of a text whose bytes come token by token, a character often in parts."""

    def __init__(self, at: int = 0):
        self.at = at            # characters that have ended
        self.held = b""         # the beginning of one that has not

    def add(self, raw: bytes) -> int:
        """Characters of the text before the first of these bytes; one that they go on with counts from where it begins, at the next place."""
        if self.held and raw and not _goes_on(self.held, raw[:1]):
            self.at += len(_text(self.held))      # it never ends: the text has replacement characters there
            self.held = b""
        at = self.at
        dec = codecs.getincrementaldecoder("utf-8")("replace")
        self.at += len(dec.decode(self.held + raw))
        self.held = dec.getstate()[0]
        return at


def _goes_on(held: bytes, byte: bytes) -> bool:
    try:
        codecs.getincrementaldecoder("utf-8")("strict").decode(held + byte)
        return True
    except UnicodeDecodeError:
        return False


def number(x: float):
    return None if math.isnan(x) else max(float(x), LOWEST)


def _text(raw: bytes) -> str:
    return raw.decode("utf-8", "replace")


def _name(raw: bytes) -> str:
    """A token's text, or its bytes where they are no text by themselves (part of a character): two tokens' are never one replacement character."""
    try:
        return raw.decode("utf-8")
    except UnicodeDecodeError:
        return "bytes:" + "".join(f"\\x{b:02x}" for b in raw)


def chat_block(tok, entries: Sequence[Entry]) -> dict:
    """``choices[0].logprobs`` of chat completions."""
    def one(token, lp):
        raw = tok.token_bytes(token)
        return {"token": _text(raw), "logprob": number(lp), "bytes": list(raw)}
    return {"content": [{**one(e.token, e.score.logprob), "top_logprobs": [one(i, lp) for i, lp in e.score.top]} for e in entries]}


def text_block(tok, entries: Sequence[Entry], top: int, offset: int) -> Tuple[dict, int]:
    """``choices[0].logprobs`` of completions for tokens whose text begins at ``offset``, and the offset behind them.  Alternatives whose texts are
    the same keep the likelier one's number; the token itself is always among them, with its own."""
    out = {"tokens": [], "token_logprobs": [], "top_logprobs": [] if top else None, "text_offset": []}
    place = Place(offset)
    for e in entries:
        text = _name(tok.token_bytes(e.token))
        at = place.add(tok.text_bytes(e.token))
        out["tokens"].append(text)
        out["text_offset"].append(at if e.at is None else e.at)
        out["token_logprobs"].append(None if e.score is None else number(e.score.logprob))
        if top:
            best = None
            if e.score is not None:
                best = {}
                for i, lp in e.score.top:
                    best.setdefault(_name(tok.token_bytes(i)), number(lp))
                best[text] = number(e.score.logprob)
            out["top_logprobs"].append(best)
    return out, place.at
