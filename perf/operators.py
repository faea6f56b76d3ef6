"""The work that the operators of log probabilities are measured on: what a model thinks of given tokens.

``rows``: log probabilities of the rows of logits that a decode or verify step left, with the entropy of each row and its top
alternatives.  ``score``: the same of a prompt's rows behind the final norm, through the head.  ``score_i8``: the same through the
8-bit head, with rows quantised per token.

The plain forms below are the definition in elementary operations; with ``own`` the calls are ``b200serve.ops.logprob``'s.

Rows, weights and their products in ``score`` lie on a grid (an 8-bit checkpoint's), so that a logit is the same 32-bit number whatever
the order of its sum: the ids of the alternatives can then be compared.  ``score_i8`` has whole numbers by itself.
"""
import math

import torch

own = False


def _rows(m, n, top, banned=0.0, pad=0):
    """``m`` rows of ``n`` logits; ``banned``: share of the vocabulary that a mask sets to minus infinity; ``pad``: columns of the
    buffer behind the vocabulary."""
    return {"op": "rows", "m": m, "n": n, "top": top, "banned": banned, "pad": pad}


def _score(op, m, n, k, top):
    """``m`` rows of ``k`` against a vocabulary of ``n``."""
    return {"op": op, "m": m, "n": n, "k": k, "top": top}


def listed():
    return [
        # the smallest call: a few rows of a toy model, launches only
        {"name": "rows-3-small", **_rows(3, 700, 2)},
        # one user's chat: the next token and its five alternatives
        {"name": "rows-1", **_rows(1, 151936, 5)},
        # a step of several requests, twenty alternatives each
        {"name": "rows-8-top20", **_rows(8, 151936, 20)},
        # a busy step with a grammar that bans nine tokens of ten, log probabilities and entropy only; odd vocabulary in a wider buffer
        {"name": "rows-64-banned", **_rows(64, 102397, 0, banned=0.9, pad=3)},
        # a batch of kept logits ranked afterwards
        {"name": "rows-500-top10", **_rows(500, 151936, 10)},
        # a toy model's prompt
        {"name": "score-130-small", **_score("score", 130, 2048, 512, 0)},
        # the likelihood of a short answer behind a prompt, model of hidden 2048: the head's bytes
        {"name": "score-77", **_score("score", 77, 102400, 2048, 0)},
        # a prompt of the 27B shape with five alternatives per token
        {"name": "score-900-top5", **_score("score", 900, 151936, 5120, 5)},
        # a long document of the 27B shape: the largest
        {"name": "score-4096", **_score("score", 4096, 151936, 5120, 0)},
        # a few rows against the 8-bit head
        {"name": "score-i8-40-top3", **_score("score_i8", 40, 64000, 4096, 3)},
        # a prompt of a model of hidden 2048, odd length and vocabulary
        {"name": "score-i8-1333", **_score("score_i8", 1333, 151933, 2048, 0)},
        # a long document, 8-bit head of the 27B shape
        {"name": "score-i8-4096", **_score("score_i8", 4096, 151936, 5120, 0)},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


#: Vocabulary and hidden size of the presets.
HEADS = ((151936, 5120), (151936, 2048), (102400, 2048), (64000, 4096), (2048, 512), (1024, 256))


def draw(rng):
    op = rng.choice(("rows", "score", "score_i8"))
    top = rng.choice((0, 0, 1, rng.randint(2, 20), 20))
    if op == "rows":
        m = _log(rng, 1, 512)
        return _rows(m, _log(rng, 600, 200000), top, banned=rng.choice((0.0, 0.0, rng.uniform(0.05, 0.95))), pad=rng.choice((0, 0, rng.randint(1, 130))))
    m = _log(rng, 1, 4096)
    if rng.random() < 0.6:
        n, k = rng.choice(HEADS)
        return _score(op, m, n - rng.choice((0, 0, rng.randint(1, 200))), k, top)
    return _score(op, m, _log(rng, 600, 151936), 16 * _log(rng, 16, 320), top)


# ------------------------------------------------------------------ what a program has in hand
def _rand(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(case, g):
    """Logits as a trained head gives them: a bell of two to three, a few candidates far above it, by another distance in every row."""
    m, n = case["m"], case["n"]
    z = torch.empty(m, n + case["pad"], device="cuda").normal_(0, 2.2, generator=g)[:, :n]
    lift = 18.0 * torch.rand(m, 1, device="cuda", generator=g)
    peaks = torch.randint(0, n, (m, 6), device="cuda", generator=g)
    z.scatter_add_(1, peaks, lift * torch.rand(m, 6, device="cuda", generator=g))
    if case["banned"]:
        ban = torch.rand(n, device="cuda", generator=g) < case["banned"]
        ban[torch.randperm(n, device="cuda", generator=g)[:64]] = False
        z.masked_fill_(ban, float("-inf"))
    u = torch.rand(m, n, device="cuda", generator=g)
    tokens = (z - (-u.clamp_(1e-9, 1 - 1e-7).log()).log()).argmax(1)       # a draw from every row
    return z, tokens.int()


def _hidden(tokens, case, g, rows_of):
    """Rows that point at their tokens, some hardly and some firmly (``rows_of``: the head's rows of given ids, of unit columns)."""
    m, k = case["m"], case["k"]
    pull = (torch.rand(m, 1, device="cuda", generator=g) * 24.0 / k) / 0.0234
    x = torch.empty(m, k, device="cuda").normal_(0, 1, generator=g) + pull * rows_of(tokens)
    return (x * 16).round_().clamp_(-127, 127).div_(16).bfloat16()


def prepare(case, seed):
    g = _rand(seed * 7919 + 17)
    m, n = case["m"], case["n"]
    state = {"case": case}
    if case["op"] == "rows":
        state["logits"], state["tokens"] = _logits(case, g)
    else:
        k = case["k"]
        w = torch.empty(n, k, dtype=torch.bfloat16, device="cuda").normal_(0, 24, generator=g).round_().clamp_(-127, 127)      # 0.0234 in steps of 2^-10
        state["tokens"] = torch.randint(0, n, (m,), device="cuda", generator=g).int()
        state["x"] = _hidden(state["tokens"].long(), case, g, lambda ids: w[ids].float() / 24)
        if case["op"] == "score":
            state["head"] = w.div_(1024)
        else:      # an 8-bit head: whole numbers and a scale per row
            state["head"] = (w.to(torch.int8), (0.5 + torch.rand(n, device="cuda", generator=g)) / 1024)
    if own:
        from b200serve.ops import logprob
        state["out"] = logprob.Logprobs.empty(m, case["top"], "cuda")
    return state


# ------------------------------------------------------------------ plain forms
def _of_logits(z, tokens, top):
    """Log probabilities of fp32 logits ``z``.  The sum of exponentials is kept without its largest term, so that the logarithm of a
    sum close to one keeps its digits."""
    best, at = z.max(1, keepdim=True)
    d = z - best
    e = d.exp().scatter_(1, at, 0.0)
    rest = e.sum(1, keepdim=True)
    lse = rest.log1p()
    entropy = lse - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / (1 + rest)
    out = {"logprob": (d.gather(1, tokens.long()[:, None]) - lse)[:, 0], "entropy": entropy[:, 0]}
    if top:
        ids = z.sort(dim=1, descending=True, stable=True).indices[:, :top]       # ties: the lower id first
        out.update(top_ids=ids.int(), top_logprobs=d.gather(1, ids) - lse)
    return out


def _pieces(n, size, f):
    """``f(first, last)`` over pieces of the rows, joined."""
    got = [f(i, min(n, i + size)) for i in range(0, n, size)]
    return {name: torch.cat([p[name] for p in got]) for name in got[0]}


def _plain(state):
    case, tokens, top = state["case"], state["tokens"], state["case"]["top"]
    if case["op"] == "rows":
        return _of_logits(state["logits"], tokens, top)
    if case["op"] == "score":
        w = state["head"].float()
        return _pieces(case["m"], 2048, lambda i, j: _of_logits(state["x"][i:j].float() @ w.T, tokens[i:j], top))
    w, scale = state["head"][0].float(), state["head"][1]
    x = state["x"].float()
    largest = x.abs().amax(1, keepdim=True)
    s = (largest / torch.full_like(largest, 127)).clamp_min(2.0 ** -126)       # (by a number torch multiplies with its rounded inverse)
    q = (x * (1 / s)).round()
    return _pieces(case["m"], 2048, lambda i, j: _of_logits(((q[i:j] @ w.T) * s[i:j]) * scale, tokens[i:j], top))


def run(state):
    if not own:
        return _plain(state)
    from b200serve.ops import logprob
    case, out = state["case"], state["out"]
    if case["op"] == "rows":
        logprob.token_logprobs(state["logits"], state["tokens"], out=out)
    elif case["op"] == "score":
        logprob.score(state["x"], state["head"], state["tokens"], out=out)
    else:
        logprob.score_i8(state["x"], state["head"], state["tokens"], out=out)
    got = {"logprob": out.logprob, "entropy": out.entropy}
    if case["top"]:
        got.update(top_ids=out.top_ids, top_logprobs=out.top_logprobs)
    return got


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    got = []
    if case["op"] == "score":
        head = state["head"].double()
    elif case["op"] == "score_i8":
        head = state["head"][0].double()
    for i in range(0, case["m"], 512):
        t = state["tokens"][i: i + 512].long()
        if case["op"] == "rows":
            z = state["logits"][i: i + 512].double()
        elif case["op"] == "score":
            z = state["x"][i: i + 512].double() @ head.T
        else:
            # the row's scale is a 32-bit number, and so is the inverse that its values are multiplied by before they are rounded
            x = state["x"][i: i + 512].float()
            s = (x.abs().max(dim=1, keepdim=True).values.double() / 127).float()
            s[s == 0] = 1
            z = (torch.round(x * torch.reciprocal(s)).double() @ head.T) * s.double() * state["head"][1].double()
        lp = torch.log_softmax(z, dim=1)
        p = lp.exp()
        one = {"logprob": lp[torch.arange(len(t), device="cuda"), t], "entropy": -(p * lp.clamp_min(-1e4)).sum(1)}
        if case["top"]:
            one["top_logprobs"] = lp.topk(case["top"], dim=1).values
        got.append(one)
    out = {name: torch.cat([p[name] for p in got]) for name in got[0]}
    if case["top"]:
        out["top_ids"] = None      # where 64 bits tell two values apart that are one in 32, the order is another
    return out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    m, n, top = case["m"], case["n"], case["top"]
    out = m * (4 + 8 + 8 * top)          # the token read; log probability, entropy and alternatives written
    each = 6.0 * m * n                   # difference, exponential, two sums, largest, comparison
    if case["op"] == "rows":
        return {"bytes": 4.0 * m * n + out, "flops": each}
    k = case["k"]
    if case["op"] == "score":
        return {"bytes": 2.0 * k * (m + n) + out, "flops": 2.0 * m * n * k + each}
    return {"bytes": 2.0 * k * m + 1.0 * k * n + 4.0 * n + out, "flops": 2.0 * m * n * k + each}
