"""Log probabilities through the engine, the adapter and the server on a GPU: the rows of steps, and prompts as they are ingested."""
import dataclasses
import http.client
import json
import math

import pytest
import torch

from b200serve.models.config import preset
from b200serve.models.weights import random_weights

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def engine(name, dtype=None, **kw):
    from b200serve.models.listed import random_listed_weights
    from b200serve.runtime.engine import Engine
    cfg = preset(name)
    w = random_listed_weights(cfg, "cuda", 3, dtype=dtype) if dtype else random_weights(cfg, device="cuda", seed=3)
    return Engine(w, max_seqs=2, max_len=512, **kw)


def prompt(cfg, n, seed=0):
    return torch.randint(0, cfg.vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


class Watch:
    """Notes the rows that the head is given, and what it makes of them in 64 bits."""

    def __init__(self, eng):
        self.rows, self.tokens, m = [], [], eng.model
        inner = m.score_rows

        def score_rows(x, tokens, out, **kw):
            self.rows.append(x.clone())
            self.tokens.append(tokens.clone())
            return inner(x, tokens, out, **kw)
        m.score_rows = score_rows

    def logits(self, head):
        x = torch.cat(self.rows)
        k = min(x.shape[1], head.shape[1])
        return x[:, :k].double() @ head[:, :k].double().T, x[:, :k].double().abs() @ head[:, :k].double().abs().T


def agree(got, z, ids, top, dz):
    """Scores of tokens 1.. against rows 0.. of 64-bit logits; dz: bound of a logit's error.  A log probability is off by twice that and by
    what fp32 sums add, below 2e-5 here (tests/test_logprob.py); of the alternatives the numbers are compared, in their order."""
    lp = torch.log_softmax(z, 1).cpu()
    h = -(lp.exp() * lp).sum(1)
    tol = 2 * float(dz) + 2e-5
    assert math.isnan(got[0].logprob) and got[0].top == []
    for i in range(1, len(ids)):
        assert abs(got[i].logprob - float(lp[i - 1, ids[i]])) <= tol, (i, got[i].logprob, float(lp[i - 1, ids[i]]))
        assert abs(got[i].entropy - float(h[i - 1])) <= tol * (1 + math.log(z.shape[1]))
        want = lp[i - 1].topk(top).values
        assert len(got[i].top) == top
        for (t, v), u in zip(got[i].top, want.tolist()):
            assert abs(v - u) <= tol and abs(v - float(lp[i - 1, t])) <= tol


# ------------------------------------------------------------------ prompts
@pytest.mark.parametrize("name,kw", [("small-dense", {}), ("small-dense", {"prefill_backend": "w4"}), ("small-dense", {"kv_dtype": "int8"}),
                                     ("small-hybrid", {}), ("small-moe", {}), ("small-windowed", {})])
@pytest.mark.parametrize("n,chunk", [(150, None), (300, 128)])
def test_prompt_through_the_gemm_pass(name, kw, n, chunk):
    """fp32 sums of 512 products, in 32 groups: each addition off by a step of what is there, 2 U of sum |x w| at most."""
    eng = engine(name, **kw)
    ids = prompt(eng.cfg, n)
    w = Watch(eng)
    for top in (0, 5):
        w.rows.clear()
        scores = eng.prompt_scores(ids, top)
        eng.reset(0)
        eng.prefill(0, ids, chunk, scores=scores)
        z, mag = w.logits(eng.model.w.lm_head)
        assert z.shape[0] == n and torch.cat(w.tokens)[: n].tolist() == ids[1:] + [-1]
        w.tokens.clear()
        agree(scores.read(), z, ids, top, float(mag.max()) * 2 * U * (eng.cfg.hidden / 16 + 16))
        # the last row is the one that the next token comes from: the same sums in another order
        last = eng.model.buf.logits[eng.last_prefill_row].double()
        assert float((last - z[-1]).abs().max()) <= float(mag.max()) * 2 * U * eng.cfg.hidden


@pytest.mark.parametrize("backend", ["int8", "bf16-resident"])
def test_prompt_through_an_int8_head(backend):
    eng = engine("small-dense", int8_head=True, prefill_backend=backend)
    ids = prompt(eng.cfg, 200)
    w = Watch(eng)
    scores = eng.prompt_scores(ids, 4)
    eng.prefill(0, ids, scores=scores)
    w8, sc = eng.model.w.lm_head_i8
    x = torch.cat(w.rows)
    if backend == "int8":      # rows quantised per token; whole sums, three roundings
        largest = x.float().abs().amax(1, keepdim=True)
        s = largest / torch.full_like(largest, 127)
        z = ((x.float() * (1 / s)).round().double() @ w8.double().T) * s.double() * sc.double()
        dz = float(z.abs().max()) * 3 * U
    else:                      # the rows of a step, as they are
        z = (x.double() @ w8.double().T) * sc.double()
        dz = float(((x.double().abs() @ w8.double().abs().T) * sc.double()).max()) * 2 * U * eng.cfg.hidden
    agree(scores.read(), z, ids, 4, dz)


@pytest.mark.parametrize("name,dtype", [("mumusun-mini", None), ("napadra-mini", None), ("pefulorn-mini", None), ("vogerax-mini", None),
                                        ("mumusun-mini", torch.float32), ("vogerax-mini", torch.float32)])
@pytest.mark.parametrize("n,chunk", [(150, None), (200, 90)])
def test_prompt_of_listed_models(name, dtype, n, chunk):
    eng = engine(name, dtype)
    ids = prompt(eng.cfg, n)
    w = Watch(eng)
    scores = eng.prompt_scores(ids, 3)
    eng.prefill(0, ids, chunk, scores=scores)
    z, mag = w.logits(eng.model.w.lm_head[: eng.cfg.vocab])
    agree(scores.read(), z, ids, 3, float(mag.max()) * 2 * U * (eng.cfg.hidden if dtype else eng.cfg.hidden / 16 + 16))


@pytest.mark.parametrize("name", ["tiny-dense", "small-dense", "small-hybrid", "tiny-moe", "napadra-mini"])
def test_prompt_in_row_steps(name):
    """Short prompts, and shapes without a GEMM pass: the steps' own logits."""
    eng = engine(name)
    n = 40 if name != "tiny-dense" else 150
    ids, seen = prompt(eng.cfg, n), []
    inner = eng.forward_rows

    def forward_rows(rows, **kw):
        out = inner(rows, **kw)
        seen.append(eng.logits(len(rows)).clone())
        return out
    eng.forward_rows = forward_rows
    agree(eng.score(ids, 6), torch.cat(seen).double(), ids, 6, 0.0)


@pytest.mark.parametrize("name", ["small-dense", "napadra-mini"])
def test_scores_belong_to_their_places(name):
    """A prompt that ends at a place has that place's distribution as its next one.  The two passes round activations differently (bf16, other
    tiles): 2^-8 of a value in each of a few sublayers moves a logit by a small part of their spread, another place's row by all of it."""
    eng = engine(name)
    ids = prompt(eng.cfg, 220, 4)
    got = eng.score(ids, 1)
    for i in (70, 128, 129, 219):
        eng.reset(0)
        eng.prefill(0, ids[:i])
        z = eng.logits(1)[0].double()
        assert abs(got[i].logprob - float(torch.log_softmax(z, 0)[ids[i]])) < 0.1 * float(z.std()) + 1e-3


def test_portions_and_refusals():
    eng = engine("small-dense")
    ids = prompt(eng.cfg, 260)
    whole = eng.score(ids, 2)
    scores = eng.prompt_scores(ids, 2)
    eng.reset(0)
    for a, b in ((0, 100), (100, 101), (101, 230), (230, 260)):      # GEMM pass and row steps in turn
        eng.prefill(0, ids[a:b], scores=scores)
    for x, y in zip(scores.read()[1:], whole[1:]):
        assert abs(x.logprob - y.logprob) < 0.1
    scores = eng.prompt_scores(ids, 2)
    with pytest.raises(ValueError, match="were ingested"):
        scores.read()
    with pytest.raises(ValueError, match="not the prompt's"):
        eng.prefill(0, ids[1:80], scores=scores)
    with pytest.raises(ValueError, match="at most"):
        eng.prompt_scores(ids, 33)
    assert math.isnan(eng.score([5], 2)[0].logprob) and len(eng.score([5], 2)) == 1 and eng.score([], 2) == []
    with pytest.raises((ValueError, RuntimeError, OverflowError)):
        eng.prompt_scores([5, 1 << 32])


# ------------------------------------------------------------------ steps
@pytest.mark.parametrize("name", ["small-dense", "small-hybrid", "napadra-mini"])
def test_rows_of_steps(name):
    from b200serve.server.adapter import EngineAdapter
    eng = engine(name)
    ad = EngineAdapter(eng)
    a, b = prompt(eng.cfg, 100, 1), prompt(eng.cfg, 70, 2)
    t0 = ad.prefill(0, a)
    z = eng.logits(1).double()
    (s,) = ad.logprobs([(0, 0, t0)], 3)
    lp = torch.log_softmax(z, 1)[0]
    assert s.top[0][0] == t0 and abs(s.logprob - float(lp[t0])) <= 2e-5 and [i for i, _ in s.top] == eng.logits(1)[0].sort(descending=True, stable=True).indices[:3].tolist()
    t1 = ad.prefill(1, b)
    ad.step({0: [t0, 5, 6], 1: [t1]})
    lp = torch.log_softmax(eng.logits(4).double(), 1)
    items = [(0, 0, 5), (0, 2, 9), (1, 0, 11)]
    for (slot, row, tok), s in zip(items, ad.logprobs(items, 1)):
        assert abs(s.logprob - float(lp[row if slot == 0 else 3, tok])) <= 2e-5
    twice = ad.logprobs([(0, 1, 5), (1, 0, 11), (0, 1, 6)], 0)      # a row asked about twice
    for (row, tok), s in zip(((1, 5), (3, 11), (1, 6)), twice):
        assert abs(s.logprob - float(lp[row, tok])) <= 2e-5
    if eng.mixed_batches:      # a prompt's portion beside decode rows
        eng.reset(1)
        tok, res = ad.step_mixed(1, b, {0: [7]})
        logits = ad._device_logits().double()
        lp = torch.log_softmax(logits, 1)
        for (slot, row, t), s, r in zip([(1, 0, tok), (0, 0, 3)], ad.logprobs([(1, 0, tok), (0, 0, 3)], 0), (1, 0)):
            assert abs(s.logprob - float(lp[r, t])) <= 2e-5


# ------------------------------------------------------------------ the server
def post(port, body):
    c = http.client.HTTPConnection("127.0.0.1", port, timeout=60)
    c.request("POST", "/v1/completions", json.dumps(body), {"Content-Type": "application/json"})
    r = c.getresponse()
    data = r.read().decode()
    c.close()
    return r.status, json.loads(data)


@pytest.mark.parametrize("spec,prefix", [("off", False), ("lookup", True), ("mtp", False), ("dflash", True)])
def test_generated_text_scored_again(spec, prefix):
    """Tokens that were generated with log probabilities, then scored as an echoed prompt: decode steps and the prompt pass, two kernels and two
    heads, say the same to rounding of the activations (bf16, as above)."""
    from b200serve.runtime.engine import Engine
    from b200serve.runtime.spec import SpecAdapter
    from b200serve.server.adapter import EngineAdapter
    from b200serve.server.app import Server, ServerOptions
    from b200serve.server.chat_template import ChatTemplate
    from b200serve.server.iface import ByteTok
    from b200serve.server.prefix import PrefixStore
    cfg = dataclasses.replace(preset("small-dense"), mtp_layers=1, vocab=259, name="small-dense-bytes")
    eng = Engine(random_weights(cfg, device="cuda", seed=8), max_seqs=2, max_len=1024, extra_kv_layers=2)
    adapter = EngineAdapter(eng, eos_ids=())
    if spec in ("mtp", "dflash"):
        adapter = SpecAdapter(adapter, spec, 3)
    store = PrefixStore(eng, host_gb=0.05, block_tokens=64) if prefix else None
    srv = Server(adapter, ByteTok(), ChatTemplate(), ServerOptions(model_name=cfg.name, spec=spec, spec_max=3), prefix=store).start()
    try:
        text = "The quick brown fox jumps over the lazy dog. " * 6
        st, a = post(srv.port, {"prompt": text, "max_tokens": 24, "ignore_eos": True, "logprobs": 4, "return_token_ids": True})
        assert st == 200
        a = a["choices"][0]
        ids, lp = a["token_ids"], a["logprobs"]
        assert len(ids) == 24 == len(lp["token_logprobs"]) and all(len(t) >= 1 for t in lp["top_logprobs"])
        whole = ByteTok().encode(text) + ids
        st, b = post(srv.port, {"prompt": whole, "max_tokens": 0, "echo": True, "logprobs": 4})
        assert st == 200
        again = b["choices"][0]["logprobs"]["token_logprobs"]
        assert len(again) == len(whole) and again[0] is None
        for x, y in zip(lp["token_logprobs"], again[-24:]):
            assert abs(x - y) < 0.1, (lp["token_logprobs"], again[-24:])
        assert b["usage"]["prompt_tokens_details"]["cached_tokens"] == 0
    finally:
        srv.stop()


def test_scored_prompt_beside_decode_rows_of_a_mixed_batch_engine():
    """A model whose prompt portions share batches with decode rows: a scored prompt has its own, and says what the engine says alone."""
    import threading
    from b200serve.server.adapter import EngineAdapter
    from b200serve.server.app import Server, ServerOptions
    from b200serve.server.chat_template import ChatTemplate
    from b200serve.server.iface import ByteTok
    eng = engine("napadra-mini")
    ids = prompt(eng.cfg, 180, 6)
    alone = eng.score(ids, 2)
    eng.reset()
    srv = Server(EngineAdapter(eng, eos_ids=()), ByteTok(), ChatTemplate(), ServerOptions(prefill_chunk=100)).start()
    try:
        other = threading.Thread(target=post, args=(srv.port, {"prompt": prompt(eng.cfg, 90, 7), "max_tokens": 200, "ignore_eos": True, "logprobs": 1}))
        other.start()
        st, body = post(srv.port, {"prompt": ids, "max_tokens": 0, "echo": True, "logprobs": 2})
        other.join()
        assert st == 200
        got = body["choices"][0]["logprobs"]["token_logprobs"]
        assert len(got) == len(ids) and got[0] is None
        # other portions, so other tiles: rounding of activations, as above
        assert max(abs(x - y.logprob) for x, y in zip(got[1:], alone[1:])) < 0.1
    finally:
        srv.stop()
