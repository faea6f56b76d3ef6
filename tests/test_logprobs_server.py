"""Log probabilities over HTTP against the stand-in engine (CPU): requests, forms of the responses, streams, echoed prompts, speculation."""
import json
import math

import numpy as np
import pytest

from b200serve.native import host as H
from b200serve.server.app import Server, ServerOptions
from b200serve.server.chat_template import ChatTemplate
from b200serve.server.iface import MockEngine
from b200serve.server.logprobs import LOWEST, Entry, Score, chat_block, host_logprob, number, text_block
from test_server import TOK, enc, post, prompt_ids

V = 259
# the stand-in's rows: one logit of 5, one of 4, the others -5
LSE = math.log(math.exp(5) + math.exp(4) + (V - 2) * math.exp(-5))
BEST, SECOND, REST = 5 - LSE, 4 - LSE, -5 - LSE


class Plain(MockEngine):
    """Without scores of its own: the server takes them from the logits, and has none for a prompt."""

    def prompt_scores(self, ids, top=0):
        return None


@pytest.fixture()
def server():
    servers = []

    def make(script=None, engine=MockEngine, prefix=None, **kw):
        eng = engine(vocab_size=V, max_len=2048, max_seqs=2, script=script or {})
        srv = Server(eng, TOK, ChatTemplate(), ServerOptions(**kw), prefix=prefix).start()
        servers.append(srv)
        return srv, eng
    yield make
    for s in servers:
        s.stop()


def close(a, b):
    return a == pytest.approx(b, abs=1e-6)      # fp32 logits, 64-bit sums


MSGS = [{"role": "user", "content": "hi"}]
KW = {"chat_template_kwargs": {"enable_thinking": False}}


def chat_server(server, text="Hey.", **kw):
    pid = prompt_ids(MSGS, enable_thinking=False)
    return server({pid: list(enc(text)) + [2]}, **kw)


@pytest.mark.parametrize("top", [0, 1, 3])
def test_chat(server, top):
    srv, _ = chat_server(server)
    st, body = post(srv.port, "/v1/chat/completions", {"messages": MSGS, "logprobs": True, "top_logprobs": top, **KW})
    assert st == 200 and body["choices"][0]["message"]["content"] == "Hey."
    content = body["choices"][0]["logprobs"]["content"]
    assert [e["token"] for e in content] == list("Hey.") and [e["bytes"] for e in content] == [[ord(c)] for c in "Hey."]
    for e, c in zip(content, "Hey."):
        assert close(e["logprob"], BEST) and len(e["top_logprobs"]) == top
        if top:
            assert e["top_logprobs"][0]["token"] == c and close(e["top_logprobs"][0]["logprob"], BEST)
        if top > 1:
            assert e["top_logprobs"][1]["token"] == chr(ord(c) + 1) and close(e["top_logprobs"][1]["logprob"], SECOND)
        if top > 2:
            assert close(e["top_logprobs"][2]["logprob"], REST)
    st, body = post(srv.port, "/v1/chat/completions", {"messages": MSGS, **KW})
    assert st == 200 and "logprobs" not in body["choices"][0]


def test_chat_stream_tells_every_token_once(server):
    srv, _ = chat_server(server, "Hey été.")
    st, frames = post(srv.port, "/v1/chat/completions", {"messages": MSGS, "logprobs": True, "top_logprobs": 1, "stream": True, **KW}, stream=True)
    told = [e for f in frames[:-1] for e in (json.loads(f)["choices"][0].get("logprobs") or {"content": []})["content"]]
    assert bytes(b for e in told for b in e["bytes"]).decode() == "Hey été."
    assert all(close(e["logprob"], BEST) for e in told)


@pytest.mark.parametrize("stream", [False, True])
def test_completions(server, stream):
    srv, _ = server({enc("ab"): list(enc("cde"))})
    body = {"prompt": "ab", "max_tokens": 3, "logprobs": 2, "stream": stream}
    if stream:
        _, frames = post(srv.port, "/v1/completions", body, stream=True)
        blocks = [b for b in (json.loads(f)["choices"][0].get("logprobs") for f in frames[:-1]) if b]
        lp = {k: sum((b[k] for b in blocks), []) for k in blocks[0]}
    else:
        lp = post(srv.port, "/v1/completions", body)[1]["choices"][0]["logprobs"]
    assert lp["tokens"] == list("cde") and lp["text_offset"] == [0, 1, 2]
    assert all(close(x, BEST) for x in lp["token_logprobs"])
    for t, c in zip(lp["top_logprobs"], "cde"):
        assert set(t) == {c, chr(ord(c) + 1)} and close(t[c], BEST) and close(t[chr(ord(c) + 1)], SECOND)


@pytest.mark.parametrize("chunk", [4096, 3])
@pytest.mark.parametrize("stream", [False, True])
def test_echo_and_scored_prompt(server, chunk, stream):
    text = "abcdefgh"
    srv, eng = server({enc("ab"): list(enc("cdXXghij"))}, prefill_chunk=chunk)
    body = {"prompt": text, "max_tokens": 2, "logprobs": 1, "echo": True, "stream": stream}
    if stream:
        _, frames = post(srv.port, "/v1/completions", body, stream=True)
        ch = [json.loads(f)["choices"][0] for f in frames[:-1]]
        out = "".join(c["text"] for c in ch)
        blocks = [c["logprobs"] for c in ch if c.get("logprobs")]
        lp = {k: sum((b[k] for b in blocks), []) for k in blocks[0]}
    else:
        ch = post(srv.port, "/v1/completions", body)[1]["choices"][0]
        out, lp = ch["text"], ch["logprobs"]
    assert out.startswith(text) and lp["tokens"][: len(text)] == list(text) and lp["text_offset"] == list(range(len(lp["tokens"])))
    assert lp["token_logprobs"][0] is None and lp["top_logprobs"][0] is None
    ids = list(enc(text))
    for i in range(1, len(ids)):      # what the stand-in says of each prefix
        want = host_logprob(eng._row(eng._next(ids[:i])), ids[i], 1)
        assert close(lp["token_logprobs"][i], want.logprob)
    assert close(lp["token_logprobs"][-1], BEST)


def test_score_only(server):
    srv, eng = server()
    st, body = post(srv.port, "/v1/completions", {"prompt": "hello", "max_tokens": 0, "echo": True, "logprobs": 0})
    ch = body["choices"][0]
    assert st == 200 and ch["text"] == "hello" and ch["finish_reason"] == "length" and body["usage"]["completion_tokens"] == 0
    assert len(ch["logprobs"]["token_logprobs"]) == 5 and ch["logprobs"]["top_logprobs"] is None and eng.steps == 0
    # without scores: the text alone
    st, body = post(srv.port, "/v1/completions", {"prompt": list(enc("hello")), "max_tokens": 0, "echo": True})
    assert body["choices"][0]["text"] == "hello" and "logprobs" not in body["choices"][0]


def test_requests_that_are_refused(server):
    srv, _ = server(engine=Plain)
    assert post(srv.port, "/v1/completions", {"prompt": "x", "max_tokens": 0})[0] == 400
    for bad in (-1, 21, 1.5, "2", [1]):
        assert post(srv.port, "/v1/completions", {"prompt": "x", "logprobs": bad})[0] == 400
        assert post(srv.port, "/v1/chat/completions", {"messages": MSGS, "logprobs": True, "top_logprobs": bad})[0] == 400
    assert post(srv.port, "/v1/chat/completions", {"messages": MSGS, "logprobs": 3})[0] == 400
    st, body = post(srv.port, "/v1/completions", {"prompt": "xyz", "echo": True, "logprobs": 1, "max_tokens": 1})
    assert st == 400 and "prompt" in body["error"]["message"]
    # what needs no scores of the prompt works
    st, body = post(srv.port, "/v1/completions", {"prompt": "xyz", "logprobs": 1, "max_tokens": 2})
    assert st == 200 and all(close(x, BEST) for x in body["choices"][0]["logprobs"]["token_logprobs"])


class Full(MockEngine):
    def prompt_scores(self, ids, top=0):
        raise RuntimeError("no room")


def test_scores_that_cannot_be_made_fail_their_request(server):
    srv, _ = server(engine=Full)
    st, body = post(srv.port, "/v1/completions", {"prompt": "xyz", "echo": True, "logprobs": 1, "max_tokens": 1})
    assert st == 400 and "no room" in body["error"]["message"]
    assert post(srv.port, "/v1/completions", {"prompt": "xyz", "max_tokens": 1})[0] == 200


def test_fields_of_requests():
    one = lambda chat, **kw: H.parse_request(json.dumps({"messages": MSGS, "prompt": "p", **kw}), chat)      # noqa: E731
    assert one(True).logprobs == -1 and one(False).logprobs == -1 and not one(False).echo
    assert one(True, logprobs=True).logprobs == 0 and one(True, logprobs=True, top_logprobs=20).logprobs == 20
    assert one(True, logprobs=False, top_logprobs=5).logprobs == -1 and one(True, logprobs=None).logprobs == -1
    assert one(False, logprobs=0).logprobs == 0 and one(False, logprobs=5).logprobs == 5 and one(False, logprobs=None).logprobs == -1
    assert one(False, logprobs=True).logprobs == 0 and one(False, logprobs=False).logprobs == -1
    r = one(False, echo=True, max_tokens=0)
    assert r.echo and r.score_only and not one(False, echo=True, max_tokens=3).score_only and not one(True, echo=True).echo



def test_drafts_keep_their_scores(server):
    """Accepted drafts and the token behind them carry the scores of their own rows, whatever the step's width."""
    text = "one two three one two three one two three one two three"
    script = {enc("go "): list(enc(text)) + [2]}
    plain, _ = server(script)
    spec, eng = server(script, spec="lookup", spec_max=4)
    body = {"prompt": "go ", "logprobs": 1, "max_tokens": 80}
    a, b = (post(s.port, "/v1/completions", body)[1]["choices"][0] for s in (plain, spec))
    assert a["text"] == text == b["text"] and a["logprobs"] == b["logprobs"] and eng.steps < len(text) - 1


class Device(MockEngine):
    """With scores of its own for the rows of a step: counts the calls."""
    calls = 0

    def logprobs(self, items, top=0):
        self.calls += 1
        assert top == 2
        return [host_logprob(self._logits[slot][row], tok, top) for slot, row, tok in items]


def test_engine_scores_are_used(server):
    srv, eng = server({enc("ab"): list(enc("cde"))}, engine=Device)
    ch = post(srv.port, "/v1/completions", {"prompt": "ab", "max_tokens": 3, "logprobs": 2})[1]["choices"][0]
    assert eng.calls == 3 and len(ch["logprobs"]["tokens"]) == 3
    post(srv.port, "/v1/completions", {"prompt": "ab", "max_tokens": 3})
    assert eng.calls == 3


def test_sessions_of_a_step_get_what_they_asked_for(server):
    from types import SimpleNamespace as N
    srv, eng = server(engine=Plain)
    eng._logits = {0: [eng._row(7), eng._row(9)], 1: [eng._row(8)]}
    of = lambda slot, n: N(slot=slot, req=N(logprobs=n))      # noqa: E731
    a, b, c = of(0, 1), of(1, 5), of(0, -1)
    got = srv._logprobs([(a, 1, 9), (c, 0, 7), (b, 0, 8), (a, 0, 3)])
    assert [g and len(g.top) for g in got] == [1, None, 5, 1] and got[0].top[0][0] == 9 and got[2].top[0][0] == 8
    assert close(got[0].logprob, BEST) and close(got[3].logprob, REST)
    assert srv._logprobs([(c, 0, 1)]) == [None]


def test_a_response_without_tokens(server):
    srv, _ = server({enc("ab"): [2]})
    ch = post(srv.port, "/v1/completions", {"prompt": "ab", "logprobs": 1})[1]["choices"][0]
    assert ch["text"] == "" and ch["logprobs"] == {"tokens": [], "token_logprobs": [], "top_logprobs": [], "text_offset": []}


class Mixed(MockEngine):
    """Prompt portions and decode rows as one batch, which notes nothing of a prompt's scores."""
    mixed_batches = True
    slow = 0.002

    def step(self, rows):
        import time
        time.sleep(self.slow)
        return super().step(rows)


def test_scored_prompts_beside_decode_rows(server):
    import threading
    srv, eng = server(engine=Mixed, prefill_chunk=4)
    busy = threading.Thread(target=post, args=(srv.port, "/v1/completions", {"prompt": "go on", "max_tokens": 150, "ignore_eos": True}))
    busy.start()
    text = "a prompt in many portions"
    got = [post(srv.port, "/v1/completions", {"prompt": text, "max_tokens": 2, "echo": True, "logprobs": 1, "ignore_eos": True})[1]["choices"][0]["logprobs"]
           for _ in range(2)]
    busy.join()
    alone = post(srv.port, "/v1/completions", {"prompt": text, "max_tokens": 2, "echo": True, "logprobs": 1, "ignore_eos": True})[1]["choices"][0]["logprobs"]
    assert got == [alone, alone] and len(alone["tokens"]) == len(text) + 2
    assert post(srv.port, "/v1/completions", {"prompt": text, "max_tokens": 2})[0] == 200


class Prefix:
    """Hands out half of a prompt as cached."""
    asked = None

    def __init__(self):
        self.asked = []

    def preferred_slot(self, ids): return -1

    def begin(self, slot, ids, split_last=False):
        self.asked.append(list(ids))
        self.eng.reset(slot)
        n = len(ids) // 2
        self.eng.seqs[slot].extend(ids[:n])
        return n

    def after_prefill(self, slot, ids): pass
    def end(self, slot, ids): pass


def test_scored_prompts_do_not_come_from_the_cache(server):
    pre = Prefix()
    srv, eng = server(prefix=pre)
    pre.eng = eng
    st, body = post(srv.port, "/v1/completions", {"prompt": "hello world", "max_tokens": 1, "echo": True, "logprobs": 0})
    assert st == 200 and len(body["choices"][0]["logprobs"]["tokens"]) == 12 and pre.asked == [[]]
    assert body["usage"]["prompt_tokens_details"]["cached_tokens"] == 0
    st, body = post(srv.port, "/v1/completions", {"prompt": "hello world", "max_tokens": 1, "echo": True})
    assert st == 200 and body["usage"]["prompt_tokens_details"]["cached_tokens"] == 5


# ------------------------------------------------------------------ the host's sums and the forms
def test_host_logprob():
    z = np.array([0.0, 3.0, -np.inf, 3.0], dtype=np.float32)
    s = host_logprob(z, 0, 3)
    assert s.logprob == pytest.approx(-math.log(1 + 2 * math.exp(3))) and [i for i, _ in s.top] == [1, 3, 0]
    assert host_logprob(z, 2, 0) == Score(-math.inf, []) and math.isnan(host_logprob(z, -1, 0).logprob)
    assert host_logprob(np.full(3, -np.inf), 1, 1) == Score(-math.inf, [(0, -math.inf)])
    assert math.isnan(host_logprob(np.array([0.0, np.nan]), 0, 0).logprob) and math.isnan(host_logprob(np.array([0.0, np.inf]), 0, 0).logprob)


def test_forms():
    assert number(-math.inf) == LOWEST and number(math.nan) is None and number(-2.5) == -2.5
    e = [Entry(enc("a")[0], None), Entry(enc("b")[0], Score(-math.inf, [(enc("c")[0], -0.5), (0, -1.0), (1, -2.0)]))]
    block, at = text_block(TOK, e, 3, 7)
    assert block == {"tokens": ["a", "b"], "token_logprobs": [None, LOWEST], "top_logprobs": [None, {"c": -0.5, "": -1.0, "b": LOWEST}], "text_offset": [7, 8]}
    assert at == 9
    one = chat_block(TOK, e[1:])["content"][0]
    assert one["token"] == "b" and one["logprob"] == LOWEST and [t["token"] for t in one["top_logprobs"]] == ["c", "", ""]
