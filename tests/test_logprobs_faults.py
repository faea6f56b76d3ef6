"""Log probabilities: what goes wrong goes wrong for the request that asked, and nothing is taken from others (CPU)."""
import threading
import time

import pytest

from b200serve.server.app import Server, ServerOptions
from b200serve.server.chat_template import ChatTemplate
from b200serve.server.iface import MockEngine
from test_server import TOK, enc, post

V = 259


@pytest.fixture()
def serve():
    servers = []

    def make(engine, prefix=None, **kw):
        srv = Server(engine, TOK, ChatTemplate(), ServerOptions(**kw), prefix=prefix).start()
        servers.append(srv)
        return srv
    yield make
    for s in servers:
        s.stop()


class Broken(MockEngine):
    """Scores fail from the n-th call on; while it is asked for scores both requests are in the step."""
    good, calls, seen = 0, 0, 0

    def step(self, rows):
        self.seen = max(self.seen, len(rows))
        return super().step(rows)

    def logprobs(self, items, top=0):
        self.calls += 1
        if self.calls > self.good:
            raise RuntimeError("no scores")
        return None


class BrokenMixed(Broken):
    mixed_batches = True


@pytest.mark.parametrize("engine", [Broken, BrokenMixed])
@pytest.mark.parametrize("good", [0, 1, 5])
@pytest.mark.parametrize("stream", [False, True])
def test_scores_that_fail_in_a_step_fail_the_request_that_asked(serve, engine, good, stream):
    """The first token's scores, or a later step's: the requests beside it go on to their end."""
    eng = engine(vocab_size=V, max_len=2048, max_seqs=3, step_delay=0.002)
    eng.good = good
    srv = serve(eng, prefill_chunk=8)
    plain = {}

    def run(i):
        plain[i] = post(srv.port, "/v1/completions", {"prompt": f"request {i} goes on", "max_tokens": 200, "ignore_eos": True})
    ts = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    until = time.time() + 5
    while eng.seen < 2 and time.time() < until:      # both are in the steps
        time.sleep(0.001)
    body = {"prompt": "and this one is scored", "max_tokens": 60, "ignore_eos": True, "logprobs": 1, "stream": stream}
    got = post(srv.port, "/v1/completions", body, stream=stream)
    for t in ts:
        t.join()
    if stream and good:
        assert not any('"finish_reason":"length"' in f for f in got[1])
    else:
        assert got[0] == 500
    assert eng.seen == 3 or good == 0
    for st, b in plain.values():
        assert st == 200 and b["usage"]["completion_tokens"] == 200
    # alone they say the same
    for i, (_, b) in plain.items():
        again = post(srv.port, "/v1/completions", {"prompt": f"request {i} goes on", "max_tokens": 200, "ignore_eos": True})[1]
        assert again["choices"][0]["text"] == b["choices"][0]["text"]
