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


def spread(kind):
    """Engines of which this GPU holds a part, as far as the checks of a call look."""
    from types import SimpleNamespace as N
    import torch
    from b200serve.parallel.pp import PipelineEngine
    from b200serve.runtime.engine import Engine
    e = object.__new__(PipelineEngine if kind == "pp" else Engine)
    e.tp, e.model, e.device = (N(world=2) if kind == "tp" else None), N(nccl=(0, 2, None) if kind == "nccl" else None), torch.device("cpu")
    e.cfg, e.broken, e.max_seqs = N(vocab=64, layer_specs=()), None, 1
    e.logits = lambda m: torch.zeros(m, 32 if kind != "pp" else 64)
    e.reset = lambda slot=None: pytest.fail("a slot was emptied for a call that is refused")
    return e


@pytest.mark.parametrize("kind", ["tp", "nccl", "pp"])
def test_part_of_a_vocabulary_is_not_scored(kind):
    """Sums over a slice of the vocabulary, or over rows that another stage holds, are no probabilities: refused, before anything is changed."""
    import torch
    e = spread(kind)
    for call in (lambda: e.logprobs([1, 2]), lambda: e.logprobs([1], 3, torch.zeros(1, 32)), lambda: e.score([1, 2, 3]), lambda: e.prompt_scores([1, 2])):
        with pytest.raises(ValueError, match="several GPUs"):
            call()
    with pytest.raises(ValueError, match="CUDA"):      # whole rows that the caller put together go to the kernel (no GPU here)
        e.logprobs([1], 0, torch.zeros(1, 64))


# ------------------------------------------------------------------ a prompt's results
def test_prompts_that_wait_hold_no_memory_of_the_device(monkeypatch):
    import torch
    from b200serve.runtime import scoring
    made = []
    buffer = scoring.ScoreBuffer
    monkeypatch.setattr(scoring, "ScoreBuffer", lambda rows, top, device: made.append((rows, top)) or buffer(rows, top, device))
    waiting = [scoring.PromptScores([5, 6, 7, 8], 3, torch.device("cpu")) for _ in range(4)]
    assert not made and all(w.buf is None and w.next is None for w in waiting)
    w = waiting[1]
    with pytest.raises(ValueError, match="not the prompt's"):
        w.expect([6])
    assert not made
    w.expect([5, 6])
    tokens, out = w.take(2)
    assert tokens.tolist() == [6, 7] and out.top_ids.shape == (2, 3)
    w.expect([7, 8])
    tokens, _ = w.take(2)
    assert tokens.tolist() == [8, -1] and made == [(4, 3)]
    assert len(w.read()) == 4
    with pytest.raises(ValueError, match="at most"):      # what can be said at once is said at once
        scoring.PromptScores([5], 33, torch.device("cpu"))
    with pytest.raises((ValueError, RuntimeError, OverflowError)):
        scoring.PromptScores([5, 1 << 32], 0, torch.device("cpu"))
    assert scoring.PromptScores([], 2, torch.device("cpu")).read() == []


def test_the_memory_plan_leaves_room_for_scored_prompts():
    from b200serve.models.config import preset
    from b200serve.ops import logprob as LP
    from b200serve.runtime import memory_plan as MP
    cfg = preset("dense-27b")
    auto = MP.plan(cfg, 64, "auto")
    slab = LP.slab_rows(4096, cfg.vocab, 5) * cfg.vocab * 4
    assert slab == 1024 * 151936 * 4 and auto.scores > slab
    assert auto.max_len < 262144 and auto.total + auto.scores <= auto.budget      # (the reserve is in the total)
    # a given length that fits beside the model is not refused; sharded models score no prompts
    most = MP.plan(cfg, 64, "auto", tp=2, budget=auto.budget)
    assert most.scores == 0
    page = MP.kv_bytes_per_page(cfg, "bf16")
    longer = auto.max_len + auto.scores // page // 64 * cfg.page_size
    assert longer > auto.max_len and MP.plan(cfg, 64, longer).total <= auto.budget
    # where they would take half of what is left, they do not
    kw = {"prefill_backend": "bf16"}
    given = MP.plan(cfg, 1, 1024, **kw)
    few = MP.plan(cfg, 1, "auto", budget=given.total, **kw)
    assert few.scores > given.kv_pool and few.max_len == 1024


@pytest.mark.gpu
def test_workspaces_are_what_the_plan_counts():
    from b200serve.ops import logprob as LP
    import ctypes
    room = LP._entry("b2_score_work", "iiiii", ctypes.c_longlong)
    for m, n, k, top, i8 in [(1, 700, 64, 0, 0), (128, 2048, 512, 3, 1), (129, 151936, 5120, 0, 0), (384, 102397, 200, 20, 1), (512, 151936, 2048, 5, 0),
                             (513, 151936, 2048, 5, 0), (1024, 151933, 5120, 32, 1), (4096, 151936, 5120, 0, 1), (32768, 2051, 128, 0, 1), (4096, 2048, 512, 5, 0)]:
        rows = LP.slab_rows(m, n, top)
        need = 4 * max(room(r, n, k, top, i8) for r in (rows, max(1, m % rows), min(rows, 512), min(rows, 256), 1))
        assert 0 < need <= LP.work_bytes(m, n, k, top, bool(i8))
        if rows > 512:
            assert LP.work_bytes(m, n, k, top, bool(i8)) <= 1.3 * need + (1 << 20)


# ------------------------------------------------------------------ what others had
def test_a_scored_prompt_leaves_the_session_it_resembles_alone(serve):
    """Nothing of a scored prompt comes from the cache: the slot that holds its beginning is not asked for, and the session there keeps it."""
    from test_logprobs_server import Prefix
    from test_prefix_store import FakeKV, run
    from b200serve.server.prefix import PrefixStore
    kv = FakeKV()
    store = PrefixStore(kv, host_gb=0, block_tokens=32)
    ids = list(range(3, 103))
    run(store, kv, 1, ids)

    class Slots(Prefix):
        granted = ()

        def preferred_slot(self, ids):
            return store.preferred_slot(ids)

        def begin(self, slot, ids, split_last=False):
            self.granted += (slot,)
            self.eng.reset(slot)
            return 0
    pre = Slots()
    eng = pre.eng = MockEngine(vocab_size=V, max_len=2048, max_seqs=2)
    srv = serve(eng, prefix=pre)
    assert store.preferred_slot(ids + [7]) == 1
    for extra, slot in (({}, 1), ({"echo": True, "logprobs": 0}, 0), ({"logprobs": 0}, 1), ({"echo": True}, 1)):
        assert post(srv.port, "/v1/completions", {"prompt": ids + [7], "max_tokens": 1, **extra})[0] == 200
        assert pre.granted[-1] == slot, extra


@pytest.mark.parametrize("chunk", [4096, 24])
def test_a_prompt_that_fills_the_context_can_be_scored(serve, chunk):
    srv = serve(MockEngine(vocab_size=V, max_len=64, max_seqs=1), prefill_chunk=chunk)
    body = {"max_tokens": 0, "echo": True, "logprobs": 1}
    st, got = post(srv.port, "/v1/completions", {"prompt": "x" * 64, **body})
    assert st == 200 and len(got["choices"][0]["logprobs"]["tokens"]) == 64 and got["usage"]["completion_tokens"] == 0
    for text, more in (("x" * 65, body), ("x" * 64, {"max_tokens": 1}), ("x" * 64, {"max_tokens": 1, "echo": True, "logprobs": 1})):
        st, got = post(srv.port, "/v1/completions", {"prompt": text, **more})
        assert st == 400 and "context holds 64" in got["error"]["message"]
    st, got = post(srv.port, "/v1/completions", {"prompt": "x" * 63, "max_tokens": 5, "ignore_eos": True})
    assert st == 200 and got["usage"]["completion_tokens"] == 1


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["small-dense", "small-hybrid", "napadra-mini"])
def test_a_prompt_that_fills_the_engine(name):
    import math
    from test_logprobs_engine import engine, prompt
    eng = engine(name)
    ids = prompt(eng.cfg, eng.max_len, 9)
    got = eng.score(ids, 1)
    assert len(got) == eng.max_len == eng.seq_len[0] and all(math.isfinite(s.logprob) for s in got[1:])
    with pytest.raises(ValueError, match="max_len"):
        eng.score(ids + [1])
    assert eng.score(ids, 1)[1:] == got[1:]


# ------------------------------------------------------------------ the host's sums
def test_the_host_puts_no_vocabulary_in_order(monkeypatch):
    """A row's alternatives on the serving thread: of 100,000 logits only those that can be among them are sorted, and none for a token alone."""
    import numpy as np
    from b200serve.server.logprobs import host_logprob
    sizes = []
    for name in ("argsort", "lexsort", "sort"):
        real = getattr(np, name)

        def noted(a, *args, real=real, **kw):
            sizes.append(np.asarray(a).shape[-1])
            return real(a, *args, **kw)
        monkeypatch.setattr(np, name, noted)
    z = np.random.default_rng(1).permutation(100000).astype(np.float32)
    assert host_logprob(z, 7, 20).top[0][0] == int(z.argmax()) and max(sizes, default=0) <= 64
    sizes.clear()
    host_logprob(z, 7, 0)
    assert not sizes


def test_host_alternatives_by_the_definition():
    """Larger first, ties to the lower id, banned ids behind numbers, NaN behind those: against a sort of the whole row."""
    import math
    import numpy as np
    from b200serve.server.logprobs import host_logprob
    rng = np.random.default_rng(2)
    for n in (1, 2, 7, 400):
        for bad in (0, 0.5, 1.0):
            for nan in (False, True):
                z = rng.integers(-3, 4, n).astype(np.float32)
                z[rng.random(n) < bad] = -np.inf
                if nan:
                    z[rng.random(n) < 0.3] = np.nan
                want = sorted(range(n), key=lambda i: (math.isnan(z[i]), -z[i] if not math.isnan(z[i]) else 0, i))
                finite = [float(v) for v in z if math.isfinite(v)]
                lse = math.log(sum(math.exp(v) for v in finite)) if finite else math.nan
                for top in (0, 1, 5, 20):
                    for t in (0, n - 1, -1, n):
                        s = host_logprob(z, t, top)
                        assert [i for i, _ in s.top] == want[:top]
                        for i, lp in [*s.top, (t, s.logprob)]:
                            if not 0 <= i < n or np.isnan(z).any():
                                assert math.isnan(lp)
                            elif not math.isfinite(z[i]):
                                assert lp == -math.inf
                            else:      # 64 bits: sums of 400 terms
                                assert abs(lp - (float(z[i]) - lse)) <= 1e-12


# ------------------------------------------------------------------ replicas
def _replicas(rank, world, port, q):
    import os
    import sys
    import torch.distributed as dist
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    from b200serve.parallel import launch as L
    from b200serve.server.iface import MockEngine
    from b200serve.server.logprobs import host_logprob
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    plane = L.ControlPlane()

    class Own(MockEngine):
        asked, mood = [], "score"

        def logprobs(self, items, top=0):
            self.asked.append((list(items), top))
            if self.mood == "fail":
                raise RuntimeError("no scores")
            return None if self.mood == "none" else [host_logprob(self._logits[s][r], t, top) for s, r, t in items]

        def set_mood(self, mood):
            self.mood = mood

        def logits(self, slot, row=0):
            assert False, "a whole row was asked for"
    eng = Own(vocab_size=259, max_seqs=2)
    if rank:
        q.put((rank, L.serve_replica_worker(eng, plane), eng.asked))
        return
    r = L.ReplicaRouter(eng, plane)
    for slot in (0, 1, 3, 4):
        r.prefill(slot, [10 + slot, 11])
    r.step({1: [7, 8], 4: [9]})
    items = [(4, 0, 5), (0, 0, 6), (1, 1, 7), (3, 0, 8), (1, 0, 9)]
    got = [r.logprobs(items, 2)]
    for mood, who in (("none", 2), ("fail", 1), ("fail", 0), ("score", 0)):
        r._call(who, "set_mood", mood)
        try:
            got.append(r.logprobs(items, 2))
        except RuntimeError as e:
            got.append(str(e))
        r._call(who, "set_mood", "score")
        assert r.length(4) == 3      # the answers are still those of their calls
    r.shutdown()
    # the same engine alone, with all slots
    one = MockEngine(vocab_size=259, max_seqs=6)
    for slot in (0, 1, 3, 4):
        one.prefill(slot, [10 + slot, 11])
    one.step({1: [7, 8], 4: [9]})
    q.put((0, got, [host_logprob(one.logits(s, row), t, 2) for s, row, t in items]))


def test_replicas_score_their_own_rows():
    import torch.multiprocessing as mp
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    ps = [ctx.Process(target=_replicas, args=(r, 3, 29709, q)) for r in range(3)]
    [p.start() for p in ps]
    res = {r[0]: r[1:] for r in (q.get(timeout=120) for _ in ps)}
    [p.join(timeout=60) for p in ps]
    assert all(p.exitcode == 0 for p in ps)
    got, want = res[0]
    assert got[0] == want == got[4] and got[1] is None and "no scores" in got[2] and "no scores" in got[3]
    assert res[1][1][0] == ([(1, 0, 8)], 2) and res[2][1][0] == ([(0, 0, 5)], 2)


# ------------------------------------------------------------------ tokens that are none
@pytest.mark.parametrize("bad", [64, 1 << 20, -1])
def test_tokens_outside_the_vocabulary_are_refused_on_the_host(bad):
    """The prompt pass gathers embeddings by token: no such id may reach the device."""
    from types import SimpleNamespace as N
    from b200serve.parallel.pp import PipelineEngine
    from b200serve.runtime.engine import Engine
    ids = [3] * 100
    ids[41] = bad

    def fake(cls):
        e = object.__new__(cls)
        e.tp, e.model, e.broken, e.max_rows, e.prefill_backend, e._prefill = None, N(nccl=None), None, 8, "bf16", None
        e.cfg, e.kv = N(vocab=64, layer_specs=(), head_dim=128, n_gdn_layers=0), N(kv_int8=False)
        e.reset = lambda slot=None: pytest.fail("a slot was emptied for a call that is refused")
        return e
    e, p = fake(Engine), fake(PipelineEngine)
    for call in (lambda: e.prefill(0, ids), lambda: e.score(ids), lambda: e.score([bad, 1]), lambda: e.prompt_scores(ids), lambda: p.prefill(0, ids)):
        with pytest.raises(ValueError, match=f"token {bad} is outside"):
            call()


@pytest.mark.parametrize("more", [{}, {"echo": True, "logprobs": 0}, {"echo": True, "max_tokens": 0}])
def test_prompt_ids_outside_the_vocabulary_are_a_bad_request(serve, more):
    srv = serve(MockEngine(vocab_size=V, max_len=512, max_seqs=1))
    for ids in ([V] * 2, [5, 6, 4000000000], [5] * 100 + [V]):
        st, body = post(srv.port, "/v1/completions", {"prompt": ids, "max_tokens": 2, **more})
        assert st == 400 and "outside the vocabulary" in body["error"]["message"]
    assert post(srv.port, "/v1/completions", {"prompt": [V - 1, 3], "max_tokens": 2, **more})[0] == 200


@pytest.mark.parametrize("bad", [(1 << 32) + 5, 1 << 32, (1 << 62) + 3])
def test_prompt_ids_of_more_than_32_bits_are_a_bad_request(serve, bad):
    """Cut to 32 bits they would be other tokens."""
    srv = serve(MockEngine(vocab_size=V, max_len=512, max_seqs=1))
    for ids in ([bad], [5, bad, 6]):
        st, body = post(srv.port, "/v1/completions", {"prompt": ids, "max_tokens": 2})
        assert st == 400 and "prompt token ids" in body["error"]["message"]
