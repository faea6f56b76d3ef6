"""Token trees through the engine: their step, settled, against plain decoding of the same models."""
import random

import pytest
import torch

from b200serve.models import config as C
from b200serve.models.weights import random_weights
from b200serve.runtime.engine import Engine, Row

gpu = pytest.mark.gpu


def engine(name, weights, **kw):
    return Engine(weights, max_len=512, use_graphs=False, **kw)


def make_tree(chain, vocab, rng, wrong=2):
    """The chain's tokens with wrong ones beside them, in an order in which parents come first."""
    tokens, parents, at = [chain[0]], [-1], 0
    for t in chain[1:]:
        places = [None] * wrong + [t]
        rng.shuffle(places)
        here = at
        for x in places:
            tokens.append(rng.randrange(vocab) if x is None else x)
            parents.append(here)
            if x is not None:
                at = len(tokens) - 1
    return tokens, parents


def path_to(parents, i):
    out = []
    while i >= 0:
        out.append(i)
        i = parents[i]
    return out[::-1]


MODELS = {"tiny-dense": C.tiny_dense, "small-dense": C.small_dense, "small-windowed": C.small_windowed, "small-moe": C.small_moe}


@gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("name", MODELS)
def test_logits_of_every_node(name, kv):
    """A node's logits are those of its path decoded row by row (the same rows but for the order of sums: tolerance of the other step kernels)."""
    cfg = MODELS[name]()
    w = random_weights(cfg, device="cuda", seed=1)
    rng = random.Random(5)
    prompt = [rng.randrange(cfg.vocab) for _ in range(61)]
    tree = ([rng.randrange(cfg.vocab) for _ in range(11)], [-1, 0, 0, 1, 1, 2, 3, 3, 6, 6, 9])
    eng = engine(name, w, max_seqs=2, kv_dtype=kv, tree_nodes=16)
    eng.prefill(1, prompt)
    got = eng.trees.forward({1: tree}).clone()
    assert eng.seq_len == [0, 61]
    plain = engine(name, w, max_seqs=1, kv_dtype=kv)
    plain.prefill(0, prompt)
    for i in (0, 4, 5, 7, 10):
        path = path_to(tree[1], i)
        plain.truncate(0, len(prompt))
        plain.forward_rows([Row(0, len(prompt) + d, tree[0][n]) for d, n in enumerate(path)])
        want = plain.logits(len(path))
        for d, n in enumerate(path):
            # both sides round each layer's activations to bf16 from sums in other orders
            assert (got[n] - want[d]).norm() <= 0.02 * want[d].norm(), (i, n)


@gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("name", ["tiny-dense", "small-dense", "small-moe"])
def test_decoding_with_trees(name, kv):
    """Several requests decoded by trees that hold the right continuation, part of it or none: the tokens are those of plain decoding as long as that
    has no near ties, and the positions count up by the accepted paths."""
    cfg = MODELS[name]()
    w = random_weights(cfg, device="cuda", seed=2)
    rng = random.Random(9)
    prompts = [[rng.randrange(cfg.vocab) for _ in range(n)] for n in (40, 7, 129)]
    plain = engine(name, w, max_seqs=1, kv_dtype=kv)
    want, clear = [], []
    for p in prompts:
        plain.reset(0)
        tokens, sure = [plain.prefill(0, p)], [True]
        for _ in range(24):
            tokens.append(plain.forward_rows([Row(0, plain.seq_len[0], tokens[-1])])[0])
            top = plain.logits(1)[0].topk(2).values
            sure.append(bool(top[0] - top[1] > 0.05 * top[0].abs()))
        want.append(tokens)
        clear.append(sure)
    eng = engine(name, w, max_seqs=4, kv_dtype=kv, tree_nodes=20)
    out = {s: [eng.prefill(s, p)] for s, p in enumerate(prompts)}
    follow = {s: out[s][0] == want[s][0] for s in out}
    for round_ in range(5):
        trees = {}
        for s in out:
            n = len(out[s])
            ahead = want[s][n - 1: n + 3] if follow[s] else [out[s][-1]]
            ahead[0] = out[s][-1]
            keep = rng.choice((len(ahead), len(ahead), 1, 2))
            trees[s] = make_tree(ahead[:keep], cfg.vocab, rng)
        before = list(eng.seq_len)
        got = eng.verify_trees(trees)
        for s, v in got.items():
            tokens, parents = trees[s]
            assert v.path[0] == 0 and all(parents[b] == a for a, b in zip(v.path, v.path[1:]))
            assert v.tokens == [tokens[i] for i in v.path] and eng.seq_len[s] == before[s] + len(v.path)
            assert len(eng.pool.table(s)) == -(-eng.seq_len[s] // 16)
            out[s] += v.tokens[1:] + [v.next_token]
    checked = 0
    for s in out:
        for i, (a, b) in enumerate(zip(out[s], want[s])):
            if not all(clear[s][: i + 1]):
                break
            assert a == b, (s, i)
            checked += 1
    assert checked >= 6       # (a seed whose first tokens are clear)


@gpu
def test_refusals():
    cfg = C.tiny_dense()
    w = random_weights(cfg, device="cuda", seed=1)
    eng = engine("", w, max_seqs=2, tree_nodes=8)
    with pytest.raises(ValueError, match="no trees"):
        eng.trees.commit()
    for bad in ({0: ([1, 2], [-1])}, {0: ([1, 2], [0, 0])}, {0: ([1, 2], [-1, 1])}, {0: ([1] * 9, [-1] + [0] * 8)}, {2: ([1], [-1])}, {0: ([], [])}, {}, {0: ([5000], [-1])}):
        with pytest.raises(ValueError):
            eng.verify_trees(bad)
    assert eng.seq_len == [0, 0]
    with pytest.raises(ValueError, match="pages for trees"):
        engine("", w, max_seqs=1).verify_trees({0: ([1], [-1])})
    hybrid = random_weights(C.small_hybrid(), device="cuda", seed=1)
    with pytest.raises(ValueError, match="attention layers"):
        engine("", hybrid, max_seqs=1, tree_nodes=8)
    # a tree of one node on an empty slot
    v = eng.verify_trees({1: ([3], [-1])})
    assert v[1].path == [0] and v[1].tokens == [3] and eng.seq_len == [0, 1]
    torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_other_slots_run_between_a_step_and_its_settling(kv):
    """A step of trees is settled with its own tokens and arg-maxes, whatever other slots have run since."""
    cfg = C.small_dense()
    w = random_weights(cfg, device="cuda", seed=1)
    rng = random.Random(9)
    prompt, other = [rng.randrange(cfg.vocab) for _ in range(45)], [rng.randrange(cfg.vocab) for _ in range(20)]
    alone, shared = (engine("", w, max_seqs=2, kv_dtype=kv, tree_nodes=16) for _ in range(2))
    first = [e.prefill(0, prompt) for e in (alone, shared)]
    assert first[0] == first[1]
    chain = [first[0]]
    for _ in range(3):      # drafts: what the model itself goes on with
        chain.append(alone.verify_trees({0: ([chain[-1]], [-1])})[0].next_token)
    alone.truncate(0, len(prompt))
    tree = make_tree(chain, cfg.vocab, rng)
    want = alone.verify_trees({0: tree})[0]
    shared.trees.forward({0: tree})
    token = shared.prefill(1, other)
    shared.forward_rows([Row(1, len(other), token)])
    got = shared.trees.commit()
    assert got == {0: want} and len(want.path) > 1
    assert shared.seq_len == [len(prompt) + len(want.path), len(other) + 1]


@gpu
def test_trees_of_a_slot_that_changed_are_not_settled():
    cfg = C.tiny_dense()
    eng = engine("", random_weights(cfg, device="cuda", seed=1), max_seqs=2, tree_nodes=8)
    prompt, tree = [1, 2, 3, 4, 5], ([3, 4], [-1, 0])
    for change in (lambda: eng.truncate(0, 4), lambda: (eng.reset(0), eng.prefill(0, prompt)), lambda: eng.forward_rows([Row(0, 5, 7)])):
        eng.reset()
        eng.prefill(0, prompt)
        eng.trees.forward({0: tree})
        change()
        held = list(eng.seq_len)
        with pytest.raises(ValueError, match="no trees"):
            eng.trees.commit()
        assert eng.seq_len == held
    eng.trees.forward({1: tree})        # another slot's changes are not this one's
    eng.truncate(0, 2)
    assert 1 in eng.trees.commit()


@gpu
def test_trees_of_a_slot_with_other_pages_are_not_settled():
    """A slot that the prefix store gave other pages is not the one whose tree has run, though it is as long."""
    from b200serve.server.prefix import EngineKV
    eng = engine("", random_weights(C.tiny_dense(), device="cuda", seed=1), max_seqs=3, tree_nodes=8)
    store, tree = EngineKV(eng), ([3, 4], [-1, 0])
    eng.prefill(0, list(range(1, 33)))
    eng.prefill(1, list(range(41, 73)))
    for slot, pages in ((0, eng.pool.table(1)), (2, [])):
        eng.trees.forward({slot: tree})
        store.set_slot(slot, list(pages), eng.seq_len[slot])
        held = eng.kv.k.clone(), list(eng.seq_len)
        with pytest.raises(ValueError, match="no trees"):
            eng.trees.commit()
        assert torch.equal(eng.kv.k, held[0]) and eng.seq_len == held[1]
    eng.trees.forward({0: tree})
    store.set_slot(2, list(eng.pool.table(1)), 32)      # another slot's
    assert 0 in eng.trees.commit()


@gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_trees_beside_decoding_from_graphs(kv):
    """Steps of trees between decode steps that are replayed: the same tokens as those steps by themselves."""
    cfg = C.small_dense()
    w = random_weights(cfg, device="cuda", seed=1)
    prompts = [list(range(1, 46)), list(range(60, 80))]
    got = []
    for graphs in (False, True):
        eng = Engine(w, max_len=512, use_graphs=graphs, max_seqs=2, tree_nodes=40, kv_dtype=kv)
        last = [eng.prefill(s, p) for s, p in enumerate(prompts)]
        tokens = [[], []]
        for step in range(6):
            eng.decode_begin([0, 1], last)
            for _ in range(2):
                last = eng.decode_step()
                for s in (0, 1):
                    tokens[s].append(last[s])
            rng = random.Random(step)
            trees = {s: make_tree([last[s], rng.randrange(cfg.vocab), rng.randrange(cfg.vocab)], cfg.vocab, rng, 1 + step) for s in (0, 1)}
            for s, v in eng.verify_trees(trees).items():
                tokens[s] += v.tokens[1:] + [v.next_token]
                last[s] = v.next_token
        got.append((tokens, list(eng.seq_len)))
    assert got[0] == got[1]


@gpu
def test_trees_of_a_slot_whose_position_was_run_again_are_not_settled():
    """A row at a position that the slot has already replaces what the tree's rows have seen, and the slot stays as long as it was."""
    eng = engine("", random_weights(C.tiny_dense(), device="cuda", seed=1), max_seqs=2, tree_nodes=8)
    for s in (0, 1):
        eng.prefill(s, [1, 2, 3, 4, 5])
    eng.trees.forward({0: ([3, 4], [-1, 0])})
    eng.forward_rows([Row(0, 2, 9)])
    assert eng.seq_len == [5, 5]
    with pytest.raises(ValueError, match="no trees"):
        eng.trees.commit()
    eng.trees.forward({0: ([3, 4], [-1, 0])})
    eng.forward_rows([Row(1, 2, 9)])
    assert 0 in eng.trees.commit()


@gpu
def test_models_over_several_gpus_are_refused():
    """A pipeline's stage has some of the layers, experts of other ranks are others' steps: no step over trees."""
    from b200serve.parallel.pp import PipelineEngine
    w = random_weights(C.small_moe(), device="cuda", seed=1)
    with pytest.raises(ValueError, match="one GPU"):
        PipelineEngine(w, 0, 2, max_len=128, tree_nodes=8)
    PipelineEngine(w, 0, 2, max_len=128)
    eng = engine("", w, max_seqs=1, tree_nodes=8)
    eng.prefill(0, [1, 2, 3])
    eng.model.ep = object()
    with pytest.raises(ValueError, match="one GPU"):
        eng.verify_trees({0: ([3, 4], [-1, 0])})
    eng.model.ep = None
    assert eng.seq_len == [3] and 0 in eng.verify_trees({0: ([3, 4], [-1, 0])})
