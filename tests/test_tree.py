"""Steps over token trees against plain references: whole numbers by a walk in Python, attention and rotation in 64 bits."""
import math
import random

import pytest
import torch

from b200serve.ops import lib as K
from b200serve.ops import tree as T

gpu = pytest.mark.gpu
PAGE = 16
INF, NAN = float("inf"), float("nan")
HALF = torch.finfo(torch.bfloat16).eps / 2          # a rounding to bf16, relative


def tree_parents(n, rng, spread=4):
    return [-1 if i == 0 else i - 1 - rng.randrange(min(i, spread)) for i in range(n)]


def ancestors(parents):
    """Mask and depth of every node."""
    masks = []
    for i, up in enumerate(parents):
        masks.append(1 << i | (masks[up] if up >= 0 else 0))
    return masks, [bin(m).count("1") - 1 for m in masks]


def signed(mask):
    return mask - (1 << 64) if mask >> 63 else mask


class State:
    """Requests of given lengths with pages in random order.  ``free``: pages that are left."""

    def __init__(self, lengths, counts, seed=0, tree=True, blocks=None, free=None, spread=4, nodes=None, reserve=0, tree_blocks=4, parents=None):
        self.rng = rng = random.Random(seed)
        self.b, self.lengths, self.counts, self.tree = len(lengths), list(lengths), list(counts), tree
        self.held = [-(-n // PAGE) for n in lengths]
        grow = [-(-(n + max(c, 0)) // PAGE) - h for n, c, h in zip(lengths, counts, self.held)]
        self.blocks = blocks or max(1, max(h + max(g, 0) for h, g in zip(self.held, grow)) + 1)
        spare = max(1, sum(max(g, 0) for g in grow) + 3) if free is None else free
        self.pages = 1 + sum(self.held) + self.b * tree_blocks + spare
        order = list(range(1, self.pages))
        rng.shuffle(order)
        take = lambda n: [order.pop() for _ in range(n)]       # noqa: E731
        self.table = [(p := take(h)) + [0] * (self.blocks - len(p)) for h in self.held]
        self.tree_table = [take(tree_blocks) for _ in range(self.b)]
        self.free, self.n_free = order + [0] * sum(self.held), len(order)       # (room for pages that come back)
        self.parents = parents if parents is not None else [tree_parents(max(c, 0), rng, spread) for c in counts]
        self.rows = sum(max(c, 0) for c in counts)
        self.max_rows = max(1, self.rows + reserve)
        self.nodes = nodes or (min(64, 16 * tree_blocks) if not tree else max(1, max(counts)))

    def cuda(self):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")       # noqa: E731
        self.t_lengths, self.t_counts, self.t_held = i32(self.lengths), i32(self.counts), i32(self.held)
        self.t_table, self.t_tree, self.t_free, self.t_n = i32(self.table), i32(self.tree_table), i32(self.free), i32([self.n_free])
        self.t_parents = i32([p for one in self.parents for p in one]) if self.tree else None
        self.pool = T.PagePool(self.t_free, self.t_n, self.t_held)
        self.step = T.TreeStep(self.t_table, self.t_tree, self.max_rows, self.pages, self.nodes)
        return self

    def plan(self, after=None):
        T.plan(self.step, self.t_lengths, self.t_counts, self.t_parents, self.pool, after)
        return self.step

    def want(self):
        """The definition, walked through: what a plan leaves."""
        table, held, free = [list(t) for t in self.table], list(self.held), self.free[: self.n_free]
        out = {"row_start": [0], "row_req": [], "row_pos": [], "slots": [], "masks": [], "parents": []}
        for r, c in enumerate(self.counts):
            if c < 0:
                free += table[r][: held[r]]
                table[r][: held[r]] = [0] * held[r]
                held[r] = 0
        for r, c in enumerate(self.counts):
            c = max(c, 0)
            masks, depth = ancestors(self.parents[r]) if self.tree else ([0] * c, list(range(c)))
            need = max(depth) + 1 if c else 0
            while need and held[r] < -(-(self.lengths[r] + need) // PAGE):
                table[r][held[r]] = free.pop()
                held[r] += 1
            for i in range(c):
                pos = self.lengths[r] + depth[i]
                page, place = (self.tree_table[r][i // PAGE], i % PAGE) if self.tree else (table[r][pos // PAGE], pos % PAGE)
                out["row_req"].append(r)
                out["row_pos"].append(pos)
                out["slots"].append(page * PAGE + place)
                out["masks"].append(signed(masks[i]))
                out["parents"].append(self.parents[r][i] if self.tree else -1)
            out["row_start"].append(out["row_start"][-1] + c)
        pad = self.max_rows - self.rows
        for name in ("row_req", "row_pos", "slots", "parents"):
            out[name] += [-1] * pad
        out["masks"] += [0] * pad
        return {**out, "table": table, "held": held, "free": free}


# ------------------------------------------------------------------ plan
PLANS = {
    "one node, empty cache": dict(lengths=[0], counts=[1]),
    "one tree": dict(lengths=[700], counts=[16]),
    "a full page before, one node": dict(lengths=[16], counts=[1]),
    "chains of 64 over page ends": dict(lengths=[15, 16, 17, 0], counts=[64, 64, 64, 64], spread=1),
    "requests without rows": dict(lengths=[40, 0, 33, 7], counts=[0, 3, 0, 0]),
    "no rows at all": dict(lengths=[40, 0], counts=[0, 0]),
    "leaving requests": dict(lengths=[100, 31, 64, 5], counts=[-1, 20, -1, 3]),
    "leaving alone": dict(lengths=[100], counts=[-1]),
    "pages that came back are taken": dict(lengths=[100, 16], counts=[-1, 30], spread=1, free=0),
    "rows behind the last": dict(lengths=[9, 200, 1000], counts=[5, 64, 1], reserve=77),
    "many": dict(lengths=[(37 * i) % 501 for i in range(1024)], counts=[(5 * i) % 9 for i in range(1024)]),
    "rows": dict(lengths=[0, 5, 16, 4000], counts=[33, 1, 0, 17], tree=False),
    "rows of a long prompt": dict(lengths=[3, 70000], counts=[5001, 700], tree=False, reserve=9),
    "rows, leaving": dict(lengths=[50, 20], counts=[-1, 50], tree=False),
    "rows of many requests": dict(lengths=[(997 * i) % 3001 for i in range(300)], counts=[(37 * i) % 53 for i in range(300)], tree=False, reserve=2000),
    "pages that came back, many rows": dict(lengths=[30000, 5, 700], counts=[-1, 9000, 20000], tree=False, free=3),
    "many trees": dict(lengths=[(997 * i) % 3001 for i in range(200)], counts=[1 + (37 * i) % 64 for i in range(200)], spread=2),
    "thirty-two nodes a tree": dict(lengths=[33, 8], counts=[32, 9], tree_blocks=2),
}


def same_plan(s, after=None):
    want, pool = s.want(), after or s.pool
    step = s.step
    step.check()
    for name in ("row_start", "row_req", "row_pos", "slots") + (("parents", "masks") if s.tree else ()):
        assert getattr(step, name).tolist() == want[name], name
    assert s.t_table.tolist() == want["table"]
    assert pool.held.tolist() == want["held"]
    assert pool.n_free.tolist() == [len(want["free"])]
    assert pool.free.tolist()[: len(want["free"])] == want["free"]
    assert step.lengths.tolist() == [n if c >= 0 else 0 for n, c in zip(s.lengths, s.counts)]


@gpu
@pytest.mark.parametrize("name", PLANS)
def test_plan(name):
    s = State(**PLANS[name]).cuda()
    s.plan()
    same_plan(s)


@gpu
def test_plan_beside_its_pool():
    """Numbers written elsewhere: the pool's own stay, and the same plan can be made again."""
    s = State([30, 31, 500], [40, 2, 9], spread=2).cuda()
    after = T.PagePool(s.t_free, torch.empty_like(s.t_n), torch.empty_like(s.t_held))
    for _ in range(2):
        s.plan(after)
        same_plan(s, after)
    assert s.t_held.tolist() == s.held and s.t_n.tolist() == [s.n_free]


@gpu
def test_plan_of_no_parents():
    """An empty tensor of parents is a step of trees without nodes, not one of consecutive rows."""
    s = State([40, 7], [3, 2]).cuda()
    s.plan()
    assert s.step.masks.tolist()[0] == 1
    T.plan(s.step, s.t_lengths, torch.zeros_like(s.t_counts), s.t_parents[:0], s.pool)
    s.step.check()
    assert s.step.masks.tolist() == [0] * 5 and s.step.parents.tolist() == [-1] * 5 and s.step.row_start.tolist() == [0, 0, 0]
    T.plan(s.step, s.t_lengths, s.t_counts, s.t_parents[:0], s.pool)
    assert s.step.status.item() == 4


FAULTS = {
    "pool": (dict(lengths=[16, 3], counts=[20, 2], spread=1, free=1), 1),
    "table": (dict(lengths=[60], counts=[20], spread=1, blocks=4), 2),
    "nodes": (dict(lengths=[5], counts=[9], nodes=8), 8),
    "own parent": (dict(lengths=[5, 5], counts=[3, 3], parents=[[-1, 0, 0], [-1, 1, 0]]), 16),
    "parent behind": (dict(lengths=[5], counts=[3], parents=[[-1, 2, 0]]), 16),
    "parent below -1": (dict(lengths=[5], counts=[2], parents=[[-1, -2]]), 16),
    "length": (dict(lengths=[-1, 4], counts=[2, 2]), 32),
    "page": (dict(lengths=[4, 4], counts=[2, 2]), 64),
    "rows": (dict(lengths=[4, 4], counts=[2, 2]), 4),
    "pool, many rows": (dict(lengths=[16, 3], counts=[2000, 2000], tree=False, free=100), 1),
    "number of free pages": (dict(lengths=[4], counts=[2]), 1),
    "held": (dict(lengths=[4], counts=[2]), 2),
}


@gpu
@pytest.mark.parametrize("name", FAULTS)
def test_plan_that_cannot_be_made(name):
    kind, bit = FAULTS[name]
    s = State(**kind)
    if name == "page":
        s.tree_table[1][0] = s.pages
    if name == "number of free pages":
        s.n_free = len(s.free) + 1
    if name == "held":
        s.held[0] = s.blocks + 1
    s.cuda()
    if name == "rows":
        s.t_parents = s.t_parents[:3]
    before = [t.clone() for t in (s.t_table, s.t_held, s.t_n, s.t_free)]
    s.plan()
    assert s.step.status.item() == bit
    with pytest.raises(K.KernelError, match="plan: "):
        s.step.check()
    if bit != 64:
        assert all(torch.equal(a, b) for a, b in zip(before, (s.t_table, s.t_held, s.t_n, s.t_free)))
        assert s.step.row_start.tolist() == [0] * (s.b + 1) and set(s.step.slots.tolist()) == {-1}
        assert torch.equal(s.step.lengths, s.t_lengths)      # (what commit says behind it, too)
    else:
        assert s.step.slots.tolist()[2:] == [-1, -1] and min(s.step.slots.tolist()[:2]) >= 0


def unchanged(s, before):
    """A plan that could not be made left nothing."""
    assert all(torch.equal(a, b) for a, b in zip(before, (s.t_table, s.t_held, s.t_n, s.t_free)))
    assert s.step.row_start.tolist() == [0] * (s.b + 1) and set(s.step.slots.tolist()) == {-1}
    assert torch.equal(s.step.lengths, s.t_lengths)


@gpu
@pytest.mark.parametrize("at", [0, 5, 199])
@pytest.mark.parametrize("nodes", [3, 41])
def test_plan_with_a_bad_parent_among_many_trees(nodes, at):
    """One warp finds it while others have not come to the trees yet, in one CTA and in a cluster: all of them go the same way, so that nothing but the
    parent is at fault, and every barrier is everyone's."""
    s = State([(37 * i) % 301 for i in range(200)], [1 + (nodes - 1) * (i % 3 == 0 or i == at) for i in range(200)])
    s.parents[at][1] = 1
    s.cuda()
    before = [t.clone() for t in (s.t_table, s.t_held, s.t_n, s.t_free)]
    for _ in range(5):
        s.plan()
        assert s.step.status.item() == 16
        unchanged(s, before)
    s.t_parents[sum(s.counts[:at]) + 1] = s.parents[at][1] = 0
    s.plan()
    same_plan(s)


@gpu
@pytest.mark.parametrize("blocks,free,status", [(40, 1000, 1), (3, 1100, 2), (3, 1000, 3)])
@pytest.mark.parametrize("tree", [True, False])
def test_plan_of_many_requests_whose_pages_do_not_suffice(tree, blocks, free, status):
    """A request's table that is too short does not change what the others need: the pool is found short or not by all of their pages."""
    s = State([16] * 1024, [1] * 1023 + [40], tree=tree, spread=1, blocks=40, free=free)
    s.table, s.blocks = [t[:blocks] for t in s.table], blocks
    s.cuda()
    before = [t.clone() for t in (s.t_table, s.t_held, s.t_n, s.t_free)]
    for _ in range(20):
        s.plan()
        assert s.step.status.item() == status
    unchanged(s, before)


@gpu
@pytest.mark.parametrize("requests", [40, 500])
@pytest.mark.parametrize("bad", [0, 17, 39])
def test_plan_with_tree_pages_that_are_not_there(requests, bad):
    """Rows in such pages have no slots, and that is all: the requests' new pages, the pool and the numbers are those of the plan, whichever warps met
    them first."""
    s = State([16 * (1 + i % 3) for i in range(requests)], [1 + i % 2 for i in range(requests)])
    s.cuda()
    s.t_tree[bad, 0] = s.pages + 7
    after = T.PagePool(s.t_free, torch.empty_like(s.t_n), torch.empty_like(s.t_held))
    want, table = s.want(), s.t_table.clone()
    lost = [r == bad for r in want["row_req"]]
    slots = [-1 if gone else slot for slot, gone in zip(want["slots"], lost)]
    assert any(lost) and sum(h > -(-n // PAGE) for h, n in zip(want["held"], s.lengths)) == requests
    for _ in range(20):
        s.t_table.copy_(table)
        s.plan(after)
        assert s.step.status.item() == 64
        assert s.step.slots.tolist() == slots and s.step.row_pos.tolist() == want["row_pos"] and s.step.masks.tolist() == want["masks"]
        assert s.t_table.tolist() == want["table"] and after.held.tolist() == want["held"] and after.n_free.tolist() == [len(want["free"])]
        assert s.step.lengths.tolist() == s.lengths and s.step.row_start.tolist() == want["row_start"]


# ------------------------------------------------------------------ caches
def make_cache(pages, n_kv, d, i8, seed=0, layers=None, fill=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = ((layers,) if layers else ()) + (pages, n_kv, PAGE, d)
    if i8:
        k, v = (torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=g) for _ in range(2))
        ks, vs = (torch.rand(shape[:-1], device="cuda", generator=g) * 0.02 + 0.004 for _ in range(2))
        if fill is not None:
            ks.fill_(fill), vs.fill_(fill)
        return T.TreeCache(k, v, ks, vs)
    k, v = (torch.randn(shape, device="cuda", generator=g).bfloat16() for _ in range(2))
    if fill is not None:
        k.fill_(fill), v.fill_(fill)
    return T.TreeCache(k, v)


def rows_at(cache, name, slots):
    """Rows of a layer at slots, in 64 bits: [slot][kv head][d]."""
    x = getattr(cache, name)[slots // PAGE, :, slots % PAGE].double()
    return x * getattr(cache, name + "_scale")[slots // PAGE, :, slots % PAGE].double()[..., None] if cache.i8 else x


# ------------------------------------------------------------------ attention
def slots_of(s, r, table):
    """Slots of a request's cached positions, then of its nodes."""
    at = [table[r][j // PAGE] * PAGE + j % PAGE for j in range(s.lengths[r])]
    return at + [s.tree_table[r][i // PAGE] * PAGE + i % PAGE for i in range(max(s.counts[r], 0))]


def attention_reference(s, q, cache, scale, window, masks=None):
    """(outputs in 64 bits, what an output may be off by).

    Scores are fp32 sums of exact products of bf16 (and whole) numbers: off by at most (D + 4) 2^-24 sum|q k| scale, with the scale's and the
    base's roundings; 2^s then by that times its weight, and by ex2.approx's 2^-22.  A weight is rounded to bf16 (2^-8) before its product with
    v, whose scale in an 8-bit cache goes onto the weight first (2^-24 more).  The sums over up to n keys add n 2^-24 and the splits' factors a
    few 2^-22.  An output is rounded to bf16 at the end."""
    n_q, d = q.shape[1] // cache.d, cache.d
    group = n_q // cache.heads
    out, tol = torch.zeros(q.shape[0], n_q, d, dtype=torch.float64, device="cuda"), torch.zeros(q.shape[0], n_q, d, dtype=torch.float64, device="cuda")
    row = 0
    for r, c in enumerate(s.counts):
        c, length = max(c, 0), s.lengths[r]
        if not c:
            continue
        at = torch.tensor(slots_of(s, r, s.table), device="cuda")
        k, v = rows_at(cache, "k", at), rows_at(cache, "v", at)
        mask, depth = ancestors(s.parents[r])
        if masks is not None:
            mask = masks[row: row + c]
        pos = list(range(length)) + [length + x for x in depth]
        sees = torch.tensor([[(j < length or mask[i] >> (j - length) & 1 == 1) and (not window or pos[j] > pos[length + i] - window) for j in range(length + c)]
                             for i in range(c)], device="cuda").reshape(c, length + c)
        for h in range(n_q):
            x, kk, vv = q[row: row + c].reshape(c, n_q, d)[:, h].double(), k[:, h // group], v[:, h // group]
            kk, vv = torch.where(sees.any(0)[:, None], kk, 0.0), torch.where(sees.any(0)[:, None], vv, 0.0)
            z = (x @ kk.T * scale).masked_fill(~sees, -INF)
            p = torch.softmax(z, 1).nan_to_num(0.0)
            off = (x.abs() @ kk.abs().T) * abs(scale) * (d + 4) * 2.0 ** -24 + 2.0 ** -21
            n = length + c
            each = off + HALF + (n + 8) * 2.0 ** -24
            out[row: row + c, h] = p @ vv
            # the weights' errors, and the sum's, which is the weights'
            tol[row: row + c, h] = (p * each) @ vv.abs() + (p * (off + (n + 8) * 2.0 ** -24)).sum(1, keepdim=True) * (p @ vv.abs())
            tol[row: row + c, h] += HALF * (out[row: row + c, h].abs() + tol[row: row + c, h]) + 1e-30
        row += c
    return out, tol


ATTENTIONS = {
    "one node, empty cache": dict(lengths=[0], counts=[1]),
    "one node, one position": dict(lengths=[1], counts=[1]),
    "a page end": dict(lengths=[15, 16, 17], counts=[3, 1, 16]),
    "tile ends": dict(lengths=[63, 64, 65, 127, 128, 129], counts=[1, 2, 3, 4, 5, 64]),
    "64 nodes": dict(lengths=[500], counts=[64]),
    "chain of 64": dict(lengths=[33], counts=[64], spread=1),
    "no rows": dict(lengths=[40, 300, 7], counts=[0, 9, 0], reserve=3),
    "leaving": dict(lengths=[40, 30], counts=[-1, 5]),
    "long": dict(lengths=[5000, 1], counts=[16, 40]),
    "many": dict(lengths=[(91 * i) % 260 for i in range(70)], counts=[1 + i % 7 for i in range(70)]),
    "two roots": dict(lengths=[20], counts=[5], parents=[[-1, 0, -1, 2, 2]]),
}
HEADS = {"gqa5": (10, 2, 128), "gqa1": (3, 3, 128), "gqa4 d64": (8, 2, 64), "gqa16": (16, 1, 128), "gqa7 d64": (7, 1, 64)}


def run_attention(s, heads, i8, window=0, scale=None, seed=0, masks=None, cache=None, pad=0, qscale=1.5, clean=None, special=None):
    n_q, n_kv, d = heads
    s.cuda()
    s.plan()
    s.step.check()
    cache = cache or make_cache(s.pages, n_kv, d, i8, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = (torch.randn(s.max_rows, n_q * d + pad, device="cuda", generator=g) * qscale).bfloat16()[:, : n_q * d]
    out = torch.full((s.max_rows, n_q * d + pad), 7.0, dtype=torch.bfloat16, device="cuda")[:, : n_q * d]
    if masks is not None:
        s.step.masks[: s.rows] = torch.tensor([signed(m) for m in masks], device="cuda")
    scale = d ** -0.5 if scale is None else scale
    T.attention(s.step, q, cache, out, scale, window)
    torch.cuda.synchronize()
    K.check_status()
    want, tol = attention_reference(s, q, clean or cache, scale, window, masks)
    got = out.double().reshape(want.shape)
    if special is not None:      # no numbers where a sum has one, numbers elsewhere
        odd = ~torch.isfinite(special)
        assert torch.equal(got[odd].nan_to_num(-7.0, 1e30, -1e30), special[odd].nan_to_num(-7.0, 1e30, -1e30))
        got = torch.where(odd, want, got)
    bad = ~((got - want).abs()[: s.rows] <= tol[: s.rows])
    assert not bad.any(), ((got - want).abs()[: s.rows] - tol[: s.rows]).max()
    assert (out[s.rows:] == 7.0).all()
    return q, cache, out


@gpu
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("name", ATTENTIONS)
def test_attention(name, heads, i8):
    run_attention(State(**ATTENTIONS[name]), HEADS[heads], i8)


@gpu
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("heads,nodes", [((8, 8, 128), 13), ((32, 8, 128), 64), ((8, 8, 64), 30), ((40, 8, 64), 64), ((64, 4, 128), 40)])
def test_attention_long_parts(heads, nodes, i8):
    """Tens of tiles to a CTA, of several requests: rings go round, segments end in them, requests of a few tiles lie between long ones."""
    run_attention(State([9000, 40, 5003, 64, 0, 8200, 700, 6111], [nodes, 1, nodes // 2, nodes, 3, nodes, nodes, 5]), heads, i8)


@gpu
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("window", [1, 2, 15, 64, 100, 100000])
def test_attention_window(window, i8):
    run_attention(State([0, 3, 64, 777, 130], [5, 20, 64, 9, 1], spread=2), (8, 2, 128), i8, window)


@gpu
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_masks(d, i8):
    """Masks that a program changed: rows that see nothing, siblings, bits behind the tree."""
    s = State([0, 40], [6, 5])
    masks = [0, 0, 0b111111, 0b100000, 1 << 63 | 0b10, 0, 0, 0b11111, 1, 0b10000, 1 << 40]
    _, _, out = run_attention(s, (4, 2, d), i8, masks=masks)
    assert (out[[0, 1, 5]] == 0).all()


@gpu
@pytest.mark.parametrize("value", [INF, NAN, -INF])
@pytest.mark.parametrize("i8", [False, True])
def test_attention_places_that_nobody_sees(value, i8):
    """Slots behind a request's last position and behind a tree's last node may hold anything."""
    s = State([37, 0, 64, 130], [5, 3, 17, 64])
    cache = make_cache(s.pages, 2, 128, i8, fill=value)
    at = torch.tensor([x for r in range(s.b) for x in slots_of(s, r, s.table)], device="cuda")
    whole = make_cache(s.pages, 2, 128, i8, 5)
    for name in ("k", "v") + (("k_scale", "v_scale") if i8 else ()):
        getattr(cache, name)[at // PAGE, :, at % PAGE] = getattr(whole, name)[at // PAGE, :, at % PAGE]
    run_attention(s, (6, 2, 128), i8, cache=cache)


MIXED = {      # requests of one tile and of many, one part and several
    "short": dict(lengths=[37, 0, 64, 130], counts=[5, 3, 17, 64]),
    "long tables": dict(lengths=[37, 0, 64, 130, 2100], counts=[5, 3, 17, 64, 30], blocks=200),
}


@gpu
@pytest.mark.parametrize("window", [0, 20, 70])
@pytest.mark.parametrize("heads", [(6, 2, 128), (8, 1, 64), (5, 5, 64), (16, 2, 128)])
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("name", MIXED)
def test_attention_values_that_some_rows_see(name, i8, heads, window):
    """Infinities and NaN among the values of a node, or of a position at a window's edge, are theirs alone who see it."""
    n_q, n_kv, d = heads
    s = State(**MIXED[name])
    cache, clean = (make_cache(s.pages, n_kv, d, i8, 5) for _ in range(2))
    special = torch.zeros(s.rows, n_q, d, dtype=torch.float64, device="cuda")
    row = 0
    for r, (length, c) in enumerate(zip(s.lengths, s.counts)):
        at, (mask, depth) = slots_of(s, r, s.table), ancestors(s.parents[r])
        near = [j for j in range(length) if window and j >= length - window - 1]
        for j in s.rng.sample(near, min(3, len(near))) + [length + x for x in s.rng.sample(range(c), min(c, 4))]:
            page, place, h, value = at[j] // PAGE, at[j] % PAGE, s.rng.randrange(n_kv), s.rng.choice([INF, -INF, NAN])
            if i8:
                cache.v_scale[page, h, place], clean.v_scale[page, h, place] = value, 0.0
                v = cache.v[page, h, place].double() * value
            else:
                dims = s.rng.sample(range(d), 5)
                cache.v[page, h, place, dims], clean.v[page, h, place, dims] = value, 0.0
                v = torch.zeros(d, dtype=torch.float64, device="cuda")
                v[dims] = value
            for i in range(c):
                pos, sees = j if j < length else length + depth[j - length], j < length or mask[i] >> (j - length) & 1
                if sees and (not window or pos > length + depth[i] - window):
                    special[row + i, h * (n_q // n_kv): (h + 1) * (n_q // n_kv)] += v
        row += c
    run_attention(s, heads, i8, window, cache=cache, clean=clean, special=special)


@gpu
@pytest.mark.parametrize("blocks", [None, 400])
@pytest.mark.parametrize("heads", [(6, 2, 128), (16, 2, 128), (5, 5, 64)])
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("where", ["node", "position"])
def test_attention_values_of_no_weight_that_are_no_numbers(where, i8, heads, blocks):
    """A value that is no number decides the sums of the rows that see it, also where its key's score lies hundreds of powers of two below others: in one
    CTA (short tables) as in parts that are added up.  (The last request's tiles of little weight are every other one: those of a softmax group.)"""
    n_q, n_kv, d = heads
    s = State([300, 130, 100], [20, 9, 7], blocks=blocks)
    g = torch.Generator(device="cuda").manual_seed(11)
    sign = torch.randint(0, 2, (n_kv, d), device="cuda", generator=g) * 2.0 - 1
    cache, clean = (make_cache(s.pages, n_kv, d, i8, 5) for _ in range(2))
    special, row = torch.zeros(s.rows, n_q, d, dtype=torch.float64, device="cuda"), 0
    for r, (length, c) in enumerate(zip(s.lengths, s.counts)):
        at, mask = slots_of(s, r, s.table), ancestors(s.parents[r])[0]
        low = [j for j in range(length + c) if (j >= length if where == "node" else j < 64 or (j >= length and r == 2))]
        for j, slot in enumerate(at):      # keys along the queries, or against them
            way = -sign if j in low else sign
            noise = torch.randn(n_kv, d, device="cuda", generator=g)
            for t in (cache, clean):
                t.k[slot // PAGE, :, slot % PAGE] = (way * 100 + noise * 3).round().to(torch.int8) if i8 else (way * 12 + noise * 0.3).bfloat16()
                if i8:
                    t.k_scale[slot // PAGE, :, slot % PAGE] = 0.12
        j = length + 2 if where == "node" else 10
        page, place, h = at[j] // PAGE, at[j] % PAGE, r % n_kv
        if i8:
            cache.v_scale[page, h, place], clean.v_scale[page, h, place] = INF, 0.0
            v = cache.v[page, h, place].double() * INF
        else:
            dims = torch.tensor([3, 40, d - 1], device="cuda")
            v = torch.zeros(d, dtype=torch.float64, device="cuda")
            v[dims] = torch.tensor([INF, -INF, NAN], dtype=torch.float64, device="cuda")
            cache.v[page, h, place, dims], clean.v[page, h, place, dims] = v[dims].bfloat16(), 0.0
        for i in range(c):
            if j < length or mask[i] >> (j - length) & 1:
                special[row + i, h * (n_q // n_kv): (h + 1) * (n_q // n_kv)] += v
        row += c
    s.cuda()
    s.plan()
    s.step.check()
    q = (sign.repeat_interleave(n_q // n_kv, 0) * (1 + torch.rand(s.rows, n_q, d, device="cuda", generator=g) / 2)).bfloat16().flatten(1)
    out = torch.empty_like(q)
    T.attention(s.step, q, cache, out, d ** -0.5)
    torch.cuda.synchronize()
    K.check_status()
    want, tol = attention_reference(s, q, clean, d ** -0.5, 0)
    got, odd = out.double().reshape(want.shape), ~torch.isfinite(special)
    assert odd.any() and not torch.isfinite(got[odd]).any()
    if where == "node":      # (where all rows see a position, 0 times what is none is NaN)
        assert torch.equal(got[odd].nan_to_num(-7.0, 1e30, -1e30), special[odd].nan_to_num(-7.0, 1e30, -1e30))
    assert ((got - want).abs() <= tol)[~odd].all()


@gpu
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("name", MIXED)
def test_attention_scores_that_are_no_numbers(name, i8):
    """A query with a NaN, a key with an infinity: no numbers in the rows that they belong to or that see them, all others as ever."""
    s = State(**MIXED[name]).cuda()
    s.plan()
    s.step.check()
    cache = make_cache(s.pages, 2, 128, i8, 5)
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(s.rows, 6 * 128, device="cuda", generator=g).bfloat16()
    want, got = torch.empty_like(q), torch.empty_like(q)
    T.attention(s.step, q, cache, want, 0.1)
    odd = torch.zeros(s.rows, 6, dtype=torch.bool, device="cuda")
    q[2, 130], q[4, 0] = NAN, INF      # heads 1 and 0
    odd[2, 1] = odd[4, 0] = True
    row = 0
    for r, c in enumerate(s.counts):
        slot, mask = slots_of(s, r, s.table)[s.lengths[r] + c - 2], ancestors(s.parents[r])[0]
        if i8:
            cache.k_scale[slot // PAGE, 1, slot % PAGE] = INF
        else:
            cache.k[slot // PAGE, 1, slot % PAGE, 9] = INF
        for i in range(c):
            odd[row + i, 3:] |= bool(mask[i] >> (c - 2) & 1)
        row += c
    T.attention(s.step, q, cache, got, 0.1)
    torch.cuda.synchronize()
    K.check_status()
    got, want = got.reshape(s.rows, 6, 128), want.reshape(s.rows, 6, 128)
    # (an infinite score above all others, or a NaN: every weight is NaN; one below all others: its weight is 0)
    x = torch.isnan(got).all(2)
    assert not (x & ~odd).any() and torch.equal(got[~odd], want[~odd])
    assert x[2, 1] and x[4, 0]
    numbers = torch.isfinite(got).all(2)
    assert (numbers | x).all() and x[odd].sum() > odd.sum() // 4


@gpu
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("heads", [(10, 2, 128), (7, 1, 64)])
@pytest.mark.parametrize("name", ATTENTIONS)
def test_attention_long_tables(name, heads, i8):
    """Tables far longer than what is in them: parts over requests instead of a CTA for each."""
    run_attention(State(**ATTENTIONS[name], blocks=400), heads, i8)


@gpu
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("blocks", [20, 100])
@pytest.mark.parametrize("heads,window", [((2, 2, 64), 0), ((12, 2, 128), 0), ((4, 1, 128), 33)])
def test_attention_many_requests(heads, window, blocks, i8):
    """More requests than a CTA keeps the numbers of."""
    run_attention(State([(91 * i) % 270 for i in range(700)], [(5 * i) % 7 - (i % 9 == 0) if (5 * i) % 7 else 0 for i in range(700)], blocks=blocks), heads, i8, window)


@gpu
@pytest.mark.parametrize("qscale", [0.0, 60.0])
def test_attention_flat_and_sharp(qscale):
    run_attention(State([300, 20], [30, 64]), (8, 2, 128), False, qscale=qscale)


@gpu
def test_attention_strides():
    run_attention(State([300, 20], [30, 64]), (8, 2, 128), False, pad=24)


@gpu
@pytest.mark.parametrize("name", MIXED)
def test_attention_over_its_queries(name):
    s = State(**MIXED[name])
    q, cache, out = run_attention(s, (6, 2, 128), False)
    T.attention(s.step, q, cache, q, 128 ** -0.5)
    assert torch.equal(q[: s.rows], out[: s.rows])


@gpu
def test_attention_pages_that_are_not_there():
    """A table that names pages outside the cache: they are nobody's, and nothing is read."""
    s = State([100], [4]).cuda()
    s.plan()
    cache = make_cache(s.pages, 2, 128, False)
    q = torch.randn(s.max_rows, 512, device="cuda").bfloat16()
    want = torch.empty_like(q)
    T.attention(s.step, q, cache, want, 0.1)
    s.t_table[0, 4], s.t_table[0, 5] = 1 << 30, -5
    out = torch.empty_like(q)
    T.attention(s.step, q, cache, out, 0.1)
    torch.cuda.synchronize()
    s.lengths[0], s.table[0] = 64, s.table[0]
    assert torch.isfinite(out).all() and not torch.equal(out, want)


@gpu
@pytest.mark.parametrize("blocks", [None, 400])
@pytest.mark.parametrize("heads", [(6, 2, 128), (16, 2, 64)])
@pytest.mark.parametrize("i8", [False, True])
def test_attention_pages_that_are_not_there_read_as_page_0(i8, heads, blocks):
    """Entries of either table that name no page of the cache, in one CTA and in parts: page 0 in their place, and nothing else changes."""
    n_q, n_kv, d = heads
    s = State([100, 37, 200], [4, 20, 40], blocks=blocks).cuda()
    s.plan()
    s.step.check()
    cache = make_cache(s.pages, n_kv, d, i8, 9)
    q = torch.randn(s.rows, n_q * d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).bfloat16()
    for r, table, at, page in ((0, "table", 4, 1 << 30), (0, "table", 5, -5), (1, "table", 0, s.pages), (2, "table", 12, -(1 << 31)), (1, "tree_table", 1, s.pages + 3), (2, "tree_table", 0, -1)):
        getattr(s, table)[r][at] = 0
        (s.t_table if table == "table" else s.t_tree)[r, at] = page
    out = torch.empty_like(q)
    T.attention(s.step, q, cache, out, d ** -0.5)
    torch.cuda.synchronize()
    K.check_status()
    want, tol = attention_reference(s, q, cache, d ** -0.5, 0)
    assert ((out.double().reshape(want.shape) - want).abs() <= tol).all()


@gpu
@pytest.mark.parametrize("blocks", [None, 400])
@pytest.mark.parametrize("rows", [1, 3, 4, 17, 24, 63])
@pytest.mark.parametrize("i8", [False, True])
def test_fewer_rows_than_the_step_has(i8, rows, blocks):
    """Calls with the first of a step's rows: those rows' results, their keys and values, and nothing behind them."""
    s = State([100, 37, 200], [4, 20, 40], blocks=blocks).cuda()
    s.plan()
    s.step.check()
    cache = make_cache(s.pages, 2, 128, i8, 9)
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv, rope = torch.randn(s.rows, 10 * 128, device="cuda", generator=g), (torch.rand(300, 64, device="cuda", generator=g), torch.rand(300, 64, device="cuda", generator=g))
    q, part = (torch.full((s.rows, 6 * 128), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    whole = T.TreeCache(*(None if t is None else t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)))
    T.rope_append(s.step, qkv, rope, q, whole)
    T.rope_append(s.step, qkv[:rows], rope, part[:rows], cache)
    assert torch.equal(part[:rows], q[:rows]) and (part[rows:] == 7.0).all()
    at = s.step.slots.long()
    for name in ("k", "v") + (("k_scale", "v_scale") if i8 else ()):
        a, b = getattr(cache, name)[at // PAGE, :, at % PAGE], getattr(whole, name)[at // PAGE, :, at % PAGE]
        assert torch.equal(a[:rows], b[:rows]) and not (a[rows:] == b[rows:]).flatten(1).all(1).any()
    out = torch.full_like(q, 7.0)
    T.attention(s.step, q[:rows], whole, out[:rows], 0.1)
    torch.cuda.synchronize()
    K.check_status()
    assert (out[rows:] == 7.0).all()
    want, tol = attention_reference(s, q, whole, 0.1, 0)
    assert ((out.double().reshape(want.shape) - want).abs() <= tol)[:rows].all()


# ------------------------------------------------------------------ rotation and append
def rope_reference(x, pos, freq, interleaved):
    """Turned heads [rows][heads][d] in 64 bits."""
    x, n = x.double().clone(), freq.numel()
    angle = pos.double()[:, None, None] * freq
    c, s = angle.cos(), angle.sin()
    a, b = (x[..., 0: 2 * n: 2].clone(), x[..., 1: 2 * n: 2].clone()) if interleaved else (x[..., :n].clone(), x[..., n: 2 * n].clone())
    lo, hi = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    x[..., lo], x[..., hi] = a * c - b * s, b * c + a * s
    return x


APPENDS = {
    "one row": dict(lengths=[0], counts=[1]),
    "trees": dict(lengths=[0, 15, 700, 31], counts=[5, 64, 1, 17], reserve=6),
    "no rows": dict(lengths=[3, 9], counts=[0, 2]),
    "rows": dict(lengths=[0, 30, 5], counts=[40, 1, 100], tree=False, reserve=3),
    "many rows": dict(lengths=[100, 0], counts=[1500, 700], tree=False),
}


@gpu
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,rot", [((10, 2, 128), 128), ((4, 4, 64), 64), ((6, 1, 128), 40), ((8, 2, 64), 24), ((3, 1, 128), 8), ((5, 1, 128), 0)])
@pytest.mark.parametrize("slices", [0, 1, 3])
@pytest.mark.parametrize("name", APPENDS)
def test_rope_append(name, heads, rot, slices, interleaved, i8):
    n_q, n_kv, d = heads
    s = State(**APPENDS[name]).cuda()
    s.plan()
    s.step.check()
    g = torch.Generator(device="cuda").manual_seed(3)
    n = (n_q + 2 * n_kv) * d
    x = torch.randn(max(slices, 1), s.max_rows, n + 16, device="cuda", generator=g)[..., :n]
    x[0, 0, n_q * d: (n_q + 1) * d] = 0          # a key of zeros
    if slices > 1:
        x[1:, 0, n_q * d: (n_q + 1) * d] = 0
    qkv = x if slices else x[0].bfloat16()
    freq = torch.tensor([1e4 ** (-2 * i / max(rot, 1)) / 2.5 for i in range(rot // 2)], dtype=torch.float64, device="cuda")
    angle = torch.arange(max(s.lengths) + 1600, device="cuda", dtype=torch.float64)[:, None] * freq
    rope = (angle.cos().float().contiguous(), angle.sin().float().contiguous())
    q = torch.full((s.max_rows, n_q * d), 7.0, dtype=torch.bfloat16, device="cuda")
    cache = make_cache(s.pages, n_kv, d, i8)
    before = [t.clone() for t in (cache.k, cache.v)]
    T.rope_append(s.step, qkv, rope, q, cache, interleaved)
    torch.cuda.synchronize()
    K.check_status()
    rows = s.rows
    y = (x.double().sum(0) if slices else qkv.double())[:rows].reshape(rows, -1, d)
    size = (x.double().abs().sum(0) if slices else qkv.double().abs())[:rows].reshape(rows, -1, d)
    pos, slots = s.step.row_pos[:rows], s.step.slots[:rows].long()
    turned = rope_reference(y[:, : n_q + n_kv], pos, freq, interleaved)
    # sums of slices, cosine and sine, two products and their sum: each rounded to fp32, of numbers no larger than the pair's
    fp32 = 2.0 ** -24 * (max(slices, 1) + 4) * 2 * (size.amax(-1, keepdim=True) + 1e-30)
    assert ((q[:rows].double().reshape(rows, n_q, d) - turned[:, :n_q]).abs() <= HALF * turned[:, :n_q].abs() + 2 * fp32[:, :n_q]).all()
    assert (q[rows:] == 7.0).all()
    for name_, want, slack in (("k", turned[:, n_q:], fp32[:, n_q: n_q + n_kv]), ("v", y[:, n_q + n_kv:], fp32[:, n_q + n_kv:])):
        got = rows_at(cache, name_, slots)
        if i8:
            largest = want.abs().amax(-1, keepdim=True)
            scale = getattr(cache, name_ + "_scale")[slots // PAGE, :, slots % PAGE].double()[..., None]
            assert ((scale - torch.where(largest > 0, largest / 127, 1.0)).abs() <= slack / 127 + largest * 2.0 ** -24).all()
            assert ((got - want).abs() <= scale * (0.5 + 127 * 2.0 ** -22) + slack).all()
        else:
            assert ((got - want).abs() <= HALF * want.abs() + 2 * slack).all()
    left = torch.ones(s.pages * PAGE, dtype=torch.bool, device="cuda")
    left[slots] = False
    for t, was in zip((cache.k, cache.v), before):       # every other slot is as it was
        flat = lambda z: z.transpose(1, 2).reshape(s.pages * PAGE, -1)[left]         # noqa: E731
        assert torch.equal(flat(t), flat(was))


@gpu
def test_rope_append_behind_the_tables():
    """Positions that the tables do not have are an error of the kernel's, and their rows are left."""
    s = State([100, 3], [4, 4], spread=1).cuda()
    s.plan()
    cache = make_cache(s.pages, 1, 64, False)
    before = cache.k.clone()
    q = torch.full((8, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    table = torch.ones(50, 32, device="cuda")
    T.rope_append(s.step, torch.randn(8, 256, device="cuda"), (table, table), q, cache)
    torch.cuda.synchronize()
    with pytest.raises(K.KernelError):
        K.check_status()
    K.status_clear()
    slots = s.step.slots[:4].long()
    assert (q[:4] == 7.0).all() and not (q[4:] == 7.0).all()
    assert torch.equal(cache.k[slots // PAGE, :, slots % PAGE], before[slots // PAGE, :, slots % PAGE])


# ------------------------------------------------------------------ commit
def commit_reference(s, tokens, targets):
    row, out = 0, []
    for r, c in enumerate(s.counts):
        c, path, following = max(c, 0), [], -1
        if c:
            at = 0
            while at is not None:
                path.append(at)
                following = targets[row + at]
                at = next((i for i in range(at + 1, c) if s.parents[r][i] == at and tokens[row + i] == following), None)
        out.append((path, following))
        row += c
    return out


COMMITS = {
    "one node, empty cache": dict(lengths=[0], counts=[1]),
    "one tree": dict(lengths=[700], counts=[16]),
    "chains over page ends": dict(lengths=[15, 16, 0, 1], counts=[64, 20, 64, 33], spread=1),
    "idle and leaving requests": dict(lengths=[40, 30, 9], counts=[0, 12, -1]),
    "many": dict(lengths=[(37 * i) % 101 for i in range(80)], counts=[(5 * i) % 13 for i in range(80)]),
    "two roots": dict(lengths=[20], counts=[5], parents=[[-1, 0, -1, 2, 2]]),
}


@gpu
@pytest.mark.parametrize("layers,n_kv,d,i8", [(None, 2, 128, False), (3, 1, 64, False), (5, 3, 128, True), (None, 2, 64, True)])
@pytest.mark.parametrize("chance", [0.0, 0.7, 1.0])
@pytest.mark.parametrize("name", COMMITS)
def test_commit(name, chance, layers, n_kv, d, i8):
    s = State(**COMMITS[name]).cuda()
    s.plan()
    s.step.check()
    rng = random.Random(7)
    tokens = [rng.randrange(4) for _ in range(s.max_rows)]      # few tokens: siblings that are alike
    targets, row = [rng.randrange(4) for _ in range(s.max_rows)], 0
    for r, c in enumerate(s.counts):
        for i in range(max(c, 0)):
            children = [j for j in range(i + 1, c) if s.parents[r][j] == i]
            if children and rng.random() < chance:
                targets[row + i] = tokens[row + rng.choice(children)]
            elif chance == 0.0:
                targets[row + i] = 9
        row += max(c, 0)
    cache = make_cache(s.pages, n_kv, d, i8, layers=layers)
    names = ("k", "v") + (("k_scale", "v_scale") if i8 else ())
    want = {n: getattr(cache, n).clone() for n in names}
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")       # noqa: E731
    got = T.commit(s.step, i32(tokens), i32(targets), cache)
    torch.cuda.synchronize()
    K.check_status()
    table = s.t_table.tolist()
    for r, (path, following) in enumerate(commit_reference(s, tokens, targets)):
        length = s.lengths[r] if s.counts[r] >= 0 else 0
        assert got.path[r].tolist() == path + [-1] * (64 - len(path))
        assert got.count[r].item() == len(path) and got.next_token[r].item() == following and got.lengths[r].item() == length + len(path)
        for i, node in enumerate(path):
            src, dst = s.tree_table[r][node // PAGE], table[r][(length + i) // PAGE]
            for n in names:
                t = want[n] if layers else want[n][None]
                t[:, dst, :, (length + i) % PAGE] = t[:, src, :, node % PAGE]
    for n in names:
        assert torch.equal(getattr(cache, n), want[n]), n


@gpu
def test_commit_results_apart_from_what_it_reads():
    """Results over the tokens, the targets or the step would be written while other layers' walks still read: refused."""
    s = State([20, 5], [7, 4]).cuda()
    s.plan()
    cache = make_cache(s.pages, 1, 64, False, layers=3)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")       # noqa: E731
    tokens, targets, room = i32(11), i32(11), i32(200)
    for count, following, lengths in ((tokens[9:], i32(2), i32(2)), (i32(2), tokens[:2], i32(2)), (i32(2), targets[3: 5], i32(2)), (i32(2), i32(2), targets[:2]),
                                      (s.step.lengths, i32(2), i32(2)), (i32(2), i32(2), s.step.lengths), (i32(2), s.step.row_start[1:], i32(2)),
                                      (i32(2), s.step.parents[8: 10], i32(2)), (s.step.slots[:2], i32(2), i32(2)), (s.step.row_pos[9:], i32(2), i32(2)),
                                      (i32(2), s.step.row_req[4: 6], i32(2)), (i32(2), i32(2), s.step.masks.view(torch.int32)[20:]), (s.t_table.view(-1)[1: 3], i32(2), i32(2)), (i32(2), s.t_tree.view(-1)[3: 5], i32(2))):
        with pytest.raises(ValueError, match="apart from"):
            T.commit(s.step, tokens, targets, cache, T.Accepted(i32(128).view(2, 64), count, following, lengths))
    with pytest.raises(ValueError, match="apart from"):
        T.commit(s.step, room[120: 131], targets, cache, T.Accepted(room[:128].view(2, 64), i32(2), i32(2), i32(2)))
    want = T.commit(s.step, tokens, targets, cache)
    got = T.commit(s.step, room[128: 139], targets, cache, T.Accepted(room[:128].view(2, 64), room[139: 141], room[141: 143], s.t_lengths))
    for name in ("path", "count", "next_token", "lengths"):
        assert torch.equal(getattr(want, name), getattr(got, name))
    K.check_status()


# ------------------------------------------------------------------ refusals
def test_refusals_on_the_host():
    """What is not on a CUDA device is refused before the library is asked."""
    z = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="free pages"):
        T.PagePool(z, z[:1], z)
    with pytest.raises(ValueError, match="block table"):
        T.TreeStep(z.reshape(2, 2), z.reshape(2, 2), 8, 10)
    with pytest.raises(ValueError):
        T.TreeCache(torch.zeros(3, 2, 16, 128, dtype=torch.bfloat16), torch.zeros(3, 2, 16, 128, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        T.Accepted.empty(3, "cpu")


@gpu
def test_refusals():
    s = State([30, 4], [5, 3]).cuda()
    step, cache = s.step, make_cache(s.pages, 2, 128, False)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")       # noqa: E731
    bf = lambda *n: torch.zeros(n, dtype=torch.bfloat16, device="cuda")     # noqa: E731
    q, out, rope = bf(8, 512), bf(8, 512), (torch.ones(200, 64, device="cuda"),) * 2
    qkv = torch.zeros(8, 1024, device="cuda")
    no = lambda f, *a, **k: pytest.raises(ValueError, f, *a, **k)      # noqa: E731
    # before a plan
    no(T.attention, step, q, cache, out, 0.1)
    no(T.rope_append, step, qkv, rope, q, cache)
    no(T.commit, step, i32(8), i32(8), cache)
    # steps, pools and plans
    no(T.TreeStep, s.t_table, s.t_tree, 0, s.pages)
    no(T.TreeStep, s.t_table, s.t_tree, 1 << 21, s.pages)
    no(T.TreeStep, s.t_table, s.t_tree, 8, s.pages, 65)
    no(T.TreeStep, s.t_table, s.t_tree[:, :1].contiguous(), 8, s.pages, 17)
    no(T.TreeStep, s.t_table, s.t_tree[:1], 8, s.pages)
    no(T.TreeStep, s.t_table.long(), s.t_tree, 8, s.pages)
    no(T.TreeStep, s.t_table, s.t_tree[:, ::2], 8, s.pages)
    no(T.TreeStep, s.t_table, s.t_tree, 8, 0)
    no(T.PagePool, s.t_free, i32(2), s.t_held)
    no(T.PagePool, s.t_free.long(), s.t_n, s.t_held)
    no(T.plan, step, i32(3), s.t_counts, s.t_parents, s.pool)
    no(T.plan, step, s.t_lengths, s.t_counts.long(), s.t_parents, s.pool)
    no(T.plan, step, s.t_lengths, s.t_counts, i32(9), s.pool)
    no(T.plan, step, s.t_lengths, s.t_counts, s.t_parents, T.PagePool(s.t_free, s.t_n, i32(3)))
    no(T.plan, step, s.t_lengths, s.t_counts, s.t_parents, s.pool, T.PagePool(s.t_free.clone(), s.t_n, s.t_held))
    s.plan()
    # caches
    k = bf(3, 2, 16, 128)
    no(T.TreeCache, k, k[:2])
    no(T.TreeCache, k.half(), k.half())
    no(T.TreeCache, bf(3, 2, 8, 128), bf(3, 2, 8, 128))
    no(T.TreeCache, bf(3, 2, 16, 96), bf(3, 2, 16, 96))
    no(T.TreeCache, k[:, :1], k[:, :1])
    no(T.TreeCache, k.to(torch.int8), k.to(torch.int8))
    no(T.TreeCache, k.to(torch.int8), k.to(torch.int8), torch.ones(3, 2, 16, device="cuda"))
    no(T.TreeCache, k.to(torch.int8), k.to(torch.int8), torch.ones(3, 2, 16, device="cuda"), torch.ones(3, 2, 15, device="cuda"))
    no(T.TreeCache, k, k, torch.ones(3, 2, 16, device="cuda"), torch.ones(3, 2, 16, device="cuda"))
    no(T.TreeCache, bf(3 * 2 * 16 * 128 + 4)[4:].reshape(3, 2, 16, 128), k)
    many = make_cache(s.pages, 2, 128, False, layers=2)
    small = make_cache(s.pages - 1, 2, 128, False)
    # attention
    for bad in ((step, q.float(), cache, out, 0.1), (step, q, cache, out[:7], 0.1), (step, bf(9, 512), cache, bf(9, 512), 0.1), (step, q[:, :500], cache, out[:, :500], 0.1),
                (step, bf(8, 384), cache, bf(8, 384), 0.1), (step, q, many, out, 0.1), (step, q, small, out, 0.1), (step, q, cache, out, 0.1, -1), (step, q, cache, out, INF), (step, q, cache, out, 0.0), (step, q, cache, out, -0.1),
                (step, q, cache, out, NAN), (step, bf(8, 513)[:, 1:], cache, out, 0.1), (step, q.cpu(), cache, out, 0.1), (step, q[:0], cache, out[:0], 0.1),
                (step, bf(8, 2 * 65 * 128), cache, bf(8, 2 * 65 * 128), 0.1), (step, q, cache, out.t().contiguous().t(), 0.1)):
        no(T.attention, *bad)
    # rotation
    for bad in ((step, qkv.half(), rope, q, cache), (step, qkv, rope, q[:7], cache), (step, qkv, rope, bf(8, 384), cache), (step, qkv[:, :1000], rope, q, cache),
                (step, torch.zeros(9, 1024, device="cuda"), rope, bf(9, 512), cache), (step, qkv, (rope[0], rope[1][:100]), q, cache), (step, qkv, (rope[0][:, :6].contiguous(),) * 2, q, cache),
                (step, qkv, (torch.ones(200, 68, device="cuda"),) * 2, q, cache), (step, qkv, rope, q, many), (step, qkv, rope, q, small), (step, qkv[:, ::2], rope, q, cache),
                (step, torch.zeros(0, 8, 1024, device="cuda"), rope, q, cache), (step, qkv, (rope[0][:0], rope[1][:0]), q, cache), (step, qkv[:, :512], rope, bf(8, 0), cache),
                (step, torch.zeros(8, 1026, device="cuda")[:, 2:], rope, q, cache)):
        no(T.rope_append, *bad)
    # commit
    own = T.Accepted(torch.zeros(2, 64, dtype=torch.int32, device="cuda"), i32(2), i32(2), step.lengths)
    for bad in ((step, i32(8).long(), i32(8), cache), (step, i32(8), i32(7), cache), (step, i32(9), i32(9), cache), (step, i32(8), i32(8), small), (step, i32(0), i32(0), cache),
                (step, i32(8), i32(8), cache, T.Accepted.empty(3, "cuda")), (step, i32(8), i32(8), cache, own), (step, i32(16)[::2], i32(8), cache)):
        no(T.commit, *bad)
    # rows that are no trees'
    r = State([30, 4], [5, 3], tree=False).cuda()
    r.plan()
    no(T.attention, r.step, q, make_cache(r.pages, 2, 128, False), out, 0.1)
    no(T.commit, r.step, i32(8), i32(8), make_cache(r.pages, 2, 128, False))
    torch.cuda.synchronize()
    K.check_status()


@gpu
def test_tables_whose_positions_pass_32_bits_are_refused():
    table, tree = torch.zeros(1, 1 << 27, dtype=torch.int32, device="cuda"), torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="pages"):
        T.TreeStep(table, tree, 8, 100)
    T.TreeStep(table[:, : (1 << 27) - 1], tree, 8, 100)


# ------------------------------------------------------------------ a run of them together
class Loop:
    """Requests that decode by trees, everything on the device: plan, one layer's append and attention, commit, lengths and pages carried from step
    to step."""

    def __init__(self, seed, i8=False, spare=40):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.b, self.nodes, self.n_q, self.n_kv, self.d = 3, 7, 4, 2, 64
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")       # noqa: E731
        held = [2, 1, 0]
        pages = 1 + 3 + 3 + spare
        self.table = torch.zeros(3, 12, dtype=torch.int32, device="cuda")
        self.table[0, :2], self.table[1, :1] = i32([1, 2]), i32([3])
        self.pool = T.PagePool(torch.arange(7, 7 + spare, dtype=torch.int32, device="cuda"), i32([spare]), i32(held))
        self.step = T.TreeStep(self.table, i32([[4], [5], [6]]), 3 * self.nodes, pages, self.nodes)
        self.lengths, self.counts = i32([20, 16, 0]), i32([self.nodes, 3, self.nodes])
        self.cache = make_cache(pages, self.n_kv, self.d, i8, seed)
        self.accepted = T.Accepted(i32([[0] * 64] * 3), i32([0] * 3), i32([0] * 3), self.lengths)
        rows = 2 * self.nodes + 3
        self.parents, self.tokens, self.targets = i32([0] * rows), i32([0] * rows), i32([0] * rows)
        self.qkv = torch.zeros(rows, (self.n_q + 2 * self.n_kv) * self.d, dtype=torch.bfloat16, device="cuda")
        self.q, self.out = (torch.zeros(rows, self.n_q * self.d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        angle = torch.arange(200, device="cuda")[:, None] * torch.tensor([0.3 ** i for i in range(32)], device="cuda")
        self.rope = (angle.cos(), angle.sin())
        self.g = g

    def draw(self, rng):
        one = [p for n in (self.nodes, 3, self.nodes) for p in tree_parents(n, rng, 2)]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32)       # noqa: E731
        self.parents.copy_(i32(one))
        self.tokens.copy_(i32([rng.randrange(2) for _ in one]))
        self.targets.copy_(i32([rng.randrange(2) for _ in one]))
        self.qkv.copy_(torch.randn(self.qkv.shape, device="cuda", generator=self.g))

    def run(self):
        T.plan(self.step, self.lengths, self.counts, self.parents, self.pool)
        T.rope_append(self.step, self.qkv, self.rope, self.q, self.cache)
        T.attention(self.step, self.q, self.cache, self.out, 0.125)
        T.commit(self.step, self.tokens, self.targets, self.cache, self.accepted)

    def state(self):
        return [t.clone() for t in (self.lengths, self.table, self.pool.n_free, self.pool.held, self.out, self.cache.k, self.cache.v, self.accepted.path, self.accepted.next_token)]


@gpu
@pytest.mark.parametrize("i8", [False, True])
def test_loop_in_a_graph(i8):
    """Steps replayed from a CUDA graph, which no host number enters, are the steps run one by one; and those are right: what is in the cache at the
    end is what attention over plain rows at the requests' positions sees."""
    a, b = Loop(1, i8), Loop(1, i8)
    ra, rb = random.Random(4), random.Random(4)
    for _ in range(2):
        a.draw(ra), b.draw(rb), a.run(), b.run()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        b.run()
    total = 0
    for _ in range(12):
        a.draw(ra), b.draw(rb)
        a.run()
        graph.replay()
        torch.cuda.synchronize()
        a.step.check(), b.step.check()
        K.check_status()
        for x, y in zip(a.state(), b.state()):
            assert torch.equal(x, y)
        assert 3 <= a.accepted.count.sum().item() <= 17
        total += a.accepted.count.sum().item()
    assert a.lengths.sum().item() >= 36 + total
    held, table = a.pool.held.tolist(), a.table.tolist()
    used = [p for r in range(3) for p in table[r][: held[r]]]
    assert len(set(used)) == len(used) and 0 not in used
    assert all(h * PAGE >= n for h, n in zip(held, a.lengths.tolist()))


@gpu
def test_keys_after_commits():
    """Keys that a loop of steps left at a request's positions are the accepted nodes' rows, turned by those positions."""
    a, rng = Loop(2), random.Random(8)
    want = {r: [] for r in range(3)}
    start = a.lengths.tolist()
    for _ in range(6):
        a.draw(rng)
        before, rows = a.lengths.tolist(), a.qkv.clone()
        a.run()
        path, count, first = a.accepted.path.tolist(), a.accepted.count.tolist(), a.step.row_start.tolist()
        for r in range(3):
            for i in range(count[r]):
                want[r].append((before[r] + i, rows[first[r] + path[r][i]]))
    table = a.table.tolist()
    freq = torch.tensor([0.3 ** i for i in range(32)], device="cuda")
    for r in range(3):
        assert [p for p, _ in want[r]] == list(range(start[r], a.lengths[r].item()))
        for pos, row in want[r]:
            key = row.reshape(-1, a.d)[a.n_q: a.n_q + a.n_kv]
            turned = rope_reference(key[None], torch.tensor([pos], device="cuda"), freq.double(), False)[0]
            got = a.cache.k[table[r][pos // PAGE], :, pos % PAGE].double()
            # tables of fp32 angles: off by 2^-24 of an angle up to 200, and the rounding to bf16
            assert ((got - turned).abs() <= HALF * turned.abs() + 200 * 2.0 ** -23 * key.double().abs().amax(-1, keepdim=True)).all()
            assert torch.equal(a.cache.v[table[r][pos // PAGE], :, pos % PAGE], row.reshape(-1, a.d)[a.n_q + a.n_kv:])


@gpu
def test_two_calls_at_once():
    """Layers of one step on two streams, and steps of their own, share nothing."""
    s = State([3000, 700, 64, 5], [16, 9, 30, 2]).cuda()
    s.plan()
    caches = [make_cache(s.pages, 8, 128, i8, seed) for seed, i8 in ((1, False), (2, True), (3, False), (4, False))]
    g = torch.Generator(device="cuda").manual_seed(3)
    q = [torch.randn(s.max_rows, 40 * 128, device="cuda", generator=g).bfloat16() for _ in caches]
    want, got = [torch.empty_like(x) for x in q], [torch.empty_like(x) for x in q]
    for x, c, o in zip(q, caches, want):
        T.attention(s.step, x, c, o, 0.09)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in caches]
    for _ in range(20):
        for x, c, o, st in zip(q, caches, got, streams):
            with torch.cuda.stream(st):
                T.attention(s.step, x, c, o, 0.09)
    torch.cuda.synchronize()
    K.check_status()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("i8", [False, True])
def test_far_pages(i8):
    """Pages whose elements lie beyond 2^32 bytes, and beyond 2^31 elements of a layer, from its beginning."""
    pages, n_kv, d = 150000, 8, 128
    s = State([200, 33], [20, 7])
    near = s.pages
    move = lambda p: p and p + pages - near       # noqa: E731  (the same pages at the end of a large cache)
    s.table, s.tree_table, s.free = [[move(p) for p in t] for t in s.table], [[move(p) for p in t] for t in s.tree_table], [move(p) for p in s.free]
    s.pages = pages
    small = make_cache(near, n_kv, d, i8, 7)
    dtype = torch.int8 if i8 else torch.bfloat16
    k, v = (torch.zeros(pages, n_kv, PAGE, d, dtype=dtype, device="cuda") for _ in range(2))
    k[pages - near:], v[pages - near:] = small.k, small.v
    if i8:
        ks, vs = (torch.ones(pages, n_kv, PAGE, device="cuda") for _ in range(2))
        ks[pages - near:], vs[pages - near:] = small.k_scale, small.v_scale
    cache = T.TreeCache(k, v, ks, vs) if i8 else T.TreeCache(k, v)
    run_attention(s, (16, n_kv, d), i8, cache=cache)
    rows = s.rows
    qkv = torch.randn(rows, (16 + 2 * n_kv) * d, device="cuda")
    q = torch.empty(rows, 16 * d, dtype=torch.bfloat16, device="cuda")
    table = torch.ones(400, 64, device="cuda"), torch.zeros(400, 64, device="cuda")
    T.rope_append(s.step, qkv, table, q, cache)
    slots = s.step.slots[:rows].long()
    y = qkv.reshape(rows, -1, d)[:, 16: 16 + n_kv]
    if not i8:
        assert torch.equal(cache.k[slots // PAGE, :, slots % PAGE], y.bfloat16())
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")       # noqa: E731
    was = cache.v[slots[0] // PAGE, :, slots[0] % PAGE].clone()
    got = T.commit(s.step, i32([1] * rows), i32([0] * rows), cache)
    assert got.count.tolist() == [1, 1]
    page = s.t_table[0, 200 // PAGE].item()
    assert page > pages - near and torch.equal(cache.v[page, :, 200 % PAGE], was)
    K.check_status()
