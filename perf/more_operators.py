"""The work that the operators of steps over token trees are measured on: several drafted continuations of a request, verified at once
over its paged cache.

``plan``: block tables, slot maps, positions and ancestor masks of a step's rows, from the requests' lengths.  ``append``: rows of a qkv
projection rotated, queries out, keys and values into the cache at their slots.  ``attention``: every node of the trees over its request's
cache and its own ancestors.  ``commit``: the accepted path of every tree, its keys and values moved to the request's positions.

The plain forms below are the definition in elementary operations; with ``own`` the calls are ``b200serve.ops.tree``'s.

Pages hold 16 positions, ``[page][kv head][16][D]``; page 0 is nobody's.  A tree's nodes stand in pages of their own (``tree_table``), in
the order in which they are given: node i of a tree has its parent among the nodes before it, or none (-1).
"""
import functools
import math

import torch

own = False

PAGE = 16
NODES = 64          # nodes of a tree, at most


def _trees(b, nodes, least_nodes=0, spread=4):
    """``b`` trees of ``least_nodes`` (0: as many as ``nodes``) to ``nodes`` nodes, whose parents lie up to ``spread`` places before them."""
    return {"b": b, "nodes": nodes, "least_nodes": least_nodes or nodes, "spread": spread}


def _plan(b, longest, least, tree=True, reserve=0, **kind):
    """Lengths from ``least`` to ``longest``; ``tree`` false: rows at consecutive positions, ``nodes`` of them at most, and ``reserve``
    columns of the row buffers that the step does not fill."""
    return {"op": "plan", "longest": longest, "least": least, "tree": tree, "reserve": reserve, **_trees(b, **kind)}


def _append(b, n_q, n_kv, d, rot, slices, i8, interleaved, longest, least, tree=True, **kind):
    """``slices``: fp32 partial sums of the projection (0: bf16 rows); ``rot``: rotated dimensions."""
    return {"op": "append", "n_q": n_q, "n_kv": n_kv, "d": d, "rot": rot, "slices": slices, "i8": i8, "interleaved": interleaved, "longest": longest,
            "least": least, "tree": tree, **_trees(b, **kind)}


def _attention(b, n_q, n_kv, d, longest, least, i8=False, window=0, **kind):
    return {"op": "attention", "n_q": n_q, "n_kv": n_kv, "d": d, "longest": longest, "least": least, "i8": i8, "window": window, **_trees(b, **kind)}


def _commit(b, planes, n_kv, d, longest, least, i8=False, **kind):
    return {"op": "commit", "planes": planes, "n_kv": n_kv, "d": d, "longest": longest, "least": least, "i8": i8, **_trees(b, **kind)}


def listed():
    return [
        # one user's chat, a tree of sixteen drafts: launches only
        {"name": "plan-1", **_plan(1, 700, 700, nodes=16)},
        # a full server: portions of prompts beside decode rows, a buffer of rows that the step does not fill
        {"name": "plan-rows-100", **_plan(100, 33000, 1, tree=False, reserve=517, nodes=160, least_nodes=1)},
        # the qkv projection of one user's tree, 27B shape: four split-K slices
        {"name": "append-16", **_append(1, 40, 8, 128, 128, 4, False, False, 4100, 4100, nodes=16)},
        # trees of many users, 8-bit cache, half of every head rotated, neighbouring pairs
        {"name": "append-i8-1008", **_append(48, 16, 4, 128, 64, 1, True, True, 2000, 700, nodes=30, least_nodes=12)},
        # portions of prompts of several users in one batch behind a long document, bf16 rows of the projection, positions far out
        {"name": "append-rows-5000", **_append(5, 32, 8, 128, 128, 0, False, False, 120000, 90000, tree=False, nodes=1300, least_nodes=700)},
        # the smallest call: a toy model's first tokens
        {"name": "attention-tiny", **_attention(1, 4, 2, 64, 37, 37, nodes=3)},
        # one user's chat, 27B shape
        {"name": "attention-1", **_attention(1, 40, 8, 128, 4100, 4100, nodes=16)},
        # wide trees: as many products as bytes
        {"name": "attention-wide", **_attention(16, 16, 4, 128, 9000, 1000, nodes=64, least_nodes=40)},
        # long documents over an 8-bit cache, 27B shape
        {"name": "attention-i8-long", **_attention(12, 40, 8, 128, 65000, 20001, i8=True, nodes=24)},
        # a full server, 27B shape: the largest
        {"name": "attention-32", **_attention(32, 40, 8, 128, 33000, 2000, nodes=16, least_nodes=5)},
        # one user's tree settled over the 64 layers of the 27B shape
        {"name": "commit-1", **_commit(1, 64, 8, 128, 4100, 4100, nodes=16)},
        # many users, 8-bit cache, 40 layers
        {"name": "commit-i8-32", **_commit(32, 40, 4, 128, 900, 30, i8=True, nodes=32, least_nodes=9)},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


#: Query heads, key/value heads and head size: the presets', and others.
HEADS = ((40, 8, 128), (16, 4, 128), (8, 2, 128), (32, 8, 128), (4, 2, 64), (16, 16, 128), (64, 4, 128), (24, 8, 64), (7, 1, 128), (12, 12, 64))
#: What a drawn attention case reads and computes at most.
MOST_BYTES, MOST_FLOPS = 2_200_000_000, 240_000_000_000


def _draw_trees(rng):
    nodes = rng.choice((_log(rng, 1, 64), rng.randint(4, 64)))
    return {"nodes": nodes, "least_nodes": rng.choice((nodes, rng.randint(1, nodes))), "spread": rng.choice((1, 2, 4, 8, 64))}


def draw(rng):
    op = rng.choice(("plan", "append", "attention", "attention", "commit"))
    b = _log(rng, 1, 64)
    longest = _log(rng, 1, 65536)
    n_q, n_kv, d = rng.choice(HEADS)
    if op == "plan" or op == "append":
        tree = rng.random() < 0.6
        kind = _draw_trees(rng) if tree else {"nodes": _log(rng, 1, 4096 // b), "least_nodes": 1}
        if op == "plan":
            return _plan(b, longest, rng.randint(0, longest), tree, rng.choice((0, rng.randint(1, 600))), **kind)
        i8 = rng.random() < 0.4
        longest = min(longest, 4000) if i8 else longest
        return _append(b, n_q, n_kv, d, rng.choice((d, d, d // 2, 16 * rng.randint(1, d // 16))), rng.choice((0, 0, 1, 2, 5)), i8, rng.random() < 0.4, longest,
                       rng.randint(0, longest), tree, **kind)
    if op == "commit":
        b = _log(rng, 1, 32)
        longest = _log(rng, 1, 2000)
        return _commit(b, _log(rng, 1, 64), min(n_kv, 8), d, longest, rng.randint(0, longest), rng.random() < 0.4, **_draw_trees(rng))
    i8 = rng.random() < 0.4
    kind = _draw_trees(rng)
    longest = max(1, min(longest, MOST_BYTES // (b * n_kv * d * (2 if i8 else 4)), MOST_FLOPS // (4 * b * kind["nodes"] * n_q * d) - kind["nodes"]))
    return _attention(b, n_q, n_kv, d, longest, rng.randint(0, longest), i8, rng.choice((0, 0, 0, _log(rng, 20, 4096))), **kind)


# ------------------------------------------------------------------ what a program has in hand
def _rand(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _spread(lo, hi, b, g):
    """``b`` whole numbers from ``lo`` to ``hi`` in even steps, in another order with every seed: their sum is the case's."""
    return _steps(lo, hi, b).to("cuda")[torch.randperm(b, device="cuda", generator=g)]


def _steps(lo, hi, b):
    return torch.tensor([hi - (hi - lo) * i // max(1, b - 1) for i in range(b)], dtype=torch.int32)


def _normal(g, *shape, scale=1.0):
    return torch.empty(shape, device="cuda").normal_(0, scale, generator=g)


def _parents(counts, spread, g):
    """Node i's parent among the ``spread`` nodes before it, all trees' nodes one after another."""
    start = counts.cumsum(0) - counts
    i = torch.arange(int(counts.sum()), device="cuda") - torch.repeat_interleave(start, counts)
    back = (torch.rand(i.shape, device="cuda", generator=g) * i.clamp(1, spread)).long()
    return torch.where(i > 0, i - 1 - back, -1).int()


def _tables(case, lengths, g, room):
    """Pages of a pool in random order: block tables that hold ``lengths``, tables of the trees' pages, what is left.  ``room``: positions
    a request can grow to.  Requests whose rows are appended share their prompt's pages, all but the last one's; the others have their own."""
    b = case["b"]
    held = (lengths + PAGE - 1) // PAGE
    cap = (room + PAGE - 1) // PAGE
    shared = cap if case["op"] == "append" else 0
    need = int(held.sum()) if not shared else b
    spare = b * (-(-case["nodes"] // PAGE) + 1) + 5
    trees = b * (NODES // PAGE)
    pages = 1 + shared + need + trees + spare
    order = (torch.randperm(pages - 1, device="cuda", generator=g) + 1).int()
    column = torch.arange(cap, device="cuda")[None, :]
    at = column < held[:, None]
    if shared:
        own_page = order[shared: shared + b, None]
        block_table = torch.where(column < held[:, None] - 1, order[:shared], torch.where(at, own_page, 0)).contiguous()
    else:
        block_table = torch.zeros(b, cap, dtype=torch.int32, device="cuda")
        block_table[at] = order[:need]
    rest = order[shared + need:]
    return {"pages": pages, "held": held.int(), "block_table": block_table, "tree_table": rest[:trees].reshape(b, -1).contiguous(), "free": rest[trees:].contiguous(),
            "n_free": torch.tensor([spare], dtype=torch.int32, device="cuda")}


def _frequencies(rot, longest):
    """Angle per position of every pair: base 1e6, slowed down four times where positions go beyond 32768."""
    f = torch.tensor([1e6 ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device="cuda")
    return f / 4 if longest > 32768 else f


def _cache(case, pages, g, planes=None):
    """Keys and values as a model leaves them in the pages, or in 8 bits with a scale for every position and head."""
    shape = (pages, case["n_kv"], PAGE, case["d"])
    shape = shape if planes is None else (planes, *shape)
    if not case["i8"]:
        return {"k": torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(0, 1.3, generator=g),
                "v": torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(0, 1, generator=g)}
    return {"k": torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=g), "v": torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=g),
            "k_scale": torch.rand(shape[:-1], device="cuda", generator=g).mul_(0.02).add_(0.005), "v_scale": torch.rand(shape[:-1], device="cuda", generator=g).mul_(0.02).add_(0.004)}


def prepare(case, seed):
    g = _rand(seed * 6007 + 29)
    op, b, nodes = case["op"], case["b"], case["nodes"]
    lengths = _spread(case["least"], case["longest"], b, g)
    counts = _spread(case["least_nodes"], nodes, b, g)
    tree = case.get("tree", True)
    rows = int(counts.sum())
    s = {"case": case, "lengths": lengths, "counts": counts, "rows": rows, "max_rows": rows + case.get("reserve", 0), **_tables(case, lengths, g, case["longest"] + nodes + 1)}
    s["parents"] = _parents(counts, case["spread"], g) if tree else None
    if op == "append":
        n = (case["n_q"] + 2 * case["n_kv"]) * case["d"]
        s["qkv"] = _normal(g, case["slices"], rows, n, scale=1.0 / case["slices"] ** 0.5) if case["slices"] else _normal(g, rows, n).bfloat16()
        angle = torch.arange(case["longest"] + nodes + 1, dtype=torch.float64, device="cuda")[:, None] * _frequencies(case["rot"], case["longest"])
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q"] = torch.zeros(rows, case["n_q"] * case["d"], dtype=torch.bfloat16, device="cuda")
        s.update(_cache(case, s["pages"], g))
    elif op == "attention":
        s["q"] = _normal(g, rows, case["n_q"] * case["d"], scale=1.5).bfloat16()
        s["out"] = torch.zeros_like(s["q"])
        s.update(_cache(case, s["pages"], g))
    elif op == "commit":
        s["tokens"] = torch.randint(0, 151936, (rows,), device="cuda", generator=g).int()
        # a node's target: most often the token of one of its children
        start = torch.repeat_interleave(counts.cumsum(0) - counts, counts)
        up = torch.where(s["parents"] < 0, rows, start + s["parents"]).long()
        key = torch.randint(0, 1 << 20, (rows,), device="cuda", generator=g) * (1 << 20) + torch.arange(rows, device="cuda")
        child = torch.full((rows + 1,), -1, device="cuda").scatter_reduce_(0, up, key, "amax")[:rows] % (1 << 20)
        follow = torch.rand(rows, device="cuda", generator=g) < 0.85
        s["targets"] = torch.where(follow, s["tokens"][child.clamp(0, rows - 1)], torch.randint(0, 151936, (rows,), device="cuda", generator=g).int()).int()
        s.update(_cache(case, s["pages"], g, case["planes"]))
    s["plan"] = _plan_rows(s)      # the plain form's tables: what a step has of its plan
    if own:
        from b200serve.ops import tree as T
        s["pool"] = T.PagePool(s["free"], s["n_free"], s["held"])
        s["after"] = T.PagePool(s["free"], torch.empty_like(s["n_free"]), torch.empty_like(s["held"]))
        s["step"] = T.TreeStep(s["block_table"], s["tree_table"], s["max_rows"], s["pages"], nodes if tree else NODES)
        if op != "plan":
            T.plan(s["step"], s["lengths"], s["counts"], s["parents"], s["pool"], s["after"])
            s["cache"] = T.TreeCache(s["k"], s["v"], s.get("k_scale"), s.get("v_scale"))
        if op == "commit":
            s["accepted"] = T.Accepted.empty(b, "cuda")
    return s


# ------------------------------------------------------------------ plain forms
def _rows_of(s):
    """(request, place among its rows) of every row."""
    counts = s["counts"].long()
    start = counts.cumsum(0) - counts
    req = torch.repeat_interleave(torch.arange(counts.numel(), device="cuda"), counts, output_size=s["rows"])
    return req, torch.arange(s["rows"], device="cuda") - start[req], start


def _ancestors(s, i, start, req):
    """Depth and ancestor mask of every node: pointers to parents doubled six times."""
    one = torch.ones_like(i)
    up = torch.where(s["parents"] < 0, s["rows"], s["parents"] + start[req]).long()       # the row behind the last one: nobody
    up = torch.cat([up, up.new_full((1,), s["rows"])])
    mask, depth = torch.cat([one << i, up.new_zeros(1)]), torch.cat([(up[:-1] < s["rows"]).long(), up.new_zeros(1)])
    for _ in range(6):
        mask, depth, up = mask | mask[up], depth + depth[up], up[up]
    return depth[:-1], mask[:-1]


def _plan_rows(s):
    tree, b = s["parents"] is not None, s["lengths"].numel()
    req, i, start = _rows_of(s)
    length, held = s["lengths"].long(), s["held"].long()
    if tree:
        depth, mask = _ancestors(s, i, start, req)
        need = torch.zeros_like(length).scatter_reduce_(0, req, depth + 1, "amax")
    else:
        depth, mask, need = i, None, s["counts"].long()
    want = torch.maximum(held, torch.where(need > 0, (length + need + PAGE - 1) // PAGE, 0))
    take = want - held
    first = take.cumsum(0) - take            # pages taken before this request's, from the end of the free list
    column = torch.arange(s["block_table"].shape[1], device="cuda")[None, :]
    new = (column >= held[:, None]) & (column < want[:, None])
    at = s["n_free"].long() - 1 - first[:, None] - (column - held[:, None])
    table = torch.where(new, s["free"][at.clamp(0, s["free"].numel() - 1)], s["block_table"])
    pos = length[req] + depth
    page = s["tree_table"][req, i // PAGE] if tree else table[req, pos // PAGE]
    fill = lambda x, t: torch.nn.functional.pad(x.to(t), (0, s["max_rows"] - s["rows"]), value=-1)      # noqa: E731
    out = {"row_start": torch.nn.functional.pad(s["counts"].cumsum(0), (1, 0)).int(), "row_req": fill(req, torch.int32), "row_pos": fill(pos, torch.int32),
           "slots": fill(page * PAGE + (i if tree else pos) % PAGE, torch.int32), "block_table": table, "held": want.int(), "n_free": (s["n_free"] - take.sum()).int()}
    if tree:
        out["masks"] = torch.nn.functional.pad(mask, (0, s["max_rows"] - s["rows"]))
    return out


def _turn(x, cos, sin, interleaved):
    """Pairs of the first 2 n dimensions of ``x`` [rows][heads][d] rotated by angles [rows][n]."""
    n = cos.shape[1]
    cos, sin = cos[:, None, :], sin[:, None, :]
    a, b = (x[..., 0: 2 * n: 2], x[..., 1: 2 * n: 2]) if interleaved else (x[..., :n], x[..., n: 2 * n])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _heads(case, x):
    x = x.reshape(x.shape[0], -1, case["d"])
    return x.split([case["n_q"], case["n_kv"], case["n_kv"]], 1)


def _quantised(x):
    """Whole numbers and the scale of every vector."""
    largest = x.abs().amax(-1, keepdim=True)
    scale = torch.where(largest > 0, largest / torch.full_like(largest, 127), torch.ones_like(largest))      # (by a number torch multiplies with its rounded inverse)
    return (x * (1 / scale)).round().to(torch.int8), scale[..., 0]


def _append_rows(s):
    case, plan = s["case"], s["plan"]
    x = functools.reduce(torch.add, s["qkv"].unbind(0)) if case["slices"] else s["qkv"].float()
    pos, slots = plan["row_pos"][: s["rows"]].long(), plan["slots"][: s["rows"]].long()
    q, k, v = _heads(case, x)
    cos, sin = s["cos"][pos], s["sin"][pos]
    s["q"].copy_(_turn(q, cos, sin, case["interleaved"]).flatten(1))
    for name, y in (("k", _turn(k, cos, sin, case["interleaved"])), ("v", v)):
        if case["i8"]:
            y, scale = _quantised(y)
            s[name + "_scale"][slots // PAGE, :, slots % PAGE] = scale
        s[name][slots // PAGE, :, slots % PAGE] = y.to(s[name].dtype)


def _append_result(s):
    if not s["case"]["i8"]:
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    return {"q": s["q"], "k": s["k"] * s["k_scale"][..., None], "v": s["v"] * s["v_scale"][..., None], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}      # (fp32)


def _pages_of(s, name, table, dtype):
    """Keys or values of tables of pages, [request][kv head][position][d]."""
    x = s[name][table.long()].to(dtype)
    if s["case"]["i8"]:
        x = x * s[name + "_scale"][table.long()][..., None].to(dtype)
    return x.transpose(1, 2).flatten(2, 3)


def _attend(s, lo, hi, dtype, soft):
    """Requests ``lo`` to ``hi`` over the longest one's pages; ``soft``: weights of masked scores."""
    case, counts, length = s["case"], s["counts"][lo:hi].long(), s["lengths"][lo:hi].long()
    b, n, nkv, d = hi - lo, int(case["nodes"]), case["n_kv"], case["d"]
    blocks, tree_blocks = -(-case["longest"] // PAGE), -(-n // PAGE)
    row = s["plan"]["row_start"][lo:hi].long()[:, None] + torch.arange(n, device="cuda")[None, :]
    live = torch.arange(n, device="cuda")[None, :] < counts[:, None]
    row = row.clamp(max=s["rows"] - 1)
    q = s["q"][row].to(dtype).reshape(b, n, nkv, -1, d).permute(0, 2, 1, 3, 4)          # [b][kv][node][head][d]
    k = torch.cat([_pages_of(s, "k", s["block_table"][lo:hi, :blocks], dtype), _pages_of(s, "k", s["tree_table"][lo:hi, :tree_blocks], dtype)[:, :, :n]], 2)
    v = torch.cat([_pages_of(s, "v", s["block_table"][lo:hi, :blocks], dtype), _pages_of(s, "v", s["tree_table"][lo:hi, :tree_blocks], dtype)[:, :, :n]], 2)
    z = (q.flatten(2, 3) @ k.transpose(2, 3)).reshape(b, nkv, n, -1, k.shape[2])
    pos = s["plan"]["row_pos"][row].long()                                               # [b][node]
    key = torch.arange(blocks * PAGE, device="cuda")[None, None, :]
    seen = (key < length[:, None, None]).expand(-1, n, -1)
    node = (s["plan"]["masks"][row][:, :, None] >> torch.arange(n, device="cuda")) & 1 == 1
    if case["window"]:
        seen = seen & (key > pos[:, :, None] - case["window"])
        node = node & (pos[:, None, :] > pos[:, :, None] - case["window"])
    seen = (torch.cat([seen, node & live[:, None, :]], 2) & live[:, :, None])[:, None, :, None, :]
    o = (soft(z * d ** -0.5, seen).flatten(2, 3) @ v).reshape(b, nkv, n, -1, d).permute(0, 2, 1, 3, 4).reshape(b, n, -1)
    return o[live]


def _softmax(z, seen):
    z = z.masked_fill(~seen, float("-inf"))
    best = z.amax(-1, keepdim=True)
    e = (z - best.clamp_min(-3e38)).exp()
    return e / e.sum(-1, keepdim=True).clamp_min(1e-38)


def _attention_rows(s):
    case = s["case"]
    each = case["n_kv"] * (case["longest"] + case["nodes"] + PAGE) * max(case["nodes"] * (case["n_q"] // case["n_kv"]), case["d"])
    step = max(1, (3 << 30) // each)          # requests at a time
    b = case["b"]
    s["out"].copy_(torch.cat([_attend(s, i, min(b, i + step), torch.float32, _softmax) for i in range(0, b, step)]))


def _commit_rows(s):
    """A node follows its parent where its token is the parent's target (of several the first does); the path is the nodes whose
    ancestors all follow, from node 0 on."""
    plan, b, rows = s["plan"], s["case"]["b"], s["rows"]
    req, i, start = _rows_of(s)
    length, mask = s["lengths"].long(), plan["masks"][:rows]
    up = torch.where(s["parents"] < 0, rows, s["parents"] + start[req]).long()
    fits = (up < rows) & (s["tokens"] == s["targets"][up.clamp(max=rows - 1)])
    first = torch.full((rows + 1,), NODES, device="cuda").scatter_reduce_(0, torch.where(fits, up, rows), i, "amin")
    follows = fits & (first[up] == i)
    bits = torch.zeros(b, dtype=torch.long, device="cuda").scatter_add_(0, req, follows.long() << i)
    on = (mask & ~bits[req]) == 1
    req, node = req[on], i[on]
    to = plan["row_pos"][:rows][on].long()
    depth = to - length[req]
    path = torch.full((b, NODES), -1, dtype=torch.int32, device="cuda")
    path[req, depth] = node.int()
    accepted = (path >= 0).sum(1)
    src, dst = s["tree_table"][req, node // PAGE].long(), plan["block_table"][req, to // PAGE].long()
    for name in ("k", "v", "k_scale", "v_scale"):
        if name in s:
            s[name][:, dst, :, to % PAGE] = s[name][:, src, :, node % PAGE]
    last = (start + path.gather(1, (accepted - 1).clamp_min(0)[:, None])[:, 0]).clamp(0, rows - 1)
    following = torch.where(s["counts"] > 0, s["targets"][last], -1)
    return {"path": path, "accepted": accepted.int(), "next_token": following.int(), "lengths": (length + accepted).int()}


def _commit_result(s, got):
    """The caches as they are: what is moved keeps its bits, 8-bit values (whole numbers) and their scales apart."""
    names = ("k", "v", "k_scale", "v_scale") if s["case"]["i8"] else ("k", "v")
    return {**got, **{name: s[name] for name in names}}


def run(s):
    op = s["case"]["op"]
    if own:
        from b200serve.ops import tree as T
        if op == "plan":
            T.plan(s["step"], s["lengths"], s["counts"], s["parents"], s["pool"], s["after"])
            step, pool = s["step"], s["after"]
            got = {"row_start": step.row_start, "row_req": step.row_req, "row_pos": step.row_pos, "slots": step.slots, "block_table": s["block_table"], "held": pool.held,
                   "n_free": pool.n_free}
            return {**got, "masks": step.masks} if s["parents"] is not None else got
        if op == "append":
            T.rope_append(s["step"], s["qkv"], (s["cos"], s["sin"]), s["q"], s["cache"], s["case"]["interleaved"])
            return _append_result(s)
        if op == "attention":
            T.attention(s["step"], s["q"], s["cache"], s["out"], s["case"]["d"] ** -0.5, s["case"]["window"])
            return s["out"]
        a = T.commit(s["step"], s["tokens"], s["targets"], s["cache"], s["accepted"])
        return _commit_result(s, {"path": a.path, "accepted": a.count, "next_token": a.next_token, "lengths": a.lengths})
    if op == "plan":
        return _plan_rows(s)
    if op == "append":
        _append_rows(s)
        return _append_result(s)
    if op == "attention":
        _attention_rows(s)
        return s["out"]
    return _commit_result(s, _commit_rows(s))


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    if case["op"] not in ("append", "attention"):
        return None                         # whole numbers, and values that are moved as they are
    s = prepare(case, seed)
    if case["op"] == "append":
        x = (s["qkv"].double().sum(0) if case["slices"] else s["qkv"].double()).reshape(s["rows"], -1, case["d"])
        pos, slots = s["plan"]["row_pos"][: s["rows"]].double(), s["plan"]["slots"][: s["rows"]].long()
        w = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), pos[:, None] * _frequencies(case["rot"], case["longest"]))[:, None, :]      # cos + i sin
        n, r = case["n_q"] + case["n_kv"], case["rot"]
        front = x[:, :n, :r]
        pairs = front.unflatten(-1, (-1, 2)) if case["interleaved"] else front.unflatten(-1, (2, -1)).transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * w)
        x[:, :n, :r] = turned.flatten(-2) if case["interleaved"] else turned.transpose(-1, -2).flatten(-2)
        out = {"q": x[:, : case["n_q"]].flatten(1)}
        for name, y in (("k", x[:, case["n_q"]: n]), ("v", x[:, n:])):
            if case["i8"]:
                # the value is a multiple of the scale: where 64 bits round another way it is another one, so that only the scales are given
                held = s[name + "_scale"].double()
                held[slots // PAGE, :, slots % PAGE] = y.abs().amax(-1) / 127
                out[name], out[name + "_scale"] = None, held
            else:
                held = s[name].double()
                held[slots // PAGE, :, slots % PAGE] = y
                out[name] = held
        return out
    out = torch.zeros(s["rows"], case["n_q"], case["d"], dtype=torch.float64, device="cuda")
    start, group = s["plan"]["row_start"].tolist(), case["n_q"] // case["n_kv"]
    value = lambda name, r, h, t, n: (s[name][t, h].double() * (s[name + "_scale"][t, h].double()[..., None] if case["i8"] else 1.0)).flatten(0, 1)[:n]     # noqa: E731
    for r in range(case["b"]):
        lo, hi, length = start[r], start[r + 1], int(s["lengths"][r])
        n = hi - lo
        pos = s["plan"]["row_pos"][lo:hi].long()
        where = torch.cat([torch.arange(length, device="cuda"), pos])                     # the positions that keys stand at
        sees = torch.zeros(n, length + n, dtype=torch.bool, device="cuda")
        sees[:, :length] = True
        up = s["parents"][lo:hi].long()
        node = torch.arange(n, device="cuda")
        while bool((node >= 0).any()):
            on = node >= 0
            sees[on.nonzero()[:, 0], length + node[on]] = True
            node = torch.where(on, up[node.clamp_min(0)], -1)
        if case["window"]:
            sees &= where[None, :] > pos[:, None] - case["window"]
        pages, nodes = s["block_table"][r, : -(-length // PAGE)].long(), s["tree_table"][r].long()
        for h in range(case["n_kv"]):
            k = torch.cat([value("k", r, h, pages, length), value("k", r, h, nodes, n)])
            v = torch.cat([value("v", r, h, pages, length), value("v", r, h, nodes, n)])
            for i in range(h * group, (h + 1) * group):
                z = (s["q"][lo:hi, i * case["d"]: (i + 1) * case["d"]].double() @ k.T) / math.sqrt(case["d"])
                out[lo:hi, i] = torch.softmax(z.masked_fill(~sees, -math.inf), 1) @ v
    return out.flatten(1)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op, b = case["op"], case["b"]
    rows = int(_steps(case["least_nodes"], case["nodes"], b).sum())
    positions = int(_steps(case["least"], case["longest"], b).sum())
    if op == "plan":
        tree = case["tree"]
        # lengths, counts and held blocks read, starts and held blocks written; of a row its parent, request, position, slot and mask
        return {"bytes": 20.0 * b + rows * (24.0 if tree else 12.0) + 12.0 * case["reserve"], "flops": 0.0}
    d, n_kv = case["d"], case["n_kv"]
    kv = n_kv * (2.0 * d + 8 if case["i8"] else 4.0 * d)          # a position's keys and values in a layer
    if op == "append":
        n_q = case["n_q"]
        read = (n_q + 2 * n_kv) * d * (4.0 * case["slices"] or 2.0) + 4.0 * case["rot"] + 8
        return {"bytes": rows * (read + 2.0 * n_q * d + kv), "flops": rows * (3.0 * (n_q + n_kv) * case["rot"] + max(0, case["slices"] - 1) * (n_q + 2 * n_kv) * d)}
    if op == "commit":
        # a path of about three nodes
        path = 3.0 * b
        return {"bytes": rows * 12.0 + b * 16.0 + 2 * path * kv * case["planes"], "flops": 0.0}
    n_q, window = case["n_q"], case["window"]
    lengths = _steps(case["least"], case["longest"], b)
    seen = lengths.clamp(max=window) if window else lengths
    nodes = rows / b
    return {"bytes": float(seen.sum()) * kv + rows * (kv + 4.0 * n_q * d + 12.0), "flops": 4.0 * n_q * d * (float(seen.sum()) * nodes + rows * min(nodes, 8.0))}
