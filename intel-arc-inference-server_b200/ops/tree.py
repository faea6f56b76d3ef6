"""Steps over token trees: several drafted continuations of a request, verified at once over its paged cache (``csrc/tree_plan.cu``,
``csrc/tree_rope.cu``, ``csrc/tree_attn.cu``).

A step's rows are the nodes of its requests' trees, a request's one after another, a parent before its children; node 0 is the request's next
token, which is not in the cache yet.  Nodes stand in pages of their own (``tree_table``), node i at place i, until the step is settled:

    plan         lengths and trees -> rows' requests, positions, cache slots and ancestors; pages for what the longest path can add
    rope_append  a layer's qkv rows turned by their positions; queries out, keys and values to the rows' slots
    attention    every row over its request's cached positions and its own ancestors
    commit       the accepted path of every tree; its keys and values move to the request's positions, in all layers

``plan`` without parents lays out rows at consecutive positions (prompt portions, decode rows) for ``rope_append``: their slots are the
request's own.  Everything happens on the current stream, nothing waits for the host: lengths, tables and the list of free pages stay on the
device, and a step can be captured into a CUDA graph.  What only the device knows is checked there; a plan that cannot be made leaves pages,
tables and lengths as they are and no rows (``TreeStep.check``); a row whose table names a page that is not there has slot -1 and is not stored.
A step's buffers are one plan's at a time: calls that read them may run on several streams, the next plan belongs behind them.

Caches are ``KVCache`` planes: ``[page][kv head][16][D]`` with D 64 or 128, bf16, or int8 with fp32 scales ``[page][kv head][16]``.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch

from . import lib as K
from .logprob import _elsewhere, _stream

PAGE = 16
MAX_NODES = 64          # nodes of a tree: an ancestor mask is one 64-bit word
MAX_REQUESTS = 1024
MAX_ROWS = 1 << 20
MAX_BLOCKS = 1 << 27    # of a table, one too many: positions are 32-bit numbers

_FAULTS = {1: "the pool has not enough pages, or no room for those that come back", 2: "a block table is too short, or a request holds more pages than its table has",
           4: "more rows than the step has room for", 8: "a tree of too many nodes", 16: "a parent that does not stand before its child",
           32: "a negative length", 64: "a table names a page that is not there"}


_P, _L, _I = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int


class _Step(ctypes.Structure):          # csrc/tree.cuh
    _fields_ = [(n, _P) for n in ("block_table", "tree_table", "lengths", "row_start", "row_req", "row_pos", "slots", "parents", "masks", "status")] + [
        (n, _I) for n in ("requests", "max_blocks", "tree_blocks", "max_rows", "max_nodes", "num_pages")]


class _Pool(ctypes.Structure):
    _fields_ = [("free", _P), ("n_free", _P), ("held", _P), ("capacity", _I)]


class _Cache(ctypes.Structure):
    _fields_ = [("maps", ctypes.c_uint8 * 256), ("k", _P), ("v", _P), ("k_scale", _P), ("v_scale", _P), ("layer_bytes", _L), ("layer_scales", _L),
                ("layers", _I), ("pages", _I), ("heads", _I), ("d", _I)]


class _Accepted(ctypes.Structure):
    _fields_ = [(n, _P) for n in ("path", "count", "next_token", "lengths")]


@functools.lru_cache(maxsize=None)
def _fn():
    """The library's entry points with their argument types."""
    out = {}
    for name, result, args in (("plan", _I, [_P] * 6 + [_I, _P]), ("rope", _I, [_P] * 3 + [_L, _L, _I, _I, _P, _P, _I, _I, _I, _I, _P, _L, _P]), ("cache", _I, [_P]),
                               ("attention", _I, [_P] * 3 + [_L, _P, _L, _P, _I, _I, _I, ctypes.c_float, _P]), ("attention_work", _L, [_P, _I, _I, _I]),
                               ("commit", _I, [_P] * 5 + [_I, _P])):
        fn = getattr(K.lib(), "b2_tree_" + name)
        fn.restype, fn.argtypes = result, args
        out[name] = fn
    return out


def _aligned(kind):
    """A structure whose first field begins at a multiple of 64 bytes."""
    room = (ctypes.c_uint8 * (ctypes.sizeof(kind) + 64))()
    at = kind.from_buffer(room, -ctypes.addressof(room) % 64)
    return at, ctypes.addressof(at)


def _flat(t: torch.Tensor, dtype, shape, what: str, device=None) -> torch.Tensor:
    if t.dtype is not dtype or t.shape != shape or not t.is_cuda or not t.is_contiguous() or device is not None and t.device != device:
        raise ValueError(f"{what}: contiguous {dtype} {list(shape)} on {device or 'a CUDA device'}, not {t.dtype} {list(t.shape)} on {t.device}")
    return t


def _matrix(t: torch.Tensor, dtype, what: str, device, dims: int = 2) -> tuple:
    """(rows, columns, elements from row to row, address) of a matrix whose rows begin at multiples of 16 bytes, or of the first of several
    (``dims`` 3: their number and the elements from one to the next behind it)."""
    if t.dtype is not dtype or t.dim() != dims or t.get_device() != device.index:
        raise ValueError(f"{what}: rows of {dtype} on {device}, not {t.dtype} {list(t.shape)} on {t.device}")
    more = ()
    if dims == 2:
        (m, n), (ld, step) = t.shape, t.stride()
    else:
        (s, m, n), (apart, ld, step) = t.shape, t.stride()
        if s < 1 or apart * dtype.itemsize % 16:
            raise ValueError(f"{what}: one slice at least, slices at multiples of 16 bytes")
        more = (s, apart)
    at = t.data_ptr()
    if m < 2:
        ld = (n + 15) // 16 * 16      # (a lone row's stride says nothing)
    if n > 1 and step != 1 or ld < n or (at | ld * dtype.itemsize) % 16:
        raise ValueError(f"{what}: one element after another, rows that do not overlap and begin at multiples of 16 bytes")
    return (m, n, ld, at) + more


def _words(t: torch.Tensor, n: int, what: str, device) -> int:
    """Address of ``n`` int32 numbers."""
    if t.dtype is not torch.int32 or t.dim() != 1 or t.numel() != n or t.get_device() != device.index or not t.is_contiguous():
        raise ValueError(f"{what}: {n} contiguous int32 numbers on {device}, not {t.dtype} {list(t.shape)} on {t.device}")
    return t.data_ptr()


class PagePool:
    """Free pages, the last of the first ``n_free`` taken first (int32 ``[capacity]`` and ``[1]``), and the pages that every request holds
    (int32 ``[requests]``)."""

    def __init__(self, free: torch.Tensor, n_free: torch.Tensor, held: torch.Tensor):
        _flat(free, torch.int32, (free.numel(),), "free pages")
        self.free, self.n_free = free, _flat(n_free, torch.int32, (1,), "number of free pages", free.device)
        self.held = _flat(held, torch.int32, (held.numel(),), "pages of the requests", free.device)
        self._c = _Pool(free.data_ptr(), n_free.data_ptr(), held.data_ptr(), free.numel())
        self._at, self._requests, self._index = ctypes.addressof(self._c), held.numel(), free.device.index


class TreeCache:
    """Keys and values of one layer, ``[pages][kv heads][16][D]``, or of several ``[layers]...``; int8 with scales."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None):
        i8 = k_scale is not None
        if k.dtype is not (torch.int8 if i8 else torch.bfloat16) or (v_scale is not None) != i8:
            raise ValueError("a cache in bf16, or in int8 with scales of keys and values")
        if k.dim() not in (4, 5) or k.shape[-2] != PAGE or k.shape[-1] not in (64, 128) or min(k.shape) < 1:
            raise ValueError(f"a cache is [layers][pages][kv heads][{PAGE}][64 or 128], not {list(k.shape)}")
        for t, dtype, shape in ((k, k.dtype, k.shape), (v, k.dtype, k.shape)) + (((k_scale, torch.float32, k.shape[:-1]), (v_scale, torch.float32, k.shape[:-1])) if i8 else ()):
            if t.shape != shape or t.dtype is not dtype or t.device != k.device or not t.is_cuda or not (t[0] if k.dim() == 5 else t).is_contiguous():
                raise ValueError("keys, values and scales of one shape, contiguous inside a layer, on one CUDA device")
        if k.dim() == 5:
            layer = k[0].numel()
            if k.shape[0] > 1 and (k.stride(0) < layer or k.stride(0) != v.stride(0) or i8 and (k_scale.stride(0) != v_scale.stride(0) or k_scale.stride(0) < layer // k.shape[-1])):
                raise ValueError("layers that do not overlap, as far apart in the values as in the keys")
        if (k.data_ptr() | v.data_ptr()) % 16 or k.dim() == 5 and k.stride(0) * k.element_size() % 16:
            raise ValueError("a layer's keys and values begin at multiples of 16 bytes")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.layers = k.shape[0] if k.dim() == 5 else 1
        self.pages, self.heads, _, self.d = k.shape[-4:]
        if self.pages * self.heads * PAGE >= 1 << 31:
            raise ValueError("a layer of fewer than 2^31 rows")
        self.device, self.i8 = k.device, i8
        if i8 and (k_scale.data_ptr() | v_scale.data_ptr() | (k_scale.stride(0) * 4 if k.dim() == 5 else 0)) % 16:
            raise ValueError("a layer's scales begin at multiples of 16 bytes")
        self._index = k.device.index
        self._c, self._at = _aligned(_Cache)
        c, five = self._c, k.dim() == 5
        c.k, c.v, c.layers, c.pages, c.heads, c.d = k.data_ptr(), v.data_ptr(), self.layers, self.pages, self.heads, self.d
        c.k_scale, c.v_scale = (k_scale.data_ptr(), v_scale.data_ptr()) if i8 else (None, None)
        c.layer_bytes, c.layer_scales = (k.stride(0) * k.element_size(), k_scale.stride(0) if i8 else 0) if five else (0, 0)
        with torch.cuda.device(k.device):
            K._check(_fn()["cache"](self._at), "tree_cache")
        K.launch_count -= 1      # (nothing is launched)


class TreeStep:
    """What ``plan`` leaves of a step, for up to ``max_rows`` rows: ``lengths`` ``[requests]`` and ``row_start`` ``[requests + 1]``; of every row
    its request ``row_req``, position ``row_pos``, cache slot ``slots`` (page x 16 + place), parent ``parents`` and, 64 bits, ancestors ``masks``
    (bit j: node j of its tree, itself among them; a program may clear or set bits before ``attention``; a plan without parents leaves these two as
    they were).  Rows behind the last request's are -1 (masks 0).

    ``block_table`` int32 ``[requests][blocks]``: pages of the requests' positions, filled up by ``plan``.  ``tree_table`` int32
    ``[requests][blocks]``: pages of their trees.  ``num_pages``: pages that tables may name.  ``max_nodes``: of a tree, at most."""

    def __init__(self, block_table: torch.Tensor, tree_table: torch.Tensor, max_rows: int, num_pages: int, max_nodes: int = MAX_NODES):
        b, dev = block_table.shape[0], block_table.device
        _flat(block_table, torch.int32, (b, block_table.shape[-1]), "block table")
        _flat(tree_table, torch.int32, (b, tree_table.shape[-1]), "tree table", dev)
        if not 1 <= b <= MAX_REQUESTS or not 1 <= block_table.shape[1] < MAX_BLOCKS:
            raise ValueError(f"a step of 1 to {MAX_REQUESTS} requests, whose tables hold 1 to {MAX_BLOCKS - 1} pages")
        if not 1 <= max_rows <= MAX_ROWS:
            raise ValueError(f"a step of 1 to {MAX_ROWS} rows")
        if not 1 <= max_nodes <= min(MAX_NODES, PAGE * tree_table.shape[1]):
            raise ValueError(f"trees of 1 to {min(MAX_NODES, PAGE * tree_table.shape[1])} nodes, not {max_nodes}")
        if not 1 <= num_pages < 1 << 27:
            raise ValueError("tables of 1 to 2^27 pages")
        self.block_table, self.tree_table, self.device = block_table, tree_table, dev
        self.requests, self.max_rows, self.num_pages, self.max_nodes = b, max_rows, num_pages, max_nodes
        one = lambda n, t=torch.int32: torch.full((n,), -1, dtype=t, device=dev)          # noqa: E731
        self.lengths = torch.zeros(b, dtype=torch.int32, device=dev)
        self.row_start = torch.zeros(b + 1, dtype=torch.int32, device=dev)
        self.row_req, self.row_pos, self.slots, self.parents = one(max_rows), one(max_rows), one(max_rows), one(max_rows)
        self.masks = torch.zeros(max_rows, dtype=torch.int64, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self.tree: Optional[bool] = None       # the last plan's rows are trees'
        self._c = _Step(*(t.data_ptr() for t in (block_table, tree_table, self.lengths, self.row_start, self.row_req, self.row_pos, self.slots, self.parents, self.masks,
                                                 self.status)), b, block_table.shape[1], tree_table.shape[1], max_rows, max_nodes, num_pages)
        self._at, self._work = ctypes.addressof(self._c), {}
        self._small = (2 * b + 2 + 3) // 4 * 4          # fp32 words of workspace of an attention that leaves no segments
        self._floats, self._index = torch.empty(0, device=dev), dev.index

    def check(self):
        """Waits for the last plan and raises where it could not be made."""
        word = int(self.status[0])
        if word:
            raise K.KernelError("plan: " + "; ".join(text for bit, text in _FAULTS.items() if word & bit))


class Accepted:
    """What ``commit`` says of every request: ``path`` ``[requests][64]`` nodes of the accepted path, -1 behind it; their number ``count``;
    ``next_token``, the target of the last one (-1: no rows); ``lengths`` with the path's."""

    def __init__(self, path: torch.Tensor, count: torch.Tensor, next_token: torch.Tensor, lengths: torch.Tensor):
        b, dev = count.numel(), count.device
        self.path, self.count = _flat(path, torch.int32, (b, MAX_NODES), "accepted path", dev), _flat(count, torch.int32, (b,), "accepted nodes")
        self.next_token, self.lengths = _flat(next_token, torch.int32, (b,), "next tokens", dev), _flat(lengths, torch.int32, (b,), "lengths", dev)
        self._c = _Accepted(path.data_ptr(), count.data_ptr(), next_token.data_ptr(), lengths.data_ptr())
        self._at, self._requests, self._index = ctypes.addressof(self._c), b, dev.index

    @staticmethod
    def empty(requests: int, device) -> "Accepted":
        f = lambda *s: torch.empty(s, dtype=torch.int32, device=device)         # noqa: E731
        return Accepted(f(requests, MAX_NODES), f(requests), f(requests), f(requests))


def plan(step: TreeStep, lengths: torch.Tensor, counts: torch.Tensor, parents: Optional[torch.Tensor], pool: PagePool, after: Optional[PagePool] = None) -> TreeStep:
    """Lays out a step.  ``lengths``: cached positions of every request; ``counts``: its rows (0: none; -1: the request leaves and its pages go
    back).  ``parents``: of all rows, one request's after another, each the number of a node before it in its tree, or -1; None: the rows of a
    request are consecutive positions from its length on.  Block tables get the pages that are missing up to a request's length and longest path
    (``parents`` None: all its rows), in the order of the requests.  ``after``: where the pool's numbers are written (over the same free
    pages; None: in place)."""
    b, dev = step.requests, step.device
    if after is None:
        after = pool
    at, counts_at = _words(lengths, b, "lengths", dev), _words(counts, b, "rows of the requests", dev)
    rows, parents_at = step.max_rows, None
    if parents is not None:
        rows = parents.numel()
        parents_at = _words(parents, rows, "parents", dev) or at      # (an empty tensor has no address, and no parents are something else)
        if rows > step.max_rows:
            raise ValueError(f"parents: of up to {step.max_rows} rows, not {rows}")
    if pool._requests != b or after._requests != b or pool._index != step._index or after._c.free != pool._c.free:
        raise ValueError(f"pools of {b} requests on {dev}, over the same free pages")
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return plan(step, lengths, counts, parents, pool, after)
    K._check(_fn()["plan"](step._at, pool._at, after._at, at, counts_at, parents_at, rows, _stream(dev)), "tree_plan")
    step.tree = parents is not None
    return step


def _check_cache(step: TreeStep, cache: TreeCache, layers: bool):
    if step.tree is None:
        raise ValueError("the step has no plan yet")
    if cache._index != step._index or cache.pages < step.num_pages or cache.layers > 1 and not layers:
        raise ValueError(f"{'a' if layers else 'one layer of a'} cache of at least {step.num_pages} pages on {step.device}")


def rope_append(step: TreeStep, qkv: torch.Tensor, rope: tuple, q: torch.Tensor, cache: TreeCache, interleaved: bool = False) -> torch.Tensor:
    """Rows of a qkv projection, ``[rows][(n_q + 2 n_kv) D]`` bf16 or fp32, or fp32 partial sums ``[slices][rows][...]``: queries turned into ``q``
    (bf16 ``[rows][n_q D]``), keys turned and values as they are into the cache at the step's slots.  ``rope``: (cos, sin) tables fp32
    ``[positions][pairs]``, for the first 2 x pairs dimensions of a head (pairs a multiple of 4): pair i is dimensions i and i + pairs, or with
    ``interleaved`` 2 i and 2 i + 1.  Scaled positions and factors are the tables' (``models.config.Rotary``).  Rows behind the step's are left."""
    _check_cache(step, cache, False)
    dev, d, n_kv = step.device, cache.d, cache.heads
    if qkv.dtype is torch.bfloat16:
        slices, slice_elems = 0, 0
        rows, n, ld, at = _matrix(qkv, torch.bfloat16, "rows", dev)
    elif qkv.dim() == 3:
        rows, n, ld, at, slices, slice_elems = _matrix(qkv, torch.float32, "rows", dev, 3)
    else:
        slices, slice_elems = 1, 0
        rows, n, ld, at = _matrix(qkv, torch.float32, "rows", dev)
    if not 1 <= rows <= step.max_rows:
        raise ValueError(f"rows: 1 to {step.max_rows}, not {rows}")
    n_q, rest = divmod(n, d)
    n_q -= 2 * n_kv
    if rest or n_q < 1 or n_q % n_kv:
        raise ValueError(f"rows of {n} columns: heads of {d}, {n_kv} of keys and of values")
    mq, cols, ldq, pq = _matrix(q, torch.bfloat16, "queries", dev)
    if mq != rows or cols != n_q * d:
        raise ValueError(f"queries: {rows} rows of {n_q * d}")
    cos, sin = rope
    positions, pairs = cos.shape if cos.dim() == 2 else (0, 0)
    cos_at, sin_at = cos.data_ptr(), sin.data_ptr()
    if positions < 1 or pairs % 4 or 2 * pairs > d or sin.shape != cos.shape or cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or (cos_at | sin_at) % 16 \
            or cos.get_device() != dev.index or sin.get_device() != dev.index or not cos.is_contiguous() or not sin.is_contiguous():
        raise ValueError(f"rotation: two contiguous fp32 tables of positions x pairs on {dev}, pairs a multiple of 4 up to {d // 2}")
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return rope_append(step, qkv, rope, q, cache, interleaved)
    K._check(_fn()["rope"](step._at, cache._at, at, ld, slice_elems, slices, rows, cos_at, sin_at, pairs, positions, bool(interleaved), n_q, pq, ldq,
                           _stream(dev)), "tree_rope")
    return q


def attention(step: TreeStep, q: torch.Tensor, cache: TreeCache, out: torch.Tensor, scale: float, window: int = 0) -> torch.Tensor:
    """Rows ``q`` ``[rows][n_q D]`` bf16 over one layer's cache into ``out`` (the same shape, bf16): softmax in fp32 over the request's cached
    positions and the nodes of the row's mask, ``window`` > 0: those less than ``window`` positions before the row.  A row that sees nothing is
    0, whatever the places hold that it does not see (infinities and NaN too); rows behind the step's are left.  ``out`` may be ``q``."""
    _check_cache(step, cache, False)
    dev, d, n_kv = step.device, cache.d, cache.heads
    if not step.tree:
        raise ValueError("the step's rows are no trees'")
    rows, n, ldq, pq = _matrix(q, torch.bfloat16, "queries", dev)
    mo, no, ldo, po = _matrix(out, torch.bfloat16, "outputs", dev)
    n_q = n // d
    if n != n_q * d or n_q < 1 or n_q % n_kv or n_q // n_kv > MAX_GROUP or not 1 <= rows <= step.max_rows:
        raise ValueError(f"queries: 1 to {step.max_rows} rows of heads of {d}, 1 to {MAX_GROUP} to each of {n_kv} key heads, on {dev}")
    if mo != rows or no != n:
        raise ValueError(f"outputs: {rows} rows of {n} on {dev}")
    if not 0 <= window < 1 << 31 or not 0 < scale < float("inf"):
        raise ValueError("a window of 0 (none) or more positions, a scale above 0")
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return attention(step, q, cache, out, scale, window)
    room = step._work.get((n_q, n_kv, d))
    if room is None:
        room = step._work[n_q, n_kv, d] = _fn()["attention_work"](step._at, n_q, n_kv, d)
    work = step._floats.new_empty(room)      # this call's own: calls of one step on several streams share nothing
    K._check(_fn()["attention"](step._at, cache._at, pq, ldq, po, ldo, work.data_ptr(), rows, n_q, window, scale, _stream(dev)), "tree_attention")
    if room > step._small:
        K.launch_count += 1      # segments added up
    return out


MAX_GROUP = 64          # query heads to a key head


def commit(step: TreeStep, tokens: torch.Tensor, targets: torch.Tensor, cache: TreeCache, accepted: Optional[Accepted] = None) -> Accepted:
    """Settles a step.  ``tokens``: the rows' tokens; ``targets``: the token that the model gives behind each row (its arg-max, or a draw), int32
    ``[rows]``.  The path begins at a tree's node 0 and goes on with the child whose token is its parent's target, of equal ones the first.
    Its keys and values move from the tree's pages to the request's positions in every layer of ``cache``; nothing else is touched.
    ``accepted.lengths`` may be the tensor that the next ``plan`` reads; no result may share memory with ``tokens``, ``targets`` or the step."""
    _check_cache(step, cache, True)
    dev, b = step.device, step.requests
    if not step.tree:
        raise ValueError("the step's rows are no trees'")
    rows = tokens.numel()
    if not 1 <= rows <= step.max_rows:
        raise ValueError(f"tokens: of 1 to {step.max_rows} rows")
    at, targets_at = _words(tokens, rows, "tokens", dev), _words(targets, rows, "targets", dev)
    if accepted is None:
        accepted = Accepted.empty(b, dev)
    elif accepted._requests != b or accepted._index != step._index:
        raise ValueError(f"results of {b} requests on {dev}")
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return commit(step, tokens, targets, cache, accepted)
    rc = _fn()["commit"](step._at, cache._at, accepted._at, at, targets_at, rows, _stream(dev))
    if rc == -3:
        raise ValueError("results apart from the tokens, the targets and the step's own")
    K._check(rc, "tree_commit")
    return accepted
