"""Token trees on the engine: several drafted continuations of each request, verified in one step (``ops/tree.py``).

A request's tree is its next token (node 0, which is not in the cache yet) and drafts behind it, each with the node it follows.  One step runs
all nodes of all trees; the path is kept that goes on, from node 0, with the child whose token is what the model gives behind its parent (of
equal children the first, whichever path is the longer) -- greedily, the tokens that plain decoding would have made, one by one -- and the rest leaves no trace.  The engine keeps pages for the trees of every slot
(``Engine(tree_nodes=...)``).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..ops import lib as K
from ..ops import tree as T

PAGE = 16


@dataclass(frozen=True)
class Verified:
    """What a step accepted of a request's tree: nodes of the path, their tokens (the first is the request's next token itself), and the token that
    the model gives behind the last one."""
    path: List[int]
    tokens: List[int]
    next_token: int


class TreeVerifier:
    """Trees of up to ``nodes`` nodes for the slots of ``eng``."""

    def __init__(self, eng, nodes: int):
        cfg = eng.cfg
        if cfg.layer_specs or cfg.n_gdn_layers or cfg.head_dim not in (64, 128) or not eng.can_score:      # (a pipeline's stage has a part of the layers)
            raise ValueError("token trees: attention layers with heads of 64 or 128 on one GPU")
        self.eng, blocks = eng, -(-nodes // PAGE)
        b = eng.max_seqs
        for s in range(b):
            eng.pool.ensure(b + s, blocks)
        self.tree_table = torch.tensor([list(eng.pool.table(b + s)) for s in range(b)], dtype=torch.int32, device=eng.device)
        kv, n = eng.kv, cfg.n_layers
        self.step = T.TreeStep(eng.block_table, self.tree_table, eng.max_rows, kv.num_pages, nodes)
        self.caches = [T.TreeCache(*kv.layer(li)) for li in range(n)]
        scales = (kv.k_scale[:n], kv.v_scale[:n]) if kv.kv_int8 else ()
        self.all = T.TreeCache(kv.k[:n], kv.v[:n], *scales)
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=eng.device)         # noqa: E731
        self.inputs = i32(3 * b + 2 * eng.max_rows)      # lengths, rows, held pages, parents, tokens
        self.staging = torch.zeros(3 * b + 2 * eng.max_rows, dtype=torch.int32).pin_memory()
        lengths, self.counts, held, self.parents, self.tokens = self.inputs.split([b, b, b, eng.max_rows, eng.max_rows])
        self.best = i32(eng.max_rows)       # arg-max of the rows: the engine's own words are the next step's, whoever makes it
        self.at_lengths: List[int] = []
        self.lengths = lengths
        self.pool = T.PagePool(i32(1), i32(1), held)       # (the host's pool has given the pages: nothing is taken here)
        self.accepted = T.Accepted.empty(b, eng.device)
        self.rows: List[Tuple[int, List[int], List[int]]] = []

    def forward(self, trees: Dict[int, Tuple[Sequence[int], Sequence[int]]]) -> torch.Tensor:
        """Runs the nodes of ``trees`` (slot -> tokens, parents; node 0's parent is -1); fp32 logits of all rows, slots in order, nodes in theirs
        (valid until the next step).  The requests' positions are as they were until ``commit``; other slots may prefill and step in between."""
        from .engine import Row
        eng = self.eng
        if eng.model.ep is not None:
            raise ValueError("token trees: experts on one GPU")
        rows, todo, self.rows = [], [], []
        for slot in sorted(trees):
            tokens, parents = list(trees[slot][0]), list(trees[slot][1])
            n = len(tokens)
            if not 0 <= slot < eng.max_seqs or not 1 <= n <= self.step.max_nodes or len(parents) != n or parents[0] != -1 or any(not 0 <= p < i for i, p in enumerate(parents) if i):
                raise ValueError(f"tree of slot {slot}: 1 to {self.step.max_nodes} tokens, each with a node before it (the first with none: -1)")
            eng.check_ids(tokens)
            depth = [0] * n
            for i in range(1, n):
                depth[i] = depth[parents[i]] + 1
            todo.append((slot, tokens, parents, max(depth) + 1))
            rows += [Row(slot, eng.seq_len[slot] + d, t) for d, t in zip(depth, tokens)]
        if not 1 <= len(rows) <= eng.max_rows:
            raise ValueError(f"a step of 1 to {eng.max_rows} rows, not {len(rows)}")
        eng.require_ok()
        for slot, _, _, deepest in todo:
            eng._ensure_pages(slot, eng.seq_len[slot] + deepest)
        b, host = eng.max_seqs, self.staging.numpy()
        torch.cuda.current_stream(eng.device).synchronize()       # (the staging of a step before is read)
        host[:b] = eng.seq_len
        host[b: 2 * b] = 0
        host[2 * b: 3 * b] = [len(eng.pool.table(s)) for s in range(b)]
        at = 3 * b
        for slot, tokens, parents, _ in todo:
            host[b + slot] = len(tokens)
            host[at: at + len(parents)] = parents
            host[at + eng.max_rows: at + eng.max_rows + len(tokens)] = tokens
            at += len(parents)
        self.inputs.copy_(self.staging, non_blocking=True)
        eng._write_rows(rows)
        eng._snap = None
        m, model = len(rows), eng.model
        T.plan(self.step, self.lengths, self.counts, self.parents[:m], self.pool)
        model.tree = self
        try:
            model.step_rows(m, eng.ctrl, eng.block_table, eng.max_blocks, eng.kv, False)
        finally:
            model.tree = None
        self.best[:m].copy_(eng.ctrl[K.CTRL_OUT_TOKEN: K.CTRL_OUT_TOKEN + m])
        self.rows, self.at_lengths = [t[:3] for t in todo], [eng.seq_len[t[0]] for t in todo]
        return eng.logits(m)

    def forget(self, slot: int):
        """The slot's positions are no longer those that the last ``forward`` saw: it cannot be settled."""
        if any(s == slot for s, _, _ in self.rows):
            self.rows = []

    def commit(self, targets: Optional[torch.Tensor] = None) -> Dict[int, Verified]:
        """Settles the last ``forward``: ``targets`` int32, the token behind every row (a draw from its logits; None: the arg-max).  The accepted
        nodes' keys and values become the requests' next positions.  Refused where one of the trees' slots has been reset, cut or run further since."""
        eng, m = self.eng, sum(len(t) for _, t, _ in self.rows)
        if [eng.seq_len[s] for s, _, _ in self.rows] != self.at_lengths[: len(self.rows)]:
            m, self.rows = 0, []
        if not m:
            raise ValueError("no trees to settle")
        if targets is None:
            targets = self.best[:m]
        got = T.commit(self.step, self.tokens[:m], targets, self.all, self.accepted)
        path, count, following = got.path.tolist(), got.count.tolist(), got.next_token.tolist()      # (waits)
        rows, self.rows = self.rows, []
        self.step.check()
        eng.check_failed("tree step")
        out = {}
        for slot, tokens, _ in rows:
            nodes = path[slot][: count[slot]]
            eng.seq_len[slot] += len(nodes)
            eng.pool.truncate(slot, -(-eng.seq_len[slot] // PAGE))
            out[slot] = Verified(nodes, [tokens[i] for i in nodes], following[slot])
        return out
