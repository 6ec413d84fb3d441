"""Trees of drafted tokens: what a speculative step hands to the model in place of one chain of guesses.

The reference's speculative decoder verifies a chain, greedily (speculative.py:83-277). Here a step's T new tokens of a
row may be the nodes of a tree: node 0 is the row's last token that stands, every other one was drafted behind an earlier
one. A cache with a tree set (KVCache.set_tree, PagedKVCache.set_tree) makes the attention module let each node see
the cache and its own branch, and the model place it at its depth; verify() says which nodes stand and what token comes
behind them; cache.keep() closes the accepted branch up. On the GPU these are ops.tree_mask, attn_tree(_paged),
verify_drafts and kv_compact(_paged); elsewhere the torch code below and in the module.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch


@dataclass
class Drafts:
    """What a drafter proposes behind the last token: `tokens`, each behind the token `parents` names (an index among them, or
    -1: behind the last token; None: a chain)."""

    tokens: list[int]
    parents: list[int] | None = None

    def nodes(self) -> list[int]:
        """Parents of the step's nodes, node 0 being the row's last token."""
        parents = self.parents if self.parents is not None else [t - 1 for t in range(len(self.tokens))]
        if len(parents) != len(self.tokens) or any(not -1 <= p < t for t, p in enumerate(parents)):
            raise ValueError("a draft's parents name earlier tokens, one for each")
        return [-1] + [p + 1 for p in parents]

    @property
    def chain(self) -> bool:
        return self.parents is None or list(self.parents) == [t - 1 for t in range(len(self.tokens))]


def _ancestors(parents: list[int]) -> tuple[torch.Tensor, list[int]]:
    """bool [T, T] (row t: t and its ancestors) and depths."""
    T = len(parents)
    see, depth = torch.eye(T, dtype=torch.bool), [0] * T
    for t, p in enumerate(parents):
        if 0 <= p < t:
            see[t] |= see[p]
            depth[t] = depth[p] + 1
    return see, depth


def _packed(parents: list[int]) -> tuple[torch.Tensor, list[int]]:
    """ops.tree_mask's bits [T, words] and depths of one tree."""
    see, depth = _ancestors(parents)
    T = len(parents)
    bits = torch.zeros(T, -(-T // 64), 64, dtype=torch.int64)
    bits.view(T, -1)[:, :T] = see
    return (bits << torch.arange(64)).sum(-1), depth


class TokenTree:
    """The trees of one pass, in buffers that a recorded graph may read: set() fills them anew for trees of as many nodes."""

    def __init__(self, parents, batch: int, device: torch.device):
        rows = self._rows(parents, batch)
        self.batch, self.T, self.device = batch, len(rows[0]), device
        self.parents = torch.empty(batch, self.T, dtype=torch.int32, device=device)
        self.depth = torch.empty_like(self.parents)
        self.mask = torch.empty(batch, self.T, -(-self.T // 64), dtype=torch.int64, device=device)
        self.set(parents)

    @staticmethod
    def _rows(parents, batch: int) -> list[list[int]]:
        rows = parents.tolist() if isinstance(parents, torch.Tensor) else [list(p) if isinstance(p, (list, tuple)) else p for p in parents]
        if rows and not isinstance(rows[0], list):
            rows = [rows] * batch
        if len(rows) != batch or not rows[0] or any(len(r) != len(rows[0]) for r in rows):
            raise ValueError(f"a tree needs parents [T], or [B, T] with B={batch}, and at least one node")
        if len(rows[0]) > 1024:
            raise ValueError("a tree has at most 1024 nodes")
        return rows

    def set(self, parents) -> None:
        rows = self._rows(parents, self.batch)
        if len(rows[0]) != self.T:
            raise ValueError(f"these buffers hold trees of {self.T} nodes, not {len(rows[0])}")
        self.rows = rows
        self.parents.copy_(torch.tensor(rows, dtype=torch.int32).clamp(-1, self.T))
        from .attention import hip_disabled

        if self.device.type == "cuda" and not hip_disabled():
            from . import ops

            mask, depth = ops.tree_mask(self.parents)
            self.mask.copy_(mask)
            self.depth.copy_(depth)
        else:
            masks, depths = zip(*(_packed(r) for r in rows))
            self.mask.copy_(torch.stack(masks))
            self.depth.copy_(torch.tensor(depths, dtype=torch.int32))

    def see(self, row: int) -> torch.Tensor:
        """bool [T, T]: which nodes each node of a row sees."""
        return _ancestors(self.rows[row])[0]


def tree_mask(tree: TokenTree, row: int, base: int, n: int, window: int, sinks: int, device) -> torch.Tensor:
    """bool [n, base + n], True = may attend: the row's nodes against the cache before them and themselves (ops.attn_tree)."""
    among, depth = _ancestors(tree.rows[row])
    see = torch.cat([torch.ones(n, base, dtype=torch.bool), among[:n, :n]], 1)
    if window:
        own = torch.tensor(depth[:n]) + base
        pos = torch.cat([torch.arange(base), own])
        see &= (pos[None] > own[:, None] - window) | (pos < sinks)[None]
    return see.to(device)


def static_tree_mask(tree: TokenTree, pos_t: torch.Tensor, length: int, window: int, sinks: int) -> torch.Tensor:
    """tree_mask of all rows against a static cache's `length` slots, bool [B, T, length], by the device's own numbers (a
    recorded graph computes it anew)."""
    T, dev = tree.T, tree.device
    slot = torch.arange(length, device=dev)
    off = slot - pos_t
    new, at = (off >= 0) & (off < T), off.clamp(0, T - 1)
    among = ((tree.mask[..., None] >> torch.arange(64, device=dev)) & 1).flatten(-2)[..., :T].bool()
    see = torch.where(new, among.index_select(2, at), off < 0)
    if window:
        own = pos_t + tree.depth
        pos = torch.where(new, own.index_select(1, at), slot)
        see &= (pos[:, None] > own[..., None] - window) | (pos < sinks)[:, None]
    return see


def verify(logits: torch.Tensor, tokens: torch.Tensor, *, parents: torch.Tensor | None = None, uniform: torch.Tensor | None = None,
           temperature: float = 0.0, draft_probs: torch.Tensor | None = None,
           new_lens: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """ops.verify_drafts, or its rule in torch where the tensors are not on the GPU (or SLEUTH_AMD_NO_HIP=1)."""
    from . import ops
    from .attention import hip_disabled

    if logits.is_cuda and not hip_disabled():
        return ops.verify_drafts(logits, tokens, parents=parents, uniform=uniform, temperature=temperature, draft_probs=draft_probs,
                                 new_lens=new_lens)
    B, T, V = logits.shape
    if temperature < 0 or not math.isfinite(temperature):
        raise ValueError(f"temperature must be 0, or positive and finite, not {temperature}")
    if temperature and uniform is None:
        raise ValueError("a temperature needs uniform, the random numbers")
    out, path = torch.full((B, T), -1), torch.full((B, T), -1, dtype=torch.int32)
    count = torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        n = T if new_lens is None else max(0, min(int(new_lens[b]), T))
        if parents is None:
            up = [t - 1 for t in range(T)]
        else:
            up = (parents if parents.dim() == 1 else parents[b]).tolist()
        news, nodes = _verify_row(logits[b], tokens[b].tolist(), up, uniform[b].tolist() if temperature else None, temperature,
                                  None if draft_probs is None else draft_probs[b], n)
        out[b, :len(news)] = torch.tensor(news, dtype=torch.long)
        path[b, :len(nodes)] = torch.tensor(nodes, dtype=torch.int32)
        count[b] = len(nodes)
    return out.to(logits.device), path.to(logits.device), count.to(logits.device)


def _verify_row(logits, tokens, parents, u, temperature, probs, n):
    """(the row's new tokens, the nodes that stand). What is left of a node's weights shrinks with every rejected child: by
    its drafter's probabilities, scaled to what was left, or by the token itself."""
    if not n:
        return [], []
    at, nodes, news = 0, [0], []
    while True:
        x = logits[at].double()
        x = x.masked_fill(x.isnan(), -math.inf)
        top, best = x.max(), int(x.argmax())
        left = None
        if temperature and top > -math.inf:
            left = (x == top).double() if top == math.inf else ((x - top) / temperature).exp()
        taken, stands, whole = 0.0, None, left
        for t in range(at + 1, n):
            v = tokens[t]
            if parents[t] != at or not 0 <= v < x.numel():
                continue
            if left is None:
                ok = not temperature and v == best
            else:
                q = 1.0 if probs is None else float(probs[at, v])
                ok = u[t] * q * float(left.sum()) < float(left[v])
            if ok:
                stands = t
                break
            if left is not None and probs is not None:
                taken += float(left.sum())
                left = (whole - taken * probs[at].double()).clamp(min=0)
            elif left is not None:
                left = left.clone()
                left[v] = 0
        if stands is None:
            break
        at = stands
        nodes.append(at)
        news.append(tokens[at])
    last = best
    if left is not None and float(left.sum()) > 0:
        over = (left.cumsum(0) > u[0] * left.sum()).nonzero()
        last = int(over[0]) if len(over) else int((left > 0).nonzero()[-1])
    return news + [last], nodes
