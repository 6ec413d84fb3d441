"""Plain 64-bit forms of what verifying trees of drafted tokens takes: who sees whom, which drafted tokens stand, and
what of the cache moves. Written row by row, in Python."""

from __future__ import annotations

import math
import random

import torch


def make_parents(rng: random.Random, T: int, shape: str) -> list[int]:
    if shape == "chain":
        return [t - 1 for t in range(T)]
    if shape == "star":
        return [-1] + [0] * (T - 1)
    if shape == "forest":   # several nodes hang on the cache alone
        return [-1 if t < 3 else rng.randrange(-1, t) for t in range(T)]
    return [-1] + [rng.randrange(max(0, t - 7), t) for t in range(1, T)]


def chain_of(parents: list[int], t: int) -> list[int]:
    """t and its ancestors, t first; a parent that is not before its child is none."""
    out = [t]
    while 0 <= parents[out[-1]] < out[-1]:
        out.append(parents[out[-1]])
    return out


def mask_of(parents: list[int], n: int) -> tuple[list[list[int]], list[int]]:
    """Words of 64 bits (as signed numbers) and depths of the first n tokens; zeros behind them."""
    T = len(parents)
    words = -(-T // 64)
    bits, depth = [[0] * words for _ in range(T)], [0] * T
    for t in range(n):
        chain = chain_of(parents, t)
        depth[t] = len(chain) - 1
        for j in chain:
            bits[t][j // 64] |= 1 << (j % 64)
    return [[x - (1 << 64) if x >> 63 else x for x in row] for row in bits], depth


def bits_to_bool(mask: torch.Tensor, T: int) -> torch.Tensor:
    """[.., T, words] -> bool [.., T, T]"""
    return ((mask[..., None] >> torch.arange(64)) & 1).flatten(-2)[..., :T].bool()


def tree_see(base: int, n: int, among: torch.Tensor, depth: list[int] | None, window: int, sinks: int) -> torch.Tensor:
    """[n, base + n] bool: what the n new tokens of a row see; among [n, n]: which new tokens each one sees."""
    see = torch.zeros(n, base + n, dtype=torch.bool)
    pos = list(range(base)) + [base + (depth[j] if depth else 0) for j in range(n)]
    for t in range(n):
        at = base + (depth[t] if depth else 0)
        for s in range(base + n):
            ok = True if s < base else bool(among[t, s - base])
            if window and not (pos[s] > at - window or pos[s] < sinks):
                ok = False
            see[t, s] = ok
    return see


def tree_see_long(base: int, n: int, among: torch.Tensor, depth: list[int] | None, window: int, sinks: int) -> torch.Tensor:
    """tree_see by whole rows, for long caches."""
    at = base + (torch.tensor(depth[:n]) if depth else torch.zeros(n, dtype=torch.long))
    pos = torch.cat([torch.arange(base), at])
    see = torch.cat([torch.ones(n, base, dtype=torch.bool), among], 1)
    return see & ((pos[None] > at[:, None] - window) | (pos < sinks)[None]) if window else see


def verify_row(logits: torch.Tensor, tokens: list[int], parents: list[int], u: list[float] | None, heat: float,
               probs: torch.Tensor | None, n: int) -> tuple[list[int], list[int]]:
    """(new tokens, path) of one row: logits [T, V], probs [>= T - 1, V] or None, n real nodes."""
    if n == 0:
        return [], []
    V = logits.shape[1]
    x = logits.double()
    x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x)
    at, path, out = 0, [0], []
    while True:
        children = [t for t in range(at + 1, n) if parents[t] == at and 0 <= tokens[t] < V]
        row = x[at]
        top = row.max()
        best = int((row == top).nonzero()[0])
        hit = None
        if heat <= 0 or math.isnan(heat) or top == -math.inf:
            if not (heat > 0):
                hit = next((t for t in children if tokens[t] == best), None)
            last = best
        else:
            e = (row == top).double() if top == math.inf else ((row - top) / heat).exp()
            left, taken, gone = e.clone(), 0.0, set()
            for t in children:
                v, W = tokens[t], float(left.sum())
                if probs is not None:
                    q = probs[at].double()
                    if u[t] * float(q[v]) * W < float(left[v]):
                        hit = t
                        break
                    taken += W
                    left = (e - taken * q).clamp(min=0)
                else:
                    if v not in gone and u[t] * W < float(left[v]):
                        hit = t
                        break
                    gone.add(v)
                    left[v] = 0
            if hit is None:
                W = float(left.sum())
                over = (left.cumsum(0) > u[0] * W).nonzero()
                last = best if W <= 0 else int(over[0]) if len(over) else int((left > 0).nonzero()[-1])
        if hit is None:
            return out + [last], path
        at = hit
        path.append(at)
        out.append(tokens[at])


def compact_row(values: torch.Tensor, base: int, path: list[int], limit: int, held=lambda s: True) -> torch.Tensor:
    """values [K, S, D] of one row with slot base + i <- slot base + path[i] where that is behind it."""
    out = values.clone()
    for i, of in enumerate(path):
        if of > i and base + of < limit and held(base + of) and held(base + i):
            out[:, base + i] = values[:, base + of]
    return out
