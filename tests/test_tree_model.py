"""Drafted trees in the caches, the module and the generators; forked rows of the paged cache."""

from __future__ import annotations

import random

import pytest
import torch

from sleuth_amd import ops
from sleuth_amd.config import ModelConfig
from sleuth_amd.gated import GatedAttention
from sleuth_amd.generate import (GraphDecoder, generate, generate_batch, ngram_draft, ngram_tree_draft, speculative_generate)
from sleuth_amd.kv_cache import KVCache
from sleuth_amd.model import Transformer
from sleuth_amd.paged_cache import OutOfPages, PagedKVCache
from sleuth_amd.tree import Drafts, TokenTree, verify
from tree_oracle import chain_of, make_parents, mask_of, verify_row

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def make(device, dtype=torch.float32, **kw):
    torch.manual_seed(0)
    base = dict(vocab_size=64, d_model=64, n_layers=2, n_heads=4, head_size=32, n_kv_heads=2, qk_norm=True, max_seq_len=128,
                init_std=0.3)   # (large weights: the argmax is no near tie)
    base.update(kw)
    return Transformer(ModelConfig(**base)).to(device, dtype).eval()


KINDS = {"full": {}, "sliding": dict(layer_types=["sliding", "full"], sliding_window=6),
         "sinks": dict(layer_types=["sliding"] * 2, sliding_window=5, sink_tokens=2), "partial": dict(rope_dim=16)}


def _branch_logits(model, prompt, tokens, parents, t):
    """Logits behind node t, by a plain pass over the prompt and the node's branch."""
    branch = [tokens[j] for j in reversed(chain_of(parents, t))]
    return model(torch.tensor([prompt + branch], device=next(model.parameters()).device)).logits[0, -1]


# (logits of 32-bit passes: a few hundred sums of some ten terms each, of size one: far below 1e-3, as the module's other
# 32-bit comparisons with the torch path)
TOL = 1e-3


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("paged", [False, True])
@torch.no_grad()
def test_a_tree_pass_is_a_pass_of_each_branch(device, kind, paged):
    model = make(device, **KINDS[kind])
    rng = random.Random(3)
    prompts = [[rng.randrange(64) for _ in range(n)] for n in (9, 21)]
    T = 7
    parents = [make_parents(rng, T, "tree"), make_parents(rng, T, "chain")]
    tokens = [[rng.randrange(64) for _ in range(T)] for _ in prompts]
    cache = (PagedKVCache if paged else KVCache).for_model(model, 2, 64, **({"page_size": 16} if paged else {}))
    if paged:
        cache.set_new([9, 21])
        model(torch.tensor([p + [0] * (21 - len(p)) for p in prompts], device=device), cache=cache)
        cache.set_new([T, T - 2])
    else:
        for b, p in enumerate(prompts):   # rows of their own lengths
            one = KVCache.for_model(model, 1, 64)
            model(torch.tensor([p], device=device), cache=one)
            for mine, his in zip(cache.k + cache.v, one.k + one.v):
                mine[b] = his[0]
        cache.set_lengths([9, 21])
    cache.set_tree(parents)
    logits = model(torch.tensor(tokens, device=device), cache=cache).logits
    ran = {blk.attn.last_path for blk in model.blocks}
    assert ran == ({"torch"} if device == "cpu" else {"hip-paged-tree" if paged else "hip-tree"})
    assert cache.seq_lens_host == [9, 21]
    real = [T, T - 2] if paged else [T, T]
    for b in range(2):
        for t in range(real[b]):
            want = _branch_logits(model, prompts[b], tokens[b], parents[b], t)
            assert (logits[b, t] - want).abs().max() < TOL, (b, t)
    # an accepted branch: the next token goes on from it
    paths = [chain_of(parents[0], T - 1)[::-1], [0, 1]]
    if paths[0][0] != 0:
        paths[0] = [0]
    path = torch.full((2, T), -1, dtype=torch.int32)
    for b, p in enumerate(paths):
        path[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
    assert cache.keep(path.to(device), torch.tensor([len(p) for p in paths], dtype=torch.int32, device=device)) == [len(p) for p in paths]
    cache.set_tree(None)
    assert cache.seq_lens_host == [9 + len(paths[0]), 23]
    if paged:
        assert cache.seq_lens.tolist() == cache.seq_lens_host
        cache.set_new(None)
    after = model(torch.tensor([[5], [6]], device=device), cache=cache).logits
    for b, tok in enumerate((5, 6)):
        full = prompts[b] + [tokens[b][j] for j in paths[b]] + [tok]
        assert (after[b, -1] - model(torch.tensor([full], device=device)).logits[0, -1]).abs().max() < TOL


@pytest.mark.parametrize("device", DEVICES)
def test_trees_that_do_not_fit(device):
    model = make(device)
    cache = KVCache.for_model(model, 1, 32)
    for bad in ([[0] * 3] * 2, [[]], [], [[-1] * 1025]):
        with pytest.raises(ValueError):
            cache.set_tree(bad)
    cache.set_tree([-1, 0, 0])
    with torch.no_grad(), pytest.raises(ValueError, match="nodes"):
        model(torch.zeros(1, 4, dtype=torch.long, device=device), cache=cache)
    one = torch.zeros(1, 3, dtype=torch.int32, device=device)
    for count in (-1, 4, 40):
        with pytest.raises(ValueError, match="keep"):
            cache.keep(one, torch.tensor([count], dtype=torch.int32, device=device))
    gated = GatedAttention(type("C", (), dict(head_dim=32, norm_eps=1e-6))(), 0)
    with pytest.raises(NotImplementedError):
        gated(torch.zeros(1, 3, 64), None, None, cache)
    with torch.no_grad(), pytest.raises(NotImplementedError):
        model.blocks[0].attn(torch.zeros(1, 3, 64, device=device), torch.zeros(3, 32, device=device), torch.zeros(3, 32, device=device),
                             cache, torch.ones(1, 1, 3, 3, dtype=torch.bool, device=device))
    cache.reset()
    assert cache.tree is None
    for d in (Drafts([1, 2], [0, -1]), Drafts([1, 2], [-1]), Drafts([1], [-2])):
        with pytest.raises(ValueError):
            d.nodes()
    assert Drafts([4, 5, 6], [-1, -1, 0]).nodes() == [-1, 0, 0, 1] and Drafts([4, 5]).chain and not Drafts([4, 5], [-1, -1]).chain


@pytest.mark.parametrize("device", DEVICES)
def test_tree_buffers(device):
    rng = random.Random(1)
    tree = TokenTree(make_parents(rng, 70, "tree"), 2, torch.device(device))
    where = tree.mask.data_ptr(), tree.depth.data_ptr(), tree.parents.data_ptr()
    rows = [make_parents(rng, 70, "tree"), make_parents(rng, 70, "forest")]
    tree.set(rows)
    assert where == (tree.mask.data_ptr(), tree.depth.data_ptr(), tree.parents.data_ptr())
    for b, p in enumerate(rows):
        assert tree.depth[b].tolist() == mask_of(p, 70)[1]
        assert all(tree.see(b)[t].nonzero().flatten().tolist() == sorted(chain_of(p, t)) for t in range(70))
        if device == "cuda":
            assert tree.mask[b].tolist() == mask_of(p, 70)[0]
    with pytest.raises(ValueError):
        tree.set([-1, 0])


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_verify_in_torch(probs, temperature):
    g, rng = torch.Generator().manual_seed(5), random.Random(5)
    B, T, V = 6, 9, 50
    logits = 2 * torch.randn(B, T, V, generator=g)
    logits[0, 0, 3] = float("nan")
    logits[1, :, 7:] = float("-inf")
    logits[2, 0] = float("-inf")
    q = (logits.nan_to_num(0, 0, -9) + 0.5 * torch.randn(B, T, V, generator=g)).softmax(-1)
    parents = [make_parents(rng, T, rng.choice(["tree", "star", "chain"])) for _ in range(B)]
    tokens = torch.randint(-1, 9, (B, T), generator=g)
    u = torch.rand(B, T, generator=g)
    news = [T, T, T, 0, 4, T]
    out, path, count = verify(logits, tokens, parents=torch.tensor(parents, dtype=torch.int32), uniform=u, temperature=temperature,
                              draft_probs=q if probs else None, new_lens=torch.tensor(news))
    for b in range(B):
        o, p = verify_row(logits[b], tokens[b].tolist(), parents[b], u[b].double().tolist(), temperature, q[b] if probs else None, news[b])
        assert out[b].tolist() == o + [-1] * (T - len(o)) and path[b].tolist() == p + [-1] * (T - len(p)) and int(count[b]) == len(p)
    with pytest.raises(ValueError):
        verify(logits, tokens, temperature=0.5)
    with pytest.raises(ValueError):
        verify(logits, tokens, uniform=u, temperature=-0.5)


# ---------------------------------------------------------------- generators
REPEATING = [3, 9, 4, 3, 9, 5, 3, 9, 4, 7, 3, 9]


def test_ngram_tree_draft():
    d = ngram_tree_draft()(REPEATING, 6)
    # behind (.., 3, 9): 4 7 3 9, then 5 3 9 4.., then 4 3 9 5..: the last one shares its 4
    assert d.tokens[0] == 4 and 5 in d.tokens and len(d.tokens) <= 6
    roots = [t for t, p in zip(d.tokens, d.parents) if p == -1]
    assert sorted(roots) == [4, 5]
    d.nodes()
    assert ngram_tree_draft()([1, 2, 3], 4).tokens == []
    for k in range(1, 9):
        d = ngram_tree_draft(branches=2)(REPEATING, k)
        assert 1 <= len(d.tokens) <= k and d.nodes()


def _tree_of_truth(model, wrong):
    """A drafter that knows what generate() would say and offers it beside wrong tokens, in the order `wrong` says."""
    def draft(ids, k):
        real = generate(model, ids, max_new_tokens=k).new_ids
        tokens, parents, at = [], [], -1
        for i, t in enumerate(real):
            for x in ([(t + 1) % 64, t] if wrong(i) else [t, (t + 1) % 64]):
                if len(tokens) < k:
                    tokens.append(x)
                    parents.append(at)
            if t not in [x for x, p in zip(tokens, parents) if p == at]:
                break
            at = max(j for j, (x, p) in enumerate(zip(tokens, parents)) if x == t and p == at)
        return Drafts(tokens, parents)
    return draft


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["full", "sliding", "sinks"])
def test_greedy_trees_say_what_decoding_says(device, kind):
    model = make(device, **KINDS[kind])
    want = generate(model, REPEATING, 20).new_ids
    got = speculative_generate(model, REPEATING, 20, k=6, draft=ngram_tree_draft())
    assert got.new_ids == want
    got = speculative_generate(model, REPEATING, 20, k=6, draft=_tree_of_truth(model, lambda i: i % 2 == 0))
    assert got.new_ids == want
    assert got.stats["speculative"]["accepted"] >= 10   # (three of six nodes a round are right)


@pytest.mark.gpu
def test_greedy_trees_from_a_graph():
    model = make("cuda", **KINDS["sliding"])
    want = generate(model, REPEATING, 24).new_ids
    for _ in range(2):   # (the second run replays the first one's graph)
        got = speculative_generate(model, REPEATING, 24, k=6, draft=_tree_of_truth(model, lambda i: i % 3 == 0), cuda_graph=True, trees=True)
        assert got.new_ids == want and got.stats["graph_replays"] > 0
    got = speculative_generate(model, REPEATING, 24, k=6, draft=_tree_of_truth(model, lambda i: True), cuda_graph=True)
    assert got.new_ids == want   # (a chain's graph: trees run eagerly)
    dec = GraphDecoder(model, 64, torch.float32, 3)
    tokens = torch.tensor([3, 9, 4], device="cuda")
    with torch.no_grad():
        model(torch.tensor([REPEATING], device="cuda"), cache=dec.cache)
        chain = dec.verify(tokens).clone()
    with pytest.raises(ValueError, match="chains"):
        dec.verify(tokens, [-1, 0, 0])
    assert torch.isfinite(chain).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("draft", [ngram_draft, ngram_tree_draft])
def test_sampled_drafts(device, draft):
    """The same seed, the same tokens; a cold temperature, the greedy ones; other seeds, others."""
    model = make(device)
    a, b, c = (speculative_generate(model, REPEATING, 16, k=5, draft=draft(), temperature=1.5, seed=s).new_ids for s in (1, 1, 2))
    assert a == b and a != c and len(a) == 16
    assert speculative_generate(model, REPEATING, 16, k=5, draft=draft(), temperature=1e-4, seed=3).new_ids == \
        generate(model, REPEATING, 16).new_ids


def test_sampled_trees_keep_the_distribution():
    """The first drafted step's token, over 1,500 seeds, against the model's own probabilities. A count is binomial: the chance
    that one of 8 is six standard deviations off is below 1e-7."""
    model = make("cpu", vocab_size=8, n_layers=1, d_model=32, init_std=0.15)
    prompt = [1, 2, 3]
    cfg = model.cfg
    first = []
    for seed in range(1500):
        r = speculative_generate(model, prompt, 2, k=1, draft=lambda ids, k: Drafts([(ids[-1] + 1) % cfg.vocab_size], [-1]),
                                 temperature=1.0, seed=seed)
        first.append(r.new_ids)
    with torch.no_grad():
        p1 = model(torch.tensor([prompt])).logits[0, -1].double().softmax(-1)
        p2 = sum(p1[t] * model(torch.tensor([prompt + [t]])).logits[0, -1].double().softmax(-1) for t in range(8))
    for i, p in enumerate((p1, p2)):
        seen = torch.bincount(torch.tensor([x[i] for x in first]), minlength=8).double()
        assert ((seen - 1500 * p).abs() <= 6 * (1500 * p * (1 - p)).sqrt()).all(), i


# ---------------------------------------------------------------- forks
@pytest.mark.parametrize("device", DEVICES)
@torch.no_grad()
def test_forked_rows_go_their_own_ways(device):
    model = make(device)
    cache = PagedKVCache.for_model(model, 3, 64, page_size=16)
    prompt = list(range(1, 22))
    cache.set_new([21, 0, 0])
    model(torch.tensor([prompt, [0] * 21, [0] * 21], device=device), cache=cache)
    assert cache.free_pages == cache.n_pages - 2
    cache.fork(0, 1)
    cache.fork(0, 2)
    assert cache.free_pages == cache.n_pages - 2 and cache.seq_lens_host == [21] * 3
    before = cache.page_table[0, 1].item()
    cache.set_new([1, 1, 0])
    logits = model(torch.tensor([[5], [6], [0]], device=device), cache=cache).logits
    # rows 0 and 1 wrote: each has a copy of the page, row 2 keeps the first one
    assert cache.free_pages == cache.n_pages - 4
    table = cache.page_table.tolist()
    assert len({table[b][1] for b in range(3)}) == 3 and table[2][1] == before and table[0][0] == table[1][0] == table[2][0]
    cache.set_new([1, 1, 1])
    after = model(torch.tensor([[7], [8], [9]], device=device), cache=cache).logits
    assert cache.free_pages == cache.n_pages - 4   # (row 2 is alone on its page)
    for b, more in enumerate(([5, 7], [6, 8], [9])):
        if b < 2:
            want = model(torch.tensor([prompt + more[:1]], device=device)).logits[0, -1]
            assert (logits[b, 0] - want).abs().max() < TOL
        want = model(torch.tensor([prompt + more], device=device)).logits[0, -1]
        assert (after[b, 0] - want).abs().max() < TOL
    cache.release(0)
    assert cache.free_pages == cache.n_pages - 3   # (the shared page stays)
    cache.rewind([0, 16, 22])
    assert cache.free_pages == cache.n_pages - 2
    cache.reset()
    assert cache.free_pages == cache.n_pages and not any(cache._users)


def test_fork_books():
    cache = PagedKVCache([(1, 32)], 3, 64, "cpu", torch.float32, 16, n_pages=3)
    cache.set_new([20, 0, 0])
    cache.reserve(20)
    cache.advance(20)
    cache.fork(0, 1)
    for bad in ((0, 1), (0, 0), (1, 0)):
        with pytest.raises(ValueError, match="empty"):
            cache.fork(*bad)
    cache.fork(1, 2)
    cache.set_new([1, 1, 1])
    table = cache.page_table.clone()
    with pytest.raises(OutOfPages):       # two copies of the last page are needed, one page is left
        cache.reserve(1)
    assert torch.equal(cache.page_table, table) and cache.free_pages == 1
    cache.set_new([0, 1, 0])
    cache.v[0][cache.page_table[0, 1].item()] = 7.0
    cache.reserve(1)
    assert cache.free_pages == 0 and (cache.v[0][cache.page_table[1, 1].item()] == 7.0).all()
    cache.release(1)
    assert cache.free_pages == 1
    cache.release(0)
    assert cache.free_pages == 1          # (row 2 holds both)
    cache.release(2)
    assert cache.free_pages == 3


def test_keep_takes_what_a_pass_has_stored():
    cache = PagedKVCache([(1, 32)], 2, 64, "cpu", torch.float32, 16)
    cache.set_new([14, 0])
    cache.reserve(14)
    cache.advance(14)
    cache.set_new([5, 0])
    cache.set_tree([-1, 0, 0, 2, 1])
    cache.reserve(5)
    cache.advance(5)
    cache.fork(0, 1)      # (shares the nodes' pages too)
    path = torch.tensor([[0, 2, 3, -1, -1]] * 2, dtype=torch.int32)
    for counts in ([3, 3], [3, 2]):
        with pytest.raises(ValueError, match="stored"):
            cache.keep(path, torch.tensor(counts))
    assert cache.keep(path, torch.tensor([3, 0])) == [3, 0] and cache.seq_lens_host == [17, 14]
    cache.release(1)
    with pytest.raises(ValueError, match="stored"):
        cache.keep(path, torch.tensor([0, 1]))


class _NoLibrary:
    def __getattr__(self, name):
        raise AssertionError(f"{name}: the library was called for")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@torch.no_grad()
def test_trees_keep_to_torch_where_the_library_is_off(kind, monkeypatch):
    """SLEUTH_AMD_NO_HIP=1: passes of trees, what they keep, forks and their copies, the generators; nothing calls the library."""
    monkeypatch.setenv("SLEUTH_AMD_NO_HIP", "1")
    for name in ("lib", "host"):
        monkeypatch.setattr(ops, name, lambda: _NoLibrary())
    for paged in (False, True):
        model = make("cuda", **KINDS[kind])
        cache = (PagedKVCache if paged else KVCache).for_model(model, 1, 64, **({"page_size": 16} if paged else {}))
        prompt, tokens, parents = list(range(1, 16)), [3, 9, 4, 8], [-1, 0, 0, 2]
        model(torch.tensor([prompt], device="cuda"), cache=cache)
        cache.set_tree(parents)
        logits = model(torch.tensor([tokens], device="cuda"), cache=cache).logits[0]
        assert {blk.attn.last_path for blk in model.blocks} == {"torch"}
        for t in range(4):
            assert (logits[t] - _branch_logits(model, prompt, tokens, parents, t)).abs().max() < TOL
        cache.keep(torch.tensor([[0, 2, 3, -1]], dtype=torch.int32, device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda"))
        cache.set_tree(None)
        after = model(torch.tensor([[7]], device="cuda"), cache=cache).logits[0, -1]
        assert (after - model(torch.tensor([prompt + [3, 4, 8, 7]], device="cuda")).logits[0, -1]).abs().max() < TOL
    test_samples_of_a_prompt("cuda", "sinks" if kind == "sinks" else "full")
    want = generate(model, REPEATING, 20).new_ids
    for graph in (False, True):
        got = speculative_generate(model, REPEATING, 20, k=6, draft=_tree_of_truth(model, lambda i: i % 2 == 0), cuda_graph=graph,
                                   trees=graph)
        assert got.new_ids == want and got.stats["speculative"]["accepted"] >= 10


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", KINDS)
@torch.no_grad()
def test_a_static_tree_pass_in_torch(device, kind, monkeypatch):
    """A static cache's tree, whose mask is the device's to compute, is the tree of a cache whose length the host knows."""
    monkeypatch.setenv("SLEUTH_AMD_NO_HIP", "1")
    model = make(device, **KINDS[kind])
    rng = random.Random(5)
    T = 9
    for past in (0, 1, 12, 55):
        parents, tokens = make_parents(rng, T, "tree"), torch.tensor([[rng.randrange(64) for _ in range(T)]], device=device)
        logits = []
        for static in (False, True):
            cache = KVCache.for_model(model, 1, 64, tokens_per_step=T)
            if past:
                model(torch.tensor([[(3 * i) % 64 for i in range(past)]], device=device), cache=cache)
            cache.set_tree(parents)
            cache.static = static
            cache.pos_t.fill_(cache.pos)
            logits.append(model(tokens, cache=cache).logits)
        assert (logits[0] - logits[1]).abs().max() < TOL


@pytest.mark.parametrize("device", DEVICES)
def test_tree_masks_in_torch(device, monkeypatch):
    monkeypatch.setenv("SLEUTH_AMD_NO_HIP", "1")
    rng = random.Random(2)
    for T in (1, 63, 64, 65, 130):
        rows = [make_parents(rng, T, shape) for shape in ("tree", "chain", "forest")]
        tree = TokenTree(rows, 3, torch.device(device))
        assert tree.mask.tolist() == [mask_of(p, T)[0] for p in rows]
        assert tree.depth.tolist() == [mask_of(p, T)[1] for p in rows]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("paged", [False, True])
def test_caches_of_odd_heads_move_in_torch(device, paged):
    """Heads that are no 16-byte pieces run on the torch path, and so do their trees' moves and their forks' copies."""
    kw = dict(page_size=16) if paged else {}
    cache = (PagedKVCache if paged else KVCache)([(2, 6)], 2, 32, device, torch.float32, **kw)
    if paged:
        cache.set_new([6, 0])
        cache.reserve(6)
        cache.advance(6)
        cache.k[0][cache.page_table[0, 0].item()] = torch.arange(16., device=device)[:, None]
        cache.fork(0, 1)
        cache.set_new(None)
    else:
        cache.pos = 6
        cache.k[0].copy_(torch.arange(32., device=device)[:, None].expand(2, 2, 32, 6))
    cache.set_tree([-1, 0, 0, 2])
    if paged:
        cache.reserve(4)
    path = torch.tensor([[0, 2, 3, -1], [0, 1, -1, -1]], dtype=torch.int32, device=device)
    assert cache.keep(path, torch.tensor([3, 2], dtype=torch.int32, device=device)) == [3, 2]
    rows = [cache.row(0, b, 9)[0] if paged else cache.k[0][b] for b in range(2)]
    assert rows[0][0, 5:9, 0].tolist() == [5, 6, 8, 9] and rows[1][1, 5:8, 3].tolist() == [5, 6, 7]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("paged", [False, True])
def test_keep_takes_real_nodes_in_order(device, paged):
    """A path that names padding, what is no node of the tree, or nodes out of order is refused and nothing moves; nor are
    there nodes without a tree, behind a fork, or once other tokens are in."""
    if paged:
        cache = PagedKVCache([(1, 32)], 2, 64, device, torch.float32, 16)
        cache.set_new([4, 9])
        cache.reserve(9)
        cache.advance(9)
        cache.set_new([2, 5])
    else:
        cache = KVCache([(1, 32)], 2, 64, device, torch.float32)
        cache.set_lengths([4, 9])
    path = [[0, 1, -1, -1, -1], [0, 2, 3, -1, -1]]

    def keep(path, count):
        return cache.keep(torch.tensor(path, dtype=torch.int32, device=device), torch.tensor(count, dtype=torch.int32, device=device))

    with pytest.raises(ValueError, match="stored"):
        keep(path, [1, 0])                       # no tree yet
    cache.set_tree([-1, 0, 0, 2, 1])
    if paged:
        cache.reserve(5)
    for pool in (*cache.k, *cache.v):
        pool.copy_(torch.arange(pool.numel(), device=device).view_as(pool))
    cache.advance(5)
    before = [pool.clone() for pool in (*cache.k, *cache.v)]
    least = ([-1, 1, -1, -1, -1], [0, 5, -1, -1, -1], [0, 2 ** 31 - 1, -1, -1, -1], [1, 0, -1, -1, -1], [0, 0, -1, -1, -1])
    for bad in least + (([0, 4, -1, -1, -1],) if paged else ()):   # (the row's pass had two real tokens)
        with pytest.raises(ValueError, match="stored"):
            keep([bad, path[1]], [2, 3])
    with pytest.raises(ValueError, match="keep"):
        keep(path[:1], [1])
    with pytest.raises(ValueError, match="keep"):
        cache.keep(torch.tensor(path[0], dtype=torch.int32, device=device), torch.tensor([1, 0], dtype=torch.int32, device=device))
    assert all(torch.equal(x, y) for x, y in zip(before, (*cache.k, *cache.v))) and cache.seq_lens_host == [4, 9]
    cache.set_tree([-1, 0])                      # (the nodes are still the last pass's)
    cache.set_tree(None)
    assert keep(path, [2, 3]) == [2, 3] and cache.seq_lens_host == [6, 12]
    cache.advance(1)                             # a pass of plain tokens
    with pytest.raises(ValueError, match="stored"):
        keep(path, [1, 0])


def test_a_copy_that_fails_leaves_the_books():
    """Out of memory, say, while a shared page is copied: the rows still share it, and the next reserve copies it."""
    cache = PagedKVCache([(1, 32)], 3, 64, "cpu", torch.float32, 16)
    cache.set_new([20, 0, 0])
    cache.reserve(20)
    cache.advance(20)
    cache.fork(0, 1)
    cache.fork(0, 2)
    shared = cache.page_table[0, 1].item()
    cache.v[0][shared] = 5.0
    copy = cache._copy

    def fails(pages):
        raise torch.cuda.OutOfMemoryError("no memory")

    cache._copy = fails
    cache.set_new([20, 1, 0])                    # copies and new pages
    free, table = list(cache._free), [list(x) for x in cache._table]
    for _ in range(2):
        with pytest.raises(torch.cuda.OutOfMemoryError):
            cache.reserve(20)
        assert (cache._free, cache._table, cache.page_table.tolist()) == (free, table, table) and cache._users[shared] == 3
    cache._copy = copy
    cache.reserve(20)
    assert (cache._users[shared], cache.page_table[2, 1].item()) == (1, shared)
    assert len({cache._table[b][1] for b in range(3)}) == 3
    assert all((cache.v[0][cache._table[b][1]] == 5.0).all() for b in range(3))
    cache.reset()
    assert sorted(cache._free) == list(range(cache.n_pages)) and not any(cache._users)


def test_a_forks_nodes_are_the_other_rows():
    """Nodes that lie in a shared page close up for the row whose pass stored them: a fork made since would keep what that
    has moved already."""
    cache = PagedKVCache([(1, 32)], 2, 64, "cpu", torch.float32, 16)
    cache.set_new([4, 0])
    cache.reserve(4)
    cache.advance(4)
    cache.set_new(None)
    cache.set_tree([-1, 0, 0, 2, 1])
    path = torch.tensor([[0, 2, 3, -1, -1], [0, 1, 4, -1, -1]], dtype=torch.int32)
    cache.release(1)
    cache.reserve(5)
    cache.release(1)
    cache.advance(5)
    cache.fork(0, 1)
    assert cache.keep(path, torch.tensor([3, 0])) == [3, 0]
    with pytest.raises(ValueError, match="stored"):
        cache.keep(path, torch.tensor([0, 3]))
    assert cache.seq_lens_host == [7, 4]
    cache.set_new([1, 0])                        # a pass that row 1 sits out
    cache.reserve(1)
    cache.set_new(None)
    with pytest.raises(ValueError, match="stored"):
        cache.keep(path, torch.tensor([0, 3]))
    cache.reserve(5)                             # row 1 gets pages of its own, and a pass
    cache.advance(5)
    assert cache.keep(path, torch.tensor([0, 3])) == [0, 3]


@pytest.mark.gpu
@torch.no_grad()
def test_a_recorded_tree_keeps_its_size():
    model = make("cuda")
    dec = GraphDecoder(model, 64, torch.float32, 3)
    model(torch.tensor([REPEATING], device="cuda"), cache=dec.cache)
    tokens = torch.tensor([3, 9, 4], device="cuda")
    for parents in ([-1, 0], [-1, 0, 0, 1]):
        with pytest.raises(ValueError, match="3 nodes"):
            dec.verify(tokens, parents)
    want = dec.verify(tokens, [-1, 0, 0]).clone()
    for parents in ([-1, 0], torch.tensor([-1, 0, 0, 1])):
        with pytest.raises(ValueError, match="3 nodes"):
            dec.verify(tokens, parents)
    assert torch.equal(dec.verify(tokens, [-1, 0, 0]), want)


@pytest.mark.gpu
@torch.no_grad()
def test_a_refused_tree_is_not_set():
    model = make("cuda")
    dec = GraphDecoder(model, 16, torch.float32, 3)
    model(torch.tensor([REPEATING[:12]], device="cuda"), cache=dec.cache)
    tokens = torch.tensor([3, 9, 4], device="cuda")
    dec.verify(tokens, [-1, 0, 0])
    dec.cache.keep(torch.tensor([[0, 1, -1]], dtype=torch.int32, device="cuda"), torch.tensor([2], dtype=torch.int32, device="cuda"))
    dec.cache.set_tree(None)
    with pytest.raises(ValueError, match="full"):
        dec.verify(tokens, [-1, 0, 0])
    assert dec.cache.tree is None
    model(torch.tensor([[5]], device="cuda"), cache=dec.cache)
    assert dec.cache.pos == 15


@pytest.mark.parametrize("device", DEVICES)
@torch.no_grad()
def test_trees_over_forked_rows(device):
    """Two rows that share a prompt verify a tree each: the nodes go to pages of their own."""
    model = make(device)
    cache = PagedKVCache.for_model(model, 2, 64, page_size=16)
    prompt = list(range(2, 16))
    cache.set_new([14, 0])
    model(torch.tensor([prompt, [0] * 14], device=device), cache=cache)
    cache.fork(0, 1)
    cache.set_new(None)
    parents = [-1, 0, 0, 2, 1]
    tokens = [[1, 2, 3, 4, 5], [6, 7, 8, 9, 10]]
    cache.set_tree(parents)
    logits = model(torch.tensor(tokens, device=device), cache=cache).logits
    for b in range(2):
        for t in range(5):
            assert (logits[b, t] - _branch_logits(model, prompt, tokens[b], parents, t)).abs().max() < TOL
    path = torch.tensor([[0, 2, 3, -1, -1], [0, 1, 4, -1, -1]], dtype=torch.int32, device=device)
    cache.keep(path, torch.tensor([3, 3], dtype=torch.int32, device=device))
    cache.set_tree(None)
    after = model(torch.tensor([[11], [12]], device=device), cache=cache).logits
    for b, branch in enumerate(([1, 3, 4, 11], [6, 7, 10, 12])):
        want = model(torch.tensor([prompt + branch], device=device)).logits[0, -1]
        assert (after[b, 0] - want).abs().max() < TOL


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["full", "sinks"])
def test_samples_of_a_prompt(device, kind):
    model = make(device, **KINDS[kind])
    prompts = [REPEATING, [1, 2, 3], list(range(40))]
    alone = [generate(model, p, 10).new_ids for p in prompts]
    got = generate_batch(model, prompts, 10, chunk=7, page_size=16, samples=3)
    assert [r.new_ids for r in got] == [x for x in alone for _ in range(3)]
    assert [r.prompt_ids for r in got] == [p for p in prompts for _ in range(3)]
    many = generate_batch(model, prompts, 10, temperature=1.5, seed=1, chunk=7, page_size=16, samples=4)
    assert len({tuple(r.new_ids) for r in many}) > 6
    # the prompt's pages are shared: fewer in use than rows of their own would take
    single = generate_batch(model, [p for p in prompts for _ in range(4)], 10, temperature=1.5, seed=1, page_size=16)
    assert many[0].stats["most_pages"] < single[0].stats["most_pages"] or kind == "sinks"
    stop = alone[0][0]
    ended = generate_batch(model, prompts[:1], 10, stop_ids={stop}, page_size=16, samples=2)
    assert [r.stop_reason for r in ended] == ["stop_token"] * 2
    with pytest.raises(ValueError):
        generate_batch(model, prompts, samples=0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_16_bit_models(dtype):
    """The module's 16-bit path runs trees on the kernels, near the branch's own pass (two layers of 16-bit activations: a few
    steps of the type of logits of size ten)."""
    model = make("cuda", dtype, d_model=128, head_size=64, init_std=0.05)
    cache = KVCache.for_model(model, 1, 64)
    with torch.no_grad():
        model(torch.tensor([REPEATING], device="cuda"), cache=cache)
        parents, tokens = [-1, 0, 0, 1, 2, 4], [3, 9, 4, 7, 1, 2]
        cache.set_tree(parents)
        logits = model(torch.tensor([tokens], device="cuda"), cache=cache).logits[0]
        assert model.blocks[0].attn.last_path == "hip-tree"
        for t in range(6):
            want = _branch_logits(model, REPEATING, tokens, parents, t)
            assert (logits[t] - want).abs().max() <= 16 * torch.finfo(dtype).eps * want.abs().max()
