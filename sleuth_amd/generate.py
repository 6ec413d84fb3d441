"""The callers the attention path has to serve: plain decoding, speculative
draft-then-verify, and graph-replayed decode steps.

generate()             the decode loop of sleuth/forge/infer/generate.py:49-136: the prompt's
                       prefill, then one token per step through the cache (greedy or
                       temperature sampling)
speculative_generate() draft-then-verify as in speculative.py:83-277: [pending] + k guesses in one
                       forward at offset cache.pos, the agreeing prefix kept by moving pos back (the
                       rewind the reference's keep() does); beyond the reference, drafts may be trees
                       (their accepted branch closes up in the cache) and a temperature's samples
generate_batch()       several prompts of different lengths at once over a paged cache: their chunks
                       of new tokens padded to one batch, then one token per step for the rows
                       still running; pages come back as rows end or leave every layer's sight;
                       several continuations of a prompt share its pages (PagedKVCache.fork)
GraphDecoder           decode/verify steps replayed from a HIP graph (the role of
                       cuda_graph.py:67-144), built for kernels that read the live length on
                       the device: the attention reads only the keys below pos_t + T, whatever
                       the graph was recorded at, so ONE graph per step size serves every
                       context length -- no length buckets, no re-recording as the context
                       grows, no masked reads of a bucket's unused tail.
Sampling policies beyond temperature act after attention and are out of scope.
"""

from __future__ import annotations

import weakref
from dataclasses import dataclass, field
from typing import Callable

import torch

from .kv_cache import KVCache
from .paged_cache import OutOfPages, PagedKVCache
from .tree import Drafts, TokenTree, verify


@dataclass
class GenerationResult:
    prompt_ids: list[int]
    new_ids: list[int]
    stop_reason: str
    stats: dict = field(default_factory=dict)


def _pick(logits: torch.Tensor, temperature: float, gen: torch.Generator) -> torch.Tensor:
    """Next token id(s) [n] from logits [n, vocab]: argmax, or a draw at `temperature`."""
    if temperature > 0:
        return torch.multinomial((logits.float() / temperature).softmax(-1), 1, generator=gen).view(-1)
    return logits.argmax(-1)


class GraphDecoder:
    """Batch-1 decode (`step`) or verify (`verify`) steps of `tokens_per_step` tokens,
    recorded into one HIP graph (torch.cuda.CUDAGraph is hipGraph on ROCm) on first use and
    replayed afterwards. The position lives in cache.pos_t on the device; the host copies the
    new token ids and the position into the graph's input buffers before each replay.
    Use `cache` for the prompt's prefill (an ordinary eager forward)."""

    def __init__(self, model, max_len: int, dtype: torch.dtype, tokens_per_step: int = 1):
        p = next(model.parameters())
        if p.device.type != "cuda":
            raise ValueError("graph decoding needs a model on the GPU")
        self.model, self.T = model, tokens_per_step
        self.cache = KVCache.for_model(model, 1, max_len, dtype, tokens_per_step)
        self._ids = torch.zeros(1, tokens_per_step, dtype=torch.long, device=p.device)
        self._graph: torch.cuda.CUDAGraph | None = None
        self._logits: torch.Tensor | None = None
        self._trees = False
        self.replays = 0

    @property
    def recorded(self) -> bool:
        return self._graph is not None

    def _pass(self) -> torch.Tensor:
        return self.model(self._ids, cache=self.cache).logits[0]

    def _record(self) -> None:
        # one eager pass first (on a side stream, as graph capture wants): first-use
        # self-checks, library workspaces and the fused projection weights are set up
        # outside the capture; it writes the same K/V the real step writes
        side = torch.cuda.Stream(self._ids.device)
        side.wait_stream(torch.cuda.current_stream(self._ids.device))
        with torch.cuda.stream(side):
            self._pass()
        torch.cuda.current_stream(self._ids.device).wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            self._logits = self._pass()
        self._graph = g

    def _room(self) -> None:
        if self.cache.pos + self.T > self.cache.max_len:
            raise ValueError(f"KV cache full ({self.cache.max_len} tokens)")

    @torch.no_grad()
    def _launch(self, tokens: torch.Tensor) -> torch.Tensor:
        c = self.cache
        self._room()
        self._ids.copy_(tokens.view(1, self.T))
        c.pos_t.fill_(c.pos)
        c.static = True
        try:
            if self._graph is None:
                self._record()
            self._graph.replay()
        finally:
            c.static = False
        self.replays += 1
        return self._logits

    def step(self, token: torch.Tensor) -> torch.Tensor:
        """Logits [1, vocab] of `token` at position cache.pos; the cache moves on by one.
        The result is the graph's output buffer: read it before the next replay."""
        if self.T != 1 or self._trees:
            raise ValueError("step() is for one token at a time; use verify()")
        logits = self._launch(token)
        self.cache.pos += 1
        return logits

    def verify(self, tokens: torch.Tensor, parents: list[int] | None = None) -> torch.Tensor:
        """Logits [T, vocab] of T tokens at positions cache.pos, ...; cache.pos stays (the
        caller sets it to what it keeps). parents: the tokens are the nodes of a drafted tree, for which
        this decoder then records (cache.keep says which nodes stand)."""
        if self._graph is not None and (parents is not None) != self._trees:
            raise ValueError("this decoder was recorded for " + ("trees" if self._trees else "chains"))
        if parents is not None and len(TokenTree._rows(parents, 1)[0]) != self.T:
            raise ValueError(f"this decoder takes trees of {self.T} nodes")   # (its graph reads their buffers)
        self._room()   # (what is refused leaves the cache's tree as it was)
        self.cache.set_tree(parents)
        self._trees = parents is not None
        return self._launch(tokens)


_decoders: "weakref.WeakKeyDictionary[torch.nn.Module, dict]" = weakref.WeakKeyDictionary()


def decoder_for(model, max_len: int, dtype: torch.dtype, tokens_per_step: int = 1, trees: bool = False) -> GraphDecoder:
    """The model's graph decoder for this context and step size (and for chains or trees), kept across
    calls (the graph is recorded once per model); its cache is rewound for the new prompt."""
    per_model = _decoders.setdefault(model, {})
    key = (max_len, tokens_per_step, dtype, trees)
    dec = per_model.get(key)
    if dec is None:
        dec = per_model[key] = GraphDecoder(model, max_len, dtype, tokens_per_step)
    dec.cache.reset()
    return dec


@torch.no_grad()
def generate(model, prompt_ids: list[int], max_new_tokens: int = 32, temperature: float = 0.0,
             stop_ids: set[int] | None = None, seed: int | None = None, cuda_graph: bool = False,
             cache_dtype: torch.dtype | None = None) -> GenerationResult:
    if not prompt_ids:
        raise ValueError("prompt must contain at least one token")
    p = next(model.parameters())
    max_len = model.cfg.max_seq_len
    gen = torch.Generator(device=p.device).manual_seed(seed or 0)
    dec = decoder_for(model, max_len, cache_dtype or p.dtype) if cuda_graph else None
    cache = dec.cache if dec is not None else KVCache.for_model(model, 1, max_len, cache_dtype or p.dtype)
    model.eval()
    logits = model(torch.tensor([prompt_ids], device=p.device), cache=cache).logits[:, -1]
    new: list[int] = []
    reason = "max_new_tokens"
    while max_new_tokens > 0:
        tok = _pick(logits, temperature, gen)
        new.append(int(tok.item()))
        if stop_ids and new[-1] in stop_ids:
            reason = "stop_token"
            break
        if len(new) == max_new_tokens:
            break
        if cache.pos >= max_len:
            reason = "context_full"
            break
        logits = dec.step(tok.view(1)) if dec is not None else model(tok.view(1, 1), cache=cache).logits[:, -1]
    stats = {"kv_cache_mb": round(cache.nbytes() / 1e6, 2)}
    if dec is not None:
        stats["graph_replays"] = dec.replays
    return GenerationResult(list(prompt_ids), new, reason, stats)


@torch.no_grad()
def generate_batch(model, prompts: list[list[int]], max_new_tokens: int = 32, temperature: float = 0.0,
                   stop_ids: set[int] | None = None, seed: int | None = None, chunk: int = 512, page_size: int = 64,
                   n_pages: int | None = None, cache_dtype: torch.dtype | None = None, samples: int = 1) -> list[GenerationResult]:
    """generate() for a batch of prompts of any lengths over a paged cache: every pass takes up to `chunk` tokens of
    each prompt that has some left (the batch is padded to the longest), then each running row decodes one token per
    pass. A row's pages come back when it ends, and, where every layer slides, as they leave the windows (the first
    cfg.sink_tokens positions stay). Where the pool is short, OutOfPages is raised with `results`: the finished rows', and
    the others' so far (stop_reason "out_of_pages").
    samples: continuations of each prompt (results in the prompts' order, a prompt's together): the prompt runs once, and its
    rows share its pages."""
    if not prompts or not all(prompts):
        raise ValueError("every prompt must contain at least one token")
    if chunk < 1 or samples < 1:
        raise ValueError("chunk and samples must be positive")
    cfg, dev = model.cfg, next(model.parameters()).device
    longest = max(map(len, prompts))
    if longest > cfg.max_seq_len:
        raise ValueError(f"sequence length {longest} exceeds max_seq_len {cfg.max_seq_len}")
    prompts = [p for p in prompts for _ in range(samples)]
    cache = PagedKVCache.for_model(model, len(prompts), cfg.max_seq_len, cache_dtype, page_size, n_pages)
    gen = torch.Generator(device=dev).manual_seed(seed or 0)
    specs = [cfg.attn_spec(i) for i in range(cfg.n_layers)]
    window = max(s.window for s in specs) if all(s.window for s in specs) else 0
    model.eval()
    # tokens that no pass has taken yet; a prompt's other rows wait for its first one
    left = [list(p) if b % samples == 0 else [] for b, p in enumerate(prompts)]
    results = [GenerationResult(list(p), [], "max_new_tokens") for p in prompts]
    running = [max_new_tokens > 0] * len(prompts)
    passes, most_pages = 0, 0
    while any(running):
        new = [min(len(x), chunk) if run else 0 for x, run in zip(left, running)]
        T = max(new)
        ids = torch.tensor([x[:n] + [0] * (T - n) for x, n in zip(left, new)], device=dev)
        cache.set_new(new)
        try:
            cache.reserve(T)
        except OutOfPages as e:
            for r, run in zip(results, running):
                r.stop_reason = "out_of_pages" if run else r.stop_reason
            e.results = _with_stats(results, cache, passes, most_pages)
            raise
        logits = model(ids, cache=cache).logits
        passes, most_pages = passes + 1, max(most_pages, cache.n_pages - cache.free_pages)
        first = list(range(len(new)))                 # the row whose logits a row draws from
        for b, n in enumerate(new):
            left[b] = left[b][n:]
            if samples > 1 and b % samples == 0 and n and not left[b] and not results[b].new_ids:
                for other in range(b + 1, b + samples):   # the prompt is in
                    cache.fork(b, other)
                    first[other] = b
        last = logits[torch.arange(len(new), device=dev), torch.tensor(new, device=dev).clamp(min=1) - 1]
        tokens = _pick(last if samples == 1 else last[torch.tensor(first, device=dev)], temperature, gen).tolist()
        for b, n in enumerate(new):
            if not (n or first[b] != b) or left[b]:
                continue                              # not running, or more of its prompt to come
            r = results[b]
            r.new_ids.append(tokens[b])
            if stop_ids and tokens[b] in stop_ids:
                r.stop_reason = "stop_token"
            elif len(r.new_ids) == max_new_tokens:
                r.stop_reason = "max_new_tokens"
            elif cache.seq_lens_host[b] >= cfg.max_seq_len:
                r.stop_reason = "context_full"
            else:
                left[b] = [tokens[b]]
                continue
            running[b] = False
            cache.release(b)
        if window:
            cache.release_unseen(window, cfg.sink_tokens)
    return _with_stats(results, cache, passes, most_pages)


def _with_stats(results, cache, passes: int, most_pages: int) -> list[GenerationResult]:
    for r in results:
        r.stats = {"kv_cache_mb": round(cache.nbytes() / 1e6, 2), "passes": passes, "most_pages": most_pages}
    return results


def ngram_draft(max_ngram: int = 3) -> Callable[[list[int], int], list[int]]:
    """Prompt-lookup drafter: the tokens that followed the latest earlier occurrence of
    the longest suffix n-gram (n <= max_ngram)."""
    def draft(ids: list[int], k: int) -> list[int]:
        for n in range(min(max_ngram, len(ids) - 1), 0, -1):
            tail = ids[-n:]
            for start in range(len(ids) - n - 1, -1, -1):
                if ids[start:start + n] == tail:
                    return ids[start + n:start + n + k]
        return []
    return draft


def ngram_tree_draft(max_ngram: int = 3, branches: int = 3) -> Callable[[list[int], int], Drafts]:
    """ngram_draft with what followed several earlier occurrences: up to `branches` of them, the latest first, as one tree of at
    most k tokens (what they begin with alike is drafted once)."""
    def draft(ids: list[int], k: int) -> Drafts:
        for n in range(min(max_ngram, len(ids) - 1), 0, -1):
            tail = ids[-n:]
            found = [s + n for s in range(len(ids) - n - 1, -1, -1) if ids[s:s + n] == tail][:min(branches, k)]
            if not found:
                continue
            tokens, parents, known = [], [], {}
            for left, start in zip(range(len(found) - 1, -1, -1), found):
                most, at = k - left * (k // len(found)), -1      # the others' shares stay
                for t in ids[start:start + k]:
                    if (at, t) not in known:
                        if len(tokens) >= most:
                            break
                        known[at, t] = len(tokens)
                        tokens.append(t)
                        parents.append(at)
                    at = known[at, t]
            return Drafts(tokens, parents)
        return Drafts([])
    return draft


@torch.no_grad()
def speculative_generate(model, prompt_ids: list[int], max_new_tokens: int = 32, k: int = 4,
                         draft: Callable[[list[int], int], list[int] | Drafts] | None = None,
                         cuda_graph: bool = False, cache_dtype: torch.dtype | None = None, temperature: float = 0.0,
                         seed: int | None = None, trees: bool = False) -> GenerationResult:
    """Draft-then-verify: each round runs [pending] + guesses in one forward at offset cache.pos (T = 1 + k) and keeps
    what stands: greedily the longest agreeing prefix (pos is rewound), at a temperature what the target would have sampled
    (tree.verify; the drafts count as not drawn). draft(ids, k) gives a list, a chain of guesses, or Drafts, a tree of them,
    whose accepted branch closes up in the cache. trees: with cuda_graph, record the passes for trees (a chain is one); a graph
    for chains leaves a tree's round to an eager pass. A tree's nodes see other slots than a decode's tokens would, so its sums have
    another order: its logits are a decode's to rounding, not bit for bit."""
    draft = draft or ngram_draft()
    p = next(model.parameters())
    max_len = model.cfg.max_seq_len
    dtype = cache_dtype or p.dtype
    dec = decoder_for(model, max_len, dtype, tokens_per_step=k + 1, trees=trees) if cuda_graph else None
    cache = dec.cache if dec is not None else KVCache.for_model(model, 1, max_len, dtype)
    gen = torch.Generator(device=p.device).manual_seed(seed or 0)
    model.eval()
    logits = model(torch.tensor([prompt_ids], device=p.device), cache=cache).logits[0, -1]
    ids = list(prompt_ids) + [int(_pick(logits[None], temperature, gen))]
    new = ids[len(prompt_ids):]
    stats = {"forwards": 0, "drafted": 0, "accepted": 0}
    while len(new) < max_new_tokens:
        room = min(k, max_new_tokens - len(new), max_len - cache.pos - 1)
        if room < 0:
            break
        drafts = draft(ids, room) if room > 0 else []
        if not isinstance(drafts, Drafts):
            drafts = Drafts(list(drafts))
        if len(drafts.tokens) > room:
            drafts = Drafts(drafts.tokens[:room], None if drafts.parents is None else drafts.parents[:room])
        guess, start = drafts.tokens, cache.pos
        graph = dec is not None and start + k + 1 <= max_len and (trees or drafts.chain)
        tree = trees if graph else not drafts.chain
        pad = k - len(guess) if graph else 0                    # fixed T: pad the guesses (with nodes that nothing reaches)
        row = torch.tensor([[new[-1]] + guess + [new[-1]] * pad], device=p.device)
        parents = drafts.nodes() + [-1] * pad
        if graph:
            out = dec.verify(row[0], parents if tree else None)
        else:
            cache.set_tree(parents if tree else None)
            out = model(row, cache=cache).logits[0]
        if tree or temperature > 0:
            news, path, count = verify(out[None], row, parents=torch.tensor([parents], dtype=torch.int32, device=p.device),
                                       uniform=torch.rand(1, row.shape[1], generator=gen, device=p.device) if temperature > 0 else None,
                                       temperature=temperature)
            n_ok = int(count) - 1
            stands = news[0, :n_ok + 1].tolist()
            if tree:
                cache.keep(path, count)
                cache.set_tree(None)
            else:
                cache.pos = start + 1 + n_ok
        else:
            choice = out[:len(guess) + 1].argmax(-1).tolist()
            n_ok = next((i for i, (c, g) in enumerate(zip(choice, guess)) if c != g), len(guess))
            stands = guess[:n_ok] + [choice[n_ok]]
            cache.pos = start + 1 + n_ok          # keep the pending token and the accepted guesses
        stats["forwards"] += 1
        stats["drafted"] += len(guess)
        stats["accepted"] += n_ok
        for t in stands[:max_new_tokens - len(new)]:
            ids.append(t)
            new.append(t)
    res = GenerationResult(list(prompt_ids), new, "max_new_tokens", {"speculative": stats})
    if dec is not None:
        res.stats["graph_replays"] = dec.replays
    return res
