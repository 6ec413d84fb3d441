"""KV cache with per-row lengths, laid out for the HIP attention kernels.

The attention module runs on any object with the reference's cache protocol
(sleuth/forge/infer/kv_cache.py:25-138) -- the host's own KVCache and StaticKVCache
included. This class is the cache of this package's callers (generate(), the graph
decoder, the benchmark); it speaks the same protocol and adds what the kernels can use:

  storage    every layer's K and V are views [B, K, max_len, hd] of ONE device allocation
             (the arena), so a whole model's cache is a single block of HBM;
  row lengths  each batch row has its own length (`set_lengths`, `seq_lens` int32 [B] on
             the device with a host mirror `seq_lens_host`); `pos` is the longest row, and
             setting it sets every row (what the speculative decoder's rewind does);
  static mode  (graph replays) the position is the device scalar `pos_t`; `positions`
             (pos_t + 0 .. tokens_per_step-1) is computed into a fixed buffer, so a
             captured graph recomputes it on every replay.

  trees  set_tree makes the next passes' tokens the nodes of drafted trees: a pass stores them behind the rows,
             whose lengths stay until keep says which nodes stand.

Protocol members: k, v, pos, max_len, update, advance, reset, nbytes, token_history,
for_model; static, pos_t, length, tokens_per_step, positions, attn_mask, new_step.
"""

from __future__ import annotations

import torch

from .tree import TokenTree


def _set_tree(cache, parents) -> None:
    """KVCache.set_tree and PagedKVCache.set_tree: the buffers of trees of one size are kept (recorded graphs read them)."""
    if parents is None:
        cache.tree = None
        return
    rows = TokenTree._rows(parents, cache.batch)
    tree = cache._trees.get(len(rows[0]))
    if tree is None:
        tree = cache._trees[len(rows[0])] = TokenTree(rows, cache.batch, cache.device)
    else:
        tree.set(rows)
    cache.tree = tree
    cache._set_nodes = tree.T


def _pieces(shapes: list[tuple[int, int]], dtype: torch.dtype) -> bool:
    """Whether heads of these shapes are the library's to move: whole pieces of 16 bytes, of its types."""
    return dtype in (torch.bfloat16, torch.float16, torch.float32) and all(hd * dtype.itemsize % 16 == 0 for _, hd in shapes)


def _native(cache) -> bool:
    """Whether moves within a cache are the library's: on the GPU, as for the attention (SLEUTH_AMD_NO_HIP=1 keeps to torch)."""
    from .attention import hip_disabled

    return cache.pieces and cache.device.type == "cuda" and not hip_disabled()


def _kept(cache, path: torch.Tensor, count: torch.Tensor, nodes: list[int]) -> list[int]:
    """The counts of a keep, whose paths must name each row's stored nodes (the first nodes[b] of its tree) in rising order."""
    B = cache.batch
    if path.dim() != 2 or path.shape[0] != B or count.shape != (B,) or path.device != count.device:
        raise ValueError(f"keep needs path [B, T] and count [B] of {B} rows on one device")
    both = torch.cat([count[:, None], path], 1).cpu()   # (one copy to the host)
    n = both[:, 0].tolist()
    if min(n) < 0 or max(n) > path.shape[1] or any(r + x > cache.max_len for r, x in zip(cache._rows, n)):
        raise ValueError(f"keep needs paths and counts of {B} rows that fit the cache")
    for row, x, most in zip(both[:, 1:max(n) + 1].tolist(), n, nodes):
        at = [-1] + row[:x]
        if at[-1] >= most or any(a >= b for a, b in zip(at, at[1:])):
            raise ValueError("keep is for nodes that the last pass has stored, in rising order")
    return n


class KVCache:
    def __init__(self, shapes: list[tuple[int, int]], batch: int, max_len: int,
                 device: torch.device | str, dtype: torch.dtype, tokens_per_step: int = 1):
        """shapes: (n_kv_heads, head_dim) of each layer."""
        if batch < 1 or max_len < 1 or tokens_per_step < 1:
            raise ValueError("batch, max_len and tokens_per_step must be positive")
        dev = torch.device(device)
        sizes = [batch * kv * max_len * hd for kv, hd in shapes]
        half = sum(sizes)
        self._arena = torch.zeros(2 * half, device=dev, dtype=dtype)   # [all K | all V]
        self.k, self.v, off = [], [], 0
        for (kv, hd), n in zip(shapes, sizes):
            self.k.append(self._arena[off:off + n].view(batch, kv, max_len, hd))
            self.v.append(self._arena[half + off:half + off + n].view(batch, kv, max_len, hd))
            off += n
        self.max_len, self.batch, self.device = max_len, batch, dev
        self.pieces = _pieces(shapes, dtype)
        self._rows = [0] * batch
        self._rows_dev: torch.Tensor | None = None   # device mirror, made when rows differ
        self._history: torch.Tensor | None = None
        self.tree: TokenTree | None = None
        # nodes of the tree that was set last and of the one that a pass ran last (a replayed pass is not seen here): keep's
        self._set_nodes = self._ran_nodes = 0
        self._trees: dict[int, TokenTree] = {}
        # static (graph) mode
        self.static = False
        self.length = max_len
        self.tokens_per_step = tokens_per_step
        self.pos_t = torch.zeros(1, dtype=torch.long, device=dev)
        self._steps = torch.arange(tokens_per_step, device=dev)
        self._pos_buf = torch.zeros(tokens_per_step, dtype=torch.long, device=dev)
        self._pass_pos: torch.Tensor | None = None
        self._pass_masks: dict[int, torch.Tensor] = {}

    @classmethod
    def for_model(cls, model, batch: int, max_len: int | None = None, dtype: torch.dtype | None = None,
                  tokens_per_step: int = 1) -> "KVCache":
        cfg = model.cfg
        p = next(model.parameters())
        specs = [cfg.attn_spec(i) for i in range(cfg.n_layers)]
        return cls([(s.kv_heads, s.head_dim) for s in specs], batch, max_len or cfg.max_seq_len,
                   p.device, dtype or p.dtype, tokens_per_step)

    # ------------------------------------------------------------------ lengths
    @property
    def pos(self) -> int:
        return max(self._rows)

    @pos.setter
    def pos(self, value: int) -> None:
        self._rows = [int(value)] * self.batch
        self._rows_dev = None

    def set_lengths(self, lengths: list[int]) -> None:
        """Give each row its own length (tokens already stored in it)."""
        rows = [int(n) for n in lengths]
        if len(rows) != self.batch:
            raise ValueError(f"{len(rows)} lengths for batch {self.batch}")
        if min(rows) < 0 or max(rows) > self.max_len:
            raise ValueError(f"lengths must be in [0, {self.max_len}]")
        self._rows = rows
        self._rows_dev = None

    @property
    def ragged(self) -> bool:
        return min(self._rows) != max(self._rows)

    @property
    def seq_lens_host(self) -> list[int]:
        return list(self._rows)

    @property
    def seq_lens(self) -> torch.Tensor:
        """int32 [B] row lengths on the device (what forge_kv_append / forge_attn_decode
        read as row_pos)."""
        if self._rows_dev is None:
            self._rows_dev = torch.tensor(self._rows, dtype=torch.int32).to(self.device)
        return self._rows_dev

    def _room_for(self, T: int) -> None:
        if self.pos + T > self.max_len:
            raise ValueError(f"KV cache full ({self.max_len} tokens)")

    # ------------------------------------------------------------------ protocol
    def update(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor):
        """Torch-path write of this step's K/V [B, K, T, hd]; returns the K/V views the
        step attends over: [:, :, :pos+T] (static mode: [:, :, :length])."""
        kc, vc = self.k[layer], self.v[layer]
        B, _, T, _ = k_new.shape
        if self.static:
            where = self.positions
            kc.index_copy_(2, where, k_new.to(kc.dtype))
            vc.index_copy_(2, where, v_new.to(vc.dtype))
            return kc[:, :, :self.length], vc[:, :, :self.length]
        self._room_for(T)
        # one scatter for all rows: row b's token t goes to position rows[b] + t
        cols = torch.tensor(self._rows, device=kc.device)[:, None] + torch.arange(T, device=kc.device)
        rows = torch.arange(B, device=kc.device)[:, None].expand(B, T)
        kc[rows, :, cols] = k_new.transpose(1, 2).to(kc.dtype)
        vc[rows, :, cols] = v_new.transpose(1, 2).to(vc.dtype)
        top = self.pos + T
        return kc[:, :, :top], vc[:, :, :top]

    def advance(self, n: int) -> None:
        """All layers have stored n more tokens per row. In static mode the caller owns
        the position (pos and pos_t), so nothing moves here; nor with a tree, whose nodes stand once keep says so."""
        if self.tree is not None:
            self._ran_nodes = self.tree.T
            return
        if self.static:
            return
        self._set_nodes = self._ran_nodes = 0
        self._rows = [r + n for r in self._rows]
        if self._rows_dev is not None:
            self._rows_dev.add_(n)

    # ------------------------------------------------------------------ trees
    def set_tree(self, parents) -> None:
        """The next passes' T tokens of each row are the nodes of a tree: parents [T] or [B, T], node 0 the row's last token,
        node t drafted behind node parents[t] < t (anything else: behind the row's tokens alone). None: tokens in a row again."""
        _set_tree(self, parents)

    def keep(self, path: torch.Tensor, count: torch.Tensor) -> list[int]:
        """Of the last pass's nodes, path[b, :count[b]] stand (tree.verify): their keys and values close up behind the row, which
        grows by count[b]. Returns the counts. ValueError, and nothing changed, where a path names what is no node of the row's
        tree, or does not rise. Once for each pass."""
        T = max(self._set_nodes, self._ran_nodes)
        n = _kept(self, path, count, [min(T, self.max_len - r) for r in self._rows])
        if _native(self):
            from . import ops

            where = dict(row_pos=self.seq_lens) if self.ragged else dict(pos=self.pos)
            ops.kv_compact(self.k, self.v, path, count, **where)
        else:
            for b, (r, x) in enumerate(zip(self._rows, n)):
                at = r + path[b, :x].long()
                for c in (*self.k, *self.v):
                    c[b, :, r:r + x] = c[b, :, at]
        self._rows = [r + x for r, x in zip(self._rows, n)]
        self._rows_dev = None
        return n

    def reset(self) -> None:
        self.pos = 0
        self.static = False
        self.tree = None
        self._set_nodes = self._ran_nodes = 0

    def nbytes(self) -> int:
        return self._arena.numel() * self._arena.element_size()

    def token_history(self, batch: int, device) -> torch.Tensor:
        """[batch, max_len] token ids by position, -1 where none yet (made on first use)."""
        if self._history is None:
            self._history = torch.full((batch, self.max_len), -1, dtype=torch.long, device=device)
        return self._history

    # ------------------------------------------------------------------ static mode
    @property
    def positions(self) -> torch.Tensor:
        """int64 [tokens_per_step]: this pass's token positions, pos_t + 0, 1, ..."""
        if self._pass_pos is None:
            torch.add(self.pos_t, self._steps, out=self._pos_buf)
            self._pass_pos = self._pos_buf
        return self._pass_pos

    def new_step(self, positions: torch.Tensor | None = None) -> None:
        """Start of a forward pass: positions are recomputed from pos_t (or taken as given)."""
        self._pass_pos = positions
        self._pass_masks = {}

    def attn_mask(self, window: int = 0) -> torch.Tensor:
        """[1, 1, T, length] bool, True where a query may see a key; one per window per pass."""
        mask = self._pass_masks.get(window)
        if mask is None:
            gap = self.positions[:, None] - torch.arange(self.length, device=self.device)[None, :]
            mask = gap >= 0
            if window:
                mask &= gap < window
            mask = self._pass_masks[window] = mask[None, None]
        return mask
