"""A paged KV cache: memory by need instead of max_len per row, for batches whose rows grow differently.

The reference's caches (sleuth/forge/infer/kv_cache.py:25-138) hold max_len positions for every row. Here each layer's
K and V are pools [n_pages, K, page_size, hd]; position s of row b is slot s % page_size of page
page_table[b, s // page_size], the same page of every layer's pools. Pages are handed out as rows grow (reserve), and
come back when a row ends (release) or when no layer can see them any more (release_unseen: every layer slides, and
keeps its first tokens). The table and the lengths live on the device in fixed buffers, so a recorded graph of the
operators or of the layers sees them change. What is the host's to say stays outside of it: reserve before a replay,
advance after it (both refuse to be recorded).

It speaks the cache protocol of the package's callers (pos, max_len, advance, seq_lens, seq_lens_host, update; `ragged`
is always true, `static` never; pos is read only, since rows differ: rewind takes each row's length) and adds `paged`,
page_table, new_lens, reserve, top, bound and row, which the attention module uses (ops.kv_append_paged, ops.attn_paged).
"""

from __future__ import annotations

import torch


class OutOfPages(ValueError):
    """The pool has fewer free pages than a pass needs. generate_batch adds `results`, what its rows have so far."""

    results: list | None = None


class PagedKVCache:
    paged = True
    ragged = True
    static = False

    def __init__(self, shapes: list[tuple[int, int]], batch: int, max_len: int, device: torch.device | str,
                 dtype: torch.dtype, page_size: int = 64, n_pages: int | None = None):
        """shapes: (n_kv_heads, head_dim) of each layer; n_pages: pages of each pool (default: max_len for every row)."""
        if batch < 1 or max_len < 1:
            raise ValueError("batch and max_len must be positive")
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two of at least 16")
        per_row = -(-max_len // page_size)
        n = per_row * batch if n_pages is None else n_pages
        if n < 1:
            raise ValueError("n_pages must be positive")
        dev = torch.device(device)
        self.batch, self.max_len, self.device, self.page_size, self.n_pages = batch, max_len, dev, page_size, n
        sizes = [n * kv * page_size * hd for kv, hd in shapes]
        half = sum(sizes)
        self._arena = torch.zeros(2 * half, device=dev, dtype=dtype)   # [all K | all V]
        self.k, self.v, off = [], [], 0
        for (kv, hd), size in zip(shapes, sizes):
            self.k.append(self._arena[off:off + size].view(n, kv, page_size, hd))
            self.v.append(self._arena[half + off:half + off + size].view(n, kv, page_size, hd))
            off += size
        self.page_table = torch.full((batch, per_row), -1, dtype=torch.int32, device=dev)
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=dev)
        self._new_buf = torch.zeros(batch, dtype=torch.int32, device=dev)
        self._table = [[-1] * per_row for _ in range(batch)]
        self._free = list(range(n - 1, -1, -1))
        self._rows = [0] * batch
        self._least = [0] * batch     # rows cannot be rewound below this: pages that it would see were given back
        self._new: list[int] | None = None

    @classmethod
    def for_model(cls, model, batch: int, max_len: int | None = None, dtype: torch.dtype | None = None,
                  page_size: int = 64, n_pages: int | None = None) -> "PagedKVCache":
        cfg = model.cfg
        p = next(model.parameters())
        specs = [cfg.attn_spec(i) for i in range(cfg.n_layers)]
        return cls([(s.kv_heads, s.head_dim) for s in specs], batch, max_len or cfg.max_seq_len, p.device,
                   dtype or p.dtype, page_size, n_pages)

    # ------------------------------------------------------------------ lengths
    @property
    def pos(self) -> int:
        """The longest row."""
        return max(self._rows)

    @property
    def seq_lens_host(self) -> list[int]:
        return list(self._rows)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def set_new(self, new_lens: list[int] | None) -> None:
        """How many of the next pass's tokens are real in each row (a padded batch); None: all of them. It holds until
        it is set again."""
        if new_lens is not None:
            new_lens = [int(n) for n in new_lens]
            if len(new_lens) != self.batch or min(new_lens) < 0:
                raise ValueError(f"new_lens needs {self.batch} counts that are not negative")
            self._new_buf.copy_(torch.tensor(new_lens, dtype=torch.int32))
        self._new = new_lens

    @property
    def new_lens(self) -> torch.Tensor | None:
        """int32 [batch] on the device for ops.kv_append_paged and attn_paged, or None."""
        return None if self._new is None else self._new_buf

    def new_tokens(self, T: int) -> list[int]:
        """Each row's real tokens in a pass of T."""
        if self._new is None:
            return [T] * self.batch
        return [min(n, T) for n in self._new]

    def top(self, T: int) -> int:
        """The longest row once a pass of T tokens is in."""
        return max(1, max(r + n for r, n in zip(self._rows, self.new_tokens(T))))

    def bound(self, T: int) -> int:
        """max_kv_len of a pass of T tokens: top(T), or, for a graph that is being recorded, all that the cache holds: its
        replays see longer rows."""
        return self.max_len if self._recording() else self.top(T)

    def _recording(self) -> bool:
        return self.device.type == "cuda" and torch.cuda.is_current_stream_capturing()

    # ------------------------------------------------------------------ pages
    def reserve(self, T: int) -> None:
        """Pages for the next pass's real tokens (every layer of a pass may call it: the first one acts). Raises
        ValueError where a row would pass max_len, OutOfPages where the pool has no page left; nothing is handed out then."""
        P = self.page_size
        need = []
        for b, (r, n) in enumerate(zip(self._rows, self.new_tokens(T))):
            if r + n > self.max_len:
                raise ValueError(f"KV cache full ({self.max_len} tokens)")
            if n:
                need += [(b, j) for j in range(r // P, (r + n - 1) // P + 1) if self._table[b][j] < 0]
        if not need:
            return
        if self._recording():
            raise RuntimeError("reserve a paged cache's pages before recording a graph")
        if len(need) > len(self._free):
            raise OutOfPages(f"KV cache out of pages ({len(need)} needed, {len(self._free)} of {self.n_pages} free)")
        for b, j in need:
            self._table[b][j] = self._free.pop()
        self._put_table()

    def release(self, row: int) -> None:
        """The row ends: its pages come back and its length is 0."""
        self._give_back([(row, j) for j, page in enumerate(self._table[row]) if page >= 0])
        self._rows[row] = self._least[row] = 0
        self.seq_lens[row] = 0

    def rewind(self, lengths: list[int]) -> None:
        """Each row keeps its first lengths[b] tokens (after a verify step: what was accepted); pages behind its new end
        come back. ValueError, and nothing changed, where a length is not the row's or one before it, or where release_unseen
        has given back a page that a row of that length would see."""
        lengths = [int(n) for n in lengths]
        if len(lengths) != self.batch or any(not 0 <= n <= r for n, r in zip(lengths, self._rows)):
            raise ValueError(f"rewind needs {self.batch} lengths of at most {self._rows}")
        for b, (n, r) in enumerate(zip(lengths, self._rows)):
            if n < r and n < self._least[b]:
                raise ValueError(f"row {b} cannot go back to {n} tokens: pages that it would see were given back")
        self._give_back([(b, j) for b, n in enumerate(lengths) for j in range(-(-n // self.page_size), len(self._table[b]))
                         if self._table[b][j] >= 0])
        self._rows = lengths
        self.seq_lens.copy_(torch.tensor(lengths, dtype=torch.int32))

    def release_unseen(self, window: int, sinks: int = 0) -> int:
        """Give back the pages that no later query sees where every layer has a window of at most `window` keys and
        keeps at most the first `sinks` tokens. Returns how many came back."""
        if window < 1 or sinks < 0:
            raise ValueError("release_unseen needs a window")
        P = self.page_size
        gone = [(b, j) for b, r in enumerate(self._rows) for j in range(-(-sinks // P), max(0, r - window + 1) // P)
                if self._table[b][j] >= 0]
        self._give_back(gone)
        for b, j in gone:
            self._least[b] = max(self._least[b], (j + 1) * P + window - 1)
        return len(gone)

    def _give_back(self, at: list[tuple[int, int]]) -> None:
        for b, j in at:
            self._free.append(self._table[b][j])
            self._table[b][j] = -1
        if at:
            self._put_table()

    def _put_table(self) -> None:
        self.page_table.copy_(torch.tensor(self._table, dtype=torch.int32))

    # ------------------------------------------------------------------ protocol
    def update(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor) -> None:
        """Torch-path write of this pass's K/V [B, K, T, hd] (real tokens only)."""
        T, P = k_new.shape[2], self.page_size
        self.reserve(T)
        rows, cols = [], []
        for b, n in enumerate(self.new_tokens(T)):
            rows += [b] * n
            cols += range(n)
        if not rows:
            return
        b = torch.tensor(rows, device=self.device)
        t = torch.tensor(cols, device=self.device)
        pos = self.seq_lens.long()[b] + t
        page = self.page_table.long()[b, pos // P]
        self.k[layer][page, :, pos % P] = k_new[b, :, t].to(self.k[layer].dtype)
        self.v[layer][page, :, pos % P] = v_new[b, :, t].to(self.v[layer].dtype)

    def row(self, layer: int, b: int, n: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """The first n positions of a row, gathered: k, v [K, n, hd] (zeros where there is no page) and which positions
        have one, bool [n]."""
        ids = self.page_table[b, :-(-n // self.page_size)].long()
        held = (ids >= 0).repeat_interleave(self.page_size)[:n]

        def dense(pool):
            x = pool[ids.clamp(min=0)].transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])[:, :n]
            return x.masked_fill(~held[None, :, None], 0)

        return dense(self.k[layer]), dense(self.v[layer]), held

    def advance(self, n: int) -> None:
        """All layers have stored this pass's tokens."""
        if self._recording():
            raise RuntimeError("advance a paged cache outside of a recorded graph: its lengths are the host's too")
        new = self.new_tokens(n)
        self._rows = [r + x for r, x in zip(self._rows, new)]
        if self._new is None:
            self.seq_lens.add_(n)
        else:
            self.seq_lens.add_(self._new_buf.clamp(max=n))

    def reset(self) -> None:
        for b in range(self.batch):
            self.release(b)
        self._new = None

    def nbytes(self) -> int:
        return self._arena.numel() * self._arena.element_size()
