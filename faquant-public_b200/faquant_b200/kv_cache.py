"""A paged HiF4 K/V cache for the Qwen3 attention adapter and for serving loops.

The reference keeps a dequantized bf16 copy of K and V per attention module and appends one
token at a time to it (``simulated_flash_attention.py:243-289``). Here every layer's K and V
live in 4.625 bits per value, in pages that sequences of different lengths share a pool of; a
step writes any number of new tokens per sequence and attends to them in one call.

A step is: :meth:`PagedKVCache.extend` (host: pages for the new tokens), then per layer
:meth:`write` and :meth:`attend`. :meth:`truncate` takes tokens back (rejected drafts),
:meth:`read` returns a layer's keys and values in bf16 (the hand-off to a bf16 model).
``past_key_values=cache`` with ``faquant_attention_kernel = "paged"`` on the attention modules
runs a Hugging Face Qwen3 on it (``qwen3.attention_forward``); the first layer of a forward
call opens the step.

:meth:`append` stands for the steps between the projections and :meth:`write` too (per-head norm,
rotation of each token's position, Smooth-QK, Hadamard) and returns the attention's queries.

With ``sparse_pages`` the attention of a long context reads that many pages per token and kv head: the
first ones, the last ones, and those whose keys' bounds allow the greatest products
(``ops.hif4_select_pages``). It pays in steps that read hundreds of thousands of keys; below, the dense step is
faster, and exact. The bounds are kept beside the pages, 2 * head_dim + 16 bytes per page
and kv head, and made anew for the pages that a step writes to.

A step is not to be captured in a CUDA graph: :meth:`extend` makes the step's device arrays anew, and
:meth:`attend` gives the step's own lengths as bounds. What a graph needs -- arrays that stay in
their place, bounds of its last replay, one workspace -- the operators take (``ops.hif4_kv_write``,
``ops.hif4_paged_attention``), from a caller that keeps them.
"""

from __future__ import annotations

import torch

from . import ops


class PagedKVCache:
    """Pages, page tables and lengths of ``max_sequences`` sequences of at most
    ``max_length`` tokens on ``layers`` attention layers."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, *, max_sequences: int = 1, max_length: int,
                 num_pages: int | None = None, page_size: int = 64, device: torch.device | str = "cuda",
                 sparse_pages: int | None = None, sparse_first: int = 1, sparse_last: int = 2,
                 sparse_max_new: int | None = None) -> None:
        """``sparse_pages``: the pages that a token attends to per kv head, among them the
        ``sparse_first`` first and ``sparse_last`` last ones; None: all. Steps in which a sequence has more
        than ``sparse_max_new`` new tokens (prompts) attend to all pages all the same (None: no step does)."""
        if sparse_pages is not None and (sparse_first < 0 or sparse_last < 1 or sparse_first + sparse_last > sparse_pages):
            raise ValueError("sparse_pages must hold the first pages and the last ones, of which there is at least one")
        if layers < 1 or max_sequences < 1 or max_length < 1:
            raise ValueError("layers, max_sequences and max_length must be positive")
        columns = -(-max_length // page_size)
        if sparse_pages is not None and columns > 32768:
            raise ValueError("the selection of pages takes sequences of at most 32768 pages")
        self.layers, self.kv_heads, self.head_dim, self.page_size = layers, kv_heads, head_dim, page_size
        self.max_length, self.device = max_length, torch.device(device)
        num_pages = columns * max_sequences if num_pages is None else num_pages
        size = ops.hif4_page_bytes(kv_heads, head_dim, page_size)
        self.pages = torch.empty((layers, num_pages, 2, kv_heads, size // (2 * kv_heads)), dtype=torch.uint8,
                                 device=self.device)
        self.sparse_pages, self.sparse_first, self.sparse_last = sparse_pages, sparse_first, sparse_last
        self.sparse_max_new = sparse_max_new
        self.bounds = None
        if sparse_pages is not None:
            self.bounds = torch.zeros((layers, num_pages, kv_heads, ops.hif4_bounds_bytes(head_dim)), dtype=torch.uint8,
                                      device=self.device)
        self.table = torch.full((max_sequences, columns), -1, dtype=torch.int32, device=self.device)
        self._free = list(range(num_pages - 1, -1, -1))
        self._held: list[list[int]] = [[] for _ in range(max_sequences)]
        self.lengths = [0] * max_sequences  # of the sequences, with the open step's tokens
        self._new = [0] * max_sequences
        self._cu = self._lens = None

    @classmethod
    def for_model(cls, model, **kwargs) -> "PagedKVCache":
        """A cache with the shape of a Hugging Face decoder's attention layers."""
        config = model.config
        return cls(config.num_hidden_layers, config.num_key_value_heads, config.head_dim, **kwargs)

    # ---------------------------------------------------------------- host side of a step
    def extend(self, counts: list[int]) -> None:
        """Open a step with ``counts[b]`` new tokens for sequence b (0: it sits the step out)."""
        if len(counts) != len(self.lengths) or min(counts) < 0:
            raise ValueError("counts must hold a non-negative number of new tokens per sequence")
        need = []
        for b, n in enumerate(counts):
            if self.lengths[b] + n > self.max_length:
                raise ValueError(f"sequence {b} would pass max_length ({self.max_length} tokens)")
            need.append(-(-(self.lengths[b] + n) // self.page_size) - len(self._held[b]))
        if sum(max(0, k) for k in need) > len(self._free):
            raise RuntimeError("the page pool is exhausted")
        rows, cols, vals = [], [], []
        for b, (n, k) in enumerate(zip(counts, need)):
            for _ in range(max(0, k)):
                rows.append(b)
                cols.append(len(self._held[b]))
                vals.append(self._free.pop())
                self._held[b].append(vals[-1])
            self.lengths[b] += n
        self._new = list(counts)
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        # one copy for the step's arrays and the table's new entries
        host = torch.tensor(cu + self.lengths + rows + cols + vals, dtype=torch.int32)
        moved = host.to(self.device, non_blocking=True)
        a, b = len(cu), len(self.lengths)
        self._cu, self._lens = moved[:a], moved[a : a + b]
        if rows:
            r, c, v = moved[a + b :].reshape(3, -1)
            self.table[r.long(), c.long()] = v

    def truncate(self, lengths: list[int]) -> None:
        """Shorten the sequences to ``lengths``: their later tokens are forgotten, whole pages
        go back to the pool. Closes the step."""
        if len(lengths) != len(self.lengths) or any(not 0 <= n <= m for n, m in zip(lengths, self.lengths)):
            raise ValueError("lengths must be between 0 and the sequences' lengths")
        for b, n in enumerate(lengths):
            keep = -(-n // self.page_size)
            self._free.extend(reversed(self._held[b][keep:]))
            del self._held[b][keep:]
            self.lengths[b] = n
        self._new = [0] * len(lengths)
        self._cu = self._lens = None

    # ---------------------------------------------------------------- device side of a step
    def _open(self) -> None:
        if self._cu is None:
            raise RuntimeError("no step is open: call extend() first")

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Quantize and store the step's ``k``/``v [tokens, kv_heads, head_dim]`` of a layer."""
        self._open()
        if k.shape[0] != sum(self._new):
            raise ValueError(f"the step has {sum(self._new)} new tokens, got {k.shape[0]}")
        ops.hif4_kv_write(k, v, self.pages[layer], self.table, self._cu, self._lens, page_size=self.page_size,
                          levels=(ops.default_levels("k"), ops.default_levels("v")))
        self._refresh(layer)

    def append(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, **transform) -> torch.Tensor:
        """From the projections of the step's tokens, ``q [tokens, heads, head_dim]`` and ``k``/``v [tokens,
        kv_heads, head_dim]``, to the layer's cache and the queries of :meth:`attend`: norms, position
        rotation, smoothing and Hadamard transform as ``transform`` asks (``ops.hif4_kv_append``: ``cos``,
        ``sin``, ``q_norm``, ``k_norm``, ``eps``, ``rotate``, ``smooth_scale``, ``key_offset``, ``out``)."""
        self._open()
        if q.shape[0] != sum(self._new):
            raise ValueError(f"the step has {sum(self._new)} new tokens, got {q.shape[0]}")
        q = ops.hif4_kv_append(q, k, v, self.pages[layer], self.table, self._cu, self._lens, page_size=self.page_size,
                               levels=(ops.default_levels("k"), ops.default_levels("v")), **transform)
        self._refresh(layer)
        return q

    def _refresh(self, layer: int) -> None:
        """The bounds of the pages that the step wrote to."""
        if self.bounds is not None:
            ops.hif4_key_bounds(self.pages[layer], self.bounds[layer], self.table, self._cu, self._lens,
                                page_size=self.page_size, total=sum(self._new))

    def attend(self, layer: int, q: torch.Tensor, scale: float | None = None) -> torch.Tensor:
        """Attention of the step's ``q [tokens, heads, head_dim]`` over the layer's cache."""
        self._open()
        if q.shape[0] != sum(self._new):
            raise ValueError(f"the step has {sum(self._new)} new tokens, got {q.shape[0]}")
        lengths = [n for n, new in zip(self.lengths, self._new) if new]  # of those that take part
        max_new, max_len = max(self._new), max(lengths, default=0)
        # where no sequence has more pages than are taken, all of them are: the dense kernels'
        if self.sparse_pages is not None and max_len > self.sparse_pages * self.page_size and (
                self.sparse_max_new is None or max_new <= self.sparse_max_new):
            selected = ops.hif4_select_pages(q, self.bounds[layer], self.table, self._cu, self._lens,
                                             page_size=self.page_size, count=self.sparse_pages, first=self.sparse_first,
                                             last=self.sparse_last)
            return ops.hif4_sparse_attention(q, self.pages[layer], self.table, self._cu, self._lens, selected,
                                             page_size=self.page_size, scale=scale)
        return ops.hif4_paged_attention(q, self.pages[layer], self.table, self._cu, self._lens,
                                        page_size=self.page_size, max_new=max_new, max_len=max_len,
                                        total_len=sum(lengths), scale=scale)

    def read(self, layer: int, dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
        """The layer's whole cache dequantized, ``(k, v)`` each ``[sum(lengths), kv_heads, head_dim]``,
        packed by sequence."""
        cu = [0]
        for n in self.lengths:
            cu.append(cu[-1] + n)
        moved = torch.tensor(cu + self.lengths, dtype=torch.int32).to(self.device, non_blocking=True)
        return ops.hif4_kv_read(self.pages[layer], self.table, moved[: len(cu)], moved[len(cu) :],
                                page_size=self.page_size, head_dim=self.head_dim, total=cu[-1], dtype=dtype)

    def forward(self, layer: int, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                scale: float | None = None) -> torch.Tensor:
        """One layer of a model's forward call: ``query [B, H, n, D]``, ``key``/``value [B, Hkv,
        n, D]`` of B = max_sequences sequences; layer 0 opens the step. Returns ``[B, n, H, D]``."""
        b, heads, n, d = query.shape
        if layer == 0:
            if b != len(self.lengths):
                raise ValueError(f"the cache holds {len(self.lengths)} sequences, the batch {b}")
            self.extend([n] * b)

        def packed(t: torch.Tensor) -> torch.Tensor:
            return t.transpose(1, 2).reshape(b * n, t.shape[1], d)

        self.write(layer, packed(key), packed(value))
        return self.attend(layer, packed(query), scale).reshape(b, n, heads, d)

    # ---------------------------------------------------------------- what Hugging Face models ask of a cache
    def get_seq_length(self, layer_idx: int = 0) -> int:
        """Length of the sequences, which a rectangular batch has in common."""
        if len(set(self.lengths)) != 1:
            raise ValueError("the sequences have different lengths: pass position_ids to the model")
        return self.lengths[0]

    def get_mask_sizes(self, query_length: int, layer_idx: int = 0) -> tuple[int, int]:
        return max(self.lengths) + query_length, 0
