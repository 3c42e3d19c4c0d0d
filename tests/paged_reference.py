"""Plain references of the paged K/V cache, its attention and draft verification: 64-bit
softmax attention, whole-number verification in Python integers, and a small pool to run on."""

from __future__ import annotations

from fractions import Fraction

import numpy as np
import torch

from oracle import hif4 as oh


class Pool:
    """A pool of pages with a table of randomly ordered pages for sequences of ``lens`` tokens."""

    def __init__(self, lens, kv_heads, head_dim, page_size, device, *, fill=0xA5, seed=0, spare=2, gap=0):
        from faquant_b200 import ops

        self.lens_host, self.kv_heads, self.d, self.page_size = list(lens), kv_heads, head_dim, page_size
        need = [-(-n // page_size) for n in lens]
        count = sum(need) + spare
        size = ops.hif4_page_bytes(kv_heads, head_dim, page_size)
        store = torch.full((count, size + gap), fill, dtype=torch.uint8, device=device)
        self.store, self.pages = store, store[:, :size]
        order = torch.randperm(count, generator=torch.Generator().manual_seed(seed)).tolist()
        table = np.full((len(lens), max(1, *need) + 1), -1, np.int32)
        for b, n in enumerate(need):
            table[b, :n] = [order.pop() for _ in range(n)]
        self.table = torch.tensor(table, device=device)
        self.lens = torch.tensor(self.lens_host, dtype=torch.int32, device=device)

    def cu(self, new):
        return torch.tensor(np.concatenate(([0], np.cumsum(new))), dtype=torch.int32, device=self.pages.device)

    def write(self, k, v, new=None, lens=None, **kw):
        from faquant_b200 import ops

        new = self.lens_host if new is None else new
        lens = self.lens if lens is None else torch.tensor(lens, dtype=torch.int32, device=self.pages.device)
        ops.hif4_kv_write(k, v, self.pages, self.table, self.cu(new), lens, page_size=self.page_size, **kw)

    def read(self, new=None, **kw):
        from faquant_b200 import ops

        new = self.lens_host if new is None else new
        return ops.hif4_kv_read(self.pages, self.table, self.cu(new), self.lens, page_size=self.page_size,
                                head_dim=self.d, total=int(sum(new)), **kw)

    def attend(self, q, new, max_len=0, **kw):
        from faquant_b200 import ops

        return ops.hif4_paged_attention(q, self.pages, self.table, self.cu(new), self.lens, page_size=self.page_size,
                                        max_new=max(new), max_len=max(max_len, *self.lens_host), **kw)


def quantized(x: torch.Tensor, levels="123") -> torch.Tensor:
    """The oracle's HiF4 values of ``x`` along its last axis, fp32 on the CPU."""
    return torch.from_numpy(oh.fake_quantize(x.float().cpu().numpy(), levels))


def attention(q, k, v, lens, new, scale=None):
    """``(O, A)`` in fp64: the attention of packed queries over packed cached keys/values (all
    tokens of every sequence), and A = sum_k p_k |v_k|, the size that rounding errors scale with."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    heads, d = q.shape[1:]
    group = heads // k.shape[1]
    scale = d**-0.5 if scale is None else scale
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    at = begin = 0
    for length, n in zip(lens, new):
        key = k[begin : begin + length].repeat_interleave(group, 1)
        value = v[begin : begin + length].repeat_interleave(group, 1)
        for i in range(n):
            seen = length - n + i + 1
            if seen > 0:
                s = torch.einsum("hd,khd->hk", q[at + i], key[:seen]) * scale
                p = torch.softmax(s, -1)
                out[at + i] = torch.einsum("hk,khd->hd", p, value[:seen])
                size[at + i] = torch.einsum("hk,khd->hd", p, value[:seen].abs())
        at += n
        begin += length
    return out, size


def _weights(row):
    """rint(2^40 r) of fp32 weights in [0, 1], exactly, ties to even."""
    return [round(Fraction(float(r)) * 2**40) for r in row]


def verify(draft, target, drafter, accept_u, sample_u, counts):
    """Draft verification token by token: fp32 for the products and differences, whole numbers
    for the sums, one fp64 product for the threshold."""
    b, k = draft.shape
    vocab = target.shape[-1]
    target = target.float().cpu().numpy()
    drafter = None if drafter is None else drafter.float().cpu().numpy()
    tokens, accepted = np.full((b, k + 1), -1, np.int64), np.zeros(b, np.int32)
    for i in range(b):
        n = 0
        while n < counts[i]:
            x = int(draft[i, n])
            if not 0 <= x < vocab:
                break
            q = np.float32(1.0) if drafter is None else drafter[i, n, x]
            if not np.float32(accept_u[i, n]) * q < target[i, n, x]:
                break
            tokens[i, n] = x
            n += 1
        accepted[i] = n
        left = target[i, n].copy()
        if n < counts[i]:
            if drafter is not None:
                left = left - drafter[i, n]
            elif 0 <= int(draft[i, n]) < vocab:
                left[int(draft[i, n])] = 0.0
        w = _weights(np.clip(left, 0.0, 1.0))
        if sum(w) == 0:
            w = _weights(np.clip(target[i, n], 0.0, 1.0))
        if sum(w) == 0:
            continue
        u = min(max(np.float32(sample_u[i]), np.float32(0.0)), np.float32(1.0 - 2.0**-24))
        limit, total = float(u) * float(sum(w)), 0
        for j, x in enumerate(w):
            total += x
            if float(total) > limit:
                tokens[i, n] = j
                break
    return tokens, accepted
