"""Plain references of appending to the paged cache and of sparse attention on it, in 64 bits on
the CPU, written from the definitions in the C header."""

from __future__ import annotations

import math

import torch

from paged_reference import quantized


def hadamard(x):
    """The Hadamard transform over the last axis (Sylvester's order) / sqrt(d), by halves."""
    d = x.shape[-1]

    def parts(y):
        if y.shape[-1] == 1:
            return y
        a, b = y.chunk(2, -1)
        return torch.cat((parts(a + b), parts(a - b)), -1)

    return parts(x) / math.sqrt(d)


def turned(x, pos, *, norm=None, eps=1e-6, cos=None, sin=None, offset=None, smooth=None, divide=False, rotate=False):
    """fp64 ``x [T, H, D]`` after norm, rotation of ``pos [T]``, offset, smoothing ``[H, D]`` and transform."""
    x = x.double().cpu()
    if norm is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * norm.double().cpu()
    if cos is not None:
        c, s = (y.double().cpu()[pos][:, None, : x.shape[-1] // 2] for y in (cos, sin))
        a, b = x.chunk(2, -1)
        x = torch.cat((a * c - b * s, b * c + a * s), -1)
    if offset is not None:
        x = x - offset.double().cpu()
    if smooth is not None:
        x = x / smooth.double().cpu() if divide else x * smooth.double().cpu()
    return hadamard(x) if rotate else x


def positions(lens, new):
    """Per packed new token (sequence, position)."""
    return [(b, length - n + i) for b, (length, n) in enumerate(zip(lens, new)) for i in range(n)]


def exponent(top: float) -> int:
    """The least e with top <= 127 * 2^e (0 for 0)."""
    if top == 0:
        return 0
    e = math.frexp(top)[1] - 8
    while top > math.ldexp(127.0, e):
        e += 1
    return e


def page_bounds(keys):
    """``(lo, hi, e)`` of a page's quantized keys ``[tokens, D]``: whole numbers in units of 2^e."""
    lo, hi = keys.double().amin(0), keys.double().amax(0)
    e = exponent(float(torch.maximum(lo.abs(), hi.abs()).max()))
    return torch.floor(lo * 2.0**-e), torch.ceil(hi * 2.0**-e), e


def select(q, keys, lens, new, page, count, first, last, missing=()):
    """``(selected [T, H, count], scores)`` from unquantized packed keys of all tokens; ``missing`` holds
    (sequence, column) pairs whose page the table does not hold."""
    keys = quantized(keys).double()
    starts = [sum(lens[:b]) for b in range(len(lens))]
    h = keys.shape[1]
    group, d = q.shape[1] // h, q.shape[2]
    out = torch.full((q.shape[0], h, count), -1, dtype=torch.int32)
    scores = torch.full((q.shape[0], h, count), -math.inf, dtype=torch.float64)
    known = {}
    for t, (b, pos) in enumerate(positions(lens, new)):
        if pos < 0:
            continue
        columns = pos // page + 1
        for j in range(h):
            if (b, j) not in known:
                parts = [page_bounds(part) for part in keys[starts[b] : starts[b] + lens[b], j].split(page)]
                lo, hi = (torch.stack([x[i] for x in parts]) for i in (0, 1))
                known[b, j] = lo, hi, torch.tensor([2.0 ** x[2] for x in parts], dtype=torch.float64)
            lo, hi, unit = (x[:columns] for x in known[b, j])
            row = q[t, j * group : (j + 1) * group].double().cpu()
            row = torch.where(row.isfinite(), row, torch.zeros_like(row))
            f = exponent(float(row.abs().max()))
            row = torch.round(row * 2.0**-f)
            score = (row.clamp(min=0) @ hi.T + row.clamp(max=0) @ lo.T).amax(0) * unit
            rank = score.clone()
            rank[:first] = rank[max(0, columns - last) :] = math.inf
            there = [c for c in range(columns) if (b, c) not in missing]
            best = torch.sort(rank[there], dim=0, descending=True, stable=True).indices[:count].tolist()
            taken = sorted(there[i] for i in best)
            out[t, j, : len(taken)] = torch.tensor(taken, dtype=torch.int32)
            scores[t, j, : len(taken)] = score[taken] * 2.0**f
    return out, scores


def attention(q, k, v, lens, new, page, selected, scale=None, missing=()):
    """``(O, A)`` in fp64 over the listed pages (each once), A = sum_k p_k |v_k|, from quantized packed keys
    and values."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    h, d = k.shape[1:]
    group = q.shape[1] // h
    scale = d**-0.5 if scale is None else scale
    starts = [sum(lens[:b]) for b in range(len(lens))]
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    for t, (b, pos) in enumerate(positions(lens, new)):
        for j in range(h):
            rows = []
            for c in sorted(set(selected[t, j].tolist())):
                if c >= 0 and (b, c) not in missing:
                    rows += range(starts[b] + c * page, starts[b] + min(pos + 1, c * page + page))
            if not rows:
                continue
            s = (q[t, j * group : (j + 1) * group] @ k[rows, j].T) * scale
            p = torch.softmax(s, -1)
            out[t, j * group : (j + 1) * group] = p @ v[rows, j]
            size[t, j * group : (j + 1) * group] = p @ v[rows, j].abs()
    return out, size
