"""Performance cases of appending to the paged HiF4 key/value cache and of sparse attention on it.

Three operators of a serving step, in the order in which a step runs them:

- ``append`` (``ops.hif4_kv_append``): the new tokens' queries and keys get their norm, position
  rotation, smoothing and Hadamard transform; the keys and values go to 4-bit pages. The new
  tokens are read back (``ops.hif4_kv_read``), so that what was stored is an output;
- ``select`` (``ops.hif4_key_bounds``, ``ops.hif4_select_pages``): the bounds of the pages that
  the step wrote to are made anew, then every new token picks the pages to attend to (columns of
  the table, and their scores);
- ``attend`` (``ops.hif4_sparse_attention``): the attention of every new token over the tokens of
  its pages.

``run`` computes them with the library's kernels where ``own`` is true, else in elementary
torch operations.

A ragged batch is described the same way everywhere: ``cu [B + 1]`` bounds each sequence's
new tokens in the packed token axis, ``lens [B]`` are the sequence lengths that include
them (new token i of n stands at position len - n + i) and ``table [B, columns]`` holds the
pages of each sequence, -1 where it has none.

A page holds, for K and then V and per kv head, blocks of 16 tokens of 592 * NG bytes (NG =
head_dim / 64 groups of a row): the codes (a nibble n = 8 + m for the element m / 4, two to
a byte, the lower channel in the low half), the exponents (2 bits per 4 channels) and one
E6M2 scale byte per group; value = (n - 8) / 4 * 2^exponent * scale. ``_places`` gives the
byte order. A page's bounds are, per kv head, the least and the greatest key of each channel in
8 bits (rounded outward) and the exponent they share: 2 * head_dim + 16 bytes, the
exponent behind the codes. A page's score is the greatest that a query of those bounds can
reach: the sum over the channels of max(q low, q high), the greatest of the kv head's query
heads, with q in 8 bits too.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

PACKAGE = str(Path(__file__).resolve().parents[1] / "faquant-public_b200")
EPS = 1e-6
FIRST, LAST = 1, 2  # pages that are always taken: the context's first and the token's last ones


# ------------------------------------------------------------------ cases
def listed():
    def append(name, heads, kv_heads, dim, page, batch, context, tokens, dtype="bf16", norm=True, rotate=False,
               smooth=False, spread=False, mixed=False):
        return {"name": name, "kind": "append", "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
                "batch": batch, "context": context, "tokens": tokens, "dtype": dtype, "norm": norm, "rotate": rotate,
                "smooth": smooth, "spread": spread, "mixed": mixed}

    def sparse(kind, name, heads, kv_heads, dim, page, batch, context, tokens, count, spread=False, mixed=False):
        return {"name": name, "kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
                "batch": batch, "context": context, "tokens": tokens, "count": count, "spread": spread, "mixed": mixed}

    return [
        # one user, one decode step (Qwen3-8B heads): latency
        append("append, one token", 32, 8, 128, 64, 1, 1000, 1),
        # a decode step of a batch whose keys are rotated by a Hadamard matrix before they are quantized
        append("append, a step of 64", 32, 8, 128, 16, 64, 4096, 1, rotate=True, spread=True),
        # a prompt (Qwen3-32B heads), the deployed transform: norm, rotation, smoothing, Hadamard
        append("append, a prompt", 64, 8, 128, 64, 1, 8192, 8192, rotate=True, smooth=True),
        # prompts, decoding and idle users mixed; heads of 64 channels without a norm, fp32 projections
        append("append, mixed, heads of 64", 16, 4, 64, 32, 6, 6000, 700, dtype="fp32", norm=False, spread=True,
               mixed=True),
        # one user with a long context, one decode step: 2048 of 32768 tokens
        sparse("select", "select, one user", 32, 8, 128, 64, 1, 32768, 1, 32),
        # a served batch at very different lengths, small pages: at most 1024 tokens each
        sparse("select", "select, ragged batch", 32, 8, 128, 16, 32, 16000, 1, 64, spread=True),
        # a chunk of a long prompt (Qwen3-32B heads)
        sparse("select", "select, prompt chunk", 64, 8, 128, 64, 1, 32768, 512, 32),
        # verification of seven drafts and the last token for sixteen users, heads of 64
        sparse("select", "select, drafts", 16, 4, 64, 32, 16, 8192, 8, 24, spread=True),
        # the attention of the same steps
        sparse("attend", "sparse, one user", 32, 8, 128, 64, 1, 32768, 1, 32),
        sparse("attend", "sparse, ragged batch", 32, 8, 128, 16, 32, 16000, 1, 64, spread=True),
        sparse("attend", "sparse, prompt chunk", 64, 8, 128, 64, 1, 32768, 512, 32),
        # a step that mixes users in their prompts, decoding and idle; heads of 64 channels
        sparse("attend", "sparse, mixed, heads of 64", 16, 4, 64, 32, 6, 6000, 300, 24, spread=True, mixed=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("append", "select", "attend"))
    page = rng.choice((16, 32, 64, 128))
    dim = rng.choice((64, 128, 128))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 8))
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page}
    if kind == "append":
        batch = _log(rng, 1, 64)
        context = _log(rng, 1, 120000 // batch)
        tokens = min(_log(rng, 1, context), 8192 // batch) if rng.random() < 0.5 else 1
        return case | {"batch": batch, "context": context, "tokens": tokens,
                       "dtype": rng.choice(("bf16", "bf16", "fp32")), "norm": rng.random() < 0.7,
                       "rotate": rng.random() < 0.5, "smooth": rng.random() < 0.3, "spread": rng.random() < 0.7,
                       "mixed": rng.random() < 0.4}
    batch = _log(rng, 1, 48)
    tokens = _log(rng, 1, max(2, 500 // batch)) if rng.random() < 0.6 else 1
    context = _log(rng, tokens, max(tokens + 1, min(32768, 32 * 16000 // batch)))
    count = rng.randint(3, max(4, 2048 // page))
    return case | {"batch": batch, "context": context, "tokens": tokens, "count": count,
                   "spread": rng.random() < 0.7, "mixed": rng.random() < 0.4}


def _batch(case):
    """(lengths, new tokens) of the case's sequences; the first one is the longest."""
    rng = random.Random("%(kind)s %(batch)d %(context)d %(tokens)d" % (case | {"kind": ""}))
    lens = [case["context"]] * case["batch"]
    new = [min(case["tokens"], case["context"])] * case["batch"]
    for b in range(1, case["batch"]):
        if case["spread"]:
            lens[b] = _log(rng, 1, case["context"])
        if case["mixed"]:  # prompts, decoding, idle
            new[b] = rng.choice((0, 1, 1, rng.randint(1, max(1, case["tokens"]))))
        new[b] = min(new[b], lens[b])
    return lens, new


def work(case):
    lens, new = _batch(case)
    total, heads, h, d, page = sum(new), case["heads"], case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "append":
        size = 4 if case["dtype"] == "fp32" else 2
        row = 2 * h * d  # values of a token in the cache: written, read back in bf16
        each = heads * d * (size + 2) + row * (size + 0.578125 + 0.578125 + 2) + 4 * d
        return {"bytes": total * each, "flops": total * (heads + h) * d * (24 if case["rotate"] else 10)}
    # pages that a new token sees: its own and those before it
    seen = [[(length - n + i) // page + 1 for i in range(n)] for length, n in zip(lens, new)]
    if case["kind"] == "select":
        pages = sum(s[-1] for s in seen if s)
        fresh = sum(s[-1] - s[0] + 1 for s in seen if s)  # pages written to
        return {"bytes": pages * h * (2 * d + 1) + fresh * h * page * d * 0.578125 + total * (heads * d * 2 + h * case["count"] * 4),
                "flops": sum(map(sum, seen)) * heads * d * 2}
    taken = [[min(c, case["count"]) for c in s] for s in seen]
    pages = sum(min(s[-1], sum(c)) for s, c in zip(seen, taken) if s)  # no page need be read twice
    return {"bytes": pages * h * page * 2 * d * 0.578125 + total * (heads * d * 4 + h * case["count"] * 4),
            "flops": sum(map(sum, taken)) * page * heads * d * 4}


# ------------------------------------------------------------------ HiF4 pages in torch
def _quantize(x):
    """HiF4 (three scale levels) of ``x [T, H, D]`` in fp32: codes n, exponents, scale bytes."""
    t, h, d = x.shape
    x = x.float().reshape(t, h, d // 64, 16, 4)
    mag = x.abs()
    m3 = mag.amax(-1)  # per 4 channels
    m2 = m3.reshape(t, h, d // 64, 8, 2).amax(-1)  # per 8
    m1 = m2.amax(-1)  # per 64
    s = (m1 * 0.142578125).bfloat16().float().clamp(2.0**-48, 49152.0)
    bits = s.view(torch.int32)
    bits = (bits + 0x000FFFFF + ((bits >> 21) & 1)) & ~0x1FFFFF  # two mantissa bits, ties to even
    s = bits.view(torch.float32)
    rec = (1.0 / s).bfloat16().float()
    lv2 = (m2 * rec[..., None] >= 4.0).float().repeat_interleave(2, -1)
    lv3 = (m3 * rec[..., None] * torch.exp2(-lv2) >= 2.0).float()
    e = lv2 + lv3
    q = mag * (rec[..., None] * torch.exp2(-e))[..., None]
    m = torch.floor(q * 4.0 + 0.5).clamp(max=7.0)
    n = (8.0 + torch.where(x < 0, -m, m)).to(torch.uint8).reshape(t, h, d)
    scale = ((bits >> 21) - ((127 - 48) << 2)).to(torch.uint8)
    return n, e.to(torch.uint8), scale


def _to_bytes(n, e, scale):
    """One token's bytes in a canonical order: codes, exponents, scales."""
    t, h, d = n.shape
    codes = n[..., 0::2] | (n[..., 1::2] << 4)
    e = e.reshape(t, h, d // 64, 8, 2).to(torch.int32)  # sub-block of 8, quad
    shift = 2 * torch.arange(8, device=n.device, dtype=torch.int32)
    half = (e << shift[:, None]).sum(3, dtype=torch.int32)  # [T, H, group, quad], 16 bits
    ebytes = torch.stack((half & 255, half >> 8), -1).to(torch.uint8).reshape(t, h, d // 16)
    return torch.cat((codes, ebytes, scale), -1)


def _from_bytes(raw, d):
    """The fp32 values ``[T, H, D]`` of canonical bytes ``[T, H, 37 D / 64]``."""
    t, h, _ = raw.shape
    g = d // 64
    codes, ebytes, scale = raw[..., : d // 2], raw[..., d // 2 : d // 2 + d // 16], raw[..., d // 2 + d // 16 :]
    n = torch.stack((codes & 15, codes >> 4), -1).reshape(t, h, g, 8, 2, 4)
    half = ebytes.reshape(t, h, g, 1, 2, 2).to(torch.int32)
    half = half[..., 0] | (half[..., 1] << 8)  # [T, H, g, 1, quad]
    shift = 2 * torch.arange(8, device=raw.device, dtype=torch.int32)
    e = (half >> shift[:, None]) & 3  # [T, H, g, 8, quad]
    s = ((scale.to(torch.int32) << 21) + (79 << 23)).view(torch.float32)
    step = (0.25 * s)[..., None, None] * torch.exp2(e.float())
    return ((n.float() - 8.0) * step[..., None]).reshape(t, h, d)


def _places(case, pages, table, seq, pos):
    """Byte offsets ``[2, T, H, bytes]`` in ``pages`` of the tokens' canonical bytes (K, V)."""
    g, page, dev = case["dim"] // 64, case["page"], pages.device
    block = 592 * g
    r = pos % 16
    group = torch.arange(g, device=dev)[:, None, None]
    sub, byte = torch.arange(8, device=dev)[:, None], torch.arange(4, device=dev)
    quad, two = torch.arange(2, device=dev)[:, None], torch.arange(2, device=dev)
    k_code = (sub // 2 * 8 * g + 8 * group + 4 * (sub % 2) + byte).reshape(-1)
    k_exp = (512 * g + 4 * group + 2 * quad + two).reshape(-1)
    pair = (r // 2)[:, None, None, None]
    v_code = (sub ^ 2 * (pair % 4)) * 8 * g + 8 * group + 4 * (byte // 2) + byte % 2  # chunks swizzled by the pair
    v_code = v_code.reshape(len(r), 32 * g)
    v_exp = (512 * g + 8 * group + 4 * quad + two).reshape(-1)
    scale = 576 * g + torch.arange(g, device=dev)
    r = r[:, None]
    k = torch.cat((32 * g * r + k_code, 4 * g * r + k_exp, g * r + scale), 1)
    v = torch.cat((64 * g * (r // 2) + 2 * (r % 2) + v_code, 8 * g * (r // 2) + 2 * (r % 2) + v_exp, g * r + scale), 1)
    number = table[seq, pos // page].clamp(min=0).long()
    head = torch.arange(case["kv_heads"], device=dev)
    which = torch.arange(2, device=dev)[:, None, None]
    unit = (which * case["kv_heads"] + head) * (page // 16) + (pos % page // 16)[:, None]
    base = number[:, None] * pages.stride(0) + unit * block  # [2, T, H]
    return base[..., None] + torch.stack((k, v))[:, :, None, :]


def _put(case, pages, table, seq, pos, k, v):
    flat = pages.view(-1)
    at = _places(case, pages, table, seq, pos)
    flat[at[0]] = _to_bytes(*_quantize(k))
    flat[at[1]] = _to_bytes(*_quantize(v))


def _get(case, pages, table, seq, pos):
    flat = pages.view(-1)
    at = _places(case, pages, table, seq, pos)
    return _from_bytes(flat[at[0]], case["dim"]), _from_bytes(flat[at[1]], case["dim"])


# ------------------------------------------------------------------ bounds of the pages in torch
def _shared_exponent(top):
    """The least e with ``top <= 127 * 2^e`` (0 where ``top`` is 0), for fp32 ``top >= 0``."""
    fraction, e = torch.frexp(top)  # top = fraction * 2^e, fraction in [0.5, 1)
    return torch.where(top > 0, e - 7 + (fraction > 127 / 128).to(e.dtype), torch.zeros_like(e))


def _put_bounds(case, pages, bounds, table, lens, seq, col):
    """Bounds of page ``table[seq, col]`` of each (sequence, column), over the tokens below the length."""
    page = case["page"]
    pos = col[:, None] * page + torch.arange(page, device=pages.device)
    k, _ = _get(case, pages, table, seq.repeat_interleave(page), pos.reshape(-1))
    k = k.reshape(len(col), page, case["kv_heads"], case["dim"])
    live = (pos < lens[seq][:, None])[:, :, None, None]
    low = torch.where(live, k, torch.full_like(k, math.inf)).amin(1)
    high = torch.where(live, k, torch.full_like(k, -math.inf)).amax(1)
    e = _shared_exponent(torch.maximum(low.abs(), high.abs()).amax(-1))
    unit = torch.exp2(-e.float())[..., None]
    codes = torch.cat((torch.floor(low * unit), torch.ceil(high * unit)), -1).to(torch.int8).view(torch.uint8)
    tail = torch.zeros(*e.shape, 16, dtype=torch.uint8, device=pages.device)
    tail[..., 0] = e.to(torch.int8).view(torch.uint8)
    bounds[table[seq, col].long()] = torch.cat((codes, tail), -1)


def _best(scores, seen, count):
    """Per row of ``scores [T, H, columns]`` the columns to attend to among the first ``seen [T]``:
    the first FIRST, the last LAST and the best others (ties to the lowest column), ascending, -1 behind."""
    columns = scores.shape[-1]
    col = torch.arange(columns, device=scores.device)
    visible = col < seen[:, None, None]
    forced = visible & ((col < FIRST) | (col >= (seen - LAST)[:, None, None]))
    scores = torch.where(forced, torch.full_like(scores, math.inf), scores)
    scores = torch.where(visible, scores, torch.full_like(scores, -math.inf))
    order = torch.sort(scores, dim=-1, descending=True, stable=True).indices[..., :count]
    order = torch.where(order < seen[:, None, None], order, torch.full_like(order, columns)).sort(-1).values
    if order.shape[-1] < count:
        order = torch.nn.functional.pad(order, (0, count - order.shape[-1]), value=columns)
    return torch.where(order < columns, order, torch.full_like(order, -1)).to(torch.int32)


# ------------------------------------------------------------------ inputs
def _where(lens, new, device):
    """(sequence, position) of the last ``new`` tokens of every sequence, packed."""
    lens, new = (torch.tensor(v, device=device) for v in (lens, new))
    seq = torch.repeat_interleave(torch.arange(len(lens), device=device), new)
    start = torch.cumsum(new, 0) - new
    pos = torch.arange(int(new.sum()), device=device) - start[seq] + (lens - new)[seq]
    return seq, pos


def _cu(counts):
    out = [0]
    out.extend(counts)
    return torch.tensor(out, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()


def _pool(case, lens, g):
    """Pages and the table of sequences of such lengths."""
    page = case["page"]
    columns = -(-max(lens) // page)
    need = [-(-n // page) for n in lens]
    count = sum(need) + 3  # a pool with a few free pages, handed out in no order
    order = torch.randperm(count, generator=g, device="cuda")[: sum(need)].to(torch.int32)
    table = torch.full((len(lens), columns), -1, dtype=torch.int32, device="cuda")
    need = torch.tensor(need, device="cuda")
    table[torch.arange(columns, device="cuda") < need[:, None]] = order
    pages = torch.zeros((count, 2, case["kv_heads"], page // 16 * 592 * case["dim"] // 64), dtype=torch.uint8,
                        device="cuda")
    return pages, table


def _raw_append(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    lens, new = _batch(case)
    total, h, d = sum(new), case["kv_heads"], case["dim"]
    dtype = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    spread = torch.exp(0.3 * rand(1, 1, d))  # channels differ
    raw = {"q": (rand(total, case["heads"], d) * spread).to(dtype), "k": (rand(total, h, d) * spread).to(dtype),
           "v": (0.6 * rand(total, h, d)).to(dtype), "q_norm": None, "k_norm": None, "smooth": None}
    if case["norm"]:
        raw["q_norm"], raw["k_norm"] = ((1 + 0.2 * rand(d)).to(torch.bfloat16) for _ in range(2))
    if case["smooth"]:
        raw["smooth"] = torch.exp(0.2 * rand(d))
    # angles of far positions need 64 bits
    angle = torch.arange(max(lens), device="cuda", dtype=torch.float64)[:, None] * 1e6 ** (
        -torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    raw["cos"], raw["sin"] = angle.cos().float(), angle.sin().float()
    return lens, new, raw, g


def _raw_sparse(case, seed):
    """The keys and values of every cached token (packed by sequence), the new tokens among them,
    the queries, and per new token and kv head the pages to attend to."""
    g = torch.Generator("cuda").manual_seed(seed)
    lens, new = _batch(case)
    total, h, d, page = sum(lens), case["kv_heads"], case["dim"], case["page"]

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    k = (rand(total, h, d) * torch.exp(0.3 * rand(1, h, d))).to(torch.bfloat16)
    v = (0.6 * rand(total, h, d)).to(torch.bfloat16)
    q = (2.0 * rand(sum(new), case["heads"], d)).to(torch.bfloat16)
    selected = None
    if case["kind"] == "attend":  # neighbouring tokens mostly want the same pages
        seq, pos = _where(lens, new, "cuda")
        columns = -(-max(lens) // page)
        wish = rand(len(lens), h, columns)[seq] + 0.3 * rand(len(seq), h, columns)
        selected = _best(wish, pos // page + 1, case["count"])
    return lens, new, k, v, q, selected, g


def prepare(case, seed):
    if case["kind"] == "append":
        lens, new, raw, g = _raw_append(case, seed)
        pages, table = _pool(case, lens, g)
        d = case["dim"]
        bit = torch.arange(d, device="cuda")
        common = (bit[:, None] & bit)[..., None] >> torch.arange(7, device="cuda") & 1
        return raw | {"case": case, "pages": pages, "table": table, "cu": _cu(new), "total": sum(new),
                      "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
                      "hadamard": (1 - 2 * (common.sum(-1) % 2)).double() / math.sqrt(d)}
    lens, new, k, v, q, selected, g = _raw_sparse(case, seed)
    pages, table = _pool(case, lens, g)
    seq, pos = _where(lens, lens, "cuda")
    _put(case, pages, table, seq, pos, k, v)
    state = {"case": case, "pages": pages, "table": table, "cu": _cu(new), "q": q, "selected": selected, "total": sum(new),
             "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "max_new": max(new)}
    if case["kind"] == "select":
        state["bounds"] = torch.zeros(pages.shape[0], case["kv_heads"], 2 * case["dim"] + 16, dtype=torch.uint8,
                                      device="cuda")
        # those of the earlier steps' pages; the step makes its own
        seq, col = (table >= 0).nonzero(as_tuple=True)
        first = (torch.tensor(lens, device="cuda") - torch.tensor(new, device="cuda")) // case["page"]
        old = col < first[seq]
        _put_bounds(case, pages, state["bounds"], table, state["lens"], seq[old], col[old])
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        ops = _ops()
        case, page = state["case"], state["case"]["page"]
        batch = (state["table"], state["cu"], state["lens"])
        if kind == "append":
            q = ops.hif4_kv_append(state["q"], state["k"], state["v"], state["pages"], *batch, page_size=page,
                                   cos=state["cos"], sin=state["sin"], q_norm=state["q_norm"], k_norm=state["k_norm"],
                                   eps=EPS, smooth_scale=state["smooth"], rotate=case["rotate"])
            return q, *ops.hif4_kv_read(state["pages"], *batch, page_size=page, head_dim=case["dim"],
                                        total=state["total"])
        if kind == "select":
            ops.hif4_key_bounds(state["pages"], state["bounds"], *batch, page_size=page, total=state["total"])
            return ops.hif4_select_pages(state["q"], state["bounds"], *batch, page_size=page, count=case["count"],
                                         first=FIRST, last=LAST, want_scores=True)
        return ops.hif4_sparse_attention(state["q"], state["pages"], *batch, state["selected"], page_size=page)
    return {"append": _append, "select": _select, "attend": _attend}[kind](state)


def _ops():
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    from faquant_b200 import ops

    return ops


def _packed(state):
    """(sequence, position) of the new tokens, from the device's arrays."""
    cu, total = state["cu"], state["total"]
    new = (cu[1:] - cu[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(len(new), device=cu.device), new, output_size=total)
    index = torch.arange(total, device=cu.device)
    return seq, index - cu[seq].long() + (state["lens"] - new)[seq].long()


def _turned(x, state, pos, norm, smooth):
    """Norm, position rotation, smoothing and Hadamard transform of ``x [T, H, D]`` in x's type."""
    half = state["case"]["dim"] // 2
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * norm.to(x.dtype)
    c, s = (state[name][pos][:, None].to(x.dtype) for name in ("cos", "sin"))
    a, b = x[..., :half], x[..., half:]
    x = torch.cat((a * c - b * s, b * c + a * s), -1)
    if smooth is not None:
        x = x * smooth
    return torch.matmul(x, state["hadamard"].to(x.dtype)) if state["case"]["rotate"] else x


def _append(state):
    seq, pos = _packed(state)
    smooth = state["smooth"]
    q = _turned(state["q"].float(), state, pos, state["q_norm"], smooth)
    # codes jump at their borders: keys in 64 bits, rounded once to the 32 that are quantized
    k = _turned(state["k"].double(), state, pos, state["k_norm"], None if smooth is None else 1 / smooth.double())
    _put(state["case"], state["pages"], state["table"], seq, pos, k.float(), state["v"])
    k, v = _get(state["case"], state["pages"], state["table"], seq, pos)
    return q.to(torch.bfloat16), k.to(torch.bfloat16), v.to(torch.bfloat16)


def _select(state):
    case, lens, page, h, d = state["case"], state["lens"].long(), state["case"]["page"], state["case"]["kv_heads"], state["case"]["dim"]
    seq, pos = _packed(state)
    group, columns = case["heads"] // h, state["table"].shape[1]
    _put_bounds(case, state["pages"], state["bounds"], state["table"], lens, seq, pos // page)
    # whole numbers below 2^24: exact in fp32 in any order
    q = state["q"].float().reshape(-1, h, group, d)
    e = _shared_exponent(q.abs().amax((-1, -2))).float()[..., None]
    q = torch.round(q * torch.exp2(-e)[..., None])
    b = len(lens)
    slot = torch.arange(len(seq), device=q.device) - state["cu"][seq].long()
    padded = torch.zeros(b, state["max_new"], h, group, d, device=q.device)
    padded[seq, slot] = q
    padded = padded.permute(0, 2, 1, 3, 4).reshape(b, h, -1, d)
    rows = state["bounds"][state["table"].clamp(min=0).long()].permute(0, 2, 1, 3)  # [B, H, columns, bytes]
    low, high = (rows[..., i * d : i * d + d].contiguous().view(torch.int8).float().mT for i in (0, 1))
    unit = torch.exp2(rows[..., 2 * d].contiguous().view(torch.int8).float())
    scores = torch.matmul(padded.clamp(min=0), high) + torch.matmul(padded.clamp(max=0), low)
    scores = scores.reshape(b, h, -1, group, columns).amax(3) * unit[:, :, None]
    scores = scores.permute(0, 2, 1, 3)[seq, slot]
    selected = _best(scores, pos // page + 1, case["count"])
    scores = torch.gather(scores, -1, selected.clamp(min=0).long()) * torch.exp2(e)
    return selected, torch.where(selected < 0, torch.full_like(scores, -math.inf), scores)


def _attend(state):
    case, q, selected = state["case"], state["q"], state["selected"].long()
    page, h, d, b = case["page"], case["kv_heads"], case["dim"], state["table"].shape[0]
    group, columns = case["heads"] // h, state["table"].shape[1]
    seq, pos = _packed(state)
    every = torch.arange(b * columns * page, device=q.device)
    k, v = _get(case, state["pages"], state["table"], every // (columns * page), every % (columns * page))
    k, v = (x.reshape(b, columns, page, h, d) for x in (k, v))
    at = (seq[:, None, None], selected.clamp(min=0), slice(None), torch.arange(h, device=q.device)[:, None])
    q = q.float().reshape(-1, h, group, d)
    s = torch.matmul(q, k[at].flatten(2, 3).mT).mul_(d**-0.5)  # [T, H, group, count * page]
    place = selected[..., None] * page + torch.arange(page, device=q.device)
    hidden = (selected[..., None] < 0) | (place > pos[:, None, None, None])
    s.masked_fill_(hidden.flatten(2)[:, :, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s, v[at].flatten(2, 3))
    return torch.where(total > 0, o / total, torch.zeros_like(o)).reshape(len(q), case["heads"], d).to(torch.bfloat16)


# ------------------------------------------------------------------ in 64 bits
def _exact_hif4(x):
    """HiF4 values in fp64: the E6M2 scale from the group's maximum, the exponents by
    comparing with it, the element as the nearest quarter up to 7 / 4 (halves away from zero)."""
    t, h, d = x.shape
    x = x.double().reshape(t, h, d // 64, 64)

    def rounded(y, digits):  # to `digits` significant bits, ties to even
        e = torch.floor(torch.log2(y))
        e = e + (torch.exp2(e + 1) <= y).double() - (torch.exp2(e) > y).double()
        step = torch.exp2(e - (digits - 1))
        return torch.round(y / step) * step

    top = x.abs().amax(-1)
    start = (top * 0.142578125).float().double()  # one fp32 product, then bf16
    s = rounded(start.clamp(min=2.0**-100), 8).clamp(2.0**-48, 49152.0)
    s = rounded(s, 3)
    rec = rounded((1.0 / s).float().double(), 8)
    # |x| <= 24 significant bits; the products round to fp32 as the definition says
    eight = (x.abs().reshape(t, h, -1, 8, 8).amax(-1) * rec[..., None]).float().double()
    four = (x.abs().reshape(t, h, -1, 16, 4).amax(-1) * rec[..., None]).float().double()
    e2 = (eight >= 4).double().repeat_interleave(2, -1)
    e3 = (four >= 2 * torch.exp2(e2)).double()
    e = (e2 + e3).repeat_interleave(4, -1)
    m = ((x.abs() * rec[..., None]).float().double() * torch.exp2(2 - e) + 0.5).float().double().floor().clamp(max=7)
    return (torch.sign(x) * m / 4 * torch.exp2(e) * s[..., None]).reshape(t, h, d)


def _exact_transform(x):
    """The Hadamard transform over the last axis, by halves."""
    d = x.shape[-1]
    if d == 1:
        return x
    a, b = x[..., : d // 2], x[..., d // 2 :]
    return torch.cat((_exact_transform(a + b), _exact_transform(a - b)), -1)


def _exact_append(case, seed):
    lens, new, raw, _ = _raw_append(case, seed)
    _, pos = _where(lens, new, "cuda")
    turn = torch.complex(raw["cos"].double(), raw["sin"].double())[pos][:, None]
    out = []
    for name in ("q", "k"):
        x = raw[name].double()
        if case["norm"]:
            x = raw[name + "_norm"].double() * x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS)
        x = torch.complex(*x.chunk(2, -1)) * turn
        x = torch.cat((x.real, x.imag), -1)
        if case["smooth"]:
            x = x * raw["smooth"].double() if name == "q" else x / raw["smooth"].double()
        out.append(_exact_transform(x) / math.sqrt(case["dim"]) if case["rotate"] else x)
    return out[0], _exact_hif4(out[1].float()), _exact_hif4(raw["v"])


def _exact_exponent(top):
    e = torch.ceil(torch.log2(top / 127))
    e = e + (top > 127 * torch.exp2(e)).double() - (top <= 127 * torch.exp2(e - 1)).double()
    return torch.where(top > 0, e, torch.zeros_like(e))


def _exact_select(case, seed):
    """The scores of the selected pages: whole numbers times powers of two."""
    lens, new, k, _, q, _, _ = _raw_sparse(case, seed)
    page, h, d, count = case["page"], case["kv_heads"], case["dim"], case["count"]
    out, at = [], 0
    for key, length, n in zip(torch.split(k, lens), lens, new):
        if not n:
            continue
        key = _exact_hif4(key)
        columns = -(-length // page)
        key = torch.cat((key, key[-1:].expand(columns * page - length, h, d))).reshape(columns, page, h, d)
        low, high = key.amin(1), key.amax(1)
        unit = torch.exp2(_exact_exponent(torch.maximum(-low, high).amax(-1)))[..., None]
        low, high = torch.floor(low / unit) * unit, torch.ceil(high / unit) * unit
        row = q[at : at + n].double().reshape(n, h, -1, d)
        unit = torch.exp2(_exact_exponent(row.abs().amax((-1, -2))))[..., None, None]
        row = torch.round(row / unit) * unit
        scores = torch.einsum("nhgd,chd->nhgc", row.clamp(min=0), high) + torch.einsum("nhgd,chd->nhgc", row.clamp(max=0), low)
        scores = scores.amax(2)
        for i in range(n):
            seen = (length - n + i) // page + 1
            mine = scores[i, :, :seen]
            rank = mine.clone()
            rank[:, :FIRST] = math.inf
            rank[:, max(0, seen - LAST) :] = math.inf
            taken = torch.argsort(-rank, dim=1, stable=True)[:, :count].sort(1).values
            full = torch.full((h, count), -math.inf, dtype=torch.float64, device=q.device)
            full[:, : taken.shape[1]] = mine.gather(1, taken)
            out.append(full)
        at += n
    return None, torch.stack(out)


def exact(case, seed):
    if case["kind"] == "select":
        return _exact_select(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, seed)
    lens, new, k, v, q, selected, _ = _raw_sparse(case, seed)
    group, d, page = case["heads"] // case["kv_heads"], case["dim"], case["page"]
    out, at = torch.zeros(q.shape, dtype=torch.float64, device=q.device), 0
    for key, value, length, n in zip(torch.split(k, lens), torch.split(v, lens), lens, new):
        if not n:
            continue
        key, value = _exact_hif4(key), _exact_hif4(value)
        place = torch.arange(length, device=q.device)
        for head in range(case["kv_heads"]):
            listed_pages = torch.zeros(n, -(-length // page) + 1, dtype=torch.bool, device=q.device)
            listed_pages.scatter_(1, selected[at : at + n, head].long() % listed_pages.shape[1], True)  # -1: the spare one
            seen = listed_pages[:, place // page] & (place <= torch.arange(length - n, length, device=q.device)[:, None])
            for row in range(head * group, head * group + group):
                s = q[at : at + n, row].double() @ key[:, head].T / math.sqrt(d)
                out[at : at + n, row] = torch.softmax(s.masked_fill(~seen, -math.inf), -1) @ value[:, head]
        at += n
    return out
