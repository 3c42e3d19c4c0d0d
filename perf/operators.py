"""Performance cases of the paged HiF4 key/value cache and of speculative decoding on it.

Four operators of a serving step: writing new tokens' K/V into 4-bit pages
(``ops.hif4_kv_write``), reading pages back as bf16 (``ops.hif4_kv_read``), the attention of a
chunk of new tokens over the pages (``ops.hif4_paged_attention``) and the verification of
drafted tokens (``ops.verify_drafts``). ``run`` computes them with the library's kernels
where ``own`` is true, else in elementary torch operations in fp32.

A ragged batch is described the same way everywhere: ``cu [B + 1]`` bounds each sequence's
new tokens in the packed token axis, ``lens [B]`` are the sequence lengths that include
them (new token i of n stands at position len - n + i) and ``table [B, columns]`` holds the
pages of each sequence, -1 where it has none.

A page holds, for K and then V and per kv head, blocks of 16 tokens of 592 * NG bytes (NG =
head_dim / 64 groups of a row): the codes (a nibble n = 8 + m for the element m / 4, two to
a byte, the lower channel in the low half), the exponents (2 bits per 4 channels) and one
E6M2 scale byte per group; value = (n - 8) / 4 * 2^exponent * scale. ``_places`` gives the
byte order.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

PACKAGE = str(Path(__file__).resolve().parents[1] / "faquant-public_b200")
FIXED_POINT = 2.0**40  # the unit of the residual weights in verify_drafts


# ------------------------------------------------------------------ cases
def listed():
    def attend(name, heads, kv_heads, dim, page, batch, context, tokens, spread=False, mixed=False):
        return {"name": name, "kind": "attend", "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
                "batch": batch, "context": context, "tokens": tokens, "spread": spread, "mixed": mixed}

    def cache(name, kv_heads, dim, page, batch, context, tokens, back, dtype="bf16", spread=False):
        return {"name": name, "kind": "cache", "kv_heads": kv_heads, "dim": dim, "page": page, "batch": batch,
                "context": context, "tokens": tokens, "back": back, "dtype": dtype, "spread": spread}

    def verify(name, batch, drafts, vocab, dtype, drafter, ragged=False):
        return {"name": name, "kind": "verify", "batch": batch, "drafts": drafts, "vocab": vocab, "dtype": dtype,
                "drafter": drafter, "ragged": ragged}

    return [
        # one user early in a conversation, one decode step (Qwen3-8B heads): latency
        attend("decode one, 1k", 32, 8, 128, 64, 1, 1000, 1),
        # one user with a long context, one decode step (Qwen3-8B heads)
        attend("decode one, 32k", 32, 8, 128, 64, 1, 32768, 1),
        # a served batch of users at very different lengths, one decode step, small pages
        attend("decode ragged batch", 32, 8, 128, 16, 32, 16000, 1, spread=True),
        # verification of seven drafts and the last token for sixteen users (Qwen3-8B heads)
        attend("drafts, batch of 16", 32, 8, 128, 32, 16, 8192, 8, spread=True),
        # a chunk of a long prompt (Qwen3-32B heads)
        attend("prompt chunk, 32k", 64, 8, 128, 64, 1, 32768, 512),
        # a step that mixes users in their prompts, decoding and idle; heads of 64 channels
        attend("mixed step, heads of 64", 16, 4, 64, 32, 6, 6000, 700, spread=True, mixed=True),
        # a decode step of a batch writes one token per user; the new rows are read back
        cache("cache, a step", 8, 128, 16, 64, 4096, 1, "new", spread=True),
        # a prompt is written and handed to a bf16 attention
        cache("cache, a prompt", 8, 128, 64, 1, 8192, 8192, "new"),
        # whole contexts leave the cache in bf16 (hand-off to a bf16 decode model); fp32 input
        cache("cache, contexts back", 8, 128, 64, 8, 20000, 3, "all", dtype="fp32", spread=True),
        # four drafts of one user, drafted by lookup in the context (no draft distribution)
        verify("verify one", 1, 4, 151936, "fp32", False),
        # seven drafts per user of a batch from a draft model
        verify("verify batch", 128, 7, 151936, "fp32", True, ragged=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "cache", "cache", "verify"))
    page = rng.choice((16, 32, 64, 128))
    dim = rng.choice((64, 128, 128))
    if kind == "attend":
        kv_heads = rng.choice((1, 2, 4, 8))
        heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 8))
        batch = _log(rng, 1, 48)
        tokens = _log(rng, 1, max(2, 600 // batch)) if rng.random() < 0.6 else 1
        # padded scores of the plain form and its cache stay below the largest listed case's
        most = min(32768, 512 * 32768 * 64 // (batch * tokens * heads), 32 * 16000 * 8 // (batch * kv_heads))
        context = _log(rng, tokens, max(tokens + 1, most))
        return {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "batch": batch,
                "context": context, "tokens": tokens, "spread": rng.random() < 0.7, "mixed": rng.random() < 0.4}
    if kind == "cache":
        kv_heads = rng.choice((1, 2, 4, 8))
        batch = _log(rng, 1, 64)
        context = _log(rng, 1, 160000 // batch)
        tokens = _log(rng, 1, context) if rng.random() < 0.5 else 1
        return {"kind": kind, "kv_heads": kv_heads, "dim": dim, "page": page, "batch": batch, "context": context,
                "tokens": tokens, "back": rng.choice(("new", "all")), "dtype": rng.choice(("bf16", "bf16", "fp32")),
                "spread": rng.random() < 0.7}
    return {"kind": kind, "batch": _log(rng, 1, 100), "drafts": rng.randint(1, 8), "vocab": _log(rng, 1000, 152000),
            "dtype": rng.choice(("fp32", "fp32", "bf16")), "drafter": rng.random() < 0.6, "ragged": rng.random() < 0.5}


def _batch(case):
    """(lengths, new tokens) of the case's sequences; the first one is the longest."""
    rng = random.Random("%(kind)s %(batch)d %(context)d %(tokens)d" % case)
    lens = [case["context"]] * case["batch"]
    new = [min(case["tokens"], case["context"])] * case["batch"]
    for b in range(1, case["batch"]):
        if case["spread"]:
            lens[b] = _log(rng, 1, case["context"])
        if case.get("mixed"):  # prompts, decoding, idle
            new[b] = rng.choice((0, 1, 1, rng.randint(1, max(1, case["tokens"]))))
        new[b] = min(new[b], lens[b])
    return lens, new


def work(case):
    if case["kind"] == "verify":
        size = 4 if case["dtype"] == "fp32" else 2
        rows = case["batch"] * case["vocab"] * size * (2 if case["drafter"] else 1)
        per = case["drafts"] * (size * 2 + 4 + 8) + 4 + 8 * (case["drafts"] + 1) + 4
        return {"bytes": rows + case["batch"] * per, "flops": 3 * case["batch"] * case["vocab"]}
    lens, new = _batch(case)
    row = 2 * case["kv_heads"] * case["dim"]  # values of a token in the cache
    if case["kind"] == "cache":
        back = sum(lens) if case["back"] == "all" else sum(new)
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": sum(new) * row * (size + 0.5625) + back * row * (0.5625 + 2), "flops": 10 * sum(new) * row}
    pairs = sum(n * (length - n) + n * (n + 1) // 2 for length, n in zip(lens, new))
    seen = sum(length for length, n in zip(lens, new) if n)
    return {"bytes": seen * row * 0.5625 + sum(new) * case["heads"] * case["dim"] * 4,
            "flops": 4 * case["dim"] * case["heads"] * pairs}


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


# ------------------------------------------------------------------ inputs
def _where(lens, new, device):
    """(sequence, position) of the last ``new`` tokens of every sequence, packed."""
    lens, new = (torch.tensor(v, device=device) for v in (lens, new))
    seq = torch.repeat_interleave(torch.arange(len(lens), device=device), new)
    start = torch.cumsum(new, 0) - new
    pos = torch.arange(int(new.sum()), device=device) - start[seq] + (lens - new)[seq]
    return seq, pos


def _raw(case, seed):
    """The keys and values of every cached token (packed by sequence), the new tokens
    among them, and the queries."""
    g = torch.Generator("cuda").manual_seed(seed)
    lens, new = _batch(case)
    total, h, d = sum(lens), case["kv_heads"], case["dim"]
    dtype = torch.float32 if case.get("dtype") == "fp32" else torch.bfloat16
    spread = torch.exp(0.3 * torch.randn(1, h, d, generator=g, device="cuda"))  # channels differ
    k = (torch.randn(total, h, d, generator=g, device="cuda") * spread).to(dtype)
    v = (torch.randn(total, h, d, generator=g, device="cuda") * 0.6).to(dtype)
    q = None
    if case["kind"] == "attend":
        q = (2.0 * torch.randn(sum(new), case["heads"], d, generator=g, device="cuda")).to(torch.bfloat16)
    return lens, new, k, v, q, g


def _cu(counts):
    out = [0]
    out.extend(counts)
    return torch.tensor(out, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()


def prepare(case, seed):
    if case["kind"] == "verify":
        return _prepare_verify(case, seed)
    lens, new, k, v, q, g = _raw(case, seed)
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
    seq, pos = _where(lens, lens, "cuda")
    state = {"case": case, "pages": pages, "table": table, "cu": _cu(new),
             "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "max_new": max(new), "max_len": max(lens)}
    if case["kind"] == "attend":
        _put(case, pages, table, seq, pos, k, v)
        state["q"] = q
        return state
    old = pos < (torch.tensor(lens, device="cuda") - torch.tensor(new, device="cuda"))[seq]
    _put(case, pages, table, seq[old], pos[old], k[old], v[old])
    back = lens if case["back"] == "all" else new
    state |= {"k": k[~old].contiguous(), "v": v[~old].contiguous(), "cu_back": _cu(back), "total_back": sum(back),
              "total_new": sum(new)}
    return state


def _prepare_verify(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    b, kk, vocab = case["batch"], case["drafts"], case["vocab"]
    dtype = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
    logits = 2.5 * torch.randn(b, kk + 1, vocab, generator=g, device="cuda")
    target = torch.softmax(logits, -1).to(dtype)
    close = logits[:, :kk] + 0.8 * torch.randn(b, kk, vocab, generator=g, device="cuda")
    noise = -torch.log(-torch.log(torch.rand(b, kk, vocab, generator=g, device="cuda").clamp(1e-12, 1 - 1e-7)))
    tokens = (close + noise).argmax(-1)  # drawn from the draft distribution
    draft = torch.softmax(close, -1).to(dtype) if case["drafter"] else None
    count = torch.full((b,), kk, dtype=torch.int32, device="cuda")
    if case["ragged"]:
        count = torch.randint(0, kk + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    return {"case": case, "tokens": tokens, "target": target, "draft": draft, "count": count,
            "accept_u": torch.rand(b, kk, generator=g, device="cuda"), "sample_u": torch.rand(b, generator=g, device="cuda")}


# ------------------------------------------------------------------ one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        ops = _ops()
        if kind == "attend":
            return ops.hif4_paged_attention(state["q"], state["pages"], state["table"], state["cu"], state["lens"],
                                            page_size=state["case"]["page"], max_new=state["max_new"],
                                            max_len=state["max_len"])
        if kind == "cache":
            ops.hif4_kv_write(state["k"], state["v"], state["pages"], state["table"], state["cu"], state["lens"],
                              page_size=state["case"]["page"])
            return ops.hif4_kv_read(state["pages"], state["table"], state["cu_back"], state["lens"],
                                    page_size=state["case"]["page"], head_dim=state["case"]["dim"],
                                    total=state["total_back"])
        return ops.verify_drafts(state["tokens"], state["target"], state["draft"], state["accept_u"],
                                 state["sample_u"], num_drafts=state["count"])
    return {"attend": _attend, "cache": _cache, "verify": _verify}[kind](state)


def _ops():
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    from faquant_b200 import ops

    return ops


def _packed(state, cu, total):
    """(sequence, position) of a packed token axis, from the device's arrays."""
    new = (cu[1:] - cu[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(len(new), device=cu.device), new, output_size=total)
    index = torch.arange(total, device=cu.device)
    return seq, index - cu[seq].long() + (state["lens"] - new)[seq].long()


def _attend(state):
    case, q, lens = state["case"], state["q"], state["lens"].long()
    b, n, length = case["batch"], state["max_new"], state["max_len"]
    heads, h, d = case["heads"], case["kv_heads"], case["dim"]
    seq, pos = _packed(state, state["cu"], q.shape[0])
    slot = torch.arange(q.shape[0], device=q.device) - state["cu"][seq].long()
    padded = torch.zeros(b, n, heads, d, device=q.device)
    padded[seq, slot] = q.float()
    at = torch.full((b, n), -1, dtype=torch.long, device=q.device)
    at[seq, slot] = pos
    every = torch.arange(b * length, device=q.device)
    k, v = _get(case, state["pages"], state["table"], every // length, every % length)
    k = k.reshape(b, length, h, d).permute(0, 2, 3, 1)
    v = v.reshape(b, length, h, d).permute(0, 2, 1, 3)
    padded = padded.reshape(b, n, h, heads // h, d).permute(0, 2, 3, 1, 4).reshape(b, h, heads // h * n, d)
    s = torch.matmul(padded, k).mul_(d**-0.5).reshape(b, h, heads // h, n, length)
    hidden = torch.arange(length, device=q.device) > at[:, None, None, :, None]
    s.masked_fill_(hidden, float("-inf"))
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.reshape(b, h, heads // h * n, length), v).reshape(b, h, heads // h, n, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 3, 1, 2, 4).reshape(b, n, heads, d)
    return o[seq, slot].to(torch.bfloat16)


def _cache(state):
    case = state["case"]
    seq, pos = _packed(state, state["cu"], state["total_new"])
    _put(case, state["pages"], state["table"], seq, pos, state["k"], state["v"])
    seq, pos = _packed(state, state["cu_back"], state["total_back"])
    k, v = _get(case, state["pages"], state["table"], seq, pos)
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


def _verify(state):
    tokens, target, draft, count = state["tokens"], state["target"], state["draft"], state["count"].long()
    b, kk = tokens.shape
    vocab = target.shape[-1]
    rows, steps = torch.arange(b, device=tokens.device), torch.arange(kk, device=tokens.device)
    p = target[rows[:, None], steps, tokens].float()
    q = draft[rows[:, None], steps, tokens].float() if draft is not None else torch.ones_like(p)
    good = (state["accept_u"] * q < p) & (steps < count[:, None])
    accepted = torch.cumprod(good.long(), 1).sum(1)
    rest = target[rows, accepted].float()
    last = torch.minimum(accepted, torch.full_like(accepted, kk - 1))
    if draft is not None:
        other = draft[rows, last].float()
    else:
        other = torch.zeros_like(rest)
        other[rows, tokens[rows, last]] = float("inf")
    left = torch.where((accepted < count)[:, None], (rest - other).clamp(min=0.0), rest)
    w = torch.round(left.clamp(max=1.0).double() * FIXED_POINT).long()
    whole = torch.round(rest.clamp(0.0, 1.0).double() * FIXED_POINT).long()
    w = torch.where(w.sum(1, keepdim=True) > 0, w, whole)
    cdf = torch.cumsum(w, 1)
    at = state["sample_u"].double() * cdf[:, -1].double()
    token = (cdf.double() <= at[:, None]).sum(1)
    token = torch.where(cdf[:, -1] > 0, token, torch.full_like(token, -1))
    out = torch.full((b, kk + 1), -1, dtype=torch.long, device=tokens.device)
    out[:, :kk] = torch.where(steps < accepted[:, None], tokens, out[:, :kk])
    out[rows, accepted] = token
    return out, accepted.int()


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
    # |x| <= 8 significant bits (bf16) or 24 (fp32); the products round to fp32 as the definition says
    eight = (x.abs().reshape(t, h, -1, 8, 8).amax(-1) * rec[..., None]).float().double()
    four = (x.abs().reshape(t, h, -1, 16, 4).amax(-1) * rec[..., None]).float().double()
    e2 = (eight >= 4).double().repeat_interleave(2, -1)
    e3 = (four >= 2 * torch.exp2(e2)).double()
    e = (e2 + e3).repeat_interleave(4, -1)
    m = ((x.abs() * rec[..., None]).float().double() * torch.exp2(2 - e) + 0.5).float().double().floor().clamp(max=7)
    return (torch.sign(x) * m / 4 * torch.exp2(e) * s[..., None]).reshape(t, h, d)


def exact(case, seed):
    if case["kind"] == "verify":
        return None  # whole numbers
    lens, new, k, v, q, _ = _raw(case, seed)
    parts_k, parts_v = torch.split(k, lens), torch.split(v, lens)
    if case["kind"] == "cache":
        back = lens if case["back"] == "all" else new
        return tuple(torch.cat([_exact_hif4(p[p.shape[0] - n :]) for p, n in zip(parts, back)])
                     for parts in (parts_k, parts_v))
    group, d = case["heads"] // case["kv_heads"], case["dim"]
    out, at = torch.zeros(q.shape, dtype=torch.float64, device=q.device), 0
    for key, value, length, n in zip(parts_k, parts_v, lens, new):
        if not n:
            continue
        key, value = _exact_hif4(key), _exact_hif4(value)
        seen = torch.arange(length, device=q.device)[None] <= torch.arange(length - n, length, device=q.device)[:, None]
        for head in range(case["heads"]):
            s = q[at : at + n, head].double() @ key[:, head // group].T / math.sqrt(d)
            s = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
            out[at : at + n, head] = s @ value[:, head // group]
        at += n
    return out
