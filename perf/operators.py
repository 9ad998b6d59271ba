"""What the operators of speculative decoding over an 8-bit cache are measured on.

Four operators: writing a paged K/V cache in e4m3 with one power-of-two scale per (token, head) and reading rows of it
back ("cache"), decode attention over such a cache ("decode"), attention of a tree of drafted tokens over a bf16 or
e4m3 cache ("tree"), and log probabilities of given tokens with the entropy and the top alternatives ("logprobs").
`run` computes them in elementary torch operations, or, with `own` set, through the framework's entry points.

Shapes are those of the engine's model family: 16 query heads, 8 KV heads, head_dim 128; 576 seats with 200 to 1200
cached tokens in 16-token pages are the talker's decode step.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
NH, NKV, HD = 16, 8, 128
GROUP = NH // NKV
SCALE = HD ** -0.5
E_MIN, E_MAX = -96, 119            # exponents a cache scale may have
BYTES = {"bf16": 2, "e4m3": 1}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the rows of one decode step go into the cache and come back (a check of what the next step will see)
        {"name": "cache_step", "kind": "cache", "seats": 24, "lo": 200, "hi": 1200, "new": 1, "page": 16, "read": "new", "lens": 1},
        # a chunk of each prompt is written, and prefix + chunk are read back for the chunk's prefill attention
        {"name": "cache_chunk", "kind": "cache", "seats": 10, "lo": 100, "hi": 900, "new": 321, "page": 16, "read": "all", "lens": 2},
        # long prompts, large pages: a whole batch of prompts written at once
        {"name": "cache_prompts", "kind": "cache", "seats": 16, "lo": 0, "hi": 64, "new": 4095, "page": 256, "read": "all", "lens": 3},
        # one listener
        {"name": "decode_one", "kind": "decode", "seats": 1, "lo": 333, "hi": 333, "page": 16, "lens": 4},
        # the talker's decode step, one layer
        {"name": "decode_batch", "kind": "decode", "seats": 576, "lo": 200, "hi": 1200, "page": 16, "lens": 5},
        # few seats with long, uneven histories
        {"name": "decode_long", "kind": "decode", "seats": 9, "lo": 1, "hi": 40000, "page": 256, "lens": 6},
        # a short chain of drafts of one listener
        {"name": "tree_one", "kind": "tree", "cache": "bf16", "seats": 1, "tokens": 4, "lo": 701, "hi": 701, "page": 16, "shared": True, "ragged": False, "lens": 7},
        # small trees over the talker's batch
        {"name": "tree_batch", "kind": "tree", "cache": "bf16", "seats": 288, "tokens": 7, "lo": 200, "hi": 1200, "page": 16, "shared": True, "ragged": False, "lens": 8},
        # trees of their own for each seat, of uneven size, over the 8-bit cache
        {"name": "tree_ragged", "kind": "tree", "cache": "e4m3", "seats": 96, "tokens": 16, "lo": 0, "hi": 2400, "page": 16, "shared": False, "ragged": True, "lens": 9},
        # the widest trees over long histories
        {"name": "tree_wide", "kind": "tree", "cache": "bf16", "seats": 24, "tokens": 64, "lo": 1000, "hi": 8000, "page": 64, "shared": False, "ragged": False, "lens": 10},
        # one seat's drafted tokens against a codebook head
        {"name": "logprobs_codes", "kind": "logprobs", "dtype": "fp32", "rows": 16, "vocab": 2048, "given": 1, "top": 5, "temperature": 0.9},
        # scoring rows against a large text vocabulary
        {"name": "logprobs_text", "kind": "logprobs", "dtype": "bf16", "rows": 1030, "vocab": 151000, "given": 3, "top": 20, "temperature": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache", "decode", "tree", "logprobs"])
    lens = rng.randrange(1 << 20)
    if kind == "cache":
        seats, new = _log(rng, 1, 200), _log(rng, 1, 2000)
        while seats * new > 60000:
            new = max(1, new // 2)
        lo = rng.choice([0, 1, 100])
        hi = lo + _log(rng, 1, max(1, min(2000, 60000 // seats)))
        return {"kind": kind, "seats": seats, "lo": lo, "hi": hi, "new": new, "page": rng.choice([1, 16, 24, 64, 256]),
                "read": rng.choice(["new", "all"]), "lens": lens}
    if kind == "decode":
        seats = _log(rng, 1, 600)
        lo = rng.choice([0, 1, 200])
        hi = lo + _log(rng, 1, max(2, min(40000, 400000 // seats)))
        return {"kind": kind, "seats": seats, "lo": lo, "hi": hi, "page": rng.choice([1, 16, 24, 64, 256]), "lens": lens}
    if kind == "tree":
        seats, tokens = _log(rng, 1, 300), _log(rng, 1, 64)
        lo = rng.choice([0, 1, 200])
        hi = lo + _log(rng, 1, max(2, min(8000, 100000 // seats)))
        return {"kind": kind, "cache": rng.choice(["bf16", "e4m3"]), "seats": seats, "tokens": tokens, "lo": lo, "hi": hi,
                "page": rng.choice([1, 16, 24, 64, 256]), "shared": rng.random() < 0.5, "ragged": rng.random() < 0.5, "lens": lens}
    vocab = _log(rng, 2, 260000)
    rows = _log(rng, 1, max(2, min(4000, 150_000_000 // vocab)))
    return {"kind": kind, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "rows": rows, "vocab": vocab, "given": rng.choice([1, 1, 2, 5]),
            "top": min(vocab, rng.choice([0, 1, 5, 20, 64])), "temperature": rng.choice([1.0, 0.9, 0.3])}


def _lens(case):
    """Cached tokens of each seat, a function of the case alone."""
    r = random.Random(case["lens"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["seats"])]


def _drafts(case):
    """Drafted tokens of each seat."""
    r = random.Random(case["lens"] + 1)
    return [r.randint(0, case["tokens"]) if case["ragged"] else case["tokens"] for _ in range(case["seats"])]


def _rows(case):
    """(seat, position) of the rows a cache case writes, and of those it reads back, as int32 arrays."""
    lens, new = np.asarray(_lens(case)), case["new"]
    seat = np.repeat(np.arange(case["seats"]), new)
    pos = np.concatenate([np.arange(n, n + new) for n in lens])
    if case["read"] == "new":
        return (seat, pos), (seat, pos)
    return (seat, pos), (np.repeat(np.arange(case["seats"]), lens + new), np.concatenate([np.arange(n + new) for n in lens]))


def work(case):
    if case["kind"] == "cache":
        w, r = _rows(case)
        row = NKV * HD
        return {"bytes": 2 * (3 * row + NKV) * len(w[0]) + 2 * (3 * row + NKV) * len(r[0]) + 12 * (len(w[0]) + len(r[0])),
                "flops": 4 * row * len(w[0]) + 2 * row * len(r[0])}
    if case["kind"] == "logprobs":
        n, v, size = case["rows"], case["vocab"], DTYPES[case["dtype"]].itemsize
        return {"bytes": n * (v * size + case["given"] * 12 + 4 + case["top"] * 12), "flops": 6 * n * v}
    lens = _lens(case)
    t = 1 if case["kind"] == "decode" else case["tokens"]
    size = 1 if case["kind"] == "decode" else BYTES[case["cache"]]
    row = 2 * (NKV * HD * size + (NKV if size == 1 else 0))
    pages = sum(-(-n // case["page"]) for n in lens)
    total = sum(lens) * row + 4 * pages + 4 * len(lens) + 2 * 2 * NH * HD * t * len(lens)
    flops = 4 * NH * HD * t * sum(lens)
    if case["kind"] == "tree":
        drafts = _drafts(case)
        total += sum(drafts) * 2 * 2 * NKV * HD + 8 * t * (1 if case["shared"] else len(lens))
        flops += sum(2 * NH * HD * d * d for d in drafts)
    return {"bytes": total, "flops": flops}


# ------------------------------------------------------------------------------------------------ inputs
def _pages(lens, page, gen):
    """Block table (int32 [seats, pages]) of seats with room for `lens` tokens: a shuffle of the pool's pages."""
    per = max(1, max(-(-n // page) for n in lens))
    table = torch.randperm(len(lens) * per, generator=gen, device=DEV).to(torch.int32).view(len(lens), per)
    return table, len(lens) * per


def _keys(n, gen):
    """Rotated, normed keys: unit-sized, a few channels larger than the rest."""
    x = torch.randn(n, NKV, HD, generator=gen, device=DEV)
    ch = torch.exp(0.7 * torch.randn(NKV, HD, generator=gen, device=DEV))
    return (x * ch).to(torch.bfloat16)


def _values(n, gen):
    """Values whose size differs from token to token."""
    x = torch.randn(n, NKV, HD, generator=gen, device=DEV)
    return (x * torch.exp(0.5 * torch.randn(n, 1, 1, generator=gen, device=DEV))).to(torch.bfloat16)


def _pool(pages, page, gen, fmt):
    k, v = _keys(pages * page, gen), _values(pages * page, gen)
    if fmt == "bf16":
        return {"k_cache": k.view(pages, page, NKV, HD), "v_cache": v.view(pages, page, NKV, HD), "k_scale": None, "v_scale": None}
    (kq, ks), (vq, vs) = _quantise(k), _quantise(v)
    return {"k_cache": kq.view(pages, page, NKV, HD), "v_cache": vq.view(pages, page, NKV, HD),
            "k_scale": ks.view(pages, page, NKV), "v_scale": vs.view(pages, page, NKV)}


def _tree(n, rng):
    """Visibility bits of a random tree of n tokens: bit j of word i says that token i sees token j."""
    words = []
    for i in range(n):
        parent = rng.randint(max(-1, i - 6), i - 1) if i else -1
        w = (words[parent] if parent >= 0 else 0) | (1 << i)
        words.append(w)
    return [w - (1 << 64) if w >> 63 else w for w in words]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed)
    if case["kind"] == "logprobs":
        n, v = case["rows"], case["vocab"]
        x = 2.5 * torch.randn(n, v, generator=gen, device=DEV)
        x[: n // 4] *= 2.0                                             # confident rows
        if v > 8:
            x[n // 2:, v - v // 8:] = -math.inf                         # suppressed ids
        ids = torch.randint(0, v, (n, case["given"]), generator=gen, device=DEV)
        ids[:, 0] = torch.where(torch.rand(n, generator=gen, device=DEV) < 0.5, x.argmax(1), ids[:, 0])
        return {"case": case, "logits": x.to(DTYPES[case["dtype"]]), "ids": ids[:, 0].contiguous() if case["given"] == 1 else ids}
    lens = _lens(case)
    if case["kind"] == "cache":
        (ws, wp), (rs, rp) = _rows(case)
        table, pages = _pages([n + case["new"] for n in lens], case["page"], gen)
        n = len(ws)
        qkv = torch.empty(n, (NH + 2 * NKV) * HD, dtype=torch.bfloat16, device=DEV)   # rows of the QKV projection
        k, v = qkv[:, NH * HD:(NH + NKV) * HD].view(n, NKV, HD), qkv[:, (NH + NKV) * HD:].view(n, NKV, HD)
        k.copy_(_keys(n, gen))
        v.copy_(_values(n, gen))
        i32 = lambda a: torch.from_numpy(a.astype(np.int32)).to(DEV)  # noqa: E731
        return {"case": case, "k": k, "v": v, "table": table, "w_seat": i32(ws), "w_pos": i32(wp), "r_seat": i32(rs), "r_pos": i32(rp),
                **_pool(pages, case["page"], gen, "e4m3")}
    table, pages = _pages(lens, case["page"], gen)
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    b = len(lens)
    if case["kind"] == "decode":
        q = (1.5 * torch.randn(b, NH, HD, generator=gen, device=DEV)).to(torch.bfloat16)
        return {"case": case, "q": q, "seq": seq, "table": table, **_pool(pages, case["page"], gen, "e4m3")}
    t = case["tokens"]
    q = (1.5 * torch.randn(b, t, NH, HD, generator=gen, device=DEV)).to(torch.bfloat16)
    masks = [_tree(t, rng) for _ in range(1 if case["shared"] else b)]
    mask = torch.tensor(masks[0] if case["shared"] else masks, dtype=torch.int64, device=DEV)
    return {"case": case, "q": q, "k": _keys(b * t, gen).view(b, t, NKV, HD), "v": _values(b * t, gen).view(b, t, NKV, HD), "mask": mask,
            "drafts": torch.tensor(_drafts(case), dtype=torch.int32, device=DEV) if case["ragged"] else None,
            "seq": seq, "table": table, **_pool(pages, case["page"], gen, case["cache"])}


# ------------------------------------------------------------------------------------------------ plain forms
def _quantise(x):
    """(e4m3 values, E8M0 scales) of rows [n, 8, 128]: the scale of a row's head is the least power of two that brings
    its largest magnitude to 448 or less, exponents held in [E_MIN, E_MAX]."""
    x = x.float()
    top = torch.where(torch.isfinite(x), x.abs(), 0).amax(-1)
    m, e = torch.frexp(top)                                            # top = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(top > 0, e - 9 + (m > 0.875).int(), E_MIN).clamp(E_MIN, E_MAX)
    y = x * ((127 - e[..., None]) << 23).view(torch.float32)           # x * 2^-e, exact
    y = torch.where(torch.isfinite(y), y.clamp(-448, 448), math.nan).to(torch.float8_e4m3fn)
    return y, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _slots(table, page, seat, pos):
    seat, pos = seat.long(), pos.long()
    return table[seat, pos // page].long() * page + pos % page


def _read(cache, scale, slots):
    """Rows `slots` of a pool as fp32 [..., 8, 128]."""
    x = cache.view(-1, NKV, HD)
    if scale is None:
        return x[slots].float()
    x = x.view(torch.uint8)[slots].view(torch.float8_e4m3fn).float()
    return x * scale.view(-1, NKV).view(torch.uint8)[slots].view(torch.float8_e8m0fnu).float()[..., None]


def _cache(s):
    page = s["case"]["page"]
    slots = _slots(s["table"], page, s["w_seat"], s["w_pos"])
    for x, cache, scale in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        y, e = _quantise(x)
        cache.view(torch.uint8).view(-1, NKV, HD)[slots] = y.view(torch.uint8)
        scale.view(torch.uint8).view(-1, NKV)[slots] = e.view(torch.uint8)
    slots = _slots(s["table"], page, s["r_seat"], s["r_pos"])
    return [_read(s[c], s[e], slots).to(torch.bfloat16) for c, e in (("k_cache", "k_scale"), ("v_cache", "v_scale"))]


def _cached(s):
    """K and V of each seat's cached tokens, padded to the longest, as fp32 [seats, tokens, 8, 128]; which are real."""
    page, seq, table = s["case"]["page"], s["seq"].long(), s["table"]
    pos = torch.arange(max(1, s["case"]["hi"]), device=DEV)
    real = pos[None] < seq[:, None]
    seat = torch.arange(len(seq), device=DEV)[:, None]
    slots = _slots(table, page, seat, torch.where(real, pos[None], 0))
    k, v = (_read(s[c], s[e], slots) for c, e in (("k_cache", "k_scale"), ("v_cache", "v_scale")))
    return k, v.masked_fill_(~real[:, :, None, None], 0), real


def _softmax(x):
    """Softmax over the last axis; rows of -inf alone give zeros."""
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0, top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1, total)


def _decode(s):
    k, v, real = _cached(s)
    q = s["q"].float().view(-1, NKV, GROUP, HD)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) * SCALE
    p = _softmax(x.masked_fill_(~real[:, None, None], -math.inf))
    return torch.matmul(p, v.permute(0, 2, 1, 3)).view(-1, NH, HD).to(torch.bfloat16)


def _visible(s, b, t):
    """[seats, tokens, tokens]: which drafted tokens a drafted token sees; which drafted tokens there are [seats, tokens]."""
    j = torch.arange(t, device=DEV)
    live = j[None] < (s["drafts"].long()[:, None] if s["drafts"] is not None else torch.full((b, 1), t, device=DEV))
    bits = ((s["mask"].view(-1, t, 1) >> j) & 1).bool()
    return bits & live[:, None], live


def _tree_attention(s):
    k, v, real = _cached(s)
    b, t = s["q"].shape[:2]
    see, live = _visible(s, b, t)
    q = s["q"].float().view(b, t, NKV, GROUP, HD).permute(0, 2, 3, 1, 4).reshape(b, NKV, GROUP * t, HD)
    new_k, new_v = s["k"].float(), s["v"].float().masked_fill(~live[:, :, None, None], 0)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)).masked_fill_(~real[:, None, None], -math.inf)
    y = torch.matmul(q, new_k.permute(0, 2, 3, 1)).view(b, NKV, GROUP, t, t)
    y = y.masked_fill_(~see[:, None, None], -math.inf).view(b, NKV, GROUP * t, t)
    p = _softmax(torch.cat([x, y], -1) * SCALE)
    o = torch.matmul(p[..., :x.shape[-1]], v.permute(0, 2, 1, 3)) + torch.matmul(p[..., x.shape[-1]:], new_v.permute(0, 2, 1, 3))
    o = o.view(b, NKV, GROUP, t, HD).permute(0, 3, 1, 2, 4).reshape(b, t, NH, HD)
    return o.masked_fill(~live[:, :, None, None], 0).to(torch.bfloat16)


def _logprobs(s):
    x, ids, top = s["logits"].float(), s["ids"], s["case"]["top"]
    peak = x.amax(-1, keepdim=True)
    y = (x - peak) / s["case"]["temperature"]
    e = torch.exp(y)
    total = e.sum(-1, keepdim=True)
    entropy = torch.log(total[:, 0]) - torch.where(e > 0, e * y, 0).sum(-1) / total[:, 0]
    given = torch.gather(y, 1, ids.view(len(x), -1)) - torch.log(total)
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top]
    return given.view(ids.shape), entropy, order, torch.gather(y, 1, order) - torch.log(total)


def _framework():
    path = os.path.join(os.getcwd(), "qwen3-tts-engine_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import q3attn
    return q3attn


def run(state):
    s, case = state, state["case"]
    if not own:
        return {"cache": _cache, "decode": _decode, "tree": _tree_attention, "logprobs": _logprobs}[case["kind"]](s)
    q3 = _framework()
    if case["kind"] == "cache":
        pool = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
        q3.kv_quant_append_paged(s["k"], s["v"], *pool, s["w_pos"], s["table"], s["w_seat"])
        return q3.kv_dequant_paged(*pool, s["r_pos"], s["table"], s["r_seat"])
    if case["kind"] == "decode":
        return q3.paged_decode_quant(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["seq"], s["table"], SCALE)
    if case["kind"] == "tree":
        return q3.paged_tree_attn(s["q"], s["k"], s["v"], s["mask"], s["k_cache"], s["v_cache"], s["seq"], s["table"], SCALE,
                                  k_scale=s["k_scale"], v_scale=s["v_scale"], draft_lens=s["drafts"])
    return q3.token_logprobs(s["logits"], s["ids"], top_n=case["top"], temperature=case["temperature"])


# ------------------------------------------------------------------------------------------------ 64 bits
def _read64(s, which, slots):
    x = s[which + "_cache"].view(-1, NKV, HD)
    if s[which + "_scale"] is None:
        return x[slots].double()
    e = s[which + "_scale"].view(-1, NKV).view(torch.uint8)[slots].long() - 127
    return x.view(torch.uint8)[slots].view(torch.float8_e4m3fn).double() * _pow2(e)[..., None]


def _pow2(e):
    """2^e as exact doubles, for whole numbers e."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _round_e4m3(x):
    """Nearest e4m3 value (ties to even) of |x| <= 448, in 64 bits: steps of 2^(e-3) in [2^e, 2^(e+1)), and of 2^-9 below 2^-6."""
    step = _pow2(torch.frexp(x.abs().clamp_min(2.0 ** -6))[1] - 4)
    return torch.round(x / step) * step


def _attend64(q, keys, values, see):
    """q [t, 16, 128] over keys / values [n, 8, 128]; see [t, n]."""
    out = torch.zeros_like(q)
    for h in range(NH if len(keys) else 0):
        x = (q[:, h] @ keys[:, h // GROUP].T) * SCALE
        w = torch.softmax(x.masked_fill(~see, -math.inf), -1).masked_fill(~see, 0)
        w[~see.any(-1)] = 0
        out[:, h] = w @ values[:, h // GROUP]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logprobs":
        x = s["logits"].double()
        z = x / case["temperature"]
        lp = z - torch.logsumexp(z, -1, keepdim=True)
        entropy = -torch.where(lp > -math.inf, lp.exp() * lp, 0).sum(-1)
        best = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :case["top"]]
        return torch.gather(lp, 1, s["ids"].view(len(x), -1)).view(s["ids"].shape), entropy, None, torch.gather(lp, 1, best)
    if case["kind"] == "cache":
        out = []
        w = _slots(s["table"], case["page"], s["w_seat"], s["w_pos"])
        r = _slots(s["table"], case["page"], s["r_seat"], s["r_pos"])
        for which in "kv":
            rows = s[which].double()
            m, e = torch.frexp(rows.abs().amax(-1, keepdim=True).clamp_min(1e-300) / 448)
            e = torch.where(m == 0.5, e - 1, e).clamp(E_MIN, E_MAX)     # the least e with 448 * 2^e at the magnitude or above
            pool = torch.empty(s[which + "_cache"].numel() // (NKV * HD), dtype=torch.int64, device=DEV).fill_(-1)
            pool[w] = torch.arange(len(w), device=DEV)
            got = _read64(s, which, r)
            written = pool[r] >= 0
            got[written] = (_round_e4m3(rows * _pow2(-e)) * _pow2(e))[pool[r][written]]
            out.append(got)
        return out
    lens = _lens(case)
    t = 1 if case["kind"] == "decode" else case["tokens"]
    if sum(lens) * t > 30_000_000:
        return None
    q = s["q"].double().view(len(lens), t, NH, HD)
    out = torch.zeros_like(q)
    drafts = _drafts(case) if case["kind"] == "tree" else None
    for b, n in enumerate(lens):
        slots = _slots(s["table"], case["page"], torch.full((n,), b, device=DEV), torch.arange(n, device=DEV))
        keys, values = _read64(s, "k", slots), _read64(s, "v", slots)
        d = 1 if drafts is None else drafts[b]
        see = torch.ones(d, n, dtype=torch.bool, device=DEV)
        if drafts is not None:
            keys, values = torch.cat([keys, s["k"][b, :d].double()]), torch.cat([values, s["v"][b, :d].double()])
            bits = s["mask"] if case["shared"] else s["mask"][b]
            see = torch.cat([see, ((bits[:d, None] >> torch.arange(d, device=DEV)) & 1).bool()], 1)
        if d:
            out[b, :d] = _attend64(q[b, :d], keys, values, see)
    return out if case["kind"] == "tree" else out.view(len(lens), NH, HD)
