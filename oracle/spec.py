"""64-bit restatement of the speculative-decoding ops: the 8-bit cache, attention of drafted trees, log probabilities.

Plain loops over seats, heads and rows; CPU tensors in, float64 out.
"""
import math

import torch

E_MIN, E_MAX = -96, 119


def round_e4m3(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value of |x| <= 448 (float64, half to even): steps of 2^(e-3) in [2^e, 2^(e+1)), of 2^-9 below 2^-6."""
    step = torch.exp2((torch.frexp(x.abs().clamp_min(2.0 ** -6))[1] - 4).double())
    return torch.round(x / step) * step


def quantise(x: torch.Tensor):
    """(values in units of the scale, exponent) of rows [..., 128]."""
    x = x.double()
    top = torch.where(torch.isfinite(x), x.abs(), 0).amax(-1)
    m, e = torch.frexp(top / 448)                       # the least e with top <= 448 * 2^e
    e = torch.where(m == 0.5, e - 1, e)
    e = torch.where(top > 0, e, E_MIN).clamp(E_MIN, E_MAX)
    y = x / torch.exp2(e.double())[..., None]
    y = torch.where(torch.isfinite(y), round_e4m3(y.clamp(-448, 448).nan_to_num()), math.nan)
    return y, e


def values(cache: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """What an 8-bit cache holds, as float64 (cache e4m3 [..., 8, 128], scale E8M0 [..., 8])."""
    e = scale.view(torch.uint8).double() - 127
    return cache.to(torch.float32).double() * torch.exp2(e)[..., None]


def rows_of(pool: torch.Tensor, table_row: torch.Tensor, n: int) -> torch.Tensor:
    """The first n token rows of a seat, [n, 8, 128] (pool [pages, page, 8, 128], any float type)."""
    page = pool.shape[1]
    pos = torch.arange(n)
    return pool[table_row.long()[pos // page], pos % page].double()


def visible(words, n: int) -> torch.Tensor:
    """[t, n] booleans of t visibility words."""
    return torch.tensor([[bool((int(w) >> j) & 1) for j in range(n)] for w in words]).view(len(words), n)


def attend(q, keys, vals, see, scale):
    """q [t, 16, 128], keys / vals [n, 8, 128], see [t, n]. Returns (out, A, R): out [t, 16, 128]; A the same with |vals|
    (how far relative errors of the probabilities reach); R [t, 16, 1] the largest weight times row maximum."""
    t, n = see.shape
    q = q.double()
    out, A, R = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(t, q.shape[1], 1, dtype=torch.float64)
    for i in range(t):
        idx = see[i].nonzero()[:, 0]
        if len(idx) == 0:
            continue
        k, v = keys[idx].repeat_interleave(2, 1), vals[idx].repeat_interleave(2, 1)       # [m, 16, 128]
        s = torch.einsum("hd,mhd->hm", q[i], k) * scale
        p = torch.softmax(s, -1)
        out[i] = torch.einsum("hm,mhd->hd", p, v)
        A[i] = torch.einsum("hm,mhd->hd", p, v.abs())
        R[i] = (p * v.abs().amax(-1).T).amax(-1, keepdim=True)
    return out, A, R


def tree_attention(q, k, v, mask, k_pool, v_pool, seqlens, table, scale, draft_lens=None):
    """q [B, T, 16, 128]; k / v [B, T, 8, 128] or None; mask [B, T] or [T]; pools as float values. -> (out, A, R)."""
    B, T = q.shape[:2]
    outs = [torch.zeros(B, T, 16, 128, dtype=torch.float64), torch.zeros(B, T, 16, 128, dtype=torch.float64),
            torch.zeros(B, T, 16, 1, dtype=torch.float64)]
    for b in range(B):
        n, d = int(seqlens[b]), T if draft_lens is None else int(draft_lens[b])
        if d == 0:
            continue
        keys, vals = rows_of(k_pool, table[b], n), rows_of(v_pool, table[b], n)
        see = torch.ones(d, n, dtype=torch.bool)
        if k is not None:
            keys, vals = torch.cat([keys, k[b, :d].double()]), torch.cat([vals, v[b, :d].double()])
            see = torch.cat([see, visible((mask if mask.dim() == 1 else mask[b])[:d].tolist(), d)], 1)
        for o, r in zip(outs, attend(q[b, :d], keys, vals, see, scale)):
            o[b, :d] = r
    return outs


def logprobs(logits, ids, top_n, temperature=1.0):
    """(log probabilities of ids [N] or [N, M], entropy [N], top ids [N, n], their log probabilities). The maximum is
    taken off first (64 bits too lose digits of the sum next to a logit of 1e38), so a row with +inf is NaN."""
    x = logits.double()
    z = (x - x.amax(-1, keepdim=True)) / temperature
    lp = z - torch.log(torch.exp(z).sum(-1, keepdim=True))
    ent = -torch.where(lp > -math.inf, lp.exp() * lp, torch.where(torch.isnan(lp), lp, 0.0)).sum(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top_n]
    return torch.gather(lp, 1, ids.view(len(x), -1)).view(ids.shape), ent, order, torch.gather(lp, 1, order)
