"""GPU parity: log probabilities of given tokens, entropy and top alternatives, against the 64-bit oracle. Top ids are
compared exactly (value descending, id ascending).

Tolerance, derived: a thread adds up to K = V / 256 + 16 fp32 terms (each sum off by 2^-24 of itself), the exponential
and z = (x - m) log2(e) / T are off by a few 2^-24 each: ln s by (K + 40) 2^-24 at most; (x - m) / T by 2^-22 of itself.
The entropy's second term t / s has the same relative error, and is at most ln V + H.
"""
import math

import pytest
import torch

from helpers import poison_allocator
from oracle import spec as OSP

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def q3():
    import q3attn
    q3attn._lib.load()
    return q3attn


def logits(n, v, seed, dtype, scale=3.0):
    return (torch.randn(n, v, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def check(q3, x, ids, top, T=1.0, dev_x=None):
    n, v = x.shape
    for _ in range(2):
        poison_allocator((n, max(top, 1)), torch.float32)
    got = q3.token_logprobs(x.to(DEV) if dev_x is None else dev_x, ids.to(DEV), top, T)
    lp, ent, best, best_lp = [t.cpu() for t in got]
    rlp, rent, rbest, rbest_lp = OSP.logprobs(x, ids.clamp(0, v - 1), top, T)
    outside = (ids < 0) | (ids >= v)
    rlp = rlp.masked_fill(outside, -math.inf)
    assert torch.equal(best, rbest)
    base = (v / 256 + 56) * 2.0 ** -24
    for g, r, tol in ((lp, rlp, base + rlp.abs() * 2.0 ** -22), (best_lp, rbest_lp, base + rbest_lp.abs() * 2.0 ** -22),
                      (ent, rent, base * (2 + math.log(v) + rent.abs()))):
        assert g.shape == r.shape and g.dtype == torch.float32
        # the outputs are fp32: (x - m) / T = -3.39e38 / 0.5 = -6.8e38 lies below its range (3.40e38) and is -inf
        fin = torch.isfinite(r.float())
        assert torch.equal(torch.isnan(g), torch.isnan(r)) and torch.equal(g[~fin & ~torch.isnan(r)], r[~fin & ~torch.isnan(r)].float())
        d = (g.double() - r).abs()[fin]
        assert (d <= tol[fin]).all(), float((d / tol[fin]).max())


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,top", [(1, 1, 1), (3, 2, 2), (5, 63, 20), (16, 2048, 5), (4, 4099, 64), (2, 8191, 0),
                                     (1, 150001, 20), (7, 40000, 64), (2400, 700, 3)])
def test_rows(q3, dtype, n, v, top):
    x = logits(n, v, n + v, dtype)
    ids = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(3))
    check(q3, x, ids, top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [0.3, 0.9, 4.0])
def test_temperature_and_several_ids(q3, dtype, T):
    x = logits(9, 5003, 4, dtype)
    ids = torch.randint(0, 5003, (9, 300), generator=torch.Generator().manual_seed(5))
    ids[2, 7], ids[3, 0], ids[8, 299] = -1, 5003, 1 << 40
    check(q3, x, ids, 11, T)
    check(q3, x, ids[:, :0], 11, T)


@pytest.mark.parametrize("dtype", DTYPES)
def test_special_rows(q3, dtype):
    v = 20000
    x = logits(16, v, 6, dtype)
    low = torch.finfo(dtype).min
    x[0] = -math.inf
    x[1, 1:] = -math.inf
    x[2] = low
    x[3, ::2] = low
    x[4, 700] = math.nan
    x[5, 19999] = math.inf
    x[6] = 0
    x[6, 3::7] = -0.0
    x[7] = torch.arange(v).to(dtype) / 1024                       # rising
    x[8] = -torch.arange(v).to(dtype) / 1024                      # falling
    x[9] = torch.finfo(dtype).max
    x[10, 5000:] = -math.inf
    x[11] = (torch.arange(v) % 8).to(dtype)                       # massive ties
    x[12, 17] = 60.0                                              # nearly certain
    x[13] = low
    x[13, 5] = 1.0
    x[14, :] = math.nan
    x[15] *= 100
    check(q3, x, torch.arange(16) * 1250, 64)
    check(q3, x, torch.arange(16), 1, 0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start", [0, 1, 3, 7])
def test_strided_rows_and_odd_starts(q3, dtype, start):
    wide = logits(6, 3011, 8, dtype)
    x = wide[:, start:start + 2999]
    d = wide.to(DEV)[:, start:start + 2999]
    check(q3, x, torch.arange(6) * 400, 30, dev_x=d)
    check(q3, x[:1], torch.arange(1), 30, dev_x=d[:1])
    t = wide.t().contiguous().to(DEV).t()[:, start:start + 2999]          # columns first: copied
    check(q3, x, torch.arange(6), 2, dev_x=t)


@pytest.mark.parametrize("n", [1, 2, 70])
def test_values_in_one_place(q3, n):
    """All of the top alternatives side by side, at the row's end, and in one thread's vectors."""
    v = 100000
    for at in (slice(0, 64), slice(v - 64, v), slice(5000, 5016)):
        x = logits(n, v, 9, torch.float32, 0.1)
        x[:, at] += 50 + torch.arange(at.stop - at.start) * 0.5
        check(q3, x, torch.full((n,), at.start), 40)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v", [(3, 30000), (200, 30000), (1, 130000)])
@pytest.mark.parametrize("threads", [40, 66, 100, 125])
def test_ties_with_candidates_of_some_threads(q3, dtype, n, v, threads):
    """Massive ties (fewer than 64 of 128 groups of two threads above them) leave the row to the selection by tiles; its
    later tiles then have candidates of `threads` of 256 threads, in all four of a thread's vectors, which are listed as
    they are."""
    vec = 16 // dtype.itemsize
    x = torch.ones(n, v, dtype=dtype)
    i = torch.arange(v)
    for tile, up in ((1, 1), (2, 1), (3, 2)):
        x[:, (i // (1024 * vec) == tile) & (i // vec % 256 < threads)] += up
    x[n // 2, -40:] = 9.0
    ids = torch.arange(n) * 7 % v
    check(q3, x, ids, 64)
    d, first = x.to(DEV), None
    for _ in range(10):
        top = q3.token_logprobs(d, ids.to(DEV), 64).top_ids
        first = top if first is None else first
        assert torch.equal(top, first)


def test_graph_replay(q3):
    x = logits(12, 30000, 10, torch.bfloat16).to(DEV)
    ids = torch.arange(12, device=DEV)
    q3.token_logprobs(x, ids, 5)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = q3.token_logprobs(x, ids, 5)
    y = logits(12, 30000, 11, torch.bfloat16)
    x.copy_(y)
    g.replay()
    want = q3.token_logprobs(y.to(DEV), ids, 5)
    for a, b in zip(out, want):
        assert torch.equal(a, b)


def test_no_rows(q3):
    got = q3.token_logprobs(torch.empty(0, 100, device=DEV), torch.empty(0, dtype=torch.int64, device=DEV), 3)
    assert got.logprobs.shape == (0,) and got.top_ids.shape == (0, 3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v", [(500, 151000), (2, 151000), (460, 40007), (1, 2000003)])
def test_many_small_probabilities_next_to_a_certain_token(q3, dtype, n, v):
    """One token at 1, all others at e^-16.75 = 0.89 * 2^-24 of it: none of them may be lost in a sum that holds the one.
    ln p and the entropy in closed form. Tolerance: V / 8192 tile sums (fp32: 4096) of 16 terms to a thread's half, and 61
    roundings of exponentials, shuffles, warps and CTAs, 2^-24 of s = 1 + V e^-16.75 < 1.11 each; t / s = ln V + H times
    that at most."""
    d = 16.75
    x = torch.zeros(n, v, dtype=dtype, device=DEV)
    ids = torch.arange(n) * 997 % v
    x[torch.arange(n), ids] = d
    got = q3.token_logprobs(x, torch.stack([ids, (ids + 1) % v], 1).to(DEV), 1)
    rest = (v - 1) * math.exp(-d)
    lp, h = -math.log1p(rest), math.log1p(rest) + rest / (1 + rest) * d
    base = 1.11 * (v / (8192 if dtype != torch.float32 else 4096) + 16 + 61) * 2.0 ** -24
    assert torch.equal(got.top_ids[:, 0].cpu(), ids)
    err = lambda a, b: float((a.cpu().double() - b).abs().max())  # noqa: E731
    assert err(got.logprobs[:, 0], lp) <= base and err(got.top_logprobs[:, 0], lp) <= base
    assert err(got.logprobs[:, 1], lp - d) <= base + d * 2.0 ** -22
    assert err(got.entropy, h) <= base * (2 + math.log(v) + h)
    if n > 400:
        assert err(got.entropy, h) <= 2 * base        # the part of t that each token has is d e^-d: no cancellation


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [1.5, 4.0, 1000.0])
def test_logits_further_apart_than_fp32_reaches(q3, dtype, T):
    """x - m = -2 * 3.4e38 leaves fp32, (x - m) / T need not."""
    x = logits(4, 3001, 21, dtype)
    x[0] = torch.finfo(dtype).min
    x[0, 77] = torch.finfo(dtype).max
    x[1, ::2], x[1, 5] = torch.finfo(dtype).min, torch.finfo(dtype).max / 2
    x[2, 9], x[2, 10], x[2, 11:] = torch.finfo(dtype).max, torch.finfo(dtype).min, -math.inf
    check(q3, x, torch.tensor([[3, 77], [4, 5], [10, 2000], [1, 2]]), 40, T)
