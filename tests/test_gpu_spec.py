"""GPU parity: the 8-bit paged cache, decode attention over it and attention of drafted trees, against the 64-bit
oracle. Quantised bytes, scales and rows read back are compared bit for bit.

Attention tolerance, derived: the output is rounded to bf16 (2^-8 of itself); a probability is rounded to bf16 (2^-8
of itself; drafted rows and bf16 caches) or fp16 (2^-11 of itself, and 2^-25 of the largest weight where it is
subnormal; e4m3 rows), which moves the output by that share of A = sum_j p_j |v_j| at most, or n * 2^-24 * R with R =
max_j p_j max_d |v_jd| (a row's largest e4m3 value is at least 224, half of 448). Scores in fp32: each of the 128
products and sums is off by 2^-24 of sum |q k| at most; with |q| |k| scale <= 64 here that is under 2^-11 in log units
for unit-sized data, twice (numerator and sum): 2^-10 A.
"""
import math

import pytest
import torch

from helpers import bits_equal, poison_allocator
from oracle import spec as OSP
from q3attn import synth

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 128 ** -0.5
BF = torch.bfloat16


@pytest.fixture(scope="module")
def q3():
    import q3attn
    q3attn._lib.load()
    q3attn._lib.read_status()
    return q3attn


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rows(n, seed, lo=-3, hi=3):
    """bf16 rows [n, 8, 128] whose size differs from row to row and whose channels differ within one."""
    g = gen(seed)
    x = torch.randn(n, 8, 128, generator=g) * torch.exp2(torch.randint(lo, hi + 1, (n, 8, 1), generator=g).float())
    return (x * torch.exp(0.5 * torch.randn(8, 128, generator=g))).to(BF)


def bits(x):
    return x.detach().cpu().contiguous().view(torch.uint8)


def expect_cache(x):
    """(e4m3 bytes, scale bytes) of rows x by the oracle. NaN bytes compare by isnan."""
    y, e = OSP.quantise(x)
    return y, (e + 127).to(torch.uint8)


def check_rows(cache, scale, slots, x):
    y, e = expect_cache(x)
    got = cache.cpu().view(-1, 8, 128)[slots].float().double()
    assert torch.equal(torch.isnan(got), torch.isnan(y))
    assert torch.equal(got.nan_to_num(), y.nan_to_num())
    assert torch.equal(bits(scale).view(-1, 8)[slots], e)


def table_for(lens, page, seed, extra=1):
    """Shuffled block table with room for max(lens), and the pool's page count."""
    per = max(1, max(-(-n // page) for n in lens)) + extra
    perm = torch.randperm(len(lens) * per, generator=gen(seed))
    return perm.view(len(lens), per).to(torch.int32), len(lens) * per


# ------------------------------------------------------------------------------------------------ the 8-bit cache
@pytest.mark.parametrize("n,page", [(1, 16), (7, 1), (33, 24), (576, 16), (1000, 256)])
def test_append_paged_and_read_back(q3, n, page):
    k, v = rows(n, 1), rows(n, 2)
    g = gen(3)
    seats = max(1, n // 3)
    pos = torch.arange(n, dtype=torch.int32) // seats
    seat = (torch.arange(n) % seats).to(torch.int32)
    bt, pages = table_for([int(pos.max()) + 1] * seats, page, 4)
    cache = q3.empty_quant_cache(pages, page, DEV)
    before = torch.randint(0, 120, (pages, page, 8, 128), generator=g, dtype=torch.uint8).to(DEV)
    cache[0].view(torch.uint8).copy_(before)
    qkv = torch.zeros(n, 32, 128, dtype=BF)                       # k and v as strided views of projection rows
    qkv[:, 16:24], qkv[:, 24:] = k, v
    d = qkv.to(DEV)
    q3.kv_quant_append_paged(d[:, 16:24], d[:, 24:], *cache, pos.to(DEV), bt.to(DEV), seat.to(DEV))
    slots = bt[seat.long(), pos.long() // page].long() * page + pos.long() % page
    check_rows(cache[0], cache[2], slots, k)
    check_rows(cache[1], cache[3], slots, v)
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[slots] = False
    assert torch.equal(bits(cache[0]).view(-1, 1024)[rest], before.cpu().view(-1, 1024)[rest])
    assert not bits(cache[2]).view(-1, 8)[rest].any()
    poison_allocator((n, 8, 128))
    kb, vb = q3.kv_dequant_paged(*cache, pos.to(DEV), bt.to(DEV), seat.to(DEV))
    for got, c, s in ((kb, cache[0], cache[2]), (vb, cache[1], cache[3])):
        assert bits_equal(got, OSP.values(c.cpu(), s.cpu()).view(-1, 8, 128)[slots].to(BF))
    assert q3._lib.read_status() == 0


def special_rows():
    g = gen(9)
    x = torch.randn(24, 8, 128, generator=g)
    x[0] = 0
    x[1, :, 5] = float("inf")
    x[2, :, 5] = float("nan")
    x[3] = float("nan")
    x[4] = float("-inf")
    x[5] *= 1e-38                                                   # bf16 subnormals, below the smallest scale
    x[6] = 3.3895313892515355e38                                    # the largest bf16: saturates
    x[7] = 0; x[7, :, 0] = 448.0
    x[8] = 0; x[8, :, 0] = 450.0                                    # just above: the next scale
    x[9] = 0; x[9, :, 127] = -0.0
    for i in range(10, 20):
        x[i] *= 2.0 ** (12 * (i - 15))
    x[20, :, ::2] *= 2.0 ** -16                                     # e4m3 subnormals
    x[21] = (torch.arange(1024).view(8, 128) - 512) / 8.0           # ties
    x[22] *= 1e-30
    x[23] = -7.0
    return x.to(BF)


def test_append_special_values(q3):
    k = special_rows()
    n = len(k)
    slots = torch.randperm(n, generator=gen(5))
    cache = q3.empty_quant_cache(n, 1, DEV)
    q3.kv_quant_append_slots(k.to(DEV), k.flip(0).to(DEV), *cache, slots.to(DEV))
    check_rows(cache[0], cache[2], slots, k)
    check_rows(cache[1], cache[3], slots, k.flip(0))
    kb, _ = q3.kv_dequant_paged(*cache, torch.zeros(n, dtype=torch.int32, device=DEV),
                                slots.to(torch.int32)[:, None].contiguous().to(DEV))
    y, e = OSP.quantise(k)
    ref = (y * torch.exp2(e.double())[..., None]).to(BF)
    assert torch.equal(torch.isnan(kb.cpu()), torch.isnan(ref))
    assert torch.equal(kb.cpu().nan_to_num().abs(), ref.nan_to_num().abs())     # -0 keeps its sign in the cache
    # one rounding: e4m3 is off by half a step at most, 2^-4 of the value or 2^-10 of the scale
    ok = torch.isfinite(k.float()) & (k.float().abs() <= 448 * 2.0 ** 119)
    err = (kb.cpu().double() - k.double()).abs()
    assert (err <= torch.maximum(k.double().abs() * 2.0 ** -4, torch.exp2(e.double() - 10)[..., None]))[ok].all()


def test_rows_out_of_range_are_skipped(q3):
    n = 8
    k = rows(n, 1)
    cache = q3.empty_quant_cache(4, 16, DEV)
    bt = torch.tensor([[0, 1], [2, 9], [-3, 3]], dtype=torch.int32)       # seat 1 page 1 and seat 2 page 0: outside
    seat = torch.tensor([0, 0, 1, 2, 3, -1, 0, 2], dtype=torch.int32)
    pos = torch.tensor([0, 32, 16, 0, 0, 0, -1, 17], dtype=torch.int32)
    q3.kv_quant_append_paged(k.to(DEV), k.to(DEV), *cache, pos.to(DEV), bt.to(DEV), seat.to(DEV))
    assert q3._lib.read_status() == q3._lib.STATUS_BAD_PAGE | q3._lib.STATUS_BAD_LENGTH
    want = torch.zeros(64, dtype=torch.bool)
    want[[0, 49]] = True
    assert torch.equal(bits(cache[2]).view(64, 8).any(1), want)
    check_rows(cache[0], cache[2], torch.tensor([0, 49]), k[[0, 7]])
    poison_allocator((n, 8, 128))
    kb, vb = q3.kv_dequant_paged(*cache, pos.to(DEV), bt.to(DEV), seat.to(DEV))
    assert q3._lib.read_status() == q3._lib.STATUS_BAD_PAGE | q3._lib.STATUS_BAD_LENGTH
    assert not kb.cpu()[1:7].float().abs().any() and not vb.cpu()[1:7].float().abs().any()
    assert kb.cpu()[0].float().abs().any() and kb.cpu()[7].float().abs().any()
    q3.kv_quant_append_slots(k.to(DEV), k.to(DEV), *cache, torch.tensor([5, 64, -1, 6, 7, 8, 1 << 40, 9], device=DEV))
    assert q3._lib.read_status() == q3._lib.STATUS_BAD_PAGE
    check_rows(cache[1], cache[3], torch.tensor([5, 6, 7, 8, 9]), k[[0, 3, 4, 5, 7]])


def test_empty_calls(q3):
    cache = q3.empty_quant_cache(2, 16, DEV)
    z, i = torch.empty(0, 8, 128, dtype=BF, device=DEV), torch.empty(0, dtype=torch.int32, device=DEV)
    bt = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    q3.kv_quant_append_paged(z, z, *cache, i, bt, i)
    q3.kv_quant_append_slots(z, z, *cache, i.long())
    assert [x.shape[0] for x in q3.kv_dequant_paged(*cache, i, bt, i)] == [0, 0]
    assert q3.paged_decode_quant(torch.empty(0, 16, 128, dtype=BF, device=DEV), *cache, i, bt[:0], SCALE).shape == (0, 16, 128)
    out = q3.paged_tree_attn(torch.empty(0, 3, 16, 128, dtype=BF, device=DEV), z.view(0, 1, 8, 128).expand(0, 3, 8, 128),
                             z.view(0, 1, 8, 128).expand(0, 3, 8, 128), torch.ones(3, dtype=torch.int64, device=DEV),
                             *cache[:2], i, bt[:0], SCALE, k_scale=cache[2], v_scale=cache[3])
    assert out.shape == (0, 3, 16, 128)


def test_far_rows_of_a_large_pool(q3):
    """Byte offsets past 2^32 in the pools."""
    pages, page = 17000, 256
    cache = q3.empty_quant_cache(pages, page, DEV)
    last = pages - 1
    bt = torch.tensor([[last, 0, pages - 9]], dtype=torch.int32)
    lens = [600]
    k, v = rows(600, 1, -1, 1), rows(600, 2, -1, 1)
    pos = torch.arange(600, dtype=torch.int32)
    q3.kv_quant_append_paged(k.to(DEV), v.to(DEV), *cache, pos.to(DEV), bt.to(DEV), torch.zeros(600, dtype=torch.int32, device=DEV))
    q = (torch.randn(1, 16, 128, generator=gen(3))).to(BF)
    got = q3.paged_decode_quant(q.to(DEV), *cache, torch.tensor(lens, dtype=torch.int32, device=DEV), bt.to(DEV), SCALE)
    small = [c.cpu() for c in (cache[0][bt[0].long().to(DEV)], cache[1][bt[0].long().to(DEV)],
                               cache[2].view(torch.uint8)[bt[0].long().to(DEV)].view(torch.float8_e8m0fnu),
                               cache[3].view(torch.uint8)[bt[0].long().to(DEV)].view(torch.float8_e8m0fnu))]
    ref = OSP.tree_attention(q[:, None], None, None, None, OSP.values(small[0], small[2]), OSP.values(small[1], small[3]),
                             lens, torch.tensor([[0, 1, 2]]), SCALE)
    check_attention(got[:, None], ref, lens, True, False)


# ------------------------------------------------------------------------------------------------ attention
def check_attention(got, ref, lens, fp8, drafted, what=""):
    out, A, R = ref
    assert torch.isfinite(got).all(), what
    n = torch.as_tensor(lens).double().view(-1, 1, 1, 1)
    tol = out.abs() * 2.0 ** -8 + A * 2.0 ** -10
    tol += A * 2.0 ** -8 if drafted or not fp8 else A * 2.0 ** -11
    if fp8:
        tol += n * 2.0 ** -24 * R
    d = (got.cpu().double() - out).abs()
    bad = d > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / tol.clamp_min(1e-30)).max()):.2f}"


def pools(pages, page, seed, fp8):
    """Caches full of rows, and the values they hold."""
    k, v = rows(pages * page, seed, -1, 1), rows(pages * page, seed + 1, -4, 2)
    if not fp8:
        return (k.view(pages, page, 8, 128), v.view(pages, page, 8, 128), None, None), (k.view(pages, page, 8, 128), v.view(pages, page, 8, 128))
    out = []
    for x in (k, v):
        y, e = OSP.quantise(x)
        out.append((y.to(torch.float32).to(torch.float8_e4m3fn).view(pages, page, 8, 128),
                    (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu).view(pages, page, 8)))
    (kq, ks), (vq, vs) = out
    return (kq, vq, ks, vs), (OSP.values(kq, ks), OSP.values(vq, vs))


def dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


@pytest.mark.parametrize("lens,page", [([0], 16), ([1], 16), ([0, 1, 15, 16, 17, 31, 33, 0], 16), ([100, 3, 700], 24),
                                       ([5, 260, 64], 1), ([2000], 256), ([40] * 200, 16), ([37, 0, 513] * 30, 64)])
def test_decode_quant(q3, lens, page):
    bt, pages = table_for(lens, page, 1)
    cache, vals = pools(pages, page, 2, True)
    q = torch.randn(len(lens), 16, 128, generator=gen(7)).to(BF)
    poison_allocator((len(lens), 16, 128))
    got = q3.paged_decode_quant(q.to(DEV), *dev(*cache), torch.tensor(lens, dtype=torch.int32, device=DEV), bt.to(DEV), SCALE)
    ref = OSP.tree_attention(q[:, None], None, None, None, *vals, lens, bt, SCALE)
    check_attention(got[:, None], ref, lens, True, False)
    assert not got.cpu()[torch.tensor(lens) == 0].float().abs().any()
    assert q3._lib.read_status() == 0


def trees(B, T, seed, shared):
    import q3attn
    g = gen(seed)
    p = torch.stack([torch.randint(-1, max(i, 1), (B,), generator=g) if i else torch.full((B,), -1) for i in range(T)], 1)
    m = q3attn.tree_mask(p)
    return m[0].clone() if shared else m


def tree_case(B, T, lens, page, seed, fp8, shared=False, drafts=None):
    g = gen(seed + 100)
    bt, pages = table_for(lens, page, seed)
    cache, vals = pools(pages, page, seed + 1, fp8)
    q = torch.randn(B, T, 16, 128, generator=g).to(BF)
    k, v = rows(B * T, seed + 3, -1, 1).view(B, T, 8, 128), rows(B * T, seed + 4, -4, 2).view(B, T, 8, 128)
    return dict(q=q, k=k, v=v, mask=trees(B, T, seed + 5, shared), cache=cache, vals=vals, bt=bt, lens=lens,
                drafts=None if drafts is None else torch.tensor(drafts, dtype=torch.int32))


def run_tree(q3, c, **over):
    q, k, v, m, bt, drafts = (over.get(n, c[n]) for n in ("q", "k", "v", "mask", "bt", "drafts"))
    kc, vc, ks, vs = dev(*c["cache"])
    poison_allocator(tuple(q.shape))
    return q3.paged_tree_attn(*dev(q, k, v, m), kc, vc, torch.tensor(c["lens"], dtype=torch.int32, device=DEV), bt.to(DEV),
                              SCALE, k_scale=ks, v_scale=vs, draft_lens=None if drafts is None else drafts.to(DEV))


def ref_tree(c, **over):
    q, k, v, m, drafts = (over.get(n, c[n]) for n in ("q", "k", "v", "mask", "drafts"))
    return OSP.tree_attention(q, k, v, m, *c["vals"], c["lens"], c["bt"], SCALE, drafts)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T", [1, 2, 4, 5, 8, 9, 16, 17, 33, 64])
@pytest.mark.parametrize("shared", [False, True])
def test_tree_attention(q3, fp8, T, shared):
    lens = [0, 1, 16, 50, 131]
    c = tree_case(5, T, lens, 16, T, fp8, shared)
    got = run_tree(q3, c)
    check_attention(got, ref_tree(c), [n + T for n in lens], fp8, True)
    assert q3._lib.read_status() == 0


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T,page,lens,drafts", [
    (7, 1, [19, 0, 44], [0, 7, 3]), (16, 24, [100, 25, 24, 23], [16, 15, 1, 0]), (64, 64, [300, 10], [64, 33]),
    (12, 16, [0, 0, 0], [0, 0, 0]), (3, 256, [900], None), (40, 16, [17] * 40, [1 + i % 40 for i in range(40)])])
def test_tree_ragged(q3, fp8, T, page, lens, drafts):
    c = tree_case(len(lens), T, lens, page, 11, fp8, drafts=drafts)
    if drafts is not None:                                   # what lies behind a seat's drafts is never looked at
        for b, d in enumerate(drafts):
            c["k"][b, d:] = float("nan")
            c["v"][b, d:] = float("inf")
            c["q"][b, d:] = float("nan")
            c["mask"][b, d:] = -1
    got = run_tree(q3, c)
    ref = ref_tree(c)
    check_attention(got, ref, [n + T for n in lens], fp8, True)
    for b, d in enumerate(drafts or []):
        assert not got[b, d:].float().abs().any()


@pytest.mark.parametrize("fp8", [False, True])
def test_tree_rows_that_see_nothing(q3, fp8):
    c = tree_case(2, 9, [0, 0], 16, 21, fp8)
    c["mask"][0] = 0
    c["mask"][1, ::2] = 0
    got = run_tree(q3, c).cpu()
    check_attention(got, ref_tree(c), [9, 9], fp8, True)
    assert not got[0].float().abs().any() and not got[1, ::2].float().abs().any()
    assert got[1, 1].float().abs().any()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 3.3e38])
def test_unseen_values_do_not_leak(q3, fp8, bad):
    """Two branches; the rows of one hold infinities or NaN: the other's tokens are as if they were not there, and the
    tokens that see them are not finite."""
    T = 12
    c = tree_case(2, T, [40, 0], 16, 31, fp8)
    even, odd = sum(1 << i for i in range(0, T, 2)), sum(1 << i for i in range(1, T, 2))
    for i in range(T):
        c["mask"][:, i] = (odd if i % 2 else even) & ((2 << i) - 1)
    clean = ref_tree(c)
    c["k"][:, 5, :, 3] = bad
    c["v"][:, 7, :, ::5] = bad
    c["v"][:, 3, 2] = bad
    got = run_tree(q3, c).cpu()
    check_attention(got[:, ::2], [x[:, ::2] for x in clean], [40 + T, T], fp8, True)
    if bad == bad and abs(bad) > 3.35e38:
        assert torch.equal(got[:, 3, 4:6] == bad, torch.ones(2, 2, 128, dtype=torch.bool))
    assert torch.isfinite(got[:, 1]).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_stale_rows_behind_the_tokens(q3, fp8):
    """NaN in the pool behind each seat's last token, and in pages no seat owns."""
    lens = [21, 16, 5, 0]
    c = tree_case(4, 6, lens, 16, 41, fp8)
    used = torch.zeros(c["cache"][0].shape[:2], dtype=torch.bool)
    for b, n in enumerate(lens):
        for t in range(n):
            used[c["bt"][b, t // 16].long(), t % 16] = True
    for x in c["cache"]:
        if x is not None:
            x.view(torch.uint8 if fp8 else torch.int16)[~used] = 0xFF if fp8 else 0x7FFF
    check_attention(run_tree(q3, c), ref_tree(c), [n + 6 for n in lens], fp8, True)


def test_strided_arguments(q3):
    """q, k, v as views of QKV rows, a mask of padded rows, a block table that is a slice of a wider one."""
    B, T = 3, 5
    c = tree_case(B, T, [30, 2, 77], 16, 51, False)
    qkv = torch.zeros(B, T + 2, 32, 128, dtype=BF)
    qkv[:, :T, :16], qkv[:, :T, 16:24], qkv[:, :T, 24:] = c["q"], c["k"], c["v"]
    d = qkv.to(DEV)
    wide = torch.full((B, 40), -1, dtype=torch.int32)
    wide[:, :c["bt"].shape[1]] = c["bt"]
    mask = torch.full((B, 9), -1, dtype=torch.int64)
    mask[:, :T] = c["mask"]
    kc, vc = dev(*c["cache"][:2])
    got = q3.paged_tree_attn(d[:, :T, :16], d[:, :T, 16:24], d[:, :T, 24:], mask.to(DEV)[:, :T], kc, vc,
                             torch.tensor(c["lens"], dtype=torch.int32, device=DEV), wide.to(DEV)[:, :c["bt"].shape[1]], SCALE)
    check_attention(got, ref_tree(c), [n + T for n in c["lens"]], False, True)


@pytest.mark.parametrize("fp8", [False, True])
def test_bad_pages_and_lengths_raise_status(q3, fp8):
    c = tree_case(2, 3, [40, 20], 16, 61, fp8)
    bt = c["bt"].clone()
    bt[0, 1] = 10000
    run_tree(q3, c, bt=bt)
    assert q3._lib.read_status() == q3._lib.STATUS_BAD_PAGE
    full = c["bt"].shape[1] * 16
    c["lens"] = [40, full + 5]                              # held to the table's capacity
    got = run_tree(q3, c)
    assert q3._lib.read_status() == q3._lib.STATUS_BAD_LENGTH
    c["lens"] = [40, full]
    assert bits_equal(got, run_tree(q3, c))
    got = run_tree(q3, c, drafts=torch.tensor([7, -2], dtype=torch.int32))
    assert q3._lib.read_status() == q3._lib.STATUS_BAD_LENGTH
    assert bits_equal(got, run_tree(q3, c, drafts=torch.tensor([3, 0], dtype=torch.int32)))


@pytest.mark.parametrize("fp8", [False, True])
def test_extreme_value_scales(q3, fp8):
    """Rows of very different size: a huge row that hardly counts must not cost the others their digits, nor tiny rows
    theirs."""
    lens = [64, 64, 64]
    c = tree_case(3, 2, lens, 64, 71, False)
    k, v = c["cache"][0].clone(), c["cache"][1].clone()
    p0, p1, p2 = (int(c["bt"][b, 0]) for b in range(3))
    v[p0, 7] = (v[p0, 7].float() * 2.0 ** 40).to(BF)
    k[p0, 7] = 0
    v[p1] = (v[p1].float() * 2.0 ** -80).to(BF)
    v[p2] = 0
    if fp8:
        out = []
        for x in (k, v):
            y, e = OSP.quantise(x)
            out.append((y.float().to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)))
        c["cache"] = (out[0][0], out[1][0], out[0][1], out[1][1])
        c["vals"] = (OSP.values(*out[0]), OSP.values(*out[1]))
    else:
        c["cache"], c["vals"] = (k, v, None, None), (k, v)
    c["v"].zero_()
    c["q"] *= 4
    check_attention(run_tree(q3, c), ref_tree(c), [66] * 3, fp8, True)


def test_graph_capture_and_two_streams(q3):
    """Two captured graphs of different calls, replayed at once on two streams, give what eager calls give."""
    cs = [tree_case(24, 5, [100 + 7 * i for i in range(24)], 16, 81, True), tree_case(9, 20, [333] * 9, 16, 82, False)]
    eager = [run_tree(q3, c) for c in cs]
    torch.cuda.synchronize()
    streams, graphs, outs, keep = [torch.cuda.Stream() for _ in cs], [], [], []
    for c, s in zip(cs, streams):
        args = dev(c["q"], c["k"], c["v"], c["mask"], *c["cache"][:2]) + [torch.tensor(c["lens"], dtype=torch.int32, device=DEV), c["bt"].to(DEV)]
        ks, vs = dev(*c["cache"][2:])
        keep.append((args, ks, vs))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(q3.paged_tree_attn(*args, SCALE, k_scale=ks, v_scale=vs))
        graphs.append(g)
    for _ in range(20):
        for o in outs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert bits_equal(o, e)


def test_deterministic(q3):
    c = tree_case(40, 6, [500 + i for i in range(40)], 16, 91, True)
    first = run_tree(q3, c)
    for _ in range(5):
        assert bits_equal(first, run_tree(q3, c))


@pytest.mark.parametrize("far", [1 << 31, 1 << 32, (1 << 32) + 5, (1 << 40) + 5, -(1 << 31) - 1, -(1 << 32), -(1 << 40) + 3, (1 << 63) - 1, -(1 << 63)])
def test_int64_positions_and_seats_do_not_wrap(q3, far):
    """What lies outside int32 is out of range like any other: skipped with its status bit, read back as zeros."""
    cache = q3.empty_quant_cache(4, 16, DEV)
    bt = torch.arange(4, dtype=torch.int32, device=DEV).view(2, 2)
    k = rows(64, 1).to(DEV)
    q3.kv_quant_append_slots(k, k, *cache, torch.arange(64, device=DEV))
    before = [bits(c) for c in cache]
    seat = torch.tensor([0, far, 1, 0], device=DEV)
    pos = torch.tensor([far, 3, far, 7], device=DEV)
    assert q3._lib.read_status() == 0
    new = rows(4, 2)
    q3.kv_quant_append_paged(new.to(DEV), new.to(DEV), *cache, pos, bt, seat)
    assert q3._lib.read_status() == q3._lib.STATUS_BAD_LENGTH
    rest = torch.arange(64) != 7
    for c, b in zip(cache, before):
        now = bits(c)
        assert torch.equal(now.reshape(64, -1)[rest], b.reshape(64, -1)[rest])
    y, e = expect_cache(new[3:])
    assert torch.equal(cache[0].cpu().view(-1, 8, 128)[7].float().double(), y[0]) and torch.equal(bits(cache[2]).view(-1, 8)[7], e[0])
    kb, vb = q3.kv_dequant_paged(*cache, pos, bt, seat)
    assert q3._lib.read_status() == q3._lib.STATUS_BAD_LENGTH
    assert not kb.cpu()[:3].float().abs().any() and not vb.cpu()[:3].float().abs().any() and kb.cpu()[3].float().abs().any()


def test_int64_positions_of_tables_past_int32_are_refused(q3):
    """A table of 2^31 tokens a seat and more: an int64 position cannot be narrowed, an int32 one is taken."""
    cache = q3.empty_quant_cache(1, 1 << 16, DEV)
    bt = torch.zeros(1, 1 << 15, dtype=torch.int32, device=DEV)
    k, seat = rows(1, 3).to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="int64 positions"):
        q3.kv_quant_append_paged(k, k, *cache, seat.long(), bt, seat)
    with pytest.raises(RuntimeError, match="int64 positions"):
        q3.kv_dequant_paged(*cache, seat.long(), bt, seat)
    q3.kv_quant_append_paged(k, k, *cache, seat, bt, seat.long())
    assert q3._lib.read_status() == 0 and bits(cache[2]).any()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T", [1, 3, 4, 7, 8, 12, 20, 64])
@pytest.mark.parametrize("infinite", [False, True])
def test_keys_that_score_minus_infinity_come_first(q3, fp8, T, infinite):
    """A seat's first keys score -inf (a product past fp32's range, or K of -inf) for every head and token, the later ones
    zero: the first have no weight. A seat of such keys alone, without visible drafts, has zero rows."""
    if infinite and fp8:
        return                                                  # an 8-bit cache holds no infinities
    lens, page = [40, 16, 17, 5], 16
    bt, pages = table_for(lens, page, 1)
    x = torch.zeros(pages * page, 8, 128)
    for b, n in enumerate(lens):
        x.view(pages, page, 8, 128)[bt[b, 0].item()] = -math.inf if infinite else 4.0
    v = rows(pages * page, 3, -1, 1)
    (kq, ks), (vq, vs) = ((lambda y, e: (y.float().to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)))(*OSP.quantise(z))
                          for z in (x.to(BF).nan_to_num(neginf=0), v))
    kp, vp = (kq, vq) if fp8 else (x.to(BF), v)
    shape = lambda z, *s: z.view(pages, page, 8, *s)  # noqa: E731
    vals = (shape(OSP.values(kq, ks), 128), shape(OSP.values(vq, vs), 128)) if fp8 else (shape(kp, 128), shape(vp, 128))
    q = torch.full((4, T, 16, 128), 1.0 if infinite else -2e38).to(BF)
    k, dv = torch.zeros(4, T, 8, 128, dtype=BF), rows(4 * T, 4, -1, 1).view(4, T, 8, 128)
    mask = torch.zeros(4, T, dtype=torch.int64)
    mask[:3] = torch.tensor([1 << i if i < 63 else -(1 << 63) for i in range(T)])
    sc = dict(k_scale=shape(ks).to(DEV), v_scale=shape(vs).to(DEV)) if fp8 else {}
    got = q3.paged_tree_attn(*dev(q, k, dv, mask), *dev(shape(kp, 128), shape(vp, 128)), torch.tensor(lens, dtype=torch.int32, device=DEV),
                             bt.to(DEV), SCALE, **sc)
    ref = OSP.tree_attention(q, k, dv, mask, *vals, lens, bt, SCALE)
    assert not got.cpu()[3].float().abs().any()
    check_attention(got[:3], [r[:3] for r in ref], lens[:3], fp8, True)
    if T == 1 and fp8:
        got = q3.paged_decode_quant(q[:, 0].to(DEV), *dev(shape(kq, 128), shape(vq, 128)), sc["k_scale"], sc["v_scale"],
                                    torch.tensor(lens, dtype=torch.int32, device=DEV), bt.to(DEV), SCALE)
        assert not got.cpu()[[1, 3]].float().abs().any()
        ref = OSP.tree_attention(q, None, None, None, *vals, lens, bt, SCALE)
        check_attention(got.cpu()[[0, 2], None], [r[[0, 2]] for r in ref], [40, 17], True, False)
    assert q3._lib.read_status() == 0


@pytest.mark.parametrize("n", [2, 300])
def test_rows_that_padding_shares_stay_finite_and_the_others_exact(q3, n):
    """Padded rows of a batch all go to one row that nothing reads: the others land as ever."""
    cache = q3.empty_quant_cache(2 * n, 16, DEV)
    k, v = rows(2 * n, 1), rows(2 * n, 2)
    slots = torch.cat([torch.arange(n) * 16 + 3, torch.zeros(n, dtype=torch.int64)])
    q3.kv_quant_append_slots(k.to(DEV), v.to(DEV), *cache, slots.to(DEV))
    y, e = expect_cache(k[:n])
    got = cache[0].cpu().view(-1, 8, 128)[slots[:n]].float().double()
    assert torch.equal(got, y) and torch.equal(bits(cache[2]).view(-1, 8)[slots[:n]], e)
    kb, vb = q3.kv_dequant_paged(*cache, torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV))
    assert torch.isfinite(kb).all() and torch.isfinite(vb).all() and q3._lib.read_status() == 0
