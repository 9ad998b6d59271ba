"""GPU: the speculative-decoding ops as they are used together (drafted-tree attention over the 8-bit cache, log
probabilities that accept a path, the accepted rows appended, decode over the grown cache), the refusals of the ops, and
calls on streams other than the tensors' own.

Tolerances are those derived in test_gpu_spec.py and test_gpu_logprobs.py; what is said to be equal is compared bit for bit.
"""
import pytest
import torch

from helpers import bits_equal
from oracle import spec as OSP
from test_gpu_spec import BF, DEV, SCALE, check_attention, dev, expect_cache, gen, pools, ref_tree, rows, run_tree, table_for, tree_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def q3():
    import q3attn
    q3attn._lib.load()
    q3attn._lib.read_status()
    return q3attn


@pytest.mark.parametrize("T", [3, 7, 20])
def test_a_speculative_step(q3, T):
    """Two steps of a batch: verify drafts, accept the longest path whose tokens are the likeliest, append its rows,
    verify again over the grown cache; then one plain decode step. Every stage against the oracle."""
    lens, page, vocab = [0, 5, 31, 64, 130, 17], 16, 700
    B = len(lens)
    bt, pages = table_for(lens, page, 3, extra=4)
    cache, _ = pools(pages, page, 4, True)
    cache = dev(*cache)
    g = gen(5)
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    table = bt.to(DEV)
    for step in range(2):
        q = torch.randn(B, T, 16, 128, generator=g).to(BF)
        k, v = rows(B * T, 60 + step, -1, 1).view(B, T, 8, 128), rows(B * T, 70 + step, -3, 2).view(B, T, 8, 128)
        parents = torch.stack([torch.randint(-1, i, (B,), generator=g) if i else torch.full((B,), -1) for i in range(T)], 1)
        drafts = torch.tensor([1 + (b * 5 + step) % T for b in range(B)], dtype=torch.int32)
        mask = q3.tree_mask(parents.to(DEV))
        vals = tuple(OSP.values(c.cpu(), s.cpu()) for c, s in zip(cache[:2], cache[2:]))
        now = seq.cpu().tolist()
        out = q3.paged_tree_attn(*dev(q, k, v), mask, *cache[:2], seq, table, SCALE, k_scale=cache[2], v_scale=cache[3],
                                 draft_lens=drafts.to(DEV))
        ref = OSP.tree_attention(q, k, v, mask.cpu(), *vals, now, bt, SCALE, drafts)
        check_attention(out, ref, [n + T for n in now], True, True)
        # scores of each draft under its parent's output, the drafted token always the likeliest under even parents
        head = torch.randn(2048, vocab, generator=g) / 45
        logits = (out.view(B * T, 2048).float() @ head.to(DEV)).to(BF)
        flat_parent = parents.clamp_min(0) + T * torch.arange(B)[:, None]
        best = logits.float().argmax(-1).cpu()
        ids = torch.where(parents % 2 == 0, best[flat_parent], torch.full_like(parents, -1))
        r = q3.token_logprobs(logits[flat_parent.view(-1).to(DEV)], ids.view(-1).to(DEV), 2)
        want = OSP.logprobs(logits.cpu()[flat_parent.view(-1)], ids.view(-1).clamp_min(0), 2)[0]
        got = r.logprobs.cpu().double()
        known = ids.view(-1) >= 0
        assert (got[~known] == -torch.inf).all()
        # fp32: the logit's difference is exact to 2^-24 of 2^5 here, the sum of 700 terms and its logarithm to 2^-20
        assert ((got - want)[known].abs() <= 2.0 ** -18).all()
        ok = (ids.view(-1) == r.top_ids[:, 0].cpu()).view(B, T)
        pos, seat, src = [], [], []
        for b in range(B):
            path, last = [0], 0           # the first draft is taken, then children that were the likeliest
            for i in range(1, int(drafts[b])):
                if int(parents[b, i]) == last and ok[b, i]:
                    path.append(i)
                    last = i
            for n, i in enumerate(path):
                pos.append(now[b] + n), seat.append(b), src.append(b * T + i)
        flat = lambda x: x.view(B * T, 8, 128)[src]  # noqa: E731
        q3.kv_quant_append_paged(flat(k).to(DEV), flat(v).to(DEV), *cache, torch.tensor(pos, device=DEV), table,
                                 torch.tensor(seat, device=DEV))
        seq = seq + torch.bincount(torch.tensor(seat), minlength=B).to(DEV, torch.int32)
        back = q3.kv_dequant_paged(*cache, torch.tensor(pos, device=DEV), table, torch.tensor(seat, device=DEV))
        for x, b_ in ((flat(k), back[0]), (flat(v), back[1])):
            y, e = expect_cache(x)
            assert torch.equal(b_.cpu().double(), y * torch.exp2(e.double() - 127)[..., None])
    vals = tuple(OSP.values(c.cpu(), s.cpu()) for c, s in zip(cache[:2], cache[2:]))
    q = torch.randn(B, 16, 128, generator=g).to(BF)
    out = q3.paged_decode_quant(q.to(DEV), *cache, seq, table, SCALE)
    ref = OSP.tree_attention(q[:, None], None, None, None, *vals, seq.cpu().tolist(), bt, SCALE)
    check_attention(out[:, None], ref, seq.cpu().tolist(), True, False)
    assert q3._lib.read_status() == 0


def test_chain_of_drafts_is_decoding(q3):
    """A chain of T drafts over the bf16 cache sees what paged_decode sees once the rows are appended, one by one."""
    lens, T, page = [0, 20, 77], 6, 16
    c = tree_case(3, T, lens, page, 21, False)
    kc, vc = dev(*c["cache"][:2])
    q, k, v = dev(c["q"], c["k"], c["v"])
    chain = q3.tree_mask(torch.arange(-1, T - 1, device=DEV))
    seq, bt = torch.tensor(lens, dtype=torch.int32, device=DEV), c["bt"].to(DEV)
    out = q3.paged_tree_attn(q, k, v, chain, kc, vc, seq, bt, SCALE)
    ref = OSP.tree_attention(c["q"], c["k"], c["v"], chain.cpu(), *c["vals"], lens, c["bt"], SCALE)
    check_attention(out, ref, [n + T for n in lens], False, True)
    for t in range(T):
        q3.kv_append_paged(k[:, t].contiguous(), v[:, t].contiguous(), kc, vc, seq + t, bt)
        one = q3.paged_decode(q[:, t].contiguous(), kc, vc, seq + t + 1, bt, SCALE)
        tol = 2 * (ref[0][:, t].abs() * 2.0 ** -8 + ref[1][:, t] * (2.0 ** -10 + 2.0 ** -8))
        assert ((one.cpu().double() - out[:, t].cpu().double()).abs() <= tol).all()


# ------------------------------------------------------------------------------------------------ streams
def test_other_streams(q3):
    """Every op on a side stream, with work queued before it on that stream only, twice at once."""
    c = tree_case(7, 11, [90 + i for i in range(7)], 16, 31, True)
    cache = dev(*c["cache"])
    seq, bt = torch.tensor(c["lens"], dtype=torch.int32, device=DEV), c["bt"].to(DEV)
    q, k, v, m = dev(c["q"], c["k"], c["v"], c["mask"])
    x = torch.randn(40, 9000, generator=gen(2)).to(DEV)
    ids = torch.arange(40, device=DEV)

    def run(q_, x_):
        o = q3.paged_tree_attn(q_, k, v, m, *cache[:2], seq, bt, SCALE, k_scale=cache[2], v_scale=cache[3])
        return [o, q3.paged_decode_quant(q_[:, 0].contiguous(), *cache, seq, bt, SCALE), *q3.token_logprobs(x_, ids, 8),
                *q3.kv_dequant_paged(*cache, seq - 1, bt)]

    eager = run(q, x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                q_, x_ = torch.zeros_like(q), torch.zeros_like(x)
                junk = torch.randn(2048, 2048, device=DEV)
                for _ in range(4):
                    junk = junk @ junk * 0.01
                q_.copy_(q), x_.copy_(x)
                got.append(run(q_, x_))
        torch.cuda.synchronize()
        for outs in got:
            assert all(bits_equal(a, b) for a, b in zip(outs, eager))


def test_graph_of_a_step_with_growing_lengths(q3):
    """One captured graph of append + decode + scores, replayed while the lengths it reads grow: the plan is made on the
    device, so every replay serves the lengths of its own time."""
    page, B = 16, 5
    lens = [0, 14, 15, 40, 100]
    bt, pages = table_for(lens, page, 8, extra=3)
    cache, _ = pools(pages, page, 9, True)
    cache = dev(*cache)
    table = bt.to(DEV)
    pos = torch.tensor(lens, dtype=torch.int32, device=DEV)
    seq = pos + 1
    k, v = torch.zeros(B, 8, 128, dtype=BF, device=DEV), torch.zeros(B, 8, 128, dtype=BF, device=DEV)
    q = torch.zeros(B, 16, 128, dtype=BF, device=DEV)
    w = (torch.randn(2048, 300, generator=gen(1)) / 45).to(DEV, BF)
    ids = torch.zeros(B, dtype=torch.int64, device=DEV)

    def step():
        q3.kv_quant_append_paged(k, v, *cache, pos, table)
        o = q3.paged_decode_quant(q, *cache, seq, table, SCALE)
        return o, q3.token_logprobs(o.view(B, 2048) @ w, ids, 3)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, sc = step()
    for t in range(6):
        kk, vv, qq = rows(B, 200 + t, -1, 1), rows(B, 300 + t, -3, 1), torch.randn(B, 16, 128, generator=gen(t)).to(BF)
        k.copy_(kk), v.copy_(vv), q.copy_(qq)
        pos.copy_(torch.tensor(lens, dtype=torch.int32) + t)
        seq.copy_(pos + 1)
        graph.replay()
        vals = tuple(OSP.values(c_.cpu(), s.cpu()) for c_, s in zip(cache[:2], cache[2:]))
        now = seq.cpu().tolist()
        for b in range(B):
            y, e = expect_cache(kk[b:b + 1])
            row = OSP.rows_of(vals[0], bt[b], now[b])[-1]
            assert torch.equal(row, y[0] * torch.exp2(e[0].double() - 127)[..., None])
        ref = OSP.tree_attention(qq[:, None], None, None, None, *vals, now, bt, SCALE)
        check_attention(out[:, None], ref, now, True, False)
        top = torch.sort((out.view(B, 2048) @ w).float(), dim=-1, descending=True, stable=True)[1][:, :3]
        assert torch.equal(sc.top_ids, top)


def test_compiled_step(q3):
    """append + tree attention + scores under torch.compile (one graph, functionalised) give what eager calls give."""
    c = tree_case(3, 5, [20, 0, 33], 16, 39, True)
    seq, bt = torch.tensor(c["lens"], dtype=torch.int32, device=DEV), c["bt"].to(DEV)
    q, k, v, m = dev(c["q"], c["k"], c["v"], c["mask"])
    w = (torch.randn(2048, 300, generator=gen(3)) / 45).to(DEV, BF)
    ids = torch.arange(15, device=DEV)

    def step(kc, vc, ks, vs):
        o = q3.paged_tree_attn(q, k, v, m, kc, vc, seq, bt, SCALE, k_scale=ks, v_scale=vs)
        q3.kv_quant_append_paged(k[:, 0], v[:, 0], kc, vc, ks, vs, seq, bt)
        o1 = q3.paged_decode_quant(q[:, 0], kc, vc, ks, vs, seq + 1, bt, SCALE)
        return (o, o1, *q3.token_logprobs(o.view(15, 2048) @ w, ids, 4))

    a, b = dev(*c["cache"]), dev(*c["cache"])
    want = step(*a)
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(*b)
    assert all(bits_equal(x, y) for x, y in zip(got, want))
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


# ------------------------------------------------------------------------------------------------ arguments
@pytest.mark.parametrize("fp8,T", [(True, 3), (True, 12), (True, 30), (False, 3), (False, 30)])
@pytest.mark.parametrize("scale", [0.0, -0.05])
def test_scales_that_are_not_positive(q3, fp8, T, scale):
    c = tree_case(4, T, [0, 9, 33, 70], 16, 41, fp8)
    kc, vc, ks, vs = dev(*c["cache"])
    got = q3.paged_tree_attn(*dev(c["q"], c["k"], c["v"], c["mask"]), kc, vc,
                             torch.tensor(c["lens"], dtype=torch.int32, device=DEV), c["bt"].to(DEV), scale, k_scale=ks, v_scale=vs)
    ref = OSP.tree_attention(c["q"], c["k"], c["v"], c["mask"], *c["vals"], c["lens"], c["bt"], scale)
    check_attention(got, ref, [n + T for n in c["lens"]], fp8, True)


def test_one_seat_with_odd_strides(q3):
    """A batch of one, whose seat strides mean nothing."""
    c = tree_case(1, 5, [50], 16, 43, False)
    q, k, v = dev(c["q"], c["k"], c["v"])
    seq, bt = torch.tensor([50], dtype=torch.int32, device=DEV), c["bt"].to(DEV)
    kc, vc = dev(*c["cache"][:2])
    m = c["mask"].to(DEV)
    want = q3.paged_tree_attn(q, k, v, m, kc, vc, seq, bt, SCALE)
    odd = [x.as_strided(x.shape, (7, *x.stride()[1:])) for x in (q, k, v)]
    assert bits_equal(q3.paged_tree_attn(*odd, m, kc, vc, seq, bt, SCALE), want)


def test_shared_rows_by_stride_zero(q3):
    """Seats that share their drafted rows and queries through a stride of zero."""
    c = tree_case(3, 6, [30, 0, 12], 16, 44, True)
    one = [c[n][:1] for n in ("q", "k", "v")]
    kc, vc, ks, vs = dev(*c["cache"])
    seq, bt = torch.tensor(c["lens"], dtype=torch.int32, device=DEV), c["bt"].to(DEV)
    exp = [x.to(DEV).expand(3, -1, -1, -1) for x in one]
    got = q3.paged_tree_attn(*exp, c["mask"][0].to(DEV), kc, vc, seq, bt, SCALE, k_scale=ks, v_scale=vs)
    ref = OSP.tree_attention(*(x.expand(3, -1, -1, -1) for x in one), c["mask"][0], *c["vals"], c["lens"], c["bt"], SCALE)
    check_attention(got, ref, [n + 6 for n in c["lens"]], True, True)


def test_refusals(q3):
    c = tree_case(2, 4, [5, 9], 16, 51, True)
    kc, vc, ks, vs = cache = dev(*c["cache"])
    q, k, v, m = dev(c["q"], c["k"], c["v"], c["mask"])
    seq, bt = torch.tensor([5, 9], dtype=torch.int32, device=DEV), c["bt"].to(DEV)

    def tree(**o):
        a = {**dict(q=q, k=k, v=v, m=m, kc=kc, vc=vc, seq=seq, bt=bt, ks=ks, vs=vs, d=None), **o}
        return q3.paged_tree_attn(a["q"], a["k"], a["v"], a["m"], a["kc"], a["vc"], a["seq"], a["bt"], SCALE, k_scale=a["ks"],
                                  v_scale=a["vs"], draft_lens=a["d"])

    big = lambda x: x.repeat(1, 17, 1, 1)[:, :65]  # noqa: E731
    for o in (dict(q=q.half()), dict(q=q[:, :, :8]), dict(q=q[0]), dict(k=k.float()), dict(k=k[:, :3]), dict(v=v[:1]),
              dict(m=m.int()), dict(m=m[:, :3]), dict(m=m[:1]), dict(kc=kc.view(torch.uint8)), dict(ks=None),
              dict(ks=None, vs=None), dict(ks=ks.view(torch.uint8)), dict(ks=ks[:1]), dict(kc=kc.transpose(0, 1)),
              dict(seq=seq.long()), dict(seq=seq[:1]), dict(bt=bt.long()), dict(bt=bt[:1]), dict(bt=bt.t().contiguous().t()),
              dict(d=seq.long()), dict(d=seq[:1]), dict(q=q.cpu()), dict(k=k.cpu()), dict(seq=seq.cpu()), dict(m=m.cpu()),
              dict(q=big(q), k=big(k), v=big(v), m=m.repeat(1, 17)[:, :65]), dict(q=q[:, :0], k=k[:, :0], v=v[:, :0], m=m[:, :0])):
        with pytest.raises(RuntimeError, match="q3"):
            tree(**o)
    rows_ = k[:, 0].contiguous()
    pos = torch.zeros(2, dtype=torch.int32, device=DEV)
    for bad in (lambda: q3.kv_quant_append_paged(rows_.float(), rows_, *cache, pos, bt),
                lambda: q3.kv_quant_append_paged(rows_[:, :4], rows_[:, :4], *cache, pos, bt),
                lambda: q3.kv_quant_append_paged(rows_, rows_, *cache, pos[:1], bt),
                lambda: q3.kv_quant_append_paged(rows_, rows_, *cache, pos.float(), bt),
                lambda: q3.kv_quant_append_paged(rows_, rows_, *cache, pos, bt[:1]),
                lambda: q3.kv_quant_append_slots(rows_, rows_, *cache, pos[:1]),
                lambda: q3.kv_quant_append_slots(rows_, rows_, *cache[2:], *cache[:2], pos),
                lambda: q3.kv_dequant_paged(*cache, pos, bt.cpu()),
                lambda: q3.kv_dequant_paged(*cache, torch.zeros(3, dtype=torch.int32, device=DEV), bt),
                lambda: q3.paged_decode_quant(q, *cache, seq, bt, SCALE),
                lambda: q3.paged_decode_quant(q[:1, 0], *cache, seq, bt, SCALE)):
        with pytest.raises(RuntimeError, match="q3"):
            bad()
    x, ids = torch.randn(4, 50, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    for bad in (lambda: q3.token_logprobs(x.double(), ids), lambda: q3.token_logprobs(x[0], ids), lambda: q3.token_logprobs(x, ids.int()),
                lambda: q3.token_logprobs(x, ids[:3]), lambda: q3.token_logprobs(x, ids, 51), lambda: q3.token_logprobs(x, ids, -1),
                lambda: q3.token_logprobs(x.repeat(1, 2), ids, 65), lambda: q3.token_logprobs(x, ids, 0, 0.0),
                lambda: q3.token_logprobs(x, ids, 0, float("inf")), lambda: q3.token_logprobs(x, ids, 0, float("nan")),
                lambda: q3.token_logprobs(x, ids.cpu()), lambda: q3.token_logprobs(x[:, :0], ids)):
        with pytest.raises(RuntimeError, match="q3"):
            bad()
    torch.cuda.synchronize()
    assert q3._lib.read_status() == 0


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T", [9, 33, 64])
@pytest.mark.parametrize("lens", [[0] * 300, [0, 64, 0, 0, 65, 0, 0, 0, 64, 1] * 40, [128 if i % 7 == 0 else 0 for i in range(200)]])
def test_short_seats_of_many_tokens(q3, fp8, T, lens):
    """Many seats per CTA of one tile (the drafted rows) or a few."""
    c = tree_case(len(lens), T, lens, 64, 71, fp8, drafts=[1 + (5 * i) % T for i in range(len(lens))])
    got = run_tree(q3, c)
    check_attention(got, ref_tree(c), [n + T for n in lens], fp8, True)
    assert q3._lib.read_status() == 0


def test_many_seats(q3):
    """More seats than threads of the planning pass, most of them padding: no rows, no drafts, a table of -1."""
    B, T = 5000, 2
    lens, g = [0] * B, gen(62)
    for b in range(0, B, 61):
        lens[b] = 1 + b % 70
    drafts = torch.tensor([1 + b % 2 if b % 61 == 0 or b % 7 == 0 else 0 for b in range(B)], dtype=torch.int32)
    bt = torch.randint(0, 64, (B, 5), generator=g).to(torch.int32)
    bt[torch.tensor(lens) == 0] = -1
    cache, vals = pools(64, 16, 63, True)
    q, k, v = torch.randn(B, T, 16, 128, generator=g).to(BF), rows(B * T, 64, -1, 1).view(B, T, 8, 128), rows(B * T, 65, -3, 2).view(B, T, 8, 128)
    mask = torch.tensor([1, 3])
    kc, vc, ks, vs = dev(*cache)
    got = q3.paged_tree_attn(*dev(q, k, v, mask), kc, vc, torch.tensor(lens, dtype=torch.int32, device=DEV), bt.to(DEV), SCALE,
                             k_scale=ks, v_scale=vs, draft_lens=drafts.to(DEV))
    ref = OSP.tree_attention(q, k, v, mask, *vals, lens, bt, SCALE, drafts)
    check_attention(got, ref, [n + T for n in lens], True, True)
    assert q3._lib.read_status() == 0


def test_a_chunk_of_a_prompt_over_an_8_bit_prefix(q3):
    """A prompt in two chunks over the 8-bit cache: the first chunk's rows are appended, read back as bf16 ahead of the
    second chunk's own rows, and `prefill` attends over both (causal, aligned to the end)."""
    first, second, page = [40, 0, 17, 130], [5, 33, 1, 70], 16
    B = len(first)
    bt, pages = table_for([a + b for a, b in zip(first, second)], page, 5)
    cache, table = q3.empty_quant_cache(pages, page, DEV), bt.to(DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    k1, v1 = rows(sum(first), 1, -1, 1), rows(sum(first), 2, -3, 2)
    pos = i32([p for n in first for p in range(n)])
    seat = i32([b for b, n in enumerate(first) for _ in range(n)])
    q3.kv_quant_append_paged(k1.to(DEV), v1.to(DEV), *cache, pos, table, seat)
    kp, vp = q3.kv_dequant_paged(*cache, pos, table, seat)
    k2, v2 = rows(sum(second), 3, -1, 1), rows(sum(second), 4, -3, 2)
    q = torch.randn(sum(second), 16, 128, generator=gen(6)).to(BF)
    split = lambda x, n: torch.split(x, n)  # noqa: E731
    join = lambda a, b: torch.cat([x for p in zip(split(a, first), split(b, second)) for x in p])  # noqa: E731
    cu = lambda n: torch.nn.functional.pad(torch.cumsum(torch.tensor(n), 0), (1, 0)).to(DEV, torch.int32)  # noqa: E731
    out = q3.prefill(q.to(DEV), join(kp, k2.to(DEV)), join(vp, v2.to(DEV)), cu(second), cu([a + b for a, b in zip(first, second)]),
                     max(second), SCALE).cpu()
    for b, (got, q_) in enumerate(zip(split(out, second), split(q, second))):
        n, m = first[b], second[b]
        keys = torch.cat([split(kp.cpu(), first)[b], split(k2, second)[b]]).double()
        vals = torch.cat([split(vp.cpu(), first)[b], split(v2, second)[b]]).double()
        see = torch.arange(n + m)[None] <= n + torch.arange(m)[:, None]
        ref = [r[None] for r in OSP.attend(q_, keys, vals, see, SCALE)]
        check_attention(got[None], ref, [n + m], False, True)
    # the second chunk's rows follow the first's, and the next token attends over all of them
    q3.kv_quant_append_paged(k2.to(DEV), v2.to(DEV), *cache, i32([n + p for n, m in zip(first, second) for p in range(m)]), table,
                             i32([b for b, m in enumerate(second) for _ in range(m)]))
    vals = tuple(OSP.values(c.cpu(), s.cpu()) for c, s in zip(cache[:2], cache[2:]))
    lens = [a + b for a, b in zip(first, second)]
    q1 = torch.randn(B, 16, 128, generator=gen(7)).to(BF)
    one = q3.paged_decode_quant(q1.to(DEV), *cache, i32(lens), table, SCALE)
    check_attention(one[:, None], OSP.tree_attention(q1[:, None], None, None, None, *vals, lens, bt, SCALE), lens, True, False)
    assert q3._lib.read_status() == 0
