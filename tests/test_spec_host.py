"""CPU: the 8-bit cache, drafted-tree and log-probability entries refuse bad arguments on the host before any CUDA call;
their ops have shape rules, refuse CPU tensors and trace as single nodes; visibility words and the 64-bit oracle are what
their formulas say."""
import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import q3attn
from oracle import spec as OSP
from q3attn import _lib
from q3attn.spec import BF16, E4M3, E8M0, _op

OK, INVALID, ALIGN, UNSUPPORTED, WORKSPACE = (_lib.Q3_OK, _lib.Q3_ERR_INVALID, _lib.Q3_ERR_ALIGNMENT,
                                              _lib.Q3_ERR_UNSUPPORTED, _lib.Q3_ERR_WORKSPACE)
A = 1 << 12   # an aligned address that nothing reads: every call below is refused first


# ------------------------------------------------------------------------------------------------ the C entries
def cache(**over):
    return _lib.QuantCache(**{**dict(k=A, v=A, k_scale=A, v_scale=A, num_pages=10, page_size=16), **over})


CACHE_BAD = [(dict(k=None), INVALID), (dict(v_scale=None), INVALID), (dict(num_pages=0), INVALID),
             (dict(page_size=-1), INVALID), (dict(k=A + 8), ALIGN), (dict(k_scale=A + 8), ALIGN)]


@pytest.mark.parametrize("over,code", CACHE_BAD)
def test_rows_refuse_bad_caches(over, code):
    lib, c = _lib.load(), ctypes.byref(cache(**over))
    assert lib.q3_kv_quant_append_slots(A, A, 1024, c, 8, 128, A, 3, None) == code
    assert lib.q3_kv_quant_append_paged(A, A, 1024, c, 8, 128, A, None, A, 4, 3, 4, 3, None) == code
    assert lib.q3_kv_dequant_paged(c, 8, 128, A, None, A, 4, 3, 4, A, A, 1024, 3, None) == code


def test_rows_refuse_bad_arguments():
    lib, c = _lib.load(), ctypes.byref(cache())
    slots = lambda k=A, v=A, st=1024, nkv=8, hd=128, s=A, n=3: lib.q3_kv_quant_append_slots(k, v, st, c, nkv, hd, s, n, None)  # noqa: E731
    assert slots(n=-1) == slots(s=None) == slots(k=None) == slots(v=None) == slots(st=1016) == INVALID
    assert slots(nkv=4) == slots(hd=64) == UNSUPPORTED
    assert slots(k=A + 2) == slots(v=A + 8) == slots(st=1028) == ALIGN
    assert slots(n=0, s=None, k=None) == OK
    paged = lambda pos=A, bt=A, bs=4, seats=3, mp=4, n=3: lib.q3_kv_quant_append_paged(A, A, 1024, c, 8, 128, pos, None, bt, bs, seats, mp, n, None)  # noqa: E731
    assert paged(pos=None) == paged(bt=None) == paged(bs=3) == paged(seats=0) == paged(mp=0) == paged(n=-2) == INVALID
    assert paged(n=0, pos=None) == OK
    back = lambda out=A, st=1024, n=3, bs=4: lib.q3_kv_dequant_paged(c, 8, 128, A, None, A, bs, 3, 4, out, A, st, n, None)  # noqa: E731
    assert back(out=None) == back(st=512) == back(n=-1) == back(bs=2) == INVALID
    assert back(out=A + 4) == back(st=1025) == ALIGN
    assert back(n=0, out=None) == OK


def tree(ws=A, nbytes=1 << 40, **over):
    base = dict(q=A, q_seat_stride=5 * 2048, q_token_stride=2048, k_new=A, v_new=A, kv_new_seat_stride=5 * 1024,
                kv_new_token_stride=1024, tree_mask=A, tree_mask_stride=5, draft_lens=None, k_pool=A, v_pool=A,
                k_scale=None, v_scale=None, num_pages=10, page_size=16, cache_seqlens=A, block_table=A,
                block_table_stride=4, max_pages_per_seat=4, batch=3, tokens=5, num_heads=16, num_kv_heads=8,
                head_dim=128, softmax_scale=0.1, out=A, out_seat_stride=5 * 2048, out_token_stride=2048)
    return _lib.load().q3_paged_tree_attn(ctypes.byref(_lib.TreeAttn(**{**base, **over})), ws, nbytes, None)


@pytest.mark.parametrize("over,code", [
    (dict(num_heads=32), UNSUPPORTED), (dict(num_kv_heads=16), UNSUPPORTED), (dict(head_dim=64), UNSUPPORTED),
    (dict(tokens=65), UNSUPPORTED), (dict(tokens=0), INVALID), (dict(batch=-1), INVALID), (dict(num_pages=0), INVALID),
    (dict(page_size=0), INVALID), (dict(max_pages_per_seat=0), INVALID), (dict(q=None), INVALID), (dict(out=None), INVALID),
    (dict(cache_seqlens=None), INVALID), (dict(block_table=None), INVALID), (dict(k_new=None), INVALID),
    (dict(v_new=None), INVALID), (dict(k_scale=A), INVALID), (dict(tree_mask=None), INVALID),
    (dict(q_token_stride=2040), INVALID), (dict(out_token_stride=1024), INVALID), (dict(q_seat_stride=-2048), INVALID),
    (dict(kv_new_token_stride=512), INVALID), (dict(kv_new_seat_stride=-8), INVALID), (dict(tree_mask_stride=-1), INVALID),
    (dict(block_table_stride=3), INVALID), (dict(max_pages_per_seat=1 << 27, block_table_stride=1 << 27), INVALID),
    (dict(batch=1 << 30), INVALID), (dict(q=A + 8), ALIGN), (dict(out=A + 2), ALIGN), (dict(k_pool=A + 8), ALIGN),
    (dict(k_new=A + 8), ALIGN), (dict(tree_mask=A + 4), ALIGN), (dict(q_seat_stride=10244), ALIGN),
    (dict(out_token_stride=2050), ALIGN), (dict(kv_new_seat_stride=5121), ALIGN), (dict(k_scale=A + 8, v_scale=A), ALIGN)])
def test_tree_refuses_bad_arguments(over, code):
    assert tree(**over) == code


def test_tree_empty_and_null():
    assert tree(batch=0, q=None, out=None) == OK
    assert _lib.load().q3_paged_tree_attn(None, A, 1 << 40, None) == INVALID


def scores(**over):
    base = dict(logits=A, logits_dtype=0, row_stride=100, rows=4, vocab=100, temperature=1.0, ids=A, ids_row_stride=2,
                given=2, logprobs=A, entropy=None, top_n=3, top_ids=A, top_logprobs=A)
    return _lib.load().q3_token_logprobs(ctypes.byref(_lib.Logprobs(**{**base, **over})), None)


@pytest.mark.parametrize("over,code", [
    (dict(rows=-1), INVALID), (dict(rows=(1 << 27) + 1), INVALID), (dict(vocab=0), INVALID),
    (dict(vocab=(1 << 30) + 1), INVALID), (dict(given=-1), INVALID), (dict(top_n=-1), INVALID), (dict(top_n=101), INVALID),
    (dict(top_n=65), UNSUPPORTED), (dict(temperature=0.0), INVALID), (dict(temperature=-1.0), INVALID),
    (dict(temperature=math.nan), INVALID), (dict(temperature=math.inf), INVALID), (dict(temperature=1e-31), INVALID),
    (dict(logits_dtype=3), INVALID), (dict(logits=None), INVALID), (dict(row_stride=99), INVALID), (dict(ids=None), INVALID),
    (dict(logprobs=None), INVALID), (dict(ids_row_stride=1), INVALID), (dict(top_ids=None), INVALID),
    (dict(top_logprobs=None), INVALID), (dict(logits=A + 1), ALIGN), (dict(logits_dtype=1, logits=A + 2), ALIGN),
    (dict(ids=A + 4), ALIGN), (dict(logprobs=A + 2), ALIGN), (dict(entropy=A + 1), ALIGN), (dict(top_ids=A + 4), ALIGN)])
def test_logprobs_refuse_bad_arguments(over, code):
    assert scores(**over) == code


def test_logprobs_without_rows():
    assert scores(rows=0, logits=None) == OK
    assert _lib.load().q3_token_logprobs(None, None) == INVALID


# ------------------------------------------------------------------------------------------------ the ops
def test_ops_refuse_cpu_tensors():
    c = q3attn.empty_quant_cache(3, 16, "cpu")
    k = torch.zeros(2, 8, 128, dtype=BF16)
    i, bt, seq = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(2, 1, 16, 128, dtype=BF16)
    for call in (lambda: q3attn.kv_quant_append_slots(k, k, *c, i.long()),
                 lambda: q3attn.kv_quant_append_paged(k, k, *c, i, bt),
                 lambda: q3attn.kv_dequant_paged(*c, i, bt),
                 lambda: q3attn.paged_decode_quant(q[:, 0], *c, seq, bt, 0.1),
                 lambda: q3attn.paged_tree_attn(q, k[:, None], k[:, None], torch.ones(2, 1, dtype=torch.int64), *c[:2], seq,
                                                bt, 0.1, k_scale=c[2], v_scale=c[3]),
                 lambda: q3attn.token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def e(*shape, dtype=BF16):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def test_op_shapes():
    _op("token_logprobs")
    i32, i64 = torch.int32, torch.int64
    with FakeTensorMode():
        c = (e(40, 16, 8, 128, dtype=E4M3), e(40, 16, 8, 128, dtype=E4M3), e(40, 16, 8, dtype=E8M0), e(40, 16, 8, dtype=E8M0))
        B, T = 5, 7
        seq, bt = e(B, dtype=i32), e(B, 8, dtype=i32)
        assert q3attn.kv_quant_append_slots(e(9, 8, 128), e(9, 8, 128), *c, e(9, dtype=i64)) is None
        assert q3attn.kv_quant_append_paged(e(9, 8, 128), e(9, 8, 128), *c, e(9, dtype=i32), bt, e(9, dtype=i32)) is None
        for o in q3attn.kv_dequant_paged(*c, e(9, dtype=i32), bt, e(9, dtype=i32)):
            assert o.shape == (9, 8, 128) and o.dtype == BF16
        o = q3attn.paged_decode_quant(e(B, 16, 128), *c, seq, bt, 0.1)
        assert o.shape == (B, 16, 128) and o.dtype == BF16
        o = q3attn.paged_tree_attn(e(B, T, 16, 128), e(B, T, 8, 128), e(B, T, 8, 128), e(B, T, dtype=i64), *c[:2], seq, bt,
                                   0.1, k_scale=c[2], v_scale=c[3])
        assert o.shape == (B, T, 16, 128) and o.dtype == BF16 and o.is_contiguous()
        r = q3attn.token_logprobs(e(6, 500, dtype=torch.float16), e(6, 2, dtype=i64), 4)
        assert [(x.shape, x.dtype) for x in r] == [((6, 2), torch.float32), ((6,), torch.float32), ((6, 4), i64),
                                                   ((6, 4), torch.float32)]


def test_ops_trace_as_single_nodes():
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(q, k, v, mask, kc, vc, ks, vs, seq, bt, logits, ids):
        o = q3attn.paged_tree_attn(q, k, v, mask, kc, vc, seq, bt, 0.1, k_scale=ks, v_scale=vs)
        q3attn.kv_quant_append_paged(k[:, 0], v[:, 0], kc, vc, ks, vs, seq, bt)
        return o.float().sum() + q3attn.token_logprobs(logits, ids).logprobs.sum()

    _op("token_logprobs")
    with FakeTensorMode():
        g = make_fx(step, tracing_mode="fake")(
            e(3, 4, 16, 128), e(3, 4, 8, 128), e(3, 4, 8, 128), e(3, 4, dtype=torch.int64), e(20, 16, 8, 128, dtype=E4M3),
            e(20, 16, 8, 128, dtype=E4M3), e(20, 16, 8, dtype=E8M0), e(20, 16, 8, dtype=E8M0), e(3, dtype=torch.int32),
            e(3, 4, dtype=torch.int32), e(6, 500), e(6, dtype=torch.int64))
    targets = [str(n.target) for n in g.graph.nodes if n.op == "call_function"]
    for op in ("paged_tree_attn", "kv_quant_append_paged", "token_logprobs"):
        assert targets.count(f"q3attn.{op}.default") == 1, targets
    assert not any("softmax" in t or "matmul" in t for t in targets)


def test_first_call_from_a_compiled_function():
    """In a process of its own: torch.compile traces the op's very first call as one graph (the CPU tensors are refused
    when it runs)."""
    src = ("import sys; sys.path.insert(0, sys.argv[1])\nimport torch, q3attn\n"
           "f = torch.compile(lambda x, i: q3attn.token_logprobs(x * 2, i, 3, 0.9).logprobs + 1, fullgraph=True, backend='eager')\n"
           "try:\n    f(torch.randn(4, 50), torch.zeros(4, dtype=torch.int64))\n"
           "except RuntimeError as e:\n    print('refused' if 'must be a CUDA tensor' in str(e) else repr(e))\n")
    pkg = os.path.dirname(os.path.dirname(os.path.abspath(_lib.__file__)))
    r = subprocess.run([sys.executable, "-c", src, pkg], capture_output=True, text=True, timeout=300)
    assert r.stdout.strip() == "refused", r.stdout + r.stderr[-2000:]


# ------------------------------------------------------------------------------------------------ visibility words
@pytest.mark.parametrize("T", [1, 2, 9, 63, 64])
def test_tree_mask_is_the_ancestors(T):
    g = torch.Generator().manual_seed(T)
    parents = torch.stack([torch.randint(-1, i, (4,), generator=g) if i else torch.full((4,), -1) for i in range(T)], 1)
    words = q3attn.tree_mask(parents)
    assert words.shape == (4, T) and words.dtype == torch.int64
    for b in range(4):
        for i in range(T):
            want, j = set(), i
            while j >= 0:
                want.add(j)
                j = int(parents[b, j])
            assert {j for j in range(64) if (int(words[b, i]) >> j) & 1} == want
    assert torch.equal(q3attn.tree_mask(parents[2].int()), words[2])


def test_tree_mask_chain_and_refusals():
    chain = q3attn.tree_mask(torch.arange(-1, 63))
    assert chain.tolist() == [(1 << (i + 1)) - 1 for i in range(63)] + [-1]
    # a parent that is not earlier than its child counts as none
    assert q3attn.tree_mask(torch.tensor([0, 5, 1])).tolist() == [1, 2, 6]
    for bad in (torch.zeros(65, dtype=torch.int64), torch.zeros(2, 0, dtype=torch.int64), torch.tensor(1)):
        with pytest.raises(RuntimeError, match="tokens a tree"):
            q3attn.tree_mask(bad)


# ------------------------------------------------------------------------------------------------ the oracle
def test_oracle_rounding_is_the_types():
    """Every finite e4m3 number is kept, and midpoints go to the even one."""
    all_bytes = torch.arange(256, dtype=torch.uint8).view(E4M3).float().double()
    x = all_bytes[torch.isfinite(all_bytes)]
    assert torch.equal(OSP.round_e4m3(x), x)
    pos = x[x >= 0].sort().values.unique()
    mid = (pos[1:] + pos[:-1]) / 2
    assert torch.equal(OSP.round_e4m3(mid), mid.float().to(E4M3).double())


def test_oracle_scale_is_the_least():
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(200, 128, generator=g) * torch.exp2(torch.randint(-80, 80, (200, 1), generator=g).float())).to(BF16)
    y, ex = OSP.quantise(x)
    top = x.double().abs().amax(-1)
    assert (top <= 448 * torch.exp2(ex.double())).all() and (top > 448 * torch.exp2(ex.double() - 1)).all()
    assert ((y * torch.exp2(ex.double())[:, None] - x.double()).abs()
            <= torch.maximum(x.double().abs() * 2.0 ** -4, torch.exp2(ex.double() - 10)[:, None])).all()


def test_oracle_attention_is_the_library_softmax():
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(n, h, 128, generator=g).double() for n, h in ((6, 16), (9, 8), (9, 8)))
    see = torch.rand(6, 9, generator=g) > 0.4
    see[2] = False
    out = OSP.attend(q, k, v, see, 0.1)[0]
    rep = lambda x: x.double().repeat_interleave(2, 1).transpose(0, 1)  # noqa: E731
    ref = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(0, 1), rep(k), rep(v), attn_mask=see,
                                                           scale=0.1).transpose(0, 1).nan_to_num()
    assert (out - ref).abs().max() < 1e-12 and not out[2].any()


def test_oracle_logprobs_are_log_softmax():
    x = torch.randn(5, 40, generator=torch.Generator().manual_seed(5))
    x[0, 3] = -math.inf
    lp, ent, ids, tl = OSP.logprobs(x, torch.arange(5), 4, 0.7)
    ref = torch.log_softmax(x.double() / 0.7, -1)
    assert (lp - ref.gather(1, torch.arange(5)[:, None])[:, 0]).abs().max() < 1e-12
    assert (ent - torch.special.entr(ref.exp()).sum(-1)).abs().max() < 1e-12
    assert torch.equal(tl, ref.topk(4).values) or (tl - ref.topk(4).values).abs().max() < 1e-12
    assert torch.equal(ids, x.topk(4).indices)


def test_the_merge_alone_refuses_what_the_call_refuses():
    lib = _lib.load()
    call = lambda p, ws=A, n=1 << 40: lib.q3_selftest_tree_merge(p, ws, n, None)  # noqa: E731
    one = lambda **kw: ctypes.byref(_lib.TreeAttn(**{**dict(  # noqa: E731
        q=A, q_seat_stride=2048, q_token_stride=2048, k_pool=A, v_pool=A, num_pages=1, page_size=16, cache_seqlens=A, block_table=A,
        block_table_stride=1, max_pages_per_seat=1, batch=1, tokens=1, num_heads=16, num_kv_heads=8, head_dim=128,
        softmax_scale=0.1, out=A, out_seat_stride=2048, out_token_stride=2048), **kw}))
    assert call(None) == call(one(q=None)) == call(one(tokens=0)) == call(one(block_table_stride=0)) == INVALID
    assert call(one(tokens=65)) == call(one(head_dim=64)) == UNSUPPORTED
    assert call(one(out=A + 8)) == ALIGN
    assert call(one(batch=0, q=None)) == OK
