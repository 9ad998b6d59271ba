"""GPU: the failure reporting every pipeline kernel shares. A bounded wait that expires must raise
Q3_STATUS_WAIT_TIMEOUT and return, leaving the context usable for the next call. The wait is made to expire on
purpose, with an mbarrier that nothing arrives on; nothing faults, traps or waits without a limit."""
import ctypes

import pytest
import torch

from helpers import assert_close_attn
from oracle import attention as OA
from q3attn import synth

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def q3():
    import q3attn
    q3attn._lib.load()
    return q3attn


def test_expired_wait_reports_and_the_context_stays_usable(q3):
    lib = q3._lib.load()
    q3._lib.read_status(clear=True)
    torch.cuda.synchronize()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.q3_selftest_bounded_wait(ctypes.c_uint64(1_000_000), stream) == 0   # 1 ms
    torch.cuda.synchronize()
    assert q3._lib.read_status(clear=True) & q3._lib.STATUS_WAIT_TIMEOUT
    # limits outside 1 ns .. 100 ms are refused on the host, before any launch
    assert lib.q3_selftest_bounded_wait(ctypes.c_uint64(0), stream) != 0
    assert lib.q3_selftest_bounded_wait(ctypes.c_uint64(200_000_000), stream) != 0
    # the next call on the same context is correct and raises nothing
    lay = synth.paged_layout(3, B=6, ctx_lo=1, ctx_hi=300, page=16, pages_per_seat=20)
    d = synth.decode_case(3, lay, scale=0.5)
    dd = {k: v.to(DEV) for k, v in d.items()}
    out = q3.paged_decode(dd["q"], dd["k_pool"], dd["v_pool"], lay.ctx.to(DEV), lay.block_table.to(DEV), 128 ** -0.5, 0)
    torch.cuda.synchronize()
    assert q3._lib.read_status(clear=True) == 0
    ref = OA.decode_attention(d["q"], d["k_pool"], d["v_pool"], lay.ctx, lay.block_table, 128 ** -0.5)
    assert_close_attn(out, ref, what="decode after an expired wait")


def tree_call(q3, B, T, fp8, fill, seed=5):
    """Arguments of a drafted-tree call over 40-token seats (host struct), its workspace (filled by `fill`) and tensors."""
    import oracle.spec as OSP
    g = torch.Generator().manual_seed(seed)
    bt = torch.randperm(3 * B, generator=g).view(B, 3).to(torch.int32).to(DEV)
    q = torch.randn(B, T, 16, 128, generator=g).to(torch.bfloat16).to(DEV)
    k, v = (torch.randn(B, T, 8, 128, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    pool = [torch.randn(3 * B * 16, 8, 128, generator=g).to(torch.bfloat16) for _ in range(2)]
    scales = [None, None]
    if fp8:
        pool, scales = zip(*[(y.float().to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)) for y, e in map(OSP.quantise, pool)])
    pool, scales = [x.to(DEV) for x in pool], [None if s is None else s.to(DEV) for s in scales]
    mask = q3.tree_mask(torch.arange(T) - 1).to(DEV)
    lens = torch.full((B,), 40, dtype=torch.int32, device=DEV)
    out = torch.full((B, T, 16, 128), 77.0, dtype=torch.bfloat16, device=DEV)
    lib = q3._lib.load()
    n = lib.q3_paged_tree_workspace_bytes(B, T, int(fp8))
    ws = fill(n).to(DEV)
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    args = q3._lib.TreeAttn(q=p(q), q_seat_stride=T * 2048, q_token_stride=2048, k_new=p(k), v_new=p(v),
                            kv_new_seat_stride=T * 1024, kv_new_token_stride=1024, tree_mask=p(mask), tree_mask_stride=0,
                            k_pool=p(pool[0]), v_pool=p(pool[1]), k_scale=p(scales[0]), v_scale=p(scales[1]),
                            num_pages=3 * B, page_size=16, cache_seqlens=p(lens), block_table=p(bt), block_table_stride=3,
                            max_pages_per_seat=3, batch=B, tokens=T, num_heads=16, num_kv_heads=8, head_dim=128,
                            softmax_scale=128 ** -0.5, out=p(out), out_seat_stride=T * 2048, out_token_stride=2048)
    return args, ws, out, (q, k, v, pool, scales, mask, lens, bt)


def words(*values):
    """Workspaces of 32-bit words that repeat `values`."""
    return lambda n: torch.tensor(values, dtype=torch.int32).repeat(n // (4 * len(values)) + 1)[:n // 4].contiguous()


@pytest.mark.parametrize("B,T", [(2, 4), (9, 7), (400, 7), (700, 3), (3, 12), (5, 40), (300, 20)])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("fill", [words(0), words(-1), words(0x7f7f7f7f), words(1, 0, 5, 0), words(0, 3, 2, 0), words(0, -7, 9, 0),
                                  words(0, 1, 1 << 30, 0), words(1 << 20, 1 << 20, 1 << 21, 0), words(-(1 << 31), 0, 3, 0)])
def test_unrecorded_partials_are_not_added(q3, B, T, fp8, fill):
    """The second kernel of a drafted-tree call over a workspace without records of its own: it reads and writes nothing for
    them, whatever the words are, and raises nothing."""
    args, ws, out, keep = tree_call(q3, B, T, fp8, fill)
    lib = q3._lib.load()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    # (1, 0, 5) is in bounds and is item 1's record: the one case where a stale record cannot be told from a new one
    own = ws.view(-1)[:3].tolist() == [1, 0, 5]
    assert lib.q3_selftest_tree_merge(ctypes.byref(args), ws.data_ptr(), ws.numel() * 4, stream) == 0
    torch.cuda.synchronize()
    two = T > 8 and fp8 and T <= 16                     # groups of eight tokens: item 1 is seat 0's second
    rest = torch.ones(B, T, dtype=torch.bool, device=DEV)
    if own:
        rest[0 if two else 1, 8 if two else 0:] = False
    assert bool((out[rest] == 77.0).all())
    # the whole call over the same workspace is right: its records are all its own
    assert lib.q3_paged_tree_attn(ctypes.byref(args), ws.data_ptr(), ws.numel() * 4, stream) == 0
    q, k, v, pool, scales, mask, lens, bt = keep
    want = q3.paged_tree_attn(q, k, v, mask, *[x.view(3 * B, 16, 8, 128) for x in pool], lens, bt, 128 ** -0.5,
                              **({} if not fp8 else {n: s.view(torch.float8_e8m0fnu).view(3 * B, 16, 8) for n, s in
                                                     zip(("k_scale", "v_scale"), scales)}))
    assert torch.equal(out, want)
    # and its partials added once more give the same rows
    assert lib.q3_selftest_tree_merge(ctypes.byref(args), ws.data_ptr(), ws.numel() * 4, stream) == 0
    assert torch.equal(out, want)
    assert q3._lib.read_status(clear=True) == 0
