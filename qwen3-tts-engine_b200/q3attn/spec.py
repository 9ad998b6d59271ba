"""Ops for speculative decoding over an 8-bit paged K/V cache (q3attn C ABI, opaque to torch.compile, graph-capturable).

  kv_quant_append_slots(k, v, k_cache, v_cache, k_scale, v_scale, slots)                          (mutates the cache)
  kv_quant_append_paged(k, v, k_cache, v_cache, k_scale, v_scale, positions, block_table, seat_of_row)     (the same)
  kv_dequant_paged(k_cache, v_cache, k_scale, v_scale, positions, block_table, seat_of_row) -> k, v [n, 8, 128]
  paged_decode_quant(q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, softmax_scale) -> out
  paged_tree_attn(q, k, v, tree_mask, k_cache, v_cache, cache_seqlens, block_table, softmax_scale, ...) -> out

The cache: k_cache / v_cache [num_pages, page_size, 8, 128] float8_e4m3fn and k_scale / v_scale [num_pages, page_size, 8]
float8_e8m0fnu (one power of two per token and head), from empty_quant_cache. Every op launches on the current stream of
its tensors' device and never synchronises. Workspaces come from the caching allocator with each call, so calls on
several streams, or in several captured graphs, never share one.
The ops are defined through torch.library.Library: with the same schema, a call costs 4 us of host time where the
custom_op decorator's costs 14 to 17 (measured with an empty body), which is most of a small call.
"""
import ctypes
from typing import Optional

import torch

from . import _lib
from .ops import HD, NH, NKV, _need, _ptr

_LIB = torch.library.Library("q3attn", "FRAGMENT")
BF16, E4M3, E8M0 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu
MAX_TREE_TOKENS = 64


def _define(schema, impl, fake):
    name = schema.split("(")[0]
    _LIB.define(schema)
    _LIB.impl(name, impl, "CompositeExplicitAutograd")
    torch.library.register_fake("q3attn::" + name, fake, lib=_LIB)
    return getattr(torch.ops.q3attn, name).default


def _cuda(dev, **tensors):
    for n, t in tensors.items():
        if t is not None and t.device != dev:
            _need(t.is_cuda, f"{n} must be a CUDA tensor (there is no CPU path)")
            _need(False, f"{n} is on {t.device}, the first argument on {dev}")


def _call(dev, fn, what, *args):
    """fn(*args, stream) on the current stream of `dev`."""
    if dev.index == torch.cuda.current_device():
        rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    if rc:
        _lib.check(rc, what)


def _workspace(dev, size_fn, *args):
    if dev.index == torch.cuda.current_device():
        n = size_fn(*args)
    else:
        with torch.cuda.device(dev):
            n = size_fn(*args)
    return torch.empty(n, dtype=torch.uint8, device=dev)


def empty_quant_cache(num_pages: int, page_size: int, device):
    """(k_cache, v_cache, k_scale, v_scale) of an 8-bit cache, every row zero."""
    z = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=device)  # noqa: E731
    return (z(num_pages, page_size, NKV, HD).view(E4M3), z(num_pages, page_size, NKV, HD).view(E4M3),
            z(num_pages, page_size, NKV).view(E8M0), z(num_pages, page_size, NKV).view(E8M0))


def _cache(k_cache, v_cache, k_scale, v_scale):
    _need(k_cache.is_cuda, "k_cache must be a CUDA tensor (there is no CPU path)")
    _cuda(k_cache.device, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale)
    _need(k_cache.dtype == E4M3 and v_cache.dtype == E4M3, "k_cache/v_cache must be float8_e4m3fn")
    _need(k_scale.dtype == E8M0 and v_scale.dtype == E8M0, "k_scale/v_scale must be float8_e8m0fnu")
    s = k_cache.shape
    _need(len(s) == 4 and s[2] == NKV and s[3] == HD and v_cache.shape == s and k_cache.is_contiguous()
          and v_cache.is_contiguous(), "k_cache/v_cache must be contiguous [num_pages, page_size, 8, 128]")
    _need(k_scale.shape == s[:3] and v_scale.shape == s[:3] and k_scale.is_contiguous() and v_scale.is_contiguous(),
          "k_scale/v_scale must be contiguous [num_pages, page_size, 8]")
    return _lib.QuantCache(k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), s[0], s[1])


def _kv_rows(k, v, dev):
    _cuda(dev, k=k, v=v)
    _need(k.dtype == BF16 and v.dtype == BF16, "k/v must be bfloat16")
    _need(k.dim() == 3 and k.shape[1] == NKV and k.shape[2] == HD and v.shape == k.shape, "k/v must be [n, 8, 128]")
    if k.stride() != v.stride() or k.stride(2) != 1 or k.stride(1) != HD:
        k, v = k.contiguous(), v.contiguous()
    return k, v


def _table(block_table, dev):
    _cuda(dev, block_table=block_table)
    _need(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.stride(1) == 1,
          "block_table must be int32 [seats, max_pages] with unit inner stride")


def _index(t, name, dev, dtype):
    _cuda(dev, **{name: t})
    return t if t.dtype == dtype and t.is_contiguous() else t.to(dtype).contiguous()


def _row_addresses(n, positions, block_table, seat_of_row, dev):
    _table(block_table, dev)
    pos = _index(positions, "positions", dev, torch.int32)
    seat = None if seat_of_row is None else _index(seat_of_row, "seat_of_row", dev, torch.int32)
    _need(pos.numel() == n and (seat is None or seat.numel() == n), "one position (and seat) per row")
    return pos, seat


def _append_slots(k, v, k_cache, v_cache, k_scale, v_scale, slots):
    cache, dev = _cache(k_cache, v_cache, k_scale, v_scale), k_cache.device
    k, v = _kv_rows(k, v, dev)
    s = _index(slots, "slots", dev, torch.int64)
    _need(s.numel() == k.shape[0], "one slot per row")
    _call(dev, _lib.load().q3_kv_quant_append_slots, "q3_kv_quant_append_slots", k.data_ptr(), v.data_ptr(),
          k.stride(0), ctypes.byref(cache), NKV, HD, s.data_ptr(), k.shape[0])


def _append_paged(k, v, k_cache, v_cache, k_scale, v_scale, positions, block_table, seat_of_row=None):
    cache, dev = _cache(k_cache, v_cache, k_scale, v_scale), k_cache.device
    k, v = _kv_rows(k, v, dev)
    n = k.shape[0]
    pos, seat = _row_addresses(n, positions, block_table, seat_of_row, dev)
    _need(seat is not None or n <= block_table.shape[0], "without seat_of_row, row i is seat i's: too few table rows")
    _call(dev, _lib.load().q3_kv_quant_append_paged, "q3_kv_quant_append_paged", k.data_ptr(), v.data_ptr(),
          k.stride(0), ctypes.byref(cache), NKV, HD, pos.data_ptr(), _ptr(seat), block_table.data_ptr(),
          block_table.stride(0), block_table.shape[0], block_table.shape[1], n)


def _dequant_paged(k_cache, v_cache, k_scale, v_scale, positions, block_table, seat_of_row=None):
    cache, dev = _cache(k_cache, v_cache, k_scale, v_scale), k_cache.device
    n = positions.numel()
    pos, seat = _row_addresses(n, positions, block_table, seat_of_row, dev)
    _need(seat is not None or n <= block_table.shape[0], "without seat_of_row, row i is seat i's: too few table rows")
    k = torch.empty(n, NKV, HD, dtype=BF16, device=dev)
    v = torch.empty(n, NKV, HD, dtype=BF16, device=dev)
    _call(dev, _lib.load().q3_kv_dequant_paged, "q3_kv_dequant_paged", ctypes.byref(cache), NKV, HD, pos.data_ptr(),
          _ptr(seat), block_table.data_ptr(), block_table.stride(0), block_table.shape[0], block_table.shape[1],
          k.data_ptr(), v.data_ptr(), NKV * HD, n)
    return k, v


def _attend(q, k, v, tree_mask, draft_lens, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, scale):
    """q [B, T, 16, 128] (any seat and token stride) -> out [B, T, 16, 128]."""
    dev = q.device
    _need(q.is_cuda, "q must be a CUDA tensor (there is no CPU path)")
    _need(q.dtype == BF16, f"q must be bfloat16, got {q.dtype}")
    B, T = q.shape[0], q.shape[1]
    _cuda(dev, k_cache=k_cache, cache_seqlens=cache_seqlens)
    if k_scale is not None:
        _cache(k_cache, v_cache, k_scale, v_scale)
    else:
        _cuda(dev, v_cache=v_cache)
        _need(v_scale is None, "k_scale and v_scale go together")
        _need(k_cache.dtype == BF16 and v_cache.dtype == BF16, "k_cache/v_cache must be bfloat16 (or e4m3 with scales)")
        _need(k_cache.dim() == 4 and k_cache.shape[2] == NKV and k_cache.shape[3] == HD and k_cache.is_contiguous()
              and v_cache.shape == k_cache.shape and v_cache.is_contiguous(),
              "k_cache/v_cache must be contiguous [num_pages, page_size, 8, 128]")
    _table(block_table, dev)
    _need(block_table.shape[0] == B, "block_table must have one row per seat")
    _need(cache_seqlens.dtype == torch.int32 and cache_seqlens.numel() == B and cache_seqlens.is_contiguous(),
          "cache_seqlens must be a contiguous int32 tensor [B]")
    kn, ks, mask_stride = None, (0, 0), 0
    if k is not None:
        _cuda(dev, k=k, v=v, tree_mask=tree_mask, draft_lens=draft_lens)
        _need(k.dtype == BF16 and v.dtype == BF16 and k.shape == (B, T, NKV, HD) and v.shape == k.shape,
              "k/v must be bfloat16 [B, T, 8, 128]")
        if k.stride() != v.stride() or k.stride(3) != 1 or k.stride(2) != HD or k.stride(1) < NKV * HD:
            k, v = k.contiguous(), v.contiguous()
        kn, ks = k.data_ptr(), k.stride()
        _need(tree_mask.dtype == torch.int64 and tree_mask.shape in ((T,), (B, T)), "tree_mask must be int64 [B, T] or [T]")
        if tree_mask.stride(-1) != 1:
            tree_mask = tree_mask.contiguous()
        mask_stride = tree_mask.stride(0) if tree_mask.dim() == 2 else 0
        _need(draft_lens is None or (draft_lens.dtype == torch.int32 and draft_lens.numel() == B
                                     and draft_lens.is_contiguous()), "draft_lens must be a contiguous int32 tensor [B]")
    if q.stride(3) != 1 or q.stride(2) != HD or q.stride(1) < NH * HD:
        q = q.contiguous()
    out = torch.empty(B, T, NH, HD, dtype=BF16, device=dev)
    if B == 0:
        return out
    lib = _lib.load()
    ws = _workspace(dev, lib.q3_paged_tree_workspace_bytes, B, T, k_scale is not None)
    p = _lib.TreeAttn(q.data_ptr(), q.stride(0), q.stride(1), kn, None if k is None else v.data_ptr(), ks[0], ks[1],
                      _ptr(tree_mask), mask_stride, _ptr(draft_lens), k_cache.data_ptr(), v_cache.data_ptr(),
                      _ptr(k_scale), _ptr(v_scale), k_cache.shape[0], k_cache.shape[1], cache_seqlens.data_ptr(),
                      block_table.data_ptr(), block_table.stride(0), block_table.shape[1], B, T, NH, NKV, HD,
                      scale, out.data_ptr(), T * NH * HD, NH * HD)
    _call(dev, lib.q3_paged_tree_attn, "q3_paged_tree_attn", ctypes.byref(p), ws.data_ptr(), ws.numel())
    return out


def _decode_quant(q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, softmax_scale):
    _need(q.dim() == 3 and q.shape[1] == NH and q.shape[2] == HD, f"q must be [B, 16, 128], got {tuple(q.shape)}")
    return _attend(q.unsqueeze(1), None, None, None, None, k_cache, v_cache, k_scale, v_scale, cache_seqlens,
                   block_table, softmax_scale).view(-1, NH, HD)


def _tree_attn(q, k, v, tree_mask, k_cache, v_cache, cache_seqlens, block_table, softmax_scale, k_scale=None,
               v_scale=None, draft_lens=None):
    _need(q.dim() == 4 and q.shape[2] == NH and q.shape[3] == HD, f"q must be [B, T, 16, 128], got {tuple(q.shape)}")
    _need(1 <= q.shape[1] <= MAX_TREE_TOKENS, f"1 to {MAX_TREE_TOKENS} drafted tokens a seat, got {q.shape[1]}")
    return _attend(q, k, v, tree_mask, draft_lens, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table,
                   softmax_scale)


_CACHE = "Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, Tensor(d!) v_scale"
_READ = "Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale"
_op_append_slots = _define(f"kv_quant_append_slots(Tensor k, Tensor v, {_CACHE}, Tensor slots) -> ()", _append_slots,
                           lambda *a, **kw: None)
_op_append_paged = _define(f"kv_quant_append_paged(Tensor k, Tensor v, {_CACHE}, Tensor positions, Tensor block_table, "
                           "Tensor? seat_of_row=None) -> ()", _append_paged, lambda *a, **kw: None)
_op_dequant = _define(f"kv_dequant_paged({_READ}, Tensor positions, Tensor block_table, Tensor? seat_of_row=None) -> "
                      "(Tensor, Tensor)", _dequant_paged,
                      lambda kc, vc, ks, vs, positions, bt, seat_of_row=None: tuple(
                          kc.new_empty(positions.numel(), NKV, HD, dtype=BF16) for _ in range(2)))
_op_decode = _define(f"paged_decode_quant(Tensor q, {_READ}, Tensor cache_seqlens, Tensor block_table, "
                     "float softmax_scale) -> Tensor", _decode_quant, lambda q, *a, **kw: q.new_empty(q.shape[0], NH, HD))
_op_tree = _define("paged_tree_attn(Tensor q, Tensor k, Tensor v, Tensor tree_mask, Tensor k_cache, Tensor v_cache, "
                   "Tensor cache_seqlens, Tensor block_table, float softmax_scale, Tensor? k_scale=None, "
                   "Tensor? v_scale=None, Tensor? draft_lens=None) -> Tensor", _tree_attn,
                   lambda q, *a, **kw: q.new_empty(q.shape[0], q.shape[1], NH, HD))


def kv_quant_append_slots(k, v, k_cache, v_cache, k_scale, v_scale, slots) -> None:
    """kv_append_slots for an 8-bit cache: row i of k/v [n, 8, 128] bf16 is quantised into flat pool row slots[i]. Each
    head's 128 values share the least power-of-two scale that brings the largest to 448 or less; one rounding to e4m3.
    The slots of a call must differ. Out-of-range ones are skipped and raise a status bit."""
    _op_append_slots(k, v, k_cache, v_cache, k_scale, v_scale, slots)


def kv_quant_append_paged(k, v, k_cache, v_cache, k_scale, v_scale, positions, block_table,
                          seat_of_row: Optional[torch.Tensor] = None) -> None:
    """kv_append_paged for an 8-bit cache: row i -> token positions[i] of seat seat_of_row[i] (default: seat i)."""
    _op_append_paged(k, v, k_cache, v_cache, k_scale, v_scale, positions, block_table, seat_of_row)


def kv_dequant_paged(k_cache, v_cache, k_scale, v_scale, positions, block_table,
                     seat_of_row: Optional[torch.Tensor] = None):
    """Rows of an 8-bit cache as bf16 (exact): row i is token positions[i] of seat seat_of_row[i] (default: seat i), e.g.
    the cached prefix that `prefill` takes ahead of a chunk's own rows. Returns (k, v), each [n, 8, 128]."""
    return _op_dequant(k_cache, v_cache, k_scale, v_scale, positions, block_table, seat_of_row)


def paged_decode_quant(q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, softmax_scale: float):
    """paged_decode over an 8-bit cache: q [B, 16, 128] over cache_seqlens[b] tokens of seat b's pages -> [B, 16, 128]
    bf16; a seat without tokens gets zeros. Append the step's rows first (kv_quant_append_paged)."""
    return _op_decode(q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, float(softmax_scale))


def paged_tree_attn(q, k, v, tree_mask, k_cache, v_cache, cache_seqlens, block_table, softmax_scale: float, *,
                    k_scale=None, v_scale=None, draft_lens=None):
    """Attention of T <= 64 drafted tokens per seat (speculative decoding): token i of seat b attends over the seat's
    cache_seqlens[b] cached tokens and over the drafted rows j with bit j of tree_mask[b, i] set (tree_mask int64
    [B, T], or [T] for one tree in every seat; `tree_mask(parents)` builds it). q [B, T, 16, 128] and the drafted rows
    k / v [B, T, 8, 128], bf16, after RoPE at the tokens' own positions. The cache is bf16, or 8-bit with
    k_scale / v_scale, and is only read: append the accepted rows afterwards (kv_append_paged, kv_quant_append_paged).
    draft_lens int32 [B]: seats with fewer than T drafts; their padded tokens get zero rows. -> [B, T, 16, 128] bf16."""
    return _op_tree(q, k, v, tree_mask, k_cache, v_cache, cache_seqlens, block_table, float(softmax_scale), k_scale,
                    v_scale, draft_lens)


def tree_mask(parents: torch.Tensor) -> torch.Tensor:
    """Visibility words of drafted trees for paged_tree_attn: parents [..., T] holds each token's parent (an earlier
    token of the draft, or -1 for a child of the last cached token); bit j of word i is set when j is i or an ancestor
    of i. int64, same shape and device."""
    _need(parents.dim() >= 1 and 1 <= parents.shape[-1] <= MAX_TREE_TOKENS, f"1 to {MAX_TREE_TOKENS} tokens a tree")
    p = parents.to(torch.int64)
    words = torch.zeros_like(p)
    for i in range(p.shape[-1]):
        up = p[..., i]
        w = torch.gather(words, -1, up.clamp(0, max(i - 1, 0)).unsqueeze(-1)).squeeze(-1)
        bit = 1 << i if i < 63 else -(1 << 63)
        words[..., i] = torch.where((up >= 0) & (up < i), w, 0) | bit
    return words
