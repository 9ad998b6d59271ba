"""Ops for speculative decoding over an 8-bit paged K/V cache (q3attn C ABI, opaque to torch.compile, graph-capturable).

  kv_quant_append_slots(k, v, k_cache, v_cache, k_scale, v_scale, slots)                          (mutates the cache)
  kv_quant_append_paged(k, v, k_cache, v_cache, k_scale, v_scale, positions, block_table, seat_of_row)     (the same)
  kv_dequant_paged(k_cache, v_cache, k_scale, v_scale, positions, block_table, seat_of_row) -> k, v [n, 8, 128]
  paged_decode_quant(q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, softmax_scale) -> out
  paged_tree_attn(q, k, v, tree_mask, k_cache, v_cache, cache_seqlens, block_table, softmax_scale, ...) -> out
  token_logprobs(logits, ids, top_n, temperature) -> logprobs, entropy, top_ids, top_logprobs

The cache: k_cache / v_cache [num_pages, page_size, 8, 128] float8_e4m3fn and k_scale / v_scale [num_pages, page_size, 8]
float8_e8m0fnu (one power of two per token and head), from empty_quant_cache. Every op launches on the current stream of
its tensors' device and never synchronises. Workspaces come from the caching allocator with each call, so calls on
several streams, or in several captured graphs, never share one. Tensors start on 16-byte boundaries, and the strides of
their rows, tokens and seats are multiples of 8 elements (block tables, lengths, masks and logits: their own type's
alignment): other views are refused, while rows that are not contiguous within a token, and k / v of different strides,
are copied first. The ops themselves (schemas, argument checks, calls)
are in csrc/torch_ops.cpp: they are short, and through Python and ctypes a call would cost more host time than GPU time.
"""
import os
import threading
from typing import NamedTuple, Optional

import torch

from . import _lib
from .ops import HD, NH, NKV, _need

BF16, E4M3, E8M0 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu
MAX_TREE_TOKENS = 64
_TORCH_LIB = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libq3torch.so")


_registered, _lock = False, threading.Lock()


def _register() -> None:
    """Load the bindings and register what tracing needs: with the first call of an op, not with the import, so that a
    process that imports the package to build the libraries does not hold the old ones."""
    global _registered
    _lib.load()
    if not os.path.exists(_TORCH_LIB):
        raise _lib.Q3Error(f"q3attn PyTorch bindings not built ({_TORCH_LIB} missing): run `python -m q3attn.build` from "
                           "qwen3-tts-engine_b200/ or __graft_entry__.build()")
    torch.ops.load_library(_TORCH_LIB)
    fake = torch.library.register_fake
    fake("q3attn::kv_quant_append_slots", lambda *a, **kw: None)
    fake("q3attn::kv_quant_append_paged", lambda *a, **kw: None)
    fake("q3attn::kv_dequant_paged", lambda kc, vc, ks, vs, positions, *a, **kw: tuple(
        kc.new_empty(positions.numel(), NKV, HD, dtype=BF16) for _ in range(2)))
    fake("q3attn::paged_decode_quant", lambda q, *a, **kw: q.new_empty(q.shape[0], NH, HD))
    fake("q3attn::paged_tree_attn", lambda q, *a, **kw: q.new_empty(q.shape[0], q.shape[1], NH, HD))
    fake("q3attn::token_logprobs", lambda x, ids, top_n=0, temperature=1.0: (
        x.new_empty(ids.shape, dtype=torch.float32), x.new_empty(x.shape[0], dtype=torch.float32),
        x.new_empty(x.shape[0], top_n, dtype=torch.int64), x.new_empty(x.shape[0], top_n, dtype=torch.float32)))
    _registered = True


@torch.compiler.assume_constant_result   # a compiled function may be an op's first caller: registering is not traced
def _ready() -> bool:
    if not _registered:
        with _lock:
            if not _registered:
                _register()
    return True


def _op(name):
    """The op `q3attn::name`."""
    if not _registered:
        _ready()
    return getattr(torch.ops.q3attn, name).default


def empty_quant_cache(num_pages: int, page_size: int, device):
    """(k_cache, v_cache, k_scale, v_scale) of an 8-bit cache, every row zero."""
    z = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=device)  # noqa: E731
    return (z(num_pages, page_size, NKV, HD).view(E4M3), z(num_pages, page_size, NKV, HD).view(E4M3),
            z(num_pages, page_size, NKV).view(E8M0), z(num_pages, page_size, NKV).view(E8M0))


def kv_quant_append_slots(k, v, k_cache, v_cache, k_scale, v_scale, slots) -> None:
    """kv_append_slots for an 8-bit cache: row i of k/v [n, 8, 128] bf16 is quantised into flat pool row slots[i]. Each
    head's 128 values share the least power-of-two scale that brings the largest to 448 or less; one rounding to e4m3.
    The slots of a call must differ (a repeated one ends up with a mix of its rows). Out-of-range ones are skipped and raise
    a status bit."""
    _op("kv_quant_append_slots")(k, v, k_cache, v_cache, k_scale, v_scale, slots)


def kv_quant_append_paged(k, v, k_cache, v_cache, k_scale, v_scale, positions, block_table,
                          seat_of_row: Optional[torch.Tensor] = None) -> None:
    """kv_append_paged for an 8-bit cache: row i -> token positions[i] of seat seat_of_row[i] (default: seat i)."""
    _op("kv_quant_append_paged")(k, v, k_cache, v_cache, k_scale, v_scale, positions, block_table, seat_of_row)


def kv_dequant_paged(k_cache, v_cache, k_scale, v_scale, positions, block_table,
                     seat_of_row: Optional[torch.Tensor] = None):
    """Rows of an 8-bit cache as bf16 (exact): row i is token positions[i] of seat seat_of_row[i] (default: seat i), e.g.
    the cached prefix that `prefill` takes ahead of a chunk's own rows. Returns (k, v), each [n, 8, 128]."""
    return _op("kv_dequant_paged")(k_cache, v_cache, k_scale, v_scale, positions, block_table, seat_of_row)


def paged_decode_quant(q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, softmax_scale: float):
    """paged_decode over an 8-bit cache: q [B, 16, 128] over cache_seqlens[b] tokens of seat b's pages -> [B, 16, 128]
    bf16; a seat without tokens gets zeros. Append the step's rows first (kv_quant_append_paged). Sums and softmax
    statistics are fp32; q and the probabilities are rounded to fp16 (include/q3attn.h)."""
    return _op("paged_decode_quant")(q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, float(softmax_scale))


def paged_tree_attn(q, k, v, tree_mask, k_cache, v_cache, cache_seqlens, block_table, softmax_scale: float, *,
                    k_scale=None, v_scale=None, draft_lens=None):
    """Attention of T <= 64 drafted tokens per seat (speculative decoding): token i of seat b attends over the seat's
    cache_seqlens[b] cached tokens and over the drafted rows j with bit j of tree_mask[b, i] set (tree_mask int64
    [B, T], or [T] for one tree in every seat; `tree_mask(parents)` builds it). q [B, T, 16, 128] and the drafted rows
    k / v [B, T, 8, 128], bf16, after RoPE at the tokens' own positions. The cache is bf16, or 8-bit with
    k_scale / v_scale, and is only read: append the accepted rows afterwards (kv_append_paged, kv_quant_append_paged).
    draft_lens int32 [B]: seats with fewer than T drafts; their padded tokens get zero rows. -> [B, T, 16, 128] bf16.
    Sums and softmax statistics are fp32, but the probabilities that meet V are rounded, which paged_decode's are not: to
    bf16 over a bf16 cache, for drafted rows and from 17 tokens on; to fp16 over an 8-bit cache's rows up to 16 tokens. So a
    draft's output is not bit for bit what single steps give: its error against 64 bits is 0.0022 in the 2-norm over bf16
    where unrounded probabilities leave 0.0017, the bf16 output's own."""
    return _op("paged_tree_attn")(q, k, v, tree_mask, k_cache, v_cache, cache_seqlens, block_table, float(softmax_scale),
                                  k_scale, v_scale, draft_lens)


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


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor       # fp32, the shape of ids
    entropy: torch.Tensor        # fp32 [rows]
    top_ids: torch.Tensor        # int64 [rows, top_n]
    top_logprobs: torch.Tensor   # fp32 [rows, top_n]


def token_logprobs(logits, ids, top_n: int = 0, temperature: float = 1.0) -> TokenLogprobs:
    """Log probabilities of given tokens under softmax(logits / temperature), the rows' entropies and their top_n
    alternatives, e.g. to accept or reject drafted tokens. logits [rows, vocab] bf16, fp16 or fp32; ids int64 [rows] or
    [rows, given] (an id outside the vocabulary, such as -1 for padding, scores -inf). top_n <= min(64, vocab), ordered
    by (logit descending, id ascending), NaN first. Logits of -inf have probability 0; a row with NaN or +inf, or of
    -inf alone, gives NaN. temperature 1e-30 to 1e30. One launch.
    Statistics are fp32 and summed tile by tile: a log probability is good to (vocab / 8192 + 80) 2^-24 absolutely (fp32
    logits: vocab / 4096), next to 2^-22 of its own size: 6e-6 at a vocabulary of 151000, 2e-6 as measured. The entropy
    is good to that times 2 + ln(vocab) + entropy, so a row that one token all but owns has one of few significant digits."""
    return TokenLogprobs(*_op("token_logprobs")(logits, ids, top_n, temperature))
