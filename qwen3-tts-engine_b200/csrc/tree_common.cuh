// Pieces shared by the drafted-tree attention kernels (paged_tree.cu: warp MMA for few tokens; paged_tree_tc.cu: tcgen05
// for many): work items, the split of their chunks over CTAs, row addresses. paged_tree.cu describes the split.
#pragma once
#include "q3_common.cuh"
#include "q3_kernels.h"

namespace q3 {

struct TreeItem {
  int seat, tok0;      // first token of the group
  int len, drafts;     // cached tokens; drafted rows
  int nc, n;           // cache chunks; all chunks
};

// Item w of a split with TOK tokens per group and chunks of ROWS cached or DROWS drafted rows.
template <int TOK, int ROWS, int DROWS>
__device__ __forceinline__ TreeItem tree_item(const TreeArgs& a, int w) {
  TreeItem it;
  it.seat = a.groups == 1 ? w : w / a.groups;
  it.tok0 = (w - it.seat * a.groups) * TOK;
  const long long cap = static_cast<long long>(a.max_pages) * a.page_size;
  const int raw = a.seqlens[it.seat];
  it.len = raw < 0 ? 0 : static_cast<int>(raw > cap ? cap : raw);
  it.drafts = a.k_new == nullptr ? 0 : a.tokens;
  int live = a.tokens;
  if (a.draft_lens != nullptr) {
    const int d = a.draft_lens[it.seat];
    live = it.drafts = d < 0 ? 0 : (d > a.tokens ? a.tokens : d);
  }
  it.nc = (it.len + ROWS - 1) / ROWS;
  it.n = it.tok0 < live ? it.nc + (it.drafts + DROWS - 1) / DROWS : 0;
  return it;
}

struct TreePlan {
  long long N, c0, c1;   // chunks of all items; this share's range
  long long first;       // global index of the first chunk of item `w`
  int Ge, w;             // shares that have chunks; the item that holds chunk c0
};

// Shares c .. c + NS - 1 of G of the chunk list, by all THREADS threads of the CTA; P receives share c + mine. Items
// without chunks (nothing to attend, or padded tokens alone) get zero rows here, for the CTA's heads [head0, head0 + heads).
// Returns false when all the shares are empty; one of several is empty when P.c0 == P.c1.
template <int TOK, int ROWS, int DROWS, int THREADS, int NS>
__device__ __forceinline__ bool tree_plan(const TreeArgs& a, TreePlan& P, int c, int G, int mine, int head0, int heads) {
  constexpr int kWarps = THREADS / 32;
  __shared__ long long sums[kWarps];
  __shared__ long long found_first[NS];
  __shared__ int found_item[NS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, W = a.B * a.groups;
  long long local = 0;
  for (int w0 = warp * 32; w0 < W; w0 += THREADS) {   // uniform in a warp
    const int w = w0 + lane;
    TreeItem it = {};
    if (w < W) {
      it = tree_item<TOK, ROWS, DROWS>(a, w);
      local += it.n;
      if (c == 0 && head0 == 0 &&
          (a.seqlens[it.seat] < 0 || a.seqlens[it.seat] > it.len ||
           (a.draft_lens != nullptr && a.draft_lens[it.seat] != it.drafts)))
        atomicOr(a.status, kStatusBadLength);
    }
    for (unsigned zero = __ballot_sync(0xffffffffu, w < W && it.n == 0 && w % G >= c && w % G < c + NS); zero != 0; zero &= zero - 1) {
      const int z = w0 + __ffs(zero) - 1, seat = z / a.groups, tok0 = (z - seat * a.groups) * TOK;
      const int per = heads * (kHeadDim / 8), n = min(TOK, a.tokens - tok0) * per;
      for (int i = lane; i < n; i += 32) {
        __nv_bfloat16* o = a.out + static_cast<long long>(seat) * a.out_seat +
                           static_cast<long long>(tok0 + i / per) * a.out_tok + head0 * kHeadDim;
        reinterpret_cast<uint4*>(o)[i % per] = make_uint4(0, 0, 0, 0);
      }
      if (a.span_by_item && head0 == 0 && lane == 0) a.ws_span[z] = make_int4(-1, 0, 0, 0);
    }
  }
  const long long own = local;   // one item per thread at most: its chunks
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) local += __shfl_xor_sync(0xffffffffu, local, o);
  if (lane == 0) sums[warp] = local;
  __syncthreads();
  long long N = 0;
#pragma unroll
  for (int k = 0; k < kWarps; ++k) N += sums[k];
  P.N = N;
  P.Ge = static_cast<int>(N < G ? N : G);
  const int active = min(P.Ge - c, NS);
  if (active <= 0) return false;
  const long long last = N * (c + active - 1) / P.Ge;   // where the last active share starts
  long long base = 0;
  for (int w0 = 0; w0 < W; w0 += THREADS) {
    const int w = w0 + tid;
    const int n = W <= THREADS ? static_cast<int>(own) : (w < W ? tree_item<TOK, ROWS, DROWS>(a, w).n : 0);
    long long incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    long long before = base, total = 0;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
      if (k < warp) before += sums[k];
      total += sums[k];
    }
    incl += before;
#pragma unroll
    for (int v = 0; v < NS; ++v) {
      const long long c0 = N * (c + v) / P.Ge;
      if (v < active && n > 0 && incl - n <= c0 && c0 < incl) {
        found_item[v] = w;
        found_first[v] = incl - n;
      }
    }
    base += total;
    if (base > last) break;   // uniform
  }
  __syncthreads();
  const int v = min(mine, active - 1);
  P.c0 = N * (c + v) / P.Ge;
  P.c1 = mine < active ? N * (c + v + 1) / P.Ge : P.c0;
  P.w = found_item[v];
  P.first = found_first[v];
  return true;
}

// Nothing starts in share c and goes on, so far (records per share; records per item are written as items end, unless a
// wait gave up: the merge checks them).
__device__ __forceinline__ void tree_no_span(const TreeArgs& a, int c) {
  if (!a.span_by_item) a.ws_span[c] = make_int4(-1, 0, 0, 0);
}
// Item w starts in share c; last: its last share.
__device__ __forceinline__ void tree_span(const TreeArgs& a, int w, int c, int last) {
  if (a.span_by_item) a.ws_span[w] = make_int4(last > c ? w : -1, c, last, 0);
  else if (last > c) a.ws_span[c] = make_int4(w, c, last, 0);
}

// The last share of an item whose last chunk is e: the largest c with N * c / Ge <= e.
__device__ __forceinline__ int tree_last_share(const TreePlan& P, long long e) {
  return static_cast<int>(((e + 1) * P.Ge + P.N - 1) / P.N - 1);
}

// Two e4m3 bytes each, the low and the high half of x, as packed fp16, exact.
__device__ __forceinline__ void e4m3x4_to_half2(uint32_t x, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(x));
}

__device__ __forceinline__ uint32_t finite_bf16x2(uint32_t w) {   // infinities and NaN replaced by zero
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0x0000ffffu;
  return w;
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

__device__ __forceinline__ float tree_exp2(float x) {   // relative error 2^-22, denormal results are zero
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void cp_async8(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
// One arrival on `bar` (counted in its expected ones) when this thread's earlier cp.async copies have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// Page and offset of token `tok`: a shift when the page size is a power of two (page_shift >= 0).
__device__ __forceinline__ int tree_page(const TreeArgs& a, int tok) {
  return a.page_shift >= 0 ? tok >> a.page_shift : tok / a.page_size;
}

// Pool rows of N tokens tok0, tok0 + STEP, ... of a seat, in two steps so that the table entries travel while other work is
// done: tree_pages asks for them (tokens at or past `len`: none), tree_row turns one into a pool row (-1: no token; an
// entry outside the pool reads page 0 and raises its status bit).
template <int N, int STEP>
__device__ __forceinline__ void tree_pages(const TreeArgs& a, int seat, int tok0, int len, int (&page)[N]) {
  const int32_t* table = a.block_table + static_cast<long long>(seat) * a.bt_stride;
#pragma unroll
  for (int x = 0; x < N; ++x) {
    const int tok = tok0 + x * STEP;
    page[x] = 0;   // asm volatile: the compiler must not move the load down to where the entry is used
    if (tok < len) asm volatile("ld.global.nc.s32 %0, [%1];" : "=r"(page[x]) : "l"(table + tree_page(a, tok)));
  }
}
__device__ __forceinline__ long long tree_row(const TreeArgs& a, int page, int tok, int len) {
  if (tok >= len) return -1;
  if (page < 0 || page >= a.num_pages) {
    atomicOr(a.status, kStatusBadPage);
    page = 0;
  }
  return static_cast<long long>(page) * a.page_size + (tok - tree_page(a, tok) * a.page_size);
}

}  // namespace q3
