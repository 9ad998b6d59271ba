// Log probabilities of given tokens, the entropy and the top alternatives of rows of logits, in one pass, sm_100a.
//
// Mathematics. With m = max_v x_v, z_v = (x_v - m) log2(e) / T, s = sum_v 2^z_v and t = sum_v z_v 2^z_v:
//   log p(v) = (x_v - m) / T - ln s          entropy = ln s - ln 2 * t / s
// Each thread keeps (m, s, t) of what it has seen; a larger m moves them by d = (m_old - m_new) log2(e) / T:
// s <- 2^d s, t <- 2^d (t + d s) (with the old s). x - m is formed before it is scaled, so logits of any size, the
// lowest finite value included, neither overflow nor lose digits. A tile's 16 (fp32: 8) terms are summed from zero before
// they join s and t: next to a term of 1, single terms below 2^-24 would be lost one by one (a row of 151000 with 150999
// tokens at e^-16.75: log probabilities off by 1.6e-5 so, by 1 to 2e-6 here, in the same time). Logits of -inf add
// nothing; a NaN or +inf makes the row's numbers NaN, and so does a row of -inf alone.
// The top n are ordered by (value descending, id ascending), NaN above everything: 64-bit keys, the value's order-
// preserving bits above the complement of the id, all different.
//
// Bound: HBM (the logits are read once). A row is shared by a cluster of 1 to 8 CTAs when there are few rows; every
// CTA streams its part in tiles of 1024 16-byte vectors, the next tile's loads in flight while one is worked on; the
// arithmetic is packed in pairs, one exponential per logit. 1030 bf16 rows of 151000 without alternatives: 64 us, 4.9
// TB/s (tiles of 512 vectors: 71); with the top 20: 74 to 78 us on four B200s; one row of 151000 with the top 64: 17 us.
// Selection needs no pass of its own. m is a thread's largest value; the n-th largest maximum of 128 groups of two
// threads bounds the top n from below, and only the few threads that reach it (n to 2n of 256) have their vectors
// read again, out of the L2 cache, shared out over all threads; a thread keeps the maxima of eight segments of its
// tiles, and only segments that reach the bound are read (all of them: the top 20 above take 83 us, the top 64 124
// instead of 88). Parts of rows where more than the list holds reach the bound (massive ties, fewer than n logits above
// -inf, values in one thread's vectors) take select_tiles, which is bounded for every row: it goes through the tiles with
// the n-th best key so far, and where more than half of the threads have candidates the n-th largest group maximum of the
// tile is a bound first, so that a tile adds n * 2 threads * 32 values at most. (The row of 151000 with the top 64 takes 92
// us instead of 17 when its last eighth, a CTA's whole part, is -inf.)
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "q3_common.cuh"
#include "q3_kernels.h"

namespace cg = cooperative_groups;

namespace q3 {

namespace {

typedef unsigned long long Key;

constexpr int kLpThreads = 256, kLpWarps = kLpThreads / 32;
constexpr int kLpVecs = 4;                          // 16-byte vectors per thread and tile
constexpr int kLpTileVecs = kLpThreads * kLpVecs;
constexpr int kLpGroups = kLpThreads / 2;           // two threads a group
constexpr int kLpMaxElems = 8 * kLpVecs;            // values per thread and tile, 16-bit types
constexpr int kLpList = 4224;                       // >= kTopMax + kTopMax * 2 * kLpMaxElems
constexpr int kLpSlack = 64;                        // the list is cut back when it holds n + this many
constexpr int kLpSegs = 8;                          // segments of a CTA's tiles
constexpr int kLpMaxCluster = 8;
static_assert(kLpList >= kLogprobMaxTop + kLogprobMaxTop * 2 * kLpMaxElems && kLpGroups >= 2 * kLogprobMaxTop, "list");
// select_tiles: what is listed before a tile and the candidates of a tile that adds them as they are
static_assert(kLpList >= kLogprobMaxTop + kLpSlack + kLpThreads / 2 * kLpMaxElems, "list of a tile without a bound of its own");

__device__ __forceinline__ uint32_t order_bits(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);      // -0 as +0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
  if (k == 0xffffffffu) return NAN;
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ Key make_key(float x, uint32_t id) {
  return (static_cast<Key>(order_bits(x)) << 32) | (0xffffffffu - id);
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// (x - m) / T. x - m may lie outside fp32's range where the quotient does not: halves first then, which
// is exact.
__device__ __forceinline__ float scaled_below(float x, float m, float inv_temp) {
  const float d = x - m;
  return d == -INFINITY ? (0.5f * x - 0.5f * m) * (2.f * inv_temp) : d * inv_temp;
}

__device__ __forceinline__ float exp2_fast(float x) {   // 2 ulp; results below 2^-126 are zero
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
struct Vec;   // one 16-byte vector of logits: kN values; pairs of them as floats; their largest (NaN if there is one)
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ float2 pair(const uint4& w, int i) {
    return i == 0 ? make_float2(__uint_as_float(w.x), __uint_as_float(w.y))
                  : make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
  }
  static __device__ __forceinline__ float top(const uint4& w) {
    return max_nan(max_nan(__uint_as_float(w.x), __uint_as_float(w.y)), max_nan(__uint_as_float(w.z), __uint_as_float(w.w)));
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int kN = 8;
  static constexpr uint32_t kNegInf = 0xff80u;
  static __device__ __forceinline__ float2 pair(const uint4& w, int i) {
    return bf16x2_to_float2(i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w);
  }
  static __device__ __forceinline__ float top(const uint4& w) {
    const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&w);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
};
template <>
struct Vec<__half> {
  static constexpr int kN = 8;
  static constexpr uint32_t kNegInf = 0xfc00u;
  static __device__ __forceinline__ float2 pair(const uint4& w, int i) {
    return __half22float2(reinterpret_cast<const __half2*>(&w)[i]);
  }
  static __device__ __forceinline__ float top(const uint4& w) {
    const __half2* p = reinterpret_cast<const __half2*>(&w);
    const __half2 m = __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
};
template <typename T>
__device__ __forceinline__ float value_at(const uint4& w, int i) {
  const float2 f = Vec<T>::pair(w, i >> 1);
  return (i & 1) ? f.y : f.x;
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

struct Stat {
  float m, s, t;
};

// Shared state of one CTA.
struct LpShared {
  Key list[kLpList];
  Key best[kLogprobMaxTop];       // the CTA's top n, best first (0: none)
  Key groups[kLpGroups];          // group maxima (select_tiles)
  alignas(16) uint32_t group_bits[kLpGroups];   // order bits of the group maxima over the CTA's part
  uint32_t warp_top[kLpWarps];
  float2 warp_sum[kLpWarps];
  Stat total;
  Key bound;                      // only keys above it can be among the top n
  uint32_t bound_bits;
  int count, reaching;
  uint32_t seg_bits[kLpSegs][kLpThreads];   // order bits of every thread's maximum in each segment
  uint16_t who[kLpSegs * kLpThreads];       // (segment, thread) pairs whose maximum reaches bound_bits
};

// The list cut back to its n largest keys, best first, and the bound raised to the n-th. By all threads; m = the
// number of keys listed. Every key's rank is the number of larger ones.
__device__ __forceinline__ void cut_list(LpShared& sh, int n, int m) {
  const int tid = threadIdx.x;
  for (int i = tid; i < m; i += kLpThreads) {
    const Key k = sh.list[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < m; ++j) rank += sh.list[j] > k;
    if (rank < n) sh.best[rank] = k;
  }
  __syncthreads();
  if (tid < n) sh.list[tid] = tid < m ? sh.best[tid] : 0ull;
  if (tid == 0) {
    sh.count = m < n ? m : n;
    if (m >= n && sh.best[n - 1] > sh.bound) sh.bound = sh.best[n - 1];
  }
  __syncthreads();
}

// A CTA's part of a row: vectors [v0, v1) of the row; vector v holds ids v N - off .. + N - 1 and is aligned in memory
// (the row's first and last may be cut).
template <typename T>
struct Part {
  const T* x;
  int vocab, off, v0, v1;
  static constexpr int N = Vec<T>::kN;

  __device__ __forceinline__ uint4 load(int v) const {   // ids outside the row, vectors outside the part: -inf
    const int id = v * N - off;
    if (v < v1 && id >= 0 && id + N <= vocab) return __ldg(reinterpret_cast<const uint4*>(x + id));
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (N == 4) {
        q[i] = 0xff800000u;
        if (v < v1 && id + i >= 0 && id + i < vocab) q[i] = reinterpret_cast<const uint32_t*>(x)[id + i];
      } else {
        uint32_t lo = Vec<T>::kNegInf, hi = Vec<T>::kNegInf;
        if (v < v1 && id + 2 * i >= 0 && id + 2 * i < vocab) lo = reinterpret_cast<const uint16_t*>(x)[id + 2 * i];
        if (v < v1 && id + 2 * i + 1 >= 0 && id + 2 * i + 1 < vocab)
          hi = reinterpret_cast<const uint16_t*>(x)[id + 2 * i + 1];
        q[i] = lo | (hi << 16);
      }
    }
    return make_uint4(q[0], q[1], q[2], q[3]);
  }
  __device__ __forceinline__ bool real(int v, int id) const { return v < v1 && id >= 0 && id < vocab; }
};

// The CTA's top n into sh.list / sh.best, whatever the values: tile by tile with the n-th best key so far.
template <typename T>
__device__ __noinline__ void select_tiles(LpShared& sh, const Part<T> part, int n) {
  constexpr int N = Vec<T>::kN;
  const int tid = threadIdx.x;
  __syncthreads();
  if (tid == 0) {
    sh.count = 0;
    sh.bound = 0ull;
  }
  __syncthreads();
  for (int tile = part.v0; tile < part.v1; tile += kLpTileVecs) {
    uint4 w[kLpVecs];
#pragma unroll
    for (int j = 0; j < kLpVecs; ++j) w[j] = part.load(tile + j * kLpThreads + tid);
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kLpVecs; ++j) top = max_nan(top, Vec<T>::top(w[j]));
    // strictly above: the bound is a value of an earlier tile, whose ids are smaller, and equal values rank by id
    const bool some = order_bits(top) > static_cast<uint32_t>(sh.bound >> 32);
    const int threads = __syncthreads_count(some);
    if (threads == 0) continue;
    Key bound = sh.bound;
    // The branch holds barriers, so it is taken on the barrier's own result: sh.count may not be looked at here, since
    // other warps may be listing keys already. At most n + kLpSlack keys are listed before a tile, and half of the threads
    // add kLpMaxElems each at most: the list holds them.
    if (threads > kLpThreads / 2) {
      // many: the n-th largest group maximum bounds the tile's part of the top n from below
      const int m = sh.count;   // no warp lists before this branch's barriers
      Key mine = 0ull;
#pragma unroll
      for (int j = 0; j < kLpVecs; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int v = tile + j * kLpThreads + tid, id = v * N - part.off + i;
          if (part.real(v, id)) {
            const Key k = make_key(value_at<T>(w[j], i), static_cast<uint32_t>(id));
            mine = k > mine ? k : mine;
          }
        }
      const Key other = __shfl_xor_sync(0xffffffffu, mine, 1);
      mine = other > mine ? other : mine;
      if ((tid & 1) == 0) sh.groups[tid >> 1] = mine;
      __syncthreads();
      if (tid < kLpGroups) {
        const Key k = sh.groups[tid];
        int rank = 0;
#pragma unroll 4
        for (int g = 0; g < kLpGroups; ++g) rank += sh.groups[g] > k || (sh.groups[g] == k && g < tid);
        if (rank == n - 1 && k > sh.bound + 1) sh.bound = k - 1;   // the n-th itself stays a candidate
      }
      __syncthreads();
      if (m > n) cut_list(sh, n, m);
      bound = sh.bound;
      __syncthreads();
    }
    if (some) {
#pragma unroll
      for (int j = 0; j < kLpVecs; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int v = tile + j * kLpThreads + tid, id = v * N - part.off + i;
          const Key k = make_key(value_at<T>(w[j], i), static_cast<uint32_t>(id));
          if (k > bound && part.real(v, id)) sh.list[atomicAdd(&sh.count, 1)] = k;
        }
    }
    __syncthreads();
    if (sh.count > n + kLpSlack) cut_list(sh, n, sh.count);
  }
  cut_list(sh, n, sh.count);
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads, 4) logprobs_kernel(const LogprobArgs a) {
  constexpr int N = Vec<T>::kN;
  __shared__ LpShared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const long long row = blockIdx.x / parts;
  const int n = a.top_n;
  const float c = a.inv_temp * kLog2e;
  Part<T> part;
  part.x = static_cast<const T*>(a.logits) + row * a.row_stride;
  part.vocab = a.vocab;
  part.off = static_cast<int>((reinterpret_cast<uintptr_t>(part.x) / sizeof(T)) % N);
  const int vecs = (a.vocab + part.off + N - 1) / N;
  part.v0 = static_cast<int>(static_cast<long long>(vecs) * rank / parts);
  part.v1 = static_cast<int>(static_cast<long long>(vecs) * (rank + 1) / parts);

  if (tid == 0) sh.count = sh.reaching = 0;
  if (tid < kLogprobMaxTop) sh.best[tid] = 0ull;

  // ---- one pass: the thread's (m, s, t), s and t in two halves
  float m = -INFINITY;
  float2 s2 = make_float2(0.f, 0.f), t2 = s2;
  const int tiles = (part.v1 - part.v0 + kLpTileVecs - 1) / kLpTileVecs, seg_tiles = (tiles + kLpSegs - 1) / kLpSegs;
  int seg = 0, left = seg_tiles;
  float seg_top = -INFINITY;
  uint4 next[kLpVecs];
#pragma unroll
  for (int j = 0; j < kLpVecs; ++j) next[j] = part.load(part.v0 + j * kLpThreads + tid);
  for (int tile = part.v0; tile < part.v1; tile += kLpTileVecs) {
    uint4 w[kLpVecs];
#pragma unroll
    for (int j = 0; j < kLpVecs; ++j) w[j] = next[j];
    if (tile + kLpTileVecs < part.v1) {
#pragma unroll
      for (int j = 0; j < kLpVecs; ++j) next[j] = part.load(tile + kLpTileVecs + j * kLpThreads + tid);
    }
    float top = Vec<T>::top(w[0]);
#pragma unroll
    for (int j = 1; j < kLpVecs; ++j) top = max_nan(top, Vec<T>::top(w[j]));
    seg_top = max_nan(seg_top, top);
    if (--left == 0 || tile + kLpTileVecs >= part.v1) {
      sh.seg_bits[seg++][tid] = order_bits(seg_top);
      seg_top = -INFINITY;
      left = seg_tiles;
    }
    if (!(top <= m)) {
      const float d = fmaxf((m - top) * c, -1000.f), f = exp2_fast(d);   // nothing yet: s = t = 0
      t2 = make_float2(f * (t2.x + d * s2.x), f * (t2.y + d * s2.y));
      s2 = make_float2(f * s2.x, f * s2.y);
      m = max_nan(m, top);   // a NaN stays
    }
    const float ref = m == -INFINITY ? 0.f : m;
    const float2 nref = make_float2(-ref, -ref), cc = make_float2(c, c);
    float2 ts = make_float2(0.f, 0.f), tt = ts;   // the tile's s and t
#pragma unroll
    for (int j = 0; j < kLpVecs; ++j)
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float2 z = __fmul2_rn(__fadd2_rn(Vec<T>::pair(w[j], i), nref), cc);
        const float2 p = make_float2(exp2_fast(z.x), exp2_fast(z.y));
        ts = __fadd2_rn(ts, p);
        tt = __ffma2_rn(p, make_float2(fmaxf(z.x, -1000.f), fmaxf(z.y, -1000.f)), tt);   // 0 * -inf would be NaN
      }
    s2 = __fadd2_rn(s2, ts);
    t2 = __fadd2_rn(t2, tt);
  }
  float s = s2.x + s2.y, t = t2.x + t2.y;

  // ---- the CTA's (m, s, t)
  const uint32_t bits = order_bits(m);
  const uint32_t wtop = __reduce_max_sync(0xffffffffu, bits);
  const uint32_t pair_top = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
  if ((tid & 1) == 0) sh.group_bits[tid >> 1] = pair_top;
  if (lane == 0) sh.warp_top[warp] = wtop;
  __syncthreads();
  uint32_t all = sh.warp_top[0];
#pragma unroll
  for (int k = 1; k < kLpWarps; ++k) all = max(all, sh.warp_top[k]);
  const float M = order_value(all);
  {
    const float d = fmaxf((m - (M == -INFINITY ? 0.f : M)) * c, -1000.f), f = exp2_fast(d);
    t = M != M ? NAN : f * (t + d * s);
    s = M != M ? NAN : f * s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      t += __shfl_xor_sync(0xffffffffu, t, o);
    }
    if (lane == 0) sh.warp_sum[warp] = make_float2(s, t);
  }
  // ---- the n-th largest group maximum, the threads that reach it, and the values of theirs that do
  if (n > 0) {
    if (tid < kLpGroups) {
      const uint32_t k = sh.group_bits[tid];
      int above = 0;
#pragma unroll 4
      for (int g = 0; g < kLpGroups; g += 4) {
        const uint4 q = *reinterpret_cast<const uint4*>(&sh.group_bits[g]);
        above += (q.x > k || (q.x == k && g < tid)) + (q.y > k || (q.y == k && g + 1 < tid)) +
                 (q.z > k || (q.z == k && g + 2 < tid)) + (q.w > k || (q.w == k && g + 3 < tid));
      }
      if (above == n - 1) sh.bound_bits = k;
    }
    __syncthreads();
    const uint32_t bound = sh.bound_bits;
    if (bits >= bound)
      for (int k = 0; k < seg; ++k)
        if (sh.seg_bits[k][tid] >= bound) sh.who[atomicAdd(&sh.reaching, 1)] = static_cast<uint16_t>(k * kLpThreads + tid);
    __syncthreads();
    const int reaching = sh.reaching, items = reaching * seg_tiles * kLpVecs;
    for (int i = tid; i < items; i += kLpThreads) {
      const int who = sh.who[i % reaching];
      const int v = part.v0 + (who / kLpThreads * seg_tiles * kLpVecs + i / reaching) * kLpThreads + who % kLpThreads;
      const uint4 w = part.load(v);
      if (order_bits(Vec<T>::top(w)) < bound) continue;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float x = value_at<T>(w, e);
        const int id = v * N - part.off + e;
        if (order_bits(x) >= bound && part.real(v, id)) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < kLpList) sh.list[at] = make_key(x, static_cast<uint32_t>(id));
        }
      }
    }
    __syncthreads();
    const int found = sh.count;
    __syncthreads();
    if (tid == 0) sh.bound = 0ull;
    if (found <= kLpList) cut_list(sh, n, found);
    else select_tiles<T>(sh, part, n);
  } else {
    __syncthreads();
  }
  if (tid == 0) {
    float2 r = sh.warp_sum[0];
    for (int k = 1; k < kLpWarps; ++k) {
      r.x += sh.warp_sum[k].x;
      r.y += sh.warp_sum[k].y;
    }
    sh.total = {M, r.x, r.y};
  }
  __syncthreads();

  // ---- joined over the row's CTAs, by the first of them
  if (parts > 1) {
    cluster.sync();
    if (rank == 0) {
      if (tid == 0) {
        float top = sh.total.m;
        for (int k = 1; k < parts; ++k) top = max_nan(top, cluster.map_shared_rank(&sh, k)->total.m);
        const float ref = top == -INFINITY ? 0.f : top;
        Stat r = {top, 0.f, 0.f};
        for (int k = 0; k < parts; ++k) {
          const Stat p = cluster.map_shared_rank(&sh, k)->total;
          const float d = fmaxf((p.m - ref) * c, -1000.f), f = exp2_fast(d);
          r.s += f * p.s;
          r.t += f * (p.t + d * p.s);
        }
        sh.total = r;
      }
      if (n > 0) {
        // with j = ceil(n / parts), at least n keys are as large as the least of the parts' j-th (0: a part has fewer)
        if (warp == 0) {
          Key k = lane < parts ? cluster.map_shared_rank(&sh, lane)->best[(n + parts - 1) / parts - 1] : ~0ull;
#pragma unroll
          for (int o = kLpMaxCluster / 2; o > 0; o >>= 1) {
            const Key other = __shfl_xor_sync(0xffffffffu, k, o);
            k = other < k ? other : k;
          }
          if (lane == 0) {
            sh.bound = k;
            sh.count = 0;
          }
        }
        __syncthreads();
        const Key bound = sh.bound;
        for (int i = tid; i < parts * n; i += kLpThreads) {
          const Key k = cluster.map_shared_rank(&sh, i / n)->best[i % n];
          if (k >= bound && k != 0ull) sh.list[atomicAdd(&sh.count, 1)] = k;
        }
        __syncthreads();
        const int found = sh.count;
        __syncthreads();
        cut_list(sh, n, found);
      }
      __syncthreads();
    }
    cluster.sync();   // the other CTAs' shared memory has been read
    if (rank != 0) return;
  }
  const Stat r = sh.total;
  const float log_s = logf(r.s);
  if (tid == 0 && a.entropy) a.entropy[row] = log_s - 0.6931471805599453f * (r.t / r.s);
  for (int i = tid; i < a.given; i += kLpThreads) {
    const long long id = a.ids[row * a.ids_stride + i];
    float lp = -INFINITY;                              // an id outside the vocabulary has no probability
    if (id >= 0 && id < a.vocab) lp = scaled_below(to_float(part.x[id]), r.m, a.inv_temp) - log_s;
    a.logprobs[row * a.given + i] = lp;
  }
  if (tid < n) {
    const Key k = sh.best[tid];
    a.top_ids[row * n + tid] = static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(k));
    a.top_logprobs[row * n + tid] = scaled_below(order_value(static_cast<uint32_t>(k >> 32)), r.m, a.inv_temp) - log_s;
  }
}

// CTAs per row: as few as fill three quarters of the 4 CTAs that an SM holds (every CTA ends with a selection, which costs
// more than an uneven last wave), as long as each keeps two tiles. The top 20 of 1030 bf16 rows of 151000: one CTA a row
// 83 us, two 98; of 250: two 33, four 40.
int logprob_parts(long long rows, int vocab, int elem_bytes, int num_sms) {
  int parts = 1;
  while (parts < kLpMaxCluster && rows * parts < 3ll * num_sms &&
         static_cast<long long>(vocab) * elem_bytes >= 2ll * 2 * parts * kLpTileVecs * 16)
    parts *= 2;
  return parts;
}

template <typename T>
cudaError_t launch_typed(const LogprobArgs& a, int num_sms, cudaStream_t stream) {
  const int parts = logprob_parts(a.rows, a.vocab, sizeof(T), num_sms);
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = parts;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3(static_cast<unsigned>(a.rows * parts));
  lc.blockDim = dim3(kLpThreads);
  lc.stream = stream;
  lc.attrs = &at;
  lc.numAttrs = 1;
  return cudaLaunchKernelEx(&lc, logprobs_kernel<T>, a);
}

}  // namespace

cudaError_t launch_logprobs(const LogprobArgs& a, int num_sms, cudaStream_t stream) {
  switch (a.dtype) {
    case 0: return launch_typed<__nv_bfloat16>(a, num_sms, stream);
    case 1: return launch_typed<float>(a, num_sms, stream);
    default: return launch_typed<__half>(a, num_sms, stream);
  }
}

}  // namespace q3
