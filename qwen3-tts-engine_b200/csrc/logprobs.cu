// Log probabilities of given tokens, the entropy and the top alternatives of rows of logits, in one pass, sm_100a.
//
// Mathematics. With m = max_v x_v, z_v = (x_v - m) log2(e) / T, s = sum_v 2^z_v and t = sum_v z_v 2^z_v:
//   log p(v) = (x_v - m) / T - ln s          entropy = ln s - ln 2 * t / s
// Each thread keeps (m, s, t) of what it has seen; a larger m moves them by d = (m_old - m_new) log2(e) / T:
// s <- 2^d s, t <- 2^d (t + d s) (with the old s). x - m is formed before it is scaled, so logits of any size, the
// lowest finite value included, neither overflow nor lose digits. Logits of -inf add nothing; a NaN or +inf makes the
// row's numbers NaN, and so does a row of -inf alone.
// The top n are ordered by (value descending, id ascending), NaN above everything: 64-bit keys, the value's order-
// preserving bits above the complement of the id, all different.
//
// Bound: HBM (the logits are read once). A row is shared by a cluster of 1 to 8 CTAs when there are few rows; every
// CTA streams its part in tiles of 512 16-byte vectors, the next tile's loads in flight while one is worked on.
// Selection rides on the same pass: a thread compares the largest of its tile values with the n-th best key found so
// far, and one counting barrier per tile says how many threads have candidates (none, for most tiles). Candidates go
// to a shared-memory list, which is cut back to n when it grows. When nearly all threads have some (the first tile, a
// rising row) the n-th largest of 128 group maxima is a bound first: at most n groups reach it, so a tile never adds
// more than n * 2 threads * 16 values.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "q3_common.cuh"
#include "q3_kernels.h"

namespace cg = cooperative_groups;

namespace q3 {

namespace {

typedef unsigned long long Key;

constexpr int kLpThreads = 256, kLpWarps = kLpThreads / 32;
constexpr int kLpVecs = 2;                          // 16-byte vectors per thread and tile
constexpr int kLpTileVecs = kLpThreads * kLpVecs;
constexpr int kLpGroups = kLpThreads / 2;           // two threads a group
constexpr int kLpMaxElems = 8 * kLpVecs;            // values per thread and tile, 16-bit types
constexpr int kLpList = 2304;                       // >= kTopMax + kTopMax * 2 * kLpMaxElems
constexpr int kLpSlack = 64;                        // the list is cut back when it holds n + this many
constexpr int kLpMaxCluster = 8;
static_assert(kLpList >= kLogprobMaxTop + kLogprobMaxTop * 2 * kLpMaxElems && kLpGroups >= 2 * kLogprobMaxTop, "list");

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

template <typename T>
struct Vec;   // one 16-byte vector of logits
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ float at(const uint4& w, int i) {
    return __uint_as_float(i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w);
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int kN = 8;
  static constexpr uint32_t kNegInf = 0xff80u;
  static __device__ __forceinline__ float at(const uint4& w, int i) {
    const uint32_t x = (i >> 1) == 0 ? w.x : (i >> 1) == 1 ? w.y : (i >> 1) == 2 ? w.z : w.w;
    return __uint_as_float((i & 1) ? (x & 0xffff0000u) : (x << 16));
  }
};
template <>
struct Vec<__half> {
  static constexpr int kN = 8;
  static constexpr uint32_t kNegInf = 0xfc00u;
  static __device__ __forceinline__ float at(const uint4& w, int i) {
    const uint32_t x = (i >> 1) == 0 ? w.x : (i >> 1) == 1 ? w.y : (i >> 1) == 2 ? w.z : w.w;
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x));
    return (i & 1) ? f.y : f.x;
  }
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

struct Stat {
  float m, s, t;
};

// (m, s, t) of two disjoint parts as of their union.
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b, float c) {
  Stat r;
  r.m = max_nan(a.m, b.m);
  const float ref = r.m == -INFINITY ? 0.f : r.m;
  const float da = fmaxf((a.m - ref) * c, -1000.f), db = fmaxf((b.m - ref) * c, -1000.f);   // -inf: s is 0
  const float fa = exp2f(da), fb = exp2f(db);
  r.s = a.s * fa + b.s * fb;
  r.t = fa * (a.t + da * a.s) + fb * (b.t + db * b.s);
  return r;
}

// Shared state of one CTA's selection.
struct LpShared {
  Key list[kLpList];
  Key best[kLogprobMaxTop];       // the CTA's top n, best first (0: none)
  Key groups[kLpGroups];
  Stat stat[kLpWarps];
  Stat total;
  Key bound;                      // only keys above it can be among the top n
  int count;
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

template <typename T>
__global__ void __launch_bounds__(kLpThreads, 4) logprobs_kernel(const LogprobArgs a) {
  constexpr int N = Vec<T>::kN;
  __shared__ LpShared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const long long row = blockIdx.x / parts;
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  const int n = a.top_n;
  const float c = a.inv_temp * kLog2e;

  // vectors of the row: vector v holds ids v N - off .. + N - 1 (aligned in memory; the first and last may be cut)
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % N);
  const int vecs = (a.vocab + off + N - 1) / N;
  const int v0 = static_cast<int>(static_cast<long long>(vecs) * part / parts);
  const int v1 = static_cast<int>(static_cast<long long>(vecs) * (part + 1) / parts);

  if (tid == 0) {
    sh.count = 0;
    sh.bound = 0ull;
  }
  __syncthreads();

  auto load = [&](int v) -> uint4 {   // ids outside the row read as -inf
    uint4 w;
    const int id = v * N - off;
    if (v < v1 && id >= 0 && id + N <= a.vocab) {
      w = __ldcs(reinterpret_cast<const uint4*>(x + id));
    } else {
      uint32_t q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (N == 4) {
          q[i] = 0xff800000u;
          if (v < v1 && id + i >= 0 && id + i < a.vocab) q[i] = __float_as_uint(to_float(x[id + i]));
        } else {
          uint32_t lo = Vec<T>::kNegInf, hi = Vec<T>::kNegInf;
          if (v < v1 && id + 2 * i >= 0 && id + 2 * i < a.vocab) lo = reinterpret_cast<const uint16_t*>(x)[id + 2 * i];
          if (v < v1 && id + 2 * i + 1 >= 0 && id + 2 * i + 1 < a.vocab)
            hi = reinterpret_cast<const uint16_t*>(x)[id + 2 * i + 1];
          q[i] = lo | (hi << 16);
        }
      }
      w = make_uint4(q[0], q[1], q[2], q[3]);
    }
    return w;
  };

  Stat st = {-INFINITY, 0.f, 0.f};
  uint4 next[kLpVecs];
#pragma unroll
  for (int j = 0; j < kLpVecs; ++j) next[j] = load(v0 + j * kLpThreads + tid);
  for (int tile = v0; tile < v1; tile += kLpTileVecs) {
    uint4 w[kLpVecs];
#pragma unroll
    for (int j = 0; j < kLpVecs; ++j) w[j] = next[j];
    if (tile + kLpTileVecs < v1) {
#pragma unroll
      for (int j = 0; j < kLpVecs; ++j) next[j] = load(tile + kLpTileVecs + j * kLpThreads + tid);
    }
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kLpVecs; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) top = max_nan(top, Vec<T>::at(w[j], i));
    if (!(top <= st.m)) {
      const float d = fmaxf((st.m - top) * c, -1000.f), f = exp2f(d);   // nothing yet: s = t = 0
      st.t = f * (st.t + d * st.s);
      st.s *= f;
      st.m = top;
    }
    const float ref = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int j = 0; j < kLpVecs; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float z = (Vec<T>::at(w[j], i) - ref) * c;
        const float p = exp2f(z);
        st.s += p;
        st.t = fmaf(p, fmaxf(z, -1000.f), st.t);   // 0 * -inf would be NaN
      }
    if (n == 0) continue;

    // ---- candidates of the tile
    const uint32_t bound_hi = static_cast<uint32_t>(sh.bound >> 32);
    // strictly above: the bound is a value of an earlier tile, whose ids are smaller, and equal values rank by id
    const bool some = order_bits(top) > bound_hi;
    const int threads = __syncthreads_count(some);
    if (threads == 0) continue;
    const int m = sh.count;
    Key bound = sh.bound;
    auto id_of = [&](int j, int i) { return (tile + j * kLpThreads + tid) * N - off + i; };
    auto real = [&](int j, int id) { return tile + j * kLpThreads + tid < v1 && id >= 0 && id < a.vocab; };
    if (m + threads * kLpVecs * N > kLpList || threads > kLpThreads / 2) {
      // many: the n-th largest group maximum bounds the tile's part of the top n from below
      Key mine = 0ull;
#pragma unroll
      for (int j = 0; j < kLpVecs; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int id = id_of(j, i);
          if (real(j, id)) {
            const Key k = make_key(Vec<T>::at(w[j], i), static_cast<uint32_t>(id));
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
          const int id = id_of(j, i);
          const Key k = make_key(Vec<T>::at(w[j], i), static_cast<uint32_t>(id));
          if (k > bound && real(j, id)) sh.list[atomicAdd(&sh.count, 1)] = k;
        }
    }
    __syncthreads();
    if (sh.count > n + kLpSlack) cut_list(sh, n, sh.count);
  }

  // ---- the CTA's (m, s, t) and top n
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Stat b = {__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
                    __shfl_xor_sync(0xffffffffu, st.t, o)};
    st = join(st, b, c);
  }
  if (lane == 0) sh.stat[warp] = st;
  __syncthreads();
  if (n > 0) {
    if (tid < n) sh.best[tid] = 0ull;
    __syncthreads();
    cut_list(sh, n, sh.count);
  }
  if (tid == 0) {
    Stat r = sh.stat[0];
    for (int k = 1; k < kLpWarps; ++k) r = join(r, sh.stat[k], c);
    sh.total = r;
  }
  __syncthreads();

  // ---- joined over the row's CTAs, by the first of them
  if (parts > 1) {
    cluster.sync();
    if (part == 0) {
      if (tid == 0) {
        Stat r = sh.total;
        for (int k = 1; k < parts; ++k) r = join(r, cluster.map_shared_rank(&sh, k)->total, c);
        sh.total = r;
      }
      if (n > 0) {
        for (int i = tid; i < parts * n; i += kLpThreads) sh.list[i] = cluster.map_shared_rank(&sh, i / n)->best[i % n];
        __syncthreads();
        // empty places (0) of short parts rank last; the row has n values at least
        cut_list(sh, n, parts * n);
      }
      __syncthreads();
    }
    cluster.sync();   // the other CTAs' shared memory has been read
    if (part != 0) return;
  }
  const Stat r = sh.total;
  const float ref = r.m, log_s = logf(r.s);
  if (tid == 0 && a.entropy) a.entropy[row] = log_s - 0.6931471805599453f * (r.t / r.s);
  for (int i = tid; i < a.given; i += kLpThreads) {
    const long long id = a.ids[row * a.ids_stride + i];
    float lp = -INFINITY;                              // an id outside the vocabulary has no probability
    if (id >= 0 && id < a.vocab) lp = (to_float(x[id]) - ref) * a.inv_temp - log_s;
    a.logprobs[row * a.given + i] = lp;
  }
  if (tid < n) {
    const Key k = sh.best[tid];
    a.top_ids[row * n + tid] = static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(k));
    a.top_logprobs[row * n + tid] = (order_value(static_cast<uint32_t>(k >> 32)) - ref) * a.inv_temp - log_s;
  }
}

// CTAs per row: enough for about four waves of the GPU's 4 CTAs per SM, as long as each keeps two tiles.
int logprob_parts(long long rows, int vocab, int elem_bytes, int num_sms) {
  int parts = 1;
  while (parts < kLpMaxCluster && rows * parts < 16ll * num_sms &&
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
