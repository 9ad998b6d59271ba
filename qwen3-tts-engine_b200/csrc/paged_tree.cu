// Attention of a few drafted tokens per seat over a paged K/V cache (bf16 or e4m3 with E8M0 scales), sm_100a; with one
// token and no draft rows it is decode attention over the 8-bit cache.
//
// Mathematics. Token i of a seat (head hq, KV head h = hq / 2) sees every cached row and those drafted rows j whose bit
// j of mask[i] is set. In log2 units s_ij = scale * log2(e) * q_i . k_j and
//   o_i = sum_j 2^(s_ij - m_i) v_j / sum_j 2^(s_ij - m_i),   m_i = max_j s_ij;   no visible row: o_i = 0,
// accumulated online over tiles of 16 keys with one pass over the cache.
// e4m3 rows: k_j = 2^ek(j) ky_j and v_j = 2^ev(j) vy_j. ek enters the score. ev must not be rounded into the 11 bits
// of an fp16 probability, so P.V runs on w_ij = 2^(s_ij + ev(j) - m'_i) with a maximum of its own, m'_i =
// max_j (s_ij + ev(j)); the sum of probabilities keeps m_i, and the result is scaled by 2^(m'_i - m_i) at the end. The
// bytes of K and V convert to fp16 exactly; q is scaled by a power of two per (token, head) into fp16, exact unless an
// element is 2^28 below the largest.
//
// Work split. A work item is a (seat, group of TOK tokens); its keys are cut into chunks of 16 cached rows and then
// the drafted rows. The chunks of all items form one list, of which CTA c takes an equal contiguous share, so ragged
// lengths balance and the grid depends only on the sizes the host knows. An item inside one CTA is written directly;
// one that spans CTAs leaves an fp32 partial (output, maximum, sum) per CTA, which a second small kernel adds in CTA
// order (deterministic; it is launched with programmatic stream serialisation, so its start-up hides under the first).
//
// Bound: HBM. A token row holds all 8 KV heads in 2048 (1024 for e4m3) contiguous bytes. One producer warp fills a ring of
// shared-memory stages by TMA: R rows of all heads in one box (R = 16, or the largest power of two that divides the page
// size, so a box never leaves its page), laid out [head or half head][R rows][128 bytes] with the 128-byte swizzle, which
// makes the fragment loads of the matrix instructions free of bank conflicts. (One bulk copy per row and lane into padded
// rows cost the producer 66 cycles each, 32 a chunk: 189 us on 576 seats, e4m3.) Eight consumer warps take one KV head each.
// One token over e4m3, 576 seats of 200 to 1200 rows: 155 to 163 us on four B200s, 5.2 to 5.4 TB/s, 80 to 83% of a copy's
// rate; 288 seats x 7 tokens, bf16: 146 to 150 us, 5.5 TB/s, 84 to 86%. Four and seven tokens over e4m3 reach half of it (119
// and 131 us): the conversions to fp16 and the softmax, latency more than issue slots (28% of them are used).
// Scores S^T = K.Q^T and outputs O^T = V^T.P^T use mma.sync m16n8k16 with the 16 keys (dims) as the rows of A and the
// 2 heads x 4 tokens as the 8 columns of B: with so few query columns the legacy tensor path is far below its limit.
//
// Roundings. P meets V in V's type, since both operands of an MMA have one: bf16 rows (cached or drafted) take it in bf16
// (half a step is 2^-8 of it), e4m3 rows in fp16 (2^-11 of it, or 2^-25 of the largest weight: a smaller one has none), while
// the sums of P stay fp32 and unrounded. That is at most 2^-8 (2^-11) of sum_j p_j |v_j| next to the output's own 2^-8 of
// itself: 0.0022 instead of 0.0017 in the 2-norm over bf16, 0.0017 over e4m3. Two bf16 pieces of P would double the MMAs of P.V.
#include <cuda.h>
#include <cuda_fp16.h>

#include <cstring>

#include "tensor_map.cuh"
#include "tree_common.cuh"

namespace q3 {

namespace {

constexpr int kTreeRows = 16;                             // cached rows per chunk

// Stage layout: K, V, then (e4m3) the scales [16][8] of K and of V. Cached rows as described above; drafted rows (bf16, 16
// or, in the e4m3 kernel's stages, 8 per chunk) plainly, 2048 bytes each.
template <bool FP8>
struct TreeStage {
  static constexpr int kRow = FP8 ? 1024 : 2048;
  static constexpr int kV = kTreeRows * kRow;
  static constexpr int kScales = 2 * kV;
  static constexpr int kBytes = kScales + (FP8 ? 1024 : 0);
  static constexpr int kDraftRows = FP8 ? 8 : 16;
  static_assert(kDraftRows * kRowBytes <= kV && kBytes % 1024 == 0, "drafted rows fit their stage");
};

// Where a consumer lane's 16-byte pieces lie in a stage: K row g (unit 2t of its head's 128 bytes, or of both halves), V
// rows 2t and 2t + 1 (unit g); rows 8 further are `eight` bytes further. The swizzle xors a 128-byte line's units with the
// line's number.
template <bool FP8>
struct TreeLane {
  uint32_t k[FP8 ? 1 : 2], v[2][FP8 ? 1 : 2], eight;
  __device__ __forceinline__ void init(int R, int h, int g, int t) {
    auto at = [&](int r, int half, int unit) -> uint32_t {
      const uint32_t line = (r / R * R * TreeStage<FP8>::kRow + (FP8 ? h : 2 * h + half) * R * 128 + r % R * 128) >> 7;
      return line * 128 + ((unit ^ (line & 7)) << 4);
    };
#pragma unroll
    for (int i = 0; i < (FP8 ? 1 : 2); ++i) {
      k[i] = at(g, i, 2 * t);
      v[0][i] = TreeStage<FP8>::kV + at(2 * t, i, g);
      v[1][i] = TreeStage<FP8>::kV + at(2 * t + 1, i, g);
    }
    eight = R == kTreeRows ? 1024 : 8 * TreeStage<FP8>::kRow;
  }
};

struct TreeParams {
  TreeArgs a;
  CUtensorMap k, v;   // the pools as [heads or half heads][rows][128 bytes]
  int box_rows;
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                         __nv_bfloat16) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// An 8x8 matrix of 16-bit values (lane 4g + t: row g, columns 2t and 2t + 1) transposed across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_half2_rn(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ float max_over_rows(float v) {   // over the lanes that hold the same columns
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float sum_over_rows(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

__device__ __forceinline__ uint32_t word4(const uint4& w, int e) {
  return e == 0 ? w.x : (e == 1 ? w.y : (e == 2 ? w.z : w.w));
}

// Minus the maximum of no scores: finite, so that a first score of -inf has probability 0 and is not -inf + inf = NaN.
constexpr float kNoMax = 3.402823466e38f;

// What a consumer warp keeps of an item: lane 4g + t owns columns 2t and 2t + 1 (both heads of token 4 nt + t of the
// group) of every 8-column tile nt, and of the outputs the dims row_dim(mt) (accumulators 0, 1) and row_dim(mt) + 1
// (2, 3).
template <bool FP8, int NT>
struct TreeState {
  uint32_t q[NT][8][2];    // B fragments of Q^T: for k-step s the four dims key_dim(t, s) .. + 3 of column g
  float cf[NT][2];         // score factor of the lane's columns
  float o[NT][8][4];
  float nm[NT][2];         // minus the maximum that the outputs are relative to (FP8: of s + ev; else of s); kNoMax: none
  float ns[NT][2];         // FP8: minus the maximum of s that l is relative to
  float l[NT][2];          // this lane's part of the sum
};

template <bool FP8>
__device__ __forceinline__ int key_dim(int t, int s) {
  return FP8 ? 32 * t + 4 * s : 64 * (s >> 2) + 16 * t + 4 * (s & 3);
}
template <bool FP8>
__device__ __forceinline__ int row_dim(int g, int mt) {
  return FP8 ? 16 * g + 2 * mt : 64 * (mt >> 2) + 8 * g + 2 * (mt & 3);
}

template <bool FP8, int NT>
__device__ __forceinline__ void tree_begin(const TreeArgs& a, int seat, int tok0, int h, int lane, TreeState<FP8, NT>& st) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int tok = tok0 + 4 * nt + (g >> 1);
    const bool have = tok < a.tokens;
    const __nv_bfloat16* src = a.q + static_cast<long long>(seat) * a.q_seat + static_cast<long long>(have ? tok : 0) * a.q_tok +
                               (2 * h + (g & 1)) * kHeadDim;
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const uint2 w = have ? __ldg(reinterpret_cast<const uint2*>(src + key_dim<FP8>(t, s))) : make_uint2(0, 0);
      st.q[nt][s][0] = w.x;
      st.q[nt][s][1] = w.y;
      if (FP8) top = __vmaxu2(__vmaxu2(top, w.x & 0x7fff7fffu), w.y & 0x7fff7fffu);
    }
    float f = a.scale_log2;
    if (FP8) {
      // the column's largest magnitude to [2^14, 2^15)
      top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = max(static_cast<int>(max(top & 0xffffu, top >> 16) >> 7) - 127, -112);
      const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 - e) << 23);   // 2^(14 - e), 14 - e in [-114, 126]
#pragma unroll
      for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 x = bf16x2_to_float2(st.q[nt][s][k]);
          st.q[nt][s][k] = pack_half2_rn(x.x * up, x.y * up);
        }
      f *= __uint_as_float(static_cast<uint32_t>(127 + e - 14 > 0 ? 127 + e - 14 : 0) << 23);   // 2^(e - 14)
    }
    // columns 2t, 2t + 1 sit in the lanes whose g is 2t, 2t + 1
    st.cf[nt][0] = __shfl_sync(0xffffffffu, f, 8 * t);
    st.cf[nt][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      st.nm[nt][k] = st.ns[nt][k] = kNoMax;
      st.l[nt][k] = 0.f;
    }
#pragma unroll
    for (int mt = 0; mt < 8; ++mt)
#pragma unroll
      for (int k = 0; k < 4; ++k) st.o[nt][mt][k] = 0.f;
  }
}

// The fp32 products of one tile (acc: keys g and g + 8 of columns 2t, 2t + 1) into the running state; returns the P^T
// fragments and the probabilities. k0, k1: score factors of the two keys; ev0, ev1: their V exponents (FP8 cache rows; 1
// and 0 for others). MASKED: hide[nt] bit 0 / 1 set: the lane's token does not see key g / g + 8.
// The maxima are lazy: they move when some score passes one by more than 2^8 (or comes first: the initial one is
// -kNoMax), which is voted on and rare, so a tile has no exchange between lanes and no rescaling.
template <bool FP8, int NT, bool HALF_P, bool MASKED>
__device__ __forceinline__ void tree_softmax(TreeState<FP8, NT>& st, const float (&acc)[NT][4], float k0, float k1,
                                             float ev0, float ev1, const uint32_t (&hide)[NT], uint32_t (&pf)[NT][2],
                                             float (&p)[NT][4]) {
  float x[NT][4], top = -INFINITY;   // p: s + ev against nm; x: s against ns
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float f = HALF_P ? (k < 2 ? k0 : k1) * st.cf[nt][k & 1] : st.cf[nt][k & 1];
      const bool hidden = MASKED && ((hide[nt] >> (k >> 1)) & 1u);
      p[nt][k] = fmaf(acc[nt][k], f, HALF_P ? st.nm[nt][k & 1] + (k < 2 ? ev0 : ev1) : st.nm[nt][k & 1]);
      if (hidden) p[nt][k] = -INFINITY;
      top = fmaxf(top, p[nt][k]);
      if (FP8) {
        x[nt][k] = fmaf(acc[nt][k], f, st.ns[nt][k & 1]);
        if (hidden) x[nt][k] = -INFINITY;
        top = fmaxf(top, x[nt][k]);
      }
    }
  if (__any_sync(0xffffffffu, top > 8.f)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float s[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float f = HALF_P ? (r ? k1 : k0) * st.cf[nt][c] : st.cf[nt][c];
          s[r] = MASKED && ((hide[nt] >> r) & 1u) ? -INFINITY : acc[nt][2 * r + c] * f;
        }
        const float w0 = HALF_P ? s[0] + ev0 : s[0], w1 = HALF_P ? s[1] + ev1 : s[1];
        const float mw = max_over_rows(fmaxf(w0, w1));
        float ref = st.nm[nt][c];
        if (mw + ref > 8.f) {   // uniform over the lanes of a column
          const float alpha = tree_exp2(-ref - mw);   // 0 at first
          ref = st.nm[nt][c] = -mw;
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            st.o[nt][mt][c] *= alpha;
            st.o[nt][mt][2 + c] *= alpha;
          }
          if (!FP8) st.l[nt][c] *= alpha;
        }
        p[nt][c] = w0 + ref;
        p[nt][2 + c] = w1 + ref;
        if (FP8) {
          const float ms = max_over_rows(fmaxf(s[0], s[1]));
          float rs = st.ns[nt][c];
          if (ms + rs > 8.f) {
            st.l[nt][c] *= tree_exp2(-rs - ms);
            rs = st.ns[nt][c] = -ms;
          }
          x[nt][c] = s[0] + rs;
          x[nt][2 + c] = s[1] + rs;
        }
      }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      p[nt][k] = tree_exp2(p[nt][k]);
      st.l[nt][k & 1] += FP8 ? tree_exp2(x[nt][k]) : p[nt][k];
    }
    pf[nt][0] = transpose8(HALF_P ? pack_half2_rn(p[nt][0], p[nt][1]) : pack_bf16x2(p[nt][0], p[nt][1]));
    pf[nt][1] = transpose8(HALF_P ? pack_half2_rn(p[nt][2], p[nt][3]) : pack_bf16x2(p[nt][2], p[nt][3]));
  }
}

// The exponent of an E8M0 byte as a float (NaN for 255).
__device__ __forceinline__ float e8m0_exponent(uint32_t s) {
  return s == 255u ? NAN : __uint_as_float(0x4b000000u | s) - (8388608.f + 127.f);
}

// 16 cached e4m3 rows; TAIL: only the first `rows` are real, what follows them is stale.
template <int NT, bool TAIL>
__device__ __forceinline__ void tree_tile_e4m3(TreeState<true, NT>& st, const uint8_t* stage, const TreeLane<true>& at, int h,
                                               int lane, int rows) {
  using SL = TreeStage<true>;
  const int g = lane >> 2, t = lane & 3;
  const uint8_t *kr = stage + at.k[0], *kx = stage + (at.k[0] ^ 16);
  const uint8_t* sc = stage + SL::kScales + g * kKvHeads + h;
  const uint32_t s0 = sc[0], s1 = sc[8 * kKvHeads], e0 = sc[16 * kKvHeads], e1 = sc[24 * kKvHeads];
  float acc[NT][4];
  {
    uint4 w[4];
    w[0] = *reinterpret_cast<const uint4*>(kr);
    w[1] = *reinterpret_cast<const uint4*>(kr + at.eight);
    w[2] = *reinterpret_cast<const uint4*>(kx);
    w[3] = *reinterpret_cast<const uint4*>(kx + at.eight);
    float part[2][NT][4] = {};
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      uint32_t af[4];
      e4m3x4_to_half2(word4(w[2 * (x >> 2)], x & 3), af[0], af[2]);
      e4m3x4_to_half2(word4(w[2 * (x >> 2) + 1], x & 3), af[1], af[3]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma16816(part[x & 1][nt], af, st.q[nt][x][0], st.q[nt][x][1], __half());
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[nt][k] = part[0][nt][k] + part[1][nt][k];
  }
  float ev0 = e8m0_exponent(e0), ev1 = e8m0_exponent(e1);
  uint32_t hide[NT];
  if (TAIL) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) hide[nt] = (g >= rows ? 1u : 0u) | (g + 8 >= rows ? 2u : 0u);
    if (g >= rows) ev0 = 0.f;
    if (g + 8 >= rows) ev1 = 0.f;
  }
  uint32_t pf[NT][2];
  float p[NT][4];
  tree_softmax<true, NT, true, TAIL>(st, acc, e8m0_to_float(s0), e8m0_to_float(s1), ev0, ev1, hide, pf, p);
  asm volatile("" ::: "memory");   // V is loaded now: held over the softmax it would not fit the registers
  uint4 v[4];   // keys 2t, 2t + 1, 2t + 8, 2t + 9: dims 16 g .. + 15
#pragma unroll
  for (int k = 0; k < 4; ++k)
    v[k] = *reinterpret_cast<const uint4*>(stage + at.v[k & 1][0] + (k >> 1) * at.eight);
  if (TAIL) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (2 * t + (k & 1) + 8 * (k >> 1) >= rows) v[k] = make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int mt = 0; mt < 8; ++mt) {
    const uint32_t sel = (mt & 1) ? 0x7362u : 0x5140u;   // the two dims' bytes of both keys: (dim 0: k, k'), (dim 1: k, k')
    uint32_t af[4];
    e4m3x4_to_half2(__byte_perm(word4(v[0], mt >> 1), word4(v[1], mt >> 1), sel), af[0], af[1]);
    e4m3x4_to_half2(__byte_perm(word4(v[2], mt >> 1), word4(v[3], mt >> 1), sel), af[2], af[3]);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) mma16816(st.o[nt][mt], af, pf[nt][0], pf[nt][1], __half());
  }
}

// A tile of bf16 rows: 16 cached ones (TAIL: the first `rows` real, what follows them stale), or drafted ones (DRAFT: 16,
// or 8 in the e4m3 kernel's stages, the first `rows` real; see[nt]: bit j set when the lane's token of tile nt sees row j).
template <bool FP8, int NT, bool TAIL, bool DRAFT>
__device__ __forceinline__ void tree_tile_bf16(TreeState<FP8, NT>& st, const uint8_t* stage, const TreeLane<FP8>& at, int h,
                                               int lane, int rows,
                                               const uint32_t (&see)[NT]) {
  using SL = TreeStage<FP8>;
  constexpr int kKeys = FP8 ? 8 : 16;
  static_assert(DRAFT || !FP8, "an e4m3 cache's rows have their own tile");
  const int g = lane >> 2, t = lane & 3;
  float acc[NT][4];
  {
    float part[2][NT][4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // eight dims: k-steps 2i and 2i + 1
      const uint8_t* kr;
      if constexpr (DRAFT) kr = stage + g * kRowBytes + h * kHeadBytes + 2 * key_dim<FP8>(t, 2 * i);
      else kr = stage + (at.k[i >> 1] ^ (16 * (i & 1)));
      const uint4 w0 = *reinterpret_cast<const uint4*>(kr);
      const uint4 w1 = kKeys == 16 ? *reinterpret_cast<const uint4*>(kr + (DRAFT ? 8 * kRowBytes : at.eight)) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint32_t af[4] = {x ? w0.z : w0.x, x ? w1.z : w1.x, x ? w0.w : w0.y, x ? w1.w : w1.y};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          uint32_t b0 = st.q[nt][2 * i + x][0], b1 = st.q[nt][2 * i + x][1];
          if (FP8) {   // the fp16 values are bf16 ones times a power of two
            const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&b0));
            const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&b1));
            b0 = pack_bf16x2(f0.x, f0.y);
            b1 = pack_bf16x2(f1.x, f1.y);
          }
          mma16816(part[x][nt], af, b0, b1, __nv_bfloat16());
        }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[nt][k] = part[0][nt][k] + part[1][nt][k];
  }
  uint4 v[4][2];   // keys 2t, 2t + 1, 2t + 8, 2t + 9: the lane's 16 dims
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int key = 2 * t + (k & 1) + 8 * (k >> 1);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint8_t* vr;
      if constexpr (DRAFT) vr = stage + SL::kV + key * kRowBytes + h * kHeadBytes + 2 * row_dim<FP8>(g, 4 * i);
      else vr = stage + at.v[k & 1][i] + (k >> 1) * at.eight;
      v[k][i] = key < kKeys ? *reinterpret_cast<const uint4*>(vr) : make_uint4(0, 0, 0, 0);
    }
  }
  bool odd = false;   // DRAFT: a value that must not meet a zero probability
  uint32_t hide[NT];
  if (DRAFT || TAIL) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      hide[nt] = 0;
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (g + 8 * r >= rows || (DRAFT && !((see[nt] >> (g + 8 * r)) & 1u))) hide[nt] |= 1u << r;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool real = 2 * t + (k & 1) + 8 * (k >> 1) < rows;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint4& w = v[k][i];
        if (!real) w = make_uint4(0, 0, 0, 0);
        if (DRAFT) {
          const uint4 f = make_uint4(finite_bf16x2(w.x), finite_bf16x2(w.y), finite_bf16x2(w.z), finite_bf16x2(w.w));
          odd |= f.x != w.x || f.y != w.y || f.z != w.z || f.w != w.w;
          w = f;
        }
      }
    }
  }
  uint32_t pf[NT][2];
  float p[NT][4];
  tree_softmax<FP8, NT, false, DRAFT || TAIL>(st, acc, 1.f, 1.f, 0.f, 0.f, hide, pf, p);
#pragma unroll
  for (int mt = 0; mt < 8; ++mt) {
    const uint32_t a0 = word4(v[0][mt >> 2], mt & 3), a1 = word4(v[1][mt >> 2], mt & 3);
    const uint32_t a2 = word4(v[2][mt >> 2], mt & 3), a3 = word4(v[3][mt >> 2], mt & 3);
    const uint32_t af[4] = {__byte_perm(a0, a1, 0x5410), __byte_perm(a0, a1, 0x7632), __byte_perm(a2, a3, 0x5410),
                            __byte_perm(a2, a3, 0x7632)};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) mma16816(st.o[nt][mt], af, pf[nt][0], pf[nt][1], __nv_bfloat16());
  }
  if (DRAFT && __any_sync(0xffffffffu, odd)) {
    // a drafted row holds an infinity or NaN: only the tokens that see the row take it (0 * inf would reach the others)
#pragma unroll 1
    for (int j = 0; j < rows; ++j) {
      const uint8_t* vr = stage + SL::kV + j * kRowBytes + h * kHeadBytes;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int src = 4 * (j & 7) + t;
        const float p0 = __shfl_sync(0xffffffffu, j < 8 ? p[nt][0] : p[nt][2], src);
        const float p1 = __shfl_sync(0xffffffffu, j < 8 ? p[nt][1] : p[nt][3], src);
        if (!((see[nt] >> j) & 1u)) continue;
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) {
          const uint32_t w = *reinterpret_cast<const uint32_t*>(vr + 2 * row_dim<FP8>(g, mt));
          const float2 x = bf16x2_to_float2(w);
          if ((w & 0x7f80u) == 0x7f80u) {
            st.o[nt][mt][0] += p0 * x.x;
            st.o[nt][mt][1] += p1 * x.x;
          }
          if ((w & 0x7f800000u) == 0x7f800000u) {
            st.o[nt][mt][2] += p0 * x.y;
            st.o[nt][mt][3] += p1 * x.y;
          }
        }
      }
    }
  }
}

// End of an item's chunks in this CTA. slot < 0: the item is complete and its rows are written; else its partial goes
// to that workspace slot: outputs [8 heads][8 NT][128] fp32 and (maximum, sum) pairs.
template <bool FP8, int NT>
__device__ __forceinline__ void tree_finish(const TreeArgs& a, const TreeItem& it, int h, int lane, TreeState<FP8, NT>& st, int slot) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int tok = it.tok0 + 4 * nt + t;
    const bool padded = a.draft_lens != nullptr && tok >= it.drafts;
    float r[2], mx[2], l[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      l[k] = sum_over_rows(st.l[nt][k]);
      mx[k] = FP8 ? -st.ns[nt][k] : -st.nm[nt][k];
      // outputs relative to the maximum that l is relative to
      r[k] = FP8 && st.nm[nt][k] != kNoMax && st.ns[nt][k] != kNoMax ? exp2f(st.ns[nt][k] - st.nm[nt][k]) : 1.f;
      if (slot < 0) r[k] = (padded || l[k] == 0.f) ? 0.f : r[k] / l[k];
    }
    if (tok >= a.tokens) continue;
    if (slot < 0) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        __nv_bfloat16* dst = a.out + static_cast<long long>(it.seat) * a.out_seat + static_cast<long long>(tok) * a.out_tok +
                             (2 * h + k) * kHeadDim;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint4 w;
          uint32_t* wp = &w.x;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float(&o)[4] = st.o[nt][4 * i + x];
            // a row without keys is zero whatever the accumulators hold
            wp[x] = r[k] == 0.f ? 0u : pack_bf16x2(o[k] * r[k], o[2 + k] * r[k]);
          }
          *reinterpret_cast<uint4*>(dst + row_dim<FP8>(g, 4 * i)) = w;
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const long long col = (static_cast<long long>(slot) * kKvHeads + h) * (8 * NT) + 8 * nt + 2 * t + k;
        float* dst = a.ws_o + col * kHeadDim;
#pragma unroll
        for (int mt = 0; mt < 8; ++mt)
          *reinterpret_cast<float2*>(dst + row_dim<FP8>(g, mt)) =
              make_float2(st.o[nt][mt][k] * r[k], st.o[nt][mt][2 + k] * r[k]);
        if (g == 0) *reinterpret_cast<float2*>(a.ws_ml + 2 * col) = make_float2(mx[k], l[k]);
      }
    }
  }
}

// The producer warp: lane b < 16 / R brings box b of the chunk's K rows (and their scales), lane 16 + b of its V rows. The
// table entries of the next chunk are asked for before the wait for a free stage. Drafted rows: a lane and a bulk copy each.
template <bool FP8, int TOK, int STAGES>
__device__ __forceinline__ void tree_produce(const TreeParams& p, const TreePlan& P, uint8_t* stages, uint64_t* full,
                                             uint64_t* empty, int lane) {
  using SL = TreeStage<FP8>;
  const TreeArgs& a = p.a;
  const int which = lane >> 4, n = static_cast<int>(P.c1 - P.c0), R = p.box_rows;
  const int row = (lane & 15) * R;              // cached rows: first of the lane's box (of 16: none past them)
  const CUtensorMap* map = which ? &p.v : &p.k;
  int w = P.w;
  TreeItem it = tree_item<TOK, kTreeRows, SL::kDraftRows>(a, w);
  int j = static_cast<int>(P.c0 - P.first);   // chunk of the item
  int page[1], rows = 0, r0 = 0;
  bool draft = false;
  auto warm = [&]() {   // a new item's queries into the L2 cache
    const int toks = min(TOK, a.tokens - it.tok0);
    for (int x = lane; x < toks * 32; x += 32)
      prefetch_l2(a.q + static_cast<long long>(it.seat) * a.q_seat + static_cast<long long>(it.tok0 + (x >> 5)) * a.q_tok + (x & 31) * 64);
  };
  auto look_up = [&]() {   // asks for the table entries of chunk j of item w
    draft = j >= it.nc;
    r0 = draft ? (j - it.nc) * SL::kDraftRows : j * kTreeRows;
    rows = draft ? min(SL::kDraftRows, it.drafts - r0) : min(kTreeRows, it.len - r0);
    tree_pages<1, 1>(a, it.seat, r0 + row, draft || row >= kTreeRows ? 0 : it.len, page);
  };
  warm();
  look_up();
  int k = 0;
  bool ok = true;
  for (; k < n; ++k) {
    const int stage = k % STAGES;
    uint8_t* base = stages + stage * SL::kBytes;
    const uint8_t* src = nullptr;
    int prow = -1;
    if (draft) {
      if ((lane & 15) < rows)
        src = reinterpret_cast<const uint8_t*>((which ? a.v_new : a.k_new) + static_cast<long long>(it.seat) * a.kv_seat +
                                               static_cast<long long>(r0 + (lane & 15)) * a.kv_tok);
    } else if (row < rows) {
      prow = static_cast<int>(tree_row(a, page[0], r0 + row, it.len));
    }
    const bool was_draft = draft;
    const int was_rows = rows;
    if (k + 1 < n) {   // the next chunk's entries travel while this one waits for its stage
      if (++j >= it.n) {
        do it = tree_item<TOK, kTreeRows, SL::kDraftRows>(a, ++w);
        while (it.n == 0);
        j = 0;
        warm();
      }
      look_up();
    }
    if (k >= STAGES && !mbar_wait_sleep(&empty[stage], static_cast<uint32_t>((k / STAGES - 1) & 1))) {
      atomicOr(a.status, kStatusWaitTimeout);
      ok = false;
    }
    if (__any_sync(0xffffffffu, !ok)) break;
    fence_proxy_async_smem();
    if (lane == 0) {
      const int boxes = (was_rows + R - 1) / R;   // cached: whole boxes, with their scales unless those come row by row
      mbar_arrive_expect_tx(&full[stage], static_cast<uint32_t>(was_draft ? 2 * was_rows * kRowBytes
                                                                : 2 * boxes * R * (SL::kRow + (FP8 && R > 1 ? kKvHeads : 0))));
    }
    __syncwarp();
    if (src != nullptr) bulk_g2s(base + which * SL::kV + (lane & 15) * kRowBytes, src, kRowBytes, &full[stage]);
    if (prow >= 0) {
      tma_load_3d(smem_addr(base) + which * SL::kV + row * SL::kRow, map, 0, prow, 0, smem_addr(&full[stage]));
      if (FP8) {
        uint8_t* dst = base + SL::kScales + (which * kTreeRows + row) * kKvHeads;
        const uint8_t* sc = (which ? a.v_scale : a.k_scale) + static_cast<long long>(prow) * kKvHeads;
        if (R > 1) bulk_g2s(dst, sc, R * kKvHeads, &full[stage]);
        else cp_async8(dst, sc);
      }
    }
    if (FP8 && R == 1) cp_async_arrive(&full[stage]);
  }
  // the last chunks issued may still be landing when this warp gives up: wait for them (bounded)
  if (k < n)
    for (int x = max(k - STAGES, 0); x < k; ++x)
      mbar_wait_bounded(&full[x % STAGES], static_cast<uint32_t>((x / STAGES) & 1), 100000000ull);
}

// One CTA per SM: STREAMS shares of the chunk list, each with a ring of STAGES stages, a producer warp (of warpgroup 0, the
// others of which leave) and a consumer warp per KV head, which takes all 4 NT tokens of a group: K and V are converted
// once, and eight tokens in one warp beat four in each of two (registers permitting: 288 seats x 7 tokens, e4m3: 147 -> 132
// us, bf16: 153 -> 148). Few tokens leave a warp waiting, so e4m3, where a chunk takes longest, has two streams then.
// Registers move from warpgroup 0 (down to 32) to the consumers: with 16 of them (640 threads at 96) up to 112, with eight
// and NT = 2 (384 threads at 168) up to 232. At these counts the compiler still spills 136 bytes a thread (stores) in the
// two-stream decode form, 264 with drafts, 44 to 48 with NT = 2: 1.7% of the instructions executed over 576 seats in decode,
// 0.3% over 288 seats x 7 tokens.
template <bool FP8, int STREAMS, int NT, int STAGES>
struct TreeShape {
  static constexpr int kConsumers = kKvHeads * STREAMS, kThreads = 128 + 32 * kConsumers;
  static constexpr bool kMoveRegs = kConsumers == 16 || NT > 1;
  static constexpr int kLaunchRegs = kConsumers == 16 ? 96 : 168, kProducerRegs = 32, kConsumerRegs = kConsumers == 16 ? 112 : 232;
  static_assert(128 * kProducerRegs + 32 * kConsumers * kConsumerRegs <= kThreads * kLaunchRegs, "the register split");
  static constexpr int kTok = 4 * NT;
  static constexpr int kStream = STAGES * TreeStage<FP8>::kBytes;
  static constexpr int kBars = STREAMS * kStream;            // per stream: full[STAGES], empty[STAGES]
  static constexpr int kBytes = kBars + STREAMS * 2 * STAGES * 8;
  static constexpr int kAlloc = kBytes + 1024;               // slack to align the base to 1024 B (swizzle atoms)
  static_assert(kAlloc + 1024 <= 232448, "shared memory");
};

template <bool FP8, bool DRAFTS, int STREAMS, int NT, int STAGES>
__global__ void __launch_bounds__(TreeShape<FP8, STREAMS, NT, STAGES>::kThreads, 1)
    paged_tree_kernel(const __grid_constant__ TreeParams p) {
  using SL = TreeStage<FP8>;
  using SH = TreeShape<FP8, STREAMS, NT, STAGES>;
  const TreeArgs& a = p.a;
  extern __shared__ __align__(1024) uint8_t tree_raw[];
  uint8_t* smem = tree_raw + ((1024u - (smem_addr(tree_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    prefetch_map(&p.k);
    prefetch_map(&p.v);
  }
  const int mine = warp < 4 ? min(warp, STREAMS - 1) : (warp - 4) / kKvHeads;   // the warp's stream
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the merge may be scheduled; it waits for this grid
  if (tid == 0) {
    for (int s = 0; s < STREAMS; ++s) {
      uint64_t* b = reinterpret_cast<uint64_t*>(smem + SH::kBars) + 2 * STAGES * s;
      for (int i = 0; i < STAGES; ++i) {
        mbar_init(&b[i], FP8 && p.box_rows == 1 ? 33 : 1);   // + each lane's scales when they come row by row
        mbar_init(&b[STAGES + i], kKvHeads);
      }
      tree_no_span(a, STREAMS * blockIdx.x + s);
    }
    fence_mbar_init();
  }
  TreePlan P;
  if (!tree_plan<SH::kTok, kTreeRows, SL::kDraftRows, SH::kThreads, STREAMS>(a, P, STREAMS * blockIdx.x, STREAMS * gridDim.x,
                                                                             mine, 0, kQHeads))
    return;   // its barriers published the barrier init
  uint8_t* stages = smem + mine * SH::kStream;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + SH::kBars) + 2 * STAGES * mine;
  uint64_t* empty = full + STAGES;
  const int n = static_cast<int>(P.c1 - P.c0);

  if (warp < 4) {
    if constexpr (SH::kMoveRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(SH::kProducerRegs));
    if (warp < STREAMS && n > 0) tree_produce<FP8, SH::kTok, STAGES>(p, P, stages, full, empty, lane);
    return;
  }
  if constexpr (SH::kMoveRegs) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SH::kConsumerRegs));
  const int h = (warp - 4) % kKvHeads, t = lane & 3, c = STREAMS * static_cast<int>(blockIdx.x) + mine;
  TreeState<FP8, NT> st;
  TreeLane<FP8> at;
  at.init(p.box_rows, h, lane >> 2, t);
  int w = P.w, k = 0;
  long long first = P.first;
  bool ok = true;
  TreeItem it = tree_item<SH::kTok, kTreeRows, SL::kDraftRows>(a, w);
  while (k < n) {
    while (P.c0 + k >= first + it.n) {
      first += it.n;
      it = tree_item<SH::kTok, kTreeRows, SL::kDraftRows>(a, ++w);
    }
    tree_begin<FP8, NT>(a, it.seat, it.tok0, h, lane, st);
    const int end = static_cast<int>(min(first + it.n, P.c1) - P.c0);
    int j = static_cast<int>(P.c0 + k - first);
    for (; k < end; ++k, ++j) {
      const int stage = k % STAGES;
      if (!mbar_wait_sleep(&full[stage], static_cast<uint32_t>((k / STAGES) & 1))) {
        atomicOr(a.status, kStatusWaitTimeout);
        ok = false;
      }
      if (__any_sync(0xffffffffu, !ok)) break;
      const uint8_t* base = stages + stage * SL::kBytes;
      uint32_t see[NT] = {};
      if (!DRAFTS || j < it.nc) {
        const int rows = it.len - j * kTreeRows;
        if constexpr (FP8) {
          if (rows >= kTreeRows) tree_tile_e4m3<NT, false>(st, base, at, h, lane, kTreeRows);
          else tree_tile_e4m3<NT, true>(st, base, at, h, lane, rows);
        } else {
          if (rows >= kTreeRows) tree_tile_bf16<false, NT, false, false>(st, base, at, h, lane, kTreeRows, see);
          else tree_tile_bf16<false, NT, true, false>(st, base, at, h, lane, rows, see);
        }
      } else if constexpr (DRAFTS) {
        const int r0 = (j - it.nc) * SL::kDraftRows;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          if (it.tok0 + 4 * nt + t < it.drafts)
            see[nt] = static_cast<uint32_t>(
                static_cast<unsigned long long>(a.mask[static_cast<long long>(it.seat) * a.mask_seat + it.tok0 + 4 * nt + t]) >> r0);
        tree_tile_bf16<FP8, NT, false, true>(st, base, at, h, lane, min(SL::kDraftRows, it.drafts - r0), see);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
    }
    if (k < end) break;   // a wait gave up
    // slot 2c + 1 holds the item that starts here and goes on, 2c the one that came in from the share before
    const bool from_before = first < P.c0, goes_on = first + it.n > P.c1;
    tree_finish<FP8, NT>(a, it, h, lane, st, from_before ? 2 * c : (goes_on ? 2 * c + 1 : -1));
    if (!from_before && h == 0 && lane == 0)
      tree_span(a, w, c, goes_on ? tree_last_share(P, first + it.n - 1) : c);
  }
  if (k < n && lane == 0)
    for (int s = 0; s < STAGES; ++s)
      mbar_wait_bounded(&full[(k + s) % STAGES], static_cast<uint32_t>(((k + s) / STAGES) & 1), 100000000ull);
}

// Adds the partials of the items that span shares. Columns: (head, 2 heads x token); 128 dims of a column are four per lane
// of a warp. WIDE: few items of many partials each; one column per CTA, the partials shared out over its eight warps.
// Otherwise a warp takes four columns, so that eight loads are in flight with two partials.
constexpr int kMergeWarps = 8;

// Running (maximum, sum, output) of one column.
struct MergeState {
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ __forceinline__ void add(float pm, float pl, const float4& v) {
    const float mn = fmaxf(m, pm), ref = mn == -INFINITY ? 0.f : mn;
    const float f = exp2f(m - ref), g = exp2f(pm - ref);
    m = mn;
    l = l * f + pl * g;
    o.x = o.x * f + v.x * g; o.y = o.y * f + v.y * g; o.z = o.z * f + v.z * g; o.w = o.w * f + v.w * g;
  }
};

template <bool WIDE>
__global__ void __launch_bounds__(kMergeWarps * 32) paged_tree_merge_kernel(const TreeArgs a, int tok_per_group, int shares) {
  constexpr int kCols = WIDE ? 1 : 4, kBatch = 8 / kCols;   // columns per warp; partials asked for at a time
  __shared__ float4 part_o[WIDE ? kMergeWarps : 1][32];
  __shared__ float2 part_ml[WIDE ? kMergeWarps : 1];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int4 span = __ldcg(&a.ws_span[blockIdx.x]);
  // x < 0: nothing to add. A share that gave up a wait leaves the records of its items as the workspace came, and these
  // words say where this kernel reads and writes: what is not an item's own record within bounds is passed over. (Cleared
  // beforehand, in the plan or by an idle warp, they cost the first kernel 2 to 15% by its registers.)
  if (span.x < 0 || span.x >= a.B * a.groups || span.y < 0 || span.y >= span.z || span.z >= shares ||
      static_cast<int>(blockIdx.x) != (a.span_by_item ? span.x : span.y))
    return;
  const int seat = span.x / a.groups, tok0 = (span.x - seat * a.groups) * tok_per_group, c = span.y, parts = span.z - c + 1;
  const int live = 2 * min(tok_per_group, a.tokens - tok0), cols = 2 * tok_per_group, pairs = kKvHeads * live;
  const int pair0 = WIDE ? blockIdx.y : (blockIdx.y * kMergeWarps + warp) * kCols;
  if (pair0 >= pairs) return;   // uniform in the CTA when WIDE
  long long at[kCols];          // the columns in slot 0
#pragma unroll
  for (int i = 0; i < kCols; ++i) {
    const int pair = min(pair0 + i, pairs - 1), h = pair / live;
    at[i] = static_cast<long long>(h) * cols + (pair - h * live);
  }
  const long long slot_cols = static_cast<long long>(kKvHeads) * cols;
  MergeState st[kCols];
  for (int x0 = WIDE ? warp * kBatch : 0; x0 < parts; x0 += (WIDE ? kMergeWarps : 1) * kBatch) {
    float4 v[kBatch][kCols];
    float2 ml[kBatch][kCols];
#pragma unroll
    for (int x = 0; x < kBatch; ++x) {   // partial x: slot 2c + 1 for x = 0, then slot 2 (c + x)
      const int y = min(x0 + x, parts - 1);
      const long long slot = (y == 0 ? 2 * c + 1 : 2 * (c + y)) * slot_cols;
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
        v[x][i] = __ldcg(reinterpret_cast<const float4*>(a.ws_o + (slot + at[i]) * kHeadDim) + lane);
        ml[x][i] = __ldcg(reinterpret_cast<const float2*>(a.ws_ml) + slot + at[i]);
      }
    }
#pragma unroll
    for (int x = 0; x < kBatch; ++x)
#pragma unroll
      for (int i = 0; i < kCols; ++i)
        if (x0 + x < parts) st[i].add(ml[x][i].x, ml[x][i].y, v[x][i]);
  }
  if (WIDE) {
    part_o[warp][lane] = st[0].o;
    if (lane == 0) part_ml[warp] = make_float2(st[0].m, st[0].l);
    __syncthreads();
    if (warp != 0) return;
    for (int x = 1; x < kMergeWarps; ++x) st[0].add(part_ml[x].x, part_ml[x].y, part_o[x][lane]);
  }
  const int drafts = a.draft_lens != nullptr ? a.draft_lens[seat] : a.tokens;
#pragma unroll
  for (int i = 0; i < kCols; ++i) {
    if (pair0 + i >= pairs) break;
    const int h = (pair0 + i) / live, col = pair0 + i - h * live, tok = tok0 + (col >> 1);
    const bool none = st[i].l == 0.f || tok >= drafts;
    const float r = 1.f / st[i].l;
    __nv_bfloat16* dst = a.out + static_cast<long long>(seat) * a.out_seat + static_cast<long long>(tok) * a.out_tok +
                         (2 * h + (col & 1)) * kHeadDim;
    *(reinterpret_cast<uint2*>(dst) + lane) =
        none ? make_uint2(0, 0) : float4_to_bf16x4(make_float4(st[i].o.x * r, st[i].o.y * r, st[i].o.z * r, st[i].o.w * r));
  }
}

struct TreeConfig {
  bool tc;               // the tcgen05 kernel
  int tok, shares;       // tokens per group; shares of the chunk list
};

// Few tokens: the kernel above, in groups of 4 or 8 that each read the cache. More: the tcgen05 kernel, whose time hardly
// grows with the tokens, one share per 8 SMs (a CTA per KV head). The number of groups decides, over long and short seats
// alike. 96 seats of 1200 to 2400 rows (288 of 200 to 1200), us, here and there: bf16, 8 tokens 132 and 163 (154 and 219), 9
// tokens 217 and 165 (276 and 222); e4m3, 8 tokens 112 and 196 (133 and 275), 16 tokens 200 and 201 (247 and 289), 17 tokens
// 286 and 203 (354 and 293). The tcgen05 kernel takes the row maximum before it scales, so a scale that is not positive
// runs here too.
TreeConfig tree_config(bool fp8, int tokens, float scale, int num_sms) {
  if (tokens > (fp8 ? 16 : 8) && scale > 0.f) return {true, tokens, max(1, num_sms / kKvHeads)};
  const int tok = tokens <= 4 ? 4 : 8;
  return {false, tok, fp8 && tok == 4 ? 2 * num_sms : num_sms};
}

// A pool as [heads (bf16: half heads)][rows][128 bytes]; box = all heads x box_rows rows, 128-byte swizzle.
template <bool FP8>
bool make_pool_map(CUtensorMap* m, const void* base, long long rows, int box_rows) {
  const EncodeTiled enc = tensor_map_encoder();
  if (!enc || rows > (1ll << 31) - 1) return false;
  const cuuint32_t parts = FP8 ? kKvHeads : 2 * kKvHeads, elems = FP8 ? 128 : 64;
  const cuuint64_t dims[3] = {elems, static_cast<cuuint64_t>(rows), parts};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(TreeStage<FP8>::kRow), 128};
  const cuuint32_t box[3] = {elems, static_cast<cuuint32_t>(box_rows), parts};
  const cuuint32_t estr[3] = {1u, 1u, 1u};
  return enc(m, FP8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims,
             strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// With the moved registers the launch is refused unless the kernel was built at exactly kLaunchRegs: a setmaxnreg.inc that
// cannot be met would wait forever. (build.py looks at the count when it compiles this file.)
template <bool FP8, bool DRAFTS, int STREAMS, int NT, int STAGES>
cudaError_t launch_tree_main(const TreeArgs& a, int shares, cudaStream_t stream) {
  using SH = TreeShape<FP8, STREAMS, NT, STAGES>;
  auto kern = paged_tree_kernel<FP8, DRAFTS, STREAMS, NT, STAGES>;
  static thread_local int configured_device = -1;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (configured_device != dev) {
    cudaFuncAttributes fa;
    if ((e = cudaFuncGetAttributes(&fa, kern)) != cudaSuccess) return e;
    if (SH::kMoveRegs && fa.numRegs != SH::kLaunchRegs) return cudaErrorInvalidConfiguration;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SH::kAlloc);
    if (e != cudaSuccess) return e;
    configured_device = dev;
  }
  TreeParams p;
  memset(&p, 0, sizeof(p));
  p.a = a;
  p.box_rows = min(a.page_size & -a.page_size, kTreeRows);
  const long long rows = static_cast<long long>(a.num_pages) * a.page_size;
  if (!make_pool_map<FP8>(&p.k, a.k_pool, rows, p.box_rows) || !make_pool_map<FP8>(&p.v, a.v_pool, rows, p.box_rows))
    return cudaErrorInvalidValue;
  kern<<<shares / STREAMS, SH::kThreads, SH::kAlloc, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

TreeWorkspace tree_workspace(bool fp8, int batch, int tokens, float scale, int num_sms) {
  TreeWorkspace w;
  const TreeConfig cfg = tree_config(fp8, tokens, scale, num_sms);
  w.tc = cfg.tc;
  w.tok = cfg.tok;
  w.shares = cfg.shares;
  w.groups = (tokens + cfg.tok - 1) / cfg.tok;
  w.span_by_item = static_cast<long long>(batch) * w.groups <= w.shares;
  const size_t cols = 2ull * w.shares * kKvHeads * 2 * cfg.tok;   // two slots per share
  w.span = 0;
  w.ml = (static_cast<size_t>(w.shares) * sizeof(int4) + 255) / 256 * 256;
  w.o = w.ml + (cols * 2 * sizeof(float) + 255) / 256 * 256;
  w.bytes = w.o + cols * kHeadDim * sizeof(float);
  return w;
}

cudaError_t launch_paged_tree(const TreeArgs& a, const TreeWorkspace& w, cudaStream_t stream) {
  const bool fp8 = a.k_scale != nullptr;
  cudaError_t e;
  if (w.tc) e = launch_paged_tree_tc(a, w.shares, stream);
  else if (fp8 && a.k_new == nullptr && w.tok == 4) e = launch_tree_main<true, false, 2, 1, 3>(a, w.shares, stream);
  else if (fp8 && w.tok == 4) e = launch_tree_main<true, true, 2, 1, 3>(a, w.shares, stream);
  else if (fp8) e = launch_tree_main<true, true, 1, 2, 6>(a, w.shares, stream);
  else if (w.tok == 4) e = launch_tree_main<false, true, 1, 1, 3>(a, w.shares, stream);
  else e = launch_tree_main<false, true, 1, 2, 3>(a, w.shares, stream);
  return e != cudaSuccess ? e : launch_paged_tree_merge(a, w, stream);
}

cudaError_t launch_paged_tree_merge(const TreeArgs& a, const TreeWorkspace& w, cudaStream_t stream) {
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t lc = {};
  // with six shares and more per item the wide form (9 seats of up to 40000 rows: 13 -> 4 us)
  const int pairs = kKvHeads * 2 * min(w.tok, a.tokens), items = a.B * a.groups;
  const bool wide = w.span_by_item && w.shares >= 6 * items;
  lc.gridDim = dim3(w.span_by_item ? items : w.shares, wide ? pairs : (pairs + 4 * kMergeWarps - 1) / (4 * kMergeWarps));
  lc.blockDim = dim3(kMergeWarps * 32);
  lc.stream = stream;
  lc.attrs = &at;
  lc.numAttrs = 1;
  return wide ? cudaLaunchKernelEx(&lc, paged_tree_merge_kernel<true>, a, w.tok, w.shares)
              : cudaLaunchKernelEx(&lc, paged_tree_merge_kernel<false>, a, w.tok, w.shares);
}

}  // namespace q3
