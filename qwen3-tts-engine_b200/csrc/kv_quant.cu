// An 8-bit paged K/V cache: rows quantised as they are written, and rows read back, sm_100a.
//
// Format. Each head of a token row (128 bf16 values x_d) is stored as 128 e4m3 bytes y_d and one E8M0 byte s = e + 127:
//   top = max |x_d| over the finite x_d;   e = the least integer with top <= 448 * 2^e, held in [-96, 119];
//   y_d = e4m3(x_d * 2^-e), half to even;  a NaN or infinite x_d is stored as NaN.
// The scale is a power of two, so x_d * 2^-e is exact and the value is rounded once, by at most 2^-4 of itself (2^-10 of
// the unit near zero); y_d * 2^e has four significant bits and, with e in that range, is a normal bf16 number or zero:
// reading back is exact. e4m3 is a floating format, so a finer scale would not make the rounding smaller. The limits
// of e keep every stored value finite in fp32 (448 * 2^119 < 2^128; larger bf16 values saturate there) and far from
// fp32 denormals (2^-9 * 2^-96); rows below 2^-87 lose low bits.
// A token row is [8 heads, 128] bytes = 1024 contiguous bytes and its 8 scales 8 contiguous bytes: a page of P tokens is
// [P, 8, 128] e4m3 and [P, 8] E8M0, for K and V each, 2064 bytes a token where bf16 takes 4096.
//
// Both kernels move bytes and are bound by HBM: a warp moves K or V of one row, 16 lanes to a head, so that every load and
// store of a warp is contiguous (512 bytes of bf16, 256 of e4m3), the row's loads all before its first store, and a grid
// of one warp per row (8 lanes to a head with 32-byte pieces, or fewer warps that go on to further rows: 168 to 181 us).
// The maximum is taken on the bf16 bit patterns (an integer order that is also the order of magnitudes), the exponent
// from its bits. 65520 rows written and then read back: 153 to 158 us on three B200s, 807 MB, 78 to 80%
// of a copy's rate; 24 rows: 2 us each way.
#include <cuda_fp8.h>

#include "q3_common.cuh"
#include "q3_kernels.h"

namespace q3 {

namespace {

constexpr int kQuantThreads = 128;
constexpr int kExpMin = -96, kExpMax = 119;

// Pool row of input row `row`, or -1 (with the status bit set by the lane that says so) when it has none.
__device__ __forceinline__ long long quant_pool_row(const KvQuantArgs& a, int row, bool report) {
  long long dst;
  if (a.slots != nullptr) {
    dst = a.slots[row];
  } else {
    const int seat = a.seat_of_row != nullptr ? a.seat_of_row[row] : row;
    const int pos = a.positions[row];
    const int pidx = pos / a.page_size;
    if (seat < 0 || seat >= a.num_seats || pos < 0 || pidx >= a.max_pages) {
      if (report) atomicOr(a.status, kStatusBadLength);
      return -1;
    }
    const int pg = a.block_table[static_cast<long long>(seat) * a.bt_stride + pidx];
    dst = pg < 0 ? -1 : static_cast<long long>(pg) * a.page_size + (pos - pidx * a.page_size);
  }
  if (dst < 0 || dst >= a.pool_rows) {
    if (report) atomicOr(a.status, kStatusBadPage);
    return -1;
  }
  return dst;
}

// The larger of the packed bf16 magnitudes (as 16-bit integers), infinities and NaN left out.
__device__ __forceinline__ uint32_t finite_max(uint32_t m, uint32_t w) {
  uint32_t b = w & 0x7fff7fffu;
  if ((b & 0x7f80u) == 0x7f80u) b &= 0xffff0000u;
  if ((b & 0x7f800000u) == 0x7f800000u) b &= 0x0000ffffu;
  return __vmaxu2(m, b);
}

__device__ __forceinline__ uint16_t quant2(uint32_t w, float inv) {
  float2 f = bf16x2_to_float2(w);
  f.x *= inv;
  f.y *= inv;
  // an infinity would saturate to 448; it is stored as NaN, as a NaN is
  if ((w & 0x7f80u) == 0x7f80u) f.x = __uint_as_float(0x7fffffffu);
  if ((w & 0x7f800000u) == 0x7f800000u) f.y = __uint_as_float(0x7fffffffu);
  return static_cast<uint16_t>(__nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3));
}

// Item i: K or V (bit 0) of row i >> 1, one warp per item: 16 lanes hold a head, 8 values a lane; step j heads 2j, 2j + 1.
constexpr int kHeadPairs = kKvHeads / 2;

__global__ void __launch_bounds__(kQuantThreads) kv_quant_append_kernel(const KvQuantArgs a) {
  const int lane = threadIdx.x & 31;
  const long long i = static_cast<long long>(blockIdx.x) * (kQuantThreads / 32) + (threadIdx.x >> 5);
  if (i >= 2ll * a.n_rows) return;
  const int row = static_cast<int>(i >> 1);
  const bool is_v = (i & 1) != 0;
  const uint4* src = reinterpret_cast<const uint4*>((is_v ? a.v_rows : a.k_rows) + row * a.rows_stride) + lane;
  uint4 w[kHeadPairs];
#pragma unroll
  for (int j = 0; j < kHeadPairs; ++j) w[j] = __ldg(src + 32 * j);
  const long long dst = quant_pool_row(a, row, lane == 0 && !is_v);
  if (dst < 0) return;
  uint2* q = reinterpret_cast<uint2*>((is_v ? a.v_pool : a.k_pool) + dst * (kKvHeads * kHeadDim)) + lane;
  uint32_t even = 0;   // lane's heads' scales, a byte each
#pragma unroll
  for (int j = 0; j < kHeadPairs; ++j) {
    uint32_t m = finite_max(finite_max(finite_max(finite_max(0, w[j].x), w[j].y), w[j].z), w[j].w);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    const int top = max(m & 0xffffu, m >> 16);             // the head's largest finite magnitude, bf16 bits
    // top = 1.M * 2^(E - 127); 448 = 1.75 * 2^8: the least e is E - 127 - 8, one more when 1.M > 1.75
    int e = (top >> 7) - 135 + ((top & 127) > 96 ? 1 : 0);
    e = min(max(e, kExpMin), kExpMax);
    const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    uint2 y;
    y.x = quant2(w[j].x, inv) | (static_cast<uint32_t>(quant2(w[j].y, inv)) << 16);
    y.y = quant2(w[j].z, inv) | (static_cast<uint32_t>(quant2(w[j].w, inv)) << 16);
    q[32 * j] = y;
    even |= static_cast<uint32_t>(e + 127) << (8 * j);
  }
  // lanes 0-15 have the scales of heads 0, 2, 4, 6, lanes 16-31 of 1, 3, 5, 7: the row's 8 bytes in head order
  const uint32_t odd = __shfl_down_sync(0xffffffffu, even, 16);
  if (lane == 0)
    *reinterpret_cast<uint2*>((is_v ? a.v_scale : a.k_scale) + dst * kKvHeads) =
        make_uint2(__byte_perm(even, odd, 0x5140), __byte_perm(even, odd, 0x7362));
}

// Two e4m3 bytes times 2^(s - 127) as bf16, exact.
__device__ __forceinline__ uint32_t dequant2(uint32_t pair, float f) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(pair & 0xffffu), __NV_E4M3);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return pack_bf16x2(x.x * f, x.y * f);
}

__global__ void __launch_bounds__(kQuantThreads) kv_dequant_kernel(const KvQuantArgs a, __nv_bfloat16* k_out,
                                                                   __nv_bfloat16* v_out, long long out_stride) {
  const int lane = threadIdx.x & 31;
  const long long i = static_cast<long long>(blockIdx.x) * (kQuantThreads / 32) + (threadIdx.x >> 5);
  if (i >= 2ll * a.n_rows) return;
  const int row = static_cast<int>(i >> 1);
  const bool is_v = (i & 1) != 0;
  const long long from = quant_pool_row(a, row, lane == 0 && !is_v);
  uint2 y[kHeadPairs];
  uint2 s = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
#pragma unroll
  for (int j = 0; j < kHeadPairs; ++j) y[j] = make_uint2(0, 0);
  if (from >= 0) {
    const uint2* src = reinterpret_cast<const uint2*>((is_v ? a.v_pool : a.k_pool) + from * (kKvHeads * kHeadDim)) + lane;
    s = __ldg(reinterpret_cast<const uint2*>((is_v ? a.v_scale : a.k_scale) + from * kKvHeads));
#pragma unroll
    for (int j = 0; j < kHeadPairs; ++j) y[j] = __ldg(src + 32 * j);
  }
  uint4* out = reinterpret_cast<uint4*>((is_v ? v_out : k_out) + row * out_stride) + lane;
#pragma unroll
  for (int j = 0; j < kHeadPairs; ++j) {
    const float f = e8m0_to_float(((j < 2 ? s.x : s.y) >> (16 * (j & 1) + 8 * (lane >> 4))) & 0xffu);
    uint4 o;
    o.x = dequant2(y[j].x, f); o.y = dequant2(y[j].x >> 16, f); o.z = dequant2(y[j].y, f); o.w = dequant2(y[j].y >> 16, f);
    out[32 * j] = o;
  }
}

unsigned quant_blocks(long long n_rows) {
  return static_cast<unsigned>((2 * n_rows + kQuantThreads / 32 - 1) / (kQuantThreads / 32));
}

}  // namespace

cudaError_t launch_kv_quant_append(const KvQuantArgs& a, cudaStream_t stream) {
  kv_quant_append_kernel<<<quant_blocks(a.n_rows), kQuantThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_kv_dequant(const KvQuantArgs& a, __nv_bfloat16* k_out, __nv_bfloat16* v_out, long long out_stride,
                              cudaStream_t stream) {
  kv_dequant_kernel<<<quant_blocks(a.n_rows), kQuantThreads, 0, stream>>>(a, k_out, v_out, out_stride);
  return cudaGetLastError();
}

}  // namespace q3
