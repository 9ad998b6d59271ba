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
// Both kernels move bytes and are bound by HBM: 8 lanes hold one head (16 values a lane: two 16-byte loads and one
// 16-byte store, or the reverse), a warp four heads. The maximum is taken on the bf16 bit patterns (an integer order
// that is also the order of magnitudes), the exponent from its bits.
#include <cuda_fp8.h>

#include "q3_common.cuh"
#include "q3_kernels.h"

namespace q3 {

namespace {

constexpr int kQuantThreads = 256;
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

// Item i: K or V (bit 0), half of the 8 heads (bit 1), row i >> 2; one warp per item.
__global__ void __launch_bounds__(kQuantThreads) kv_quant_append_kernel(const KvQuantArgs a) {
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (kQuantThreads / 32);
  const long long items = 4ll * a.n_rows;
  for (long long i = static_cast<long long>(blockIdx.x) * (kQuantThreads / 32) + (threadIdx.x >> 5); i < items;
       i += warps) {
    const int row = static_cast<int>(i >> 2), which = static_cast<int>(i & 1), half = static_cast<int>((i >> 1) & 1);
    const __nv_bfloat16* src = (which ? a.v_rows : a.k_rows) + static_cast<long long>(row) * a.rows_stride +
                               half * (kKvHeads / 2 * kHeadDim) + lane * 16;
    const uint4 w0 = __ldg(reinterpret_cast<const uint4*>(src)), w1 = __ldg(reinterpret_cast<const uint4*>(src) + 1);
    const long long dst = quant_pool_row(a, row, lane == 0 && (i & 3) == 0);
    uint32_t m = 0;
    m = finite_max(m, w0.x); m = finite_max(m, w0.y); m = finite_max(m, w0.z); m = finite_max(m, w0.w);
    m = finite_max(m, w1.x); m = finite_max(m, w1.y); m = finite_max(m, w1.z); m = finite_max(m, w1.w);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    const int top = max(m & 0xffffu, m >> 16);             // the head's largest finite magnitude, bf16 bits
    // top = 1.M * 2^(E - 127); 448 = 1.75 * 2^8: the least e is E - 127 - 8, one more when 1.M > 1.75
    int e = (top >> 7) - 135 + ((top & 127) > 96 ? 1 : 0);
    e = min(max(e, kExpMin), kExpMax);
    const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    uint4 y;
    y.x = quant2(w0.x, inv) | (static_cast<uint32_t>(quant2(w0.y, inv)) << 16);
    y.y = quant2(w0.z, inv) | (static_cast<uint32_t>(quant2(w0.w, inv)) << 16);
    y.z = quant2(w1.x, inv) | (static_cast<uint32_t>(quant2(w1.y, inv)) << 16);
    y.w = quant2(w1.z, inv) | (static_cast<uint32_t>(quant2(w1.w, inv)) << 16);
    // the four heads' scales as one 32-bit word, in head order
    uint32_t s = static_cast<uint32_t>(e + 127) << (8 * (lane >> 3));
    s |= __shfl_xor_sync(0xffffffffu, s, 8);
    s |= __shfl_xor_sync(0xffffffffu, s, 16);
    if (dst < 0) continue;
    uint8_t* q = (which ? a.v_pool : a.k_pool) + dst * (kKvHeads * kHeadDim) + half * (kKvHeads / 2 * kHeadDim) + lane * 16;
    *reinterpret_cast<uint4*>(q) = y;
    uint8_t* sc = (which ? a.v_scale : a.k_scale) + dst * kKvHeads + half * (kKvHeads / 2);
    if (lane == 0) *reinterpret_cast<uint32_t*>(sc) = s;
  }
}

// Sixteen e4m3 bytes times 2^(s - 127) as bf16, exact.
__device__ __forceinline__ uint32_t dequant2(uint32_t pair, float f) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(pair & 0xffffu), __NV_E4M3);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return pack_bf16x2(x.x * f, x.y * f);
}

__global__ void __launch_bounds__(kQuantThreads) kv_dequant_kernel(const KvQuantArgs a, __nv_bfloat16* k_out,
                                                                   __nv_bfloat16* v_out, long long out_stride) {
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (kQuantThreads / 32);
  const long long items = 4ll * a.n_rows;
  for (long long i = static_cast<long long>(blockIdx.x) * (kQuantThreads / 32) + (threadIdx.x >> 5); i < items;
       i += warps) {
    const int row = static_cast<int>(i >> 2), which = static_cast<int>(i & 1), half = static_cast<int>((i >> 1) & 1);
    const long long from = quant_pool_row(a, row, lane == 0 && (i & 3) == 0);
    uint4 y = make_uint4(0, 0, 0, 0);
    uint32_t s = 127;
    if (from >= 0) {
      y = __ldg(reinterpret_cast<const uint4*>((which ? a.v_pool : a.k_pool) + from * (kKvHeads * kHeadDim) +
                                              half * (kKvHeads / 2 * kHeadDim) + lane * 16));
      s = __ldg((which ? a.v_scale : a.k_scale) + from * kKvHeads + half * (kKvHeads / 2) + (lane >> 3));
    }
    const float f = e8m0_to_float(s);
    uint4 o0, o1;
    o0.x = dequant2(y.x, f); o0.y = dequant2(y.x >> 16, f); o0.z = dequant2(y.y, f); o0.w = dequant2(y.y >> 16, f);
    o1.x = dequant2(y.z, f); o1.y = dequant2(y.z >> 16, f); o1.z = dequant2(y.w, f); o1.w = dequant2(y.w >> 16, f);
    __nv_bfloat16* out = (which ? v_out : k_out) + static_cast<long long>(row) * out_stride +
                         half * (kKvHeads / 2 * kHeadDim) + lane * 16;
    reinterpret_cast<uint4*>(out)[0] = o0;
    reinterpret_cast<uint4*>(out)[1] = o1;
  }
}

int quant_blocks(long long n_rows, int num_sms) {
  const long long blocks = (4 * n_rows + kQuantThreads / 32 - 1) / (kQuantThreads / 32);
  const long long cap = static_cast<long long>(num_sms) * 8;
  return static_cast<int>(blocks < cap ? blocks : cap);
}

}  // namespace

cudaError_t launch_kv_quant_append(const KvQuantArgs& a, int num_sms, cudaStream_t stream) {
  kv_quant_append_kernel<<<quant_blocks(a.n_rows, num_sms), kQuantThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_kv_dequant(const KvQuantArgs& a, __nv_bfloat16* k_out, __nv_bfloat16* v_out, long long out_stride,
                              int num_sms, cudaStream_t stream) {
  kv_dequant_kernel<<<quant_blocks(a.n_rows, num_sms), kQuantThreads, 0, stream>>>(a, k_out, v_out, out_stride);
  return cudaGetLastError();
}

}  // namespace q3
