// Attention of many drafted tokens (up to 64) per seat over a paged K/V cache (bf16 or e4m3), on the 5th-generation tensor
// cores (tcgen05 + TMEM), sm_100a. The mathematics, the contract and the chunk list are those of paged_tree.cu.
//
// One CTA = (share of the chunk list, KV head h). Accumulator row r = 2 token + (q head & 1): the up to 128 rows of a seat
// share every K/V tile, so the cache is read once however many tokens were drafted. Tiles of 64 keys:
//   S = Q K^T      M = 128 rows, N = 64 keys:  A = Q from TMEM, B = K from shared memory (128-byte swizzle)
//   O += P V       M = 128, N = 128 dims:      A = P (bf16) from TMEM, B = V from shared memory
// The 8 CTAs of a share walk the same keys at the same time, one head each, so the 256 (128) contiguous bytes a CTA
// takes of a token row join the other heads' in the DRAM page. Warps:
//   copies (2)    bring the head's part of 64 token rows by TMA tensor copies of 128 bytes x R rows, R the largest
//                 power of two up to 64 that divides the page size (a box never leaves its page), with the table
//                 entries looked up a tile ahead. bf16 rows land swizzled, as operands. e4m3 rows (and their scales)
//                 land in a ring of raw tiles. (Four-row gathers serve any page the same way but took 66 cycles each,
//                 64 of them a tile: 341 us on 24 seats x 64 tokens x 1000 to 8000 rows.) Issuing a tile's copies
//                 takes a warp longer than the tile's bytes take HBM, so the warps take tiles in turn.
//   loaders (4/8) turn raw e4m3 tiles into bf16 operands (exact: four significant bits times a power of two); write the
//                 drafted rows (the last tile of a seat); zero V rows past a seat's last token.
//   MMA (2)       one issues S(t), up to three tiles ahead of the softmax (three S / P buffers), the other P(t) V(t).
//   softmax (2 x 4) set t & 1 takes tile t: thread r of a set owns row r: online softmax with a lazy maximum (the set's O is
//                 rescaled in TMEM when it grows by more than 2^8), P(t) as bf16 into TMEM over S(t). Each set has an O,
//                 maximum and sum of its own, so that the sets never wait for one another within a seat (one set alone
//                 took 2000 cycles a tile, most of them latency, where HBM takes 1424); at a seat's end both add the two
//                 up, half of the dims each, to the output or as a partial to the workspace. The set with a seat's last
//                 tile writes the next seat's Q into TMEM
//                 (with Q in shared memory an S took 600 cycles: the tensor core reads 6 KB per 16 dims instead of 2).
//                 Warps without live rows have no part in any of it.
// Five kinds of warps in one kernel miss the instruction cache: long waits are calls out of line, rows that see part of
// a tile are masked in TMEM by a small loop of their own, drafted rows come in by a function, and the e4m3 path is rolled
// up (96 seats of 1200 to 2400 rows, 32 tokens: bf16 193 -> 149 us, e4m3 282 -> 200).
// An infinity or NaN in a drafted V row would reach rows that do not see it as 0 * inf: the loaders write zero in its
// place and raise a flag, and the rows that do see it get it back at the end.
//
// Bound: HBM for few tokens; for 64 the exponentials come near it (128 x 64 per tile against 32 KB of K and V: 512 of
// 1424 cycles of the SM's share of the measured copy rate). 24 seats x 64 tokens x 1000 to 8000 rows, bf16: 104 to 117 us on
// four B200s, 3.8 to 4.2 TB/s (28% of all issue slots, the tensor pipe active 26% of the time); over e4m3 132 us. e4m3 is
// bound by instruction issue (the conversion to bf16 and the softmax: 51% of all issue slots over 96 seats x 64 tokens, 232
// us; 0.8% of the instructions there are the 84 bytes a thread that the compiler spills at 96 registers).
//
// Roundings. P is bf16 (half a step is 2^-8 of it) over either cache, since e4m3 rows are bf16 operands here; its sums stay
// fp32 and unrounded. K, V and Q are exact.
#include <cuda.h>
#include <cuda_fp16.h>

#include <cstring>

#include "prefill_common.cuh"
#include "tensor_map.cuh"
#include "tree_common.cuh"

namespace q3 {

namespace {

constexpr int kTcRows = 64;                     // keys per tile (cached rows, or all drafted rows)
constexpr int kTcTok = kTreeMaxTokens;          // tokens per item: the whole draft
constexpr int kTcTmemCols = 512;
constexpr int kTcScores = 3;                    // S / P buffers
// S(t), P(t) at column 64 (t % 3); Q after them; O of set s at 256 + 128 s
constexpr uint32_t kTcQCol = 64 * kTcScores, kTcOCol = 256;
static_assert(kTcQCol + 64 <= kTcOCol && kTcOCol + 256 <= kTcTmemCols, "TMEM columns");
constexpr int kTcOddSlots = 16;                 // more than the stages: see where it is read
constexpr int kTcLoaderWarp = 8;                // after the softmax warps 0-7

template <bool FP8>
struct TcSmem {
  static constexpr int kLoaders = FP8 ? 8 : 4;               // loader warps
  static constexpr int kCopyWarps = 2;                       // 16 warps of 128 registers; e4m3: 20 of 96
  static constexpr int kMmaWarp = kTcLoaderWarp + kLoaders, kCopyWarp = kMmaWarp + 2;
  static constexpr int kThreads = (kCopyWarp + kCopyWarps) * 32;
  static constexpr int kStages = FP8 ? 4 : 6;                // operand tiles
  static constexpr int kRawSlots = FP8 ? 5 : 0;
  static constexpr int kCopySlots = FP8 ? kRawSlots : kStages;   // tiles the copies fill
  static constexpr int kTile = 16384, kHalf = 8192;
  static constexpr int kKv = 0;                              // stage s: K then V, [2 dim halves][64 keys][128 B] each
  static constexpr int kRaw = kKv + kStages * 2 * kTile;     // raw e4m3: K then V [64 rows][128 B], scales [2][64][8]
  static constexpr int kRawBytes = 2 * kTcRows * kHeadDim + 2 * kTcRows * kKvHeads;
  static constexpr int kMl = kRaw + kRawSlots * kRawBytes;   // (maximum, sum) of each set's rows, by item & 1
  static constexpr int kBars = kMl + 2 * 2 * 128 * 8;
  static constexpr int kFull = 0, kEmpty = kStages, kCopied = 2 * kStages, kRawFree = kCopied + kCopySlots,
                       kSFull = kRawFree + kRawSlots, kPFull = kSFull + kTcScores, kPvDone = kPFull + kTcScores,
                       kQFull = kPvDone + kTcScores, kOFree = kQFull + 1, kSets = kOFree + 1, kFinal = kSets + 4, kNumBars = kFinal + 2;
  static constexpr int kTmemSlot = kBars + 8 * kNumBars;
  static constexpr int kAbort = kTmemSlot + 4;
  static constexpr int kIssued = kAbort + 4;                 // per copy warp, 1 + its last tile issued (abort path)
  static constexpr int kOdd = kIssued + 4 * kCopyWarps;
  static constexpr int kBytes = kOdd + 4 * kTcOddSlots;
  static constexpr int kAlloc = kBytes + 1024;               // slack to align the base to 1024 B (swizzle atoms)
  // 1 KB of static shared memory (the plan's) and 1 KB the system keeps come on top
  static_assert(kAlloc + 1024 <= 232448 && kRawBytes % 1024 == 0 && kMl % 8 == 0 && kBars % 8 == 0,
                "shared memory");
};

struct TcParams {
  TreeArgs a;
  CUtensorMap k, v;    // the pools as [rows][1024]: boxes of box_rows rows x 128 bytes
  int box_rows;
};

// A box of rows from `row` on, 128 bytes each from column x.
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int row, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(row), "r"(bar)
      : "memory");
}
__device__ __forceinline__ bool tc_poll(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(20000u)
      : "memory");
  return ok != 0;
}
// Wait for phase `parity` of `bar`; false after 2 s or once another role has raised the abort flag. The waits sleep in the
// barrier (up to 20 us at a time): 14 to 16 warps that poll instead take the issue slots the softmax warps need.
__device__ __noinline__ bool tc_wait_on(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  const uint64_t t0 = global_timer_ns();
#pragma unroll 1
  while (!tc_poll(bar, parity))
    if (*abort_flag || global_timer_ns() - t0 > 2000000000ull) return false;
  return true;
}
__device__ __forceinline__ bool tc_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  const uint32_t b = smem_addr(bar);
  return __builtin_expect(tc_poll(b, parity), 1) || tc_wait_on(b, parity, abort_flag);
}

// 16 consecutive 32-bit columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_st16u(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(
          taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// 8 consecutive 32-bit columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const float (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "f"(v[0]), "f"(v[1]),
               "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// D += A B with A in TMEM, issued by the lane whose `leader` is not 0. The whole warp runs the code around it, so that
// addresses and descriptors stay in uniform registers (inside a branch for one lane an MMA took 70 cycles to issue).
__device__ __forceinline__ void tc_mma_tmem_a(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t leader, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
      "r"(leader)
      : "memory");
}
__device__ __forceinline__ uint32_t tc_elect() {
  uint32_t x;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(x));
  return x;
}
__device__ __forceinline__ void st_shared16(uint32_t dst, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t src) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src) : "memory");
  return v;
}
// 16 bytes of shared memory from `bytes` (16 or 0) bytes at src and zeros.
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16_at(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8_at(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}

// Byte offset of 16-byte unit c (0..15) of a row in an operand tile whose dim halves are `half` bytes apart.
__device__ __forceinline__ uint32_t tc_unit(int row, int c, int half) {
  return static_cast<uint32_t>((c >> 3) * half + row * 128 + (((c & 7) ^ (row & 7)) << 4));
}

// Where a warp stands in the CTA's tiles 0 .. n - 1 (tile k = chunk P.c0 + k): the item that holds tile k, its tiles here
// [begin, end) and the item's chunk index of tile `begin`. Each role walks the tiles on its own; a step within an item is a
// comparison (one warp's instructions run one after another, five cycles or so each, and every role is on the tile's path).
struct TcCursor {
  int w, index;          // item; how many items of this CTA came before it
  int begin, end, j0;
  long long first;
  TreeItem it;
};
__device__ __forceinline__ void tc_enter(const TreePlan& P, TcCursor& c) {
  c.begin = static_cast<int>(max(c.first - P.c0, 0ll));
  c.end = static_cast<int>(min(c.first + c.it.n, P.c1) - P.c0);
  c.j0 = static_cast<int>(max(P.c0 - c.first, 0ll));
}
// To tile k >= the present one; true when that is another item.
__device__ __forceinline__ bool tc_seek(const TreeArgs& a, const TreePlan& P, TcCursor& c, int k) {
  if (__builtin_expect(k < c.end, 1)) return false;
  while (P.c0 + k >= c.first + c.it.n) {
    c.first += c.it.n;
    c.it = tree_item<kTcTok, kTcRows, kTcTok>(a, ++c.w);
    c.index += c.it.n > 0;
  }
  tc_enter(P, c);
  return true;
}
__device__ __forceinline__ int tc_chunk(const TcCursor& c, int k) { return c.j0 + k - c.begin; }

// Four e4m3 bytes times f as two packed bf16 words, exact.
__device__ __forceinline__ uint2 dequant4(uint32_t w, float2 f) {
  uint32_t lo, hi;
  e4m3x4_to_half2(w, lo, hi);
  const float2 x = __fmul2_rn(__half22float2(*reinterpret_cast<const __half2*>(&lo)), f);
  const float2 y = __fmul2_rn(__half22float2(*reinterpret_cast<const __half2*>(&hi)), f);
  return make_uint2(pack_bf16x2(x.x, x.y), pack_bf16x2(y.x, y.y));
}

// ------------------------------------------------------------------ the copy warps: warp cw, tiles cw, cw + kCopyWarps, ..
// Lane l looks after rows 4 (l & 15) .. + 3 of a tile, of K (l < 16) or V, and copies the boxes that start there. With
// boxes of four rows or more those rows are neighbours in the pool: one table entry, one box at most. All of a tile's
// addresses are ready before its slot is waited for.
template <bool FP8>
__device__ __forceinline__ void tc_copies(const TcParams& p, const TreePlan& P, TcCursor cur, uint8_t* smem, uint64_t* bars,
                                          volatile int* abort_flag, volatile int* issued, int h, int cw, int lane) {
  using SM = TcSmem<FP8>;
  const TreeArgs& a = p.a;
  const int n = static_cast<int>(P.c1 - P.c0), which = lane >> 4, r0 = 4 * (lane & 15);
  const CUtensorMap* map = which ? &p.v : &p.k;
  const uint32_t base = smem_addr(smem) + (FP8 ? SM::kRaw + which * kTcRows * kHeadDim : SM::kKv + which * SM::kTile) + r0 * 128;
  const uint8_t* scale = FP8 ? (which ? a.v_scale : a.k_scale) : nullptr;
  const uint32_t scale_dst = smem_addr(smem) + SM::kRaw + 2 * kTcRows * kHeadDim + (which * kTcRows + r0) * kKvHeads;
  const int x0 = h * kHeadDim, R = p.box_rows;
  const bool wide = R >= 4, copies = !wide || r0 % R == 0;
  const int slot_bytes = FP8 ? SM::kRawBytes : 2 * SM::kTile;
  int pages[4], len = 0, tok = 0;
  bool starts = true;
  auto look_up = [&](int k) {   // asks for the table entries of tile k; len: 0 for a drafted tile
    starts = tc_seek(a, P, cur, k) || k == 0;
    const int j = tc_chunk(cur, k);
    len = j < cur.it.nc ? cur.it.len : 0;
    tok = j * kTcRows + r0;
    if (wide) {
      int first[1];
      tree_pages<1, 1>(a, cur.it.seat, tok, len, first);
      pages[0] = first[0];
    } else {
      tree_pages<4, 1>(a, cur.it.seat, tok, len, pages);
    }
  };
  if (cw >= n) return;
  look_up(cw);
  for (int k = cw; k < n; k += SM::kCopyWarps) {
    const int slot = k % SM::kCopySlots;
    const bool cached = len > 0;
    // rows past the last token: any row of the pool (their scores are not kept, their V rows are zeroed)
    int rows[4];
    rows[0] = static_cast<int>(max(tree_row(a, pages[0], tok, len), 0ll));
    if (!wide) {
#pragma unroll
      for (int x = 1; x < 4; ++x) rows[x] = static_cast<int>(max(tree_row(a, pages[x], tok + x, len), 0ll));
    }
    if (starts) {   // a new seat's Q into the L2 cache
      for (int r = lane; r < 4 * a.tokens; r += 32)
        prefetch_l2(a.q + static_cast<long long>(cur.it.seat) * a.q_seat + static_cast<long long>(r >> 2) * a.q_tok +
                    (2 * h + ((r >> 1) & 1)) * kHeadDim + (r & 1) * (kHeadDim / 2));
    }
    if (!cached) {   // so are drafted rows: the loaders read them
      const __nv_bfloat16* src = (which ? a.v_new : a.k_new) + static_cast<long long>(cur.it.seat) * a.kv_seat + x0;
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (r0 + x < cur.it.drafts) {
          prefetch_l2(src + static_cast<long long>(r0 + x) * a.kv_tok);
          prefetch_l2(src + static_cast<long long>(r0 + x) * a.kv_tok + kHeadDim / 2);
        }
    }
    if (k + SM::kCopyWarps < n) look_up(k + SM::kCopyWarps);
    if (k >= SM::kCopySlots) {
      const int bar = FP8 ? SM::kRawFree + slot : SM::kEmpty + slot;
      if (!__all_sync(0xffffffffu, tc_wait(&bars[bar], (k / SM::kCopySlots - 1) & 1, abort_flag))) {
        if (lane == 0) tw_fail(a.status, abort_flag);
        return;
      }
      fence_proxy_async_smem();   // generic reads and writes of the slot before the copies overwrite it
    }
    uint64_t* bar = &bars[SM::kCopied + slot];
    if (lane == 0) {
      if (cached) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(FP8 ? 2 * kTcRows * kHeadDim : 2 * SM::kTile));
      else mbar_arrive(bar);
      issued[cw] = k + 1;
    }
    __syncwarp();
    if (cached) {
      const uint32_t dst = base + slot * slot_bytes, b = smem_addr(bar);
      if (wide) {
        if (copies) {
          tma_load_2d(dst, map, x0, rows[0], b);
          if (!FP8) tma_load_2d(dst + SM::kHalf, map, x0 + 64, rows[0], b);
        }
        if (FP8) {
          const uint8_t* src = scale + static_cast<long long>(rows[0]) * kKvHeads;
          cp_async16_at(scale_dst + slot * slot_bytes, src);
          cp_async16_at(scale_dst + slot * slot_bytes + 16, src + 16);
        }
      } else {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (x % R == 0) {
            tma_load_2d(dst + x * 128, map, x0, rows[x], b);
            if (!FP8) tma_load_2d(dst + SM::kHalf + x * 128, map, x0 + 64, rows[x], b);
          }
          if (FP8) cp_async8_at(scale_dst + slot * slot_bytes + x * kKvHeads, scale + static_cast<long long>(rows[x]) * kKvHeads);
        }
      }
    }
    if (FP8) cp_async_arrive(bar);
  }
}

// ------------------------------------------------------------------ the loader warps
// A seat's drafted rows (one head of each, kv_tok elements apart) as one operand tile at dst, by 128 threads; true when a V
// value was an infinity or NaN (zero is written in its place). Out of line, like all that runs once per seat.
__device__ __noinline__ bool tc_load_draft(const __nv_bfloat16* k, const __nv_bfloat16* v, long long kv_tok, int drafts, uint32_t dst,
                                           int v_off, int half, int tid) {
  const int u = tid & 15;
#pragma unroll 1
  for (int r = tid >> 4; r < kTcRows; r += 8) {
    const uint32_t at = dst + tc_unit(r, u, half), bytes = r < drafts ? 16u : 0u;   // 0: zeros
    const long long off = min(r, drafts - 1) * kv_tok + 8 * u;
    cp_async16_zfill(at, k + off, bytes);
    cp_async16_zfill(at + v_off, v + off, bytes);
  }
  cp_async_wait_all();
  bool odd = false;
#pragma unroll 1
  for (int r = tid >> 4; r < drafts; r += 8) {   // the thread's own pieces
    const uint32_t at = dst + v_off + tc_unit(r, u, half);
    const uint4 x = ld_shared16(at);
    const uint4 f = make_uint4(finite_bf16x2(x.x), finite_bf16x2(x.y), finite_bf16x2(x.z), finite_bf16x2(x.w));
    if (f.x != x.x || f.y != x.y || f.z != x.z || f.w != x.w) {
      odd = true;
      st_shared16(at, f);
    }
  }
  return odd;
}

template <bool FP8>
struct TcLoader {
  using SM = TcSmem<FP8>;
  static constexpr int kThreads = 128;   // of a drafted tile: the first four warps
  const TreeArgs& a;
  const TreePlan& P;
  uint32_t sbase;
  uint8_t* smem;
  uint64_t* bars;
  volatile int* abort_flag;
  int h, tid;

  // Everything of tile k that the copies do not write, then the tile is handed to the tensor core.
  __device__ __forceinline__ bool tile(int k, TcCursor& c, volatile int* odd) {
    const int stage = k % SM::kStages;
    tc_seek(a, P, c, k);
    const int j = tc_chunk(c, k);
    const uint32_t dst = sbase + SM::kKv + static_cast<uint32_t>(stage) * 2 * SM::kTile;
    if (k >= SM::kStages && !wait(SM::kEmpty + stage, (k / SM::kStages - 1) & 1)) return false;
    const int real = c.it.len - j * kTcRows;   // cached tiles: rows that hold a token
    bool wrote = FP8;
    if (FP8) {
      const int slot = k % (SM::kRawSlots + !FP8);
      if (!wait(SM::kCopied + slot, (k / (SM::kRawSlots + !FP8)) & 1)) return false;
      if (j < c.it.nc) convert(smem + SM::kRaw + slot * SM::kRawBytes, dst, real);
      __syncwarp();
      if ((tid & 31) == 0) mbar_arrive(&bars[SM::kRawFree + slot]);
    } else if (j < c.it.nc && real < kTcRows) {
      // whatever lies in the rows behind the last token, their probability 0 must meet a 0
      if (!wait(SM::kCopied + stage, (k / SM::kStages) & 1)) return false;
      for (int i = tid; i < (kTcRows - real) * 16; i += kThreads)
        st_shared16(dst + SM::kTile + tc_unit(real + (i >> 4), i & 15, SM::kHalf), make_uint4(0, 0, 0, 0));
      wrote = true;
    }
    if (j >= c.it.nc && tid < kThreads) {
      const long long off = static_cast<long long>(c.it.seat) * a.kv_seat + h * kHeadDim;
      if (tc_load_draft(a.k_new + off, a.v_new + off, a.kv_tok, c.it.drafts, dst, SM::kTile, SM::kHalf, tid)) odd[c.index % kTcOddSlots] = c.index + 1;
      wrote = true;
    }
    if (wrote) fence_proxy_async_smem();   // this thread's writes before the tensor core reads
    __syncwarp();
    if ((tid & 31) == 0) mbar_arrive(&bars[SM::kFull + stage]);
    return true;
  }

  // A raw e4m3 tile as bf16 operands; rows past `real` as zeros. 8 threads per row, 16 values each.
  __device__ __forceinline__ void convert(const uint8_t* raw, uint32_t dst, int real) {
    constexpr int kAll = SM::kLoaders * 32, kPer = 2 * kTcRows * 8 / kAll, kStep = kAll / 8;
    const int u = tid & 7;
    // dims 16u .. + 15 are units 2u and 2u + 1; the lanes of the second half write the odd unit first (banks)
    const bool swap = u >= 4;
    static_assert(kPer % 2 == 0, "two pieces at a time");
#pragma unroll 1
    for (int x0 = 0; x0 < kPer; x0 += 2) {   // rows 0 .. 63 are K's, 64 .. 127 V's
      uint4 w[2];
      uint32_t s[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int i = (tid >> 3) + kStep * (x0 + x);
        w[x] = *reinterpret_cast<const uint4*>(raw + i * kHeadDim + u * 16);
        s[x] = raw[2 * kTcRows * kHeadDim + i * kKvHeads + h];
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int i = (tid >> 3) + kStep * (x0 + x), r = i % kTcRows;
        const float sc = e8m0_to_float(s[x]);
        const float2 f = make_float2(sc, sc);
        const uint2 p0 = dequant4(w[x].x, f), p1 = dequant4(w[x].y, f), p2 = dequant4(w[x].z, f), p3 = dequant4(w[x].w, f);
        uint4 lo = make_uint4(p0.x, p0.y, p1.x, p1.y), hi = make_uint4(p2.x, p2.y, p3.x, p3.y);
        if (r >= real) lo = hi = make_uint4(0, 0, 0, 0);
        const uint32_t first = dst + i / kTcRows * SM::kTile + tc_unit(r, 2 * u + swap, SM::kHalf);
        st_shared16(first, swap ? hi : lo);
        st_shared16(first ^ 16u, swap ? lo : hi);
      }
    }
  }

  __device__ __forceinline__ bool wait(int bar, uint32_t parity) {
    if (__all_sync(0xffffffffu, tc_wait(&bars[bar], parity, abort_flag))) return true;
    tw_fail(a.status, abort_flag);
    return false;
  }
};

template <bool FP8>
__global__ void __launch_bounds__(TcSmem<FP8>::kThreads, 1) paged_tree_tc_kernel(const __grid_constant__ TcParams p) {
  using SM = TcSmem<FP8>;
  const TreeArgs& a = p.a;
  constexpr int kSt = SM::kStages;
  extern __shared__ __align__(1024) uint8_t tc_raw[];
  uint8_t* smem = tc_raw + ((1024u - (smem_addr(tc_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::kBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + SM::kTmemSlot);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + SM::kAbort);
  volatile int* odd = reinterpret_cast<volatile int*>(smem + SM::kOdd);
  volatile int* issued = reinterpret_cast<volatile int*>(smem + SM::kIssued);
  const uint32_t sbase = smem_addr(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int h = blockIdx.x & 7, share = blockIdx.x >> 3, shares = gridDim.x >> 3;
  const int live_warps = (2 * a.tokens + 31) / 32;              // of each softmax set
  if (tid == 32) {
    prefetch_map(&p.k);
    prefetch_map(&p.v);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the merge may be scheduled; it waits for this grid
  if (tid == 0) {
    for (int i = 0; i < kSt; ++i) {
      mbar_init(&bars[SM::kFull + i], SM::kLoaders);            // one arrival per loader warp
      mbar_init(&bars[SM::kEmpty + i], 1);
    }
    for (int i = 0; i < SM::kCopySlots; ++i) mbar_init(&bars[SM::kCopied + i], FP8 ? 33 : 1);   // + a lane's scales each
    for (int i = 0; i < SM::kRawSlots; ++i) mbar_init(&bars[SM::kRawFree + i], SM::kLoaders);
    for (int i = 0; i < kTcScores; ++i) {
      mbar_init(&bars[SM::kSFull + i], 1);
      mbar_init(&bars[SM::kPFull + i], live_warps);
      mbar_init(&bars[SM::kPvDone + i], 1);
    }
    mbar_init(&bars[SM::kQFull], live_warps);
    mbar_init(&bars[SM::kOFree], 2 * live_warps);
    for (int i = 0; i < 4; ++i) mbar_init(&bars[SM::kSets + i], 2);
    for (int i = 0; i < 2; ++i) mbar_init(&bars[SM::kFinal + i], 1);
    *abort_flag = 0;
    for (int i = 0; i < SM::kCopyWarps; ++i) issued[i] = 0;
    for (int i = 0; i < kTcOddSlots; ++i) odd[i] = 0;
    if (h == 0) tree_no_span(a, share);
    fence_mbar_init();
  }
  TreePlan P;
  if (!tree_plan<kTcTok, kTcRows, kTcTok, SM::kThreads, 1>(a, P, share, shares, 0, 2 * h, 2)) return;   // nothing allocated yet
  if (warp == SM::kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(kTcTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int n = static_cast<int>(P.c1 - P.c0);
  TcCursor cur = {P.w, 0, 0, 0, 0, P.first, tree_item<kTcTok, kTcRows, kTcTok>(a, P.w)};
  tc_enter(P, cur);

  if (warp >= SM::kCopyWarp) {
    tc_copies<FP8>(p, P, cur, smem, bars, abort_flag, issued, h, warp - SM::kCopyWarp, lane);
  } else if (warp >= kTcLoaderWarp && warp < SM::kMmaWarp) {
    TcLoader<FP8> ld{a, P, sbase, smem, bars, abort_flag, h, tid - 32 * kTcLoaderWarp};
    for (int k = 0; k < n; ++k)
      if (!ld.tile(k, cur, odd)) break;
  } else if (warp == SM::kMmaWarp || warp == SM::kMmaWarp + 1) {
    // two warps: S(k) and P(k) V(k), each tile after tile
    const bool scores = warp == SM::kMmaWarp;
    const uint32_t leader = tc_elect(), bar0 = smem_addr(bars);
    constexpr uint32_t kIdescQK = umma_idesc_bf16(128, kTcRows, 0, 0);
    constexpr uint32_t kIdescPV = umma_idesc_bf16(128, kHeadDim, 0, 1);
    const uint64_t dk = sw128_desc(sbase + SM::kKv, 1024, 16);
    const uint64_t dv = sw128_desc(sbase + SM::kKv + SM::kTile, 1024, SM::kHalf);
    bool ok = true;
    auto wait = [&](int bar, int phase) {
      return __all_sync(0xffffffffu, tc_wait(&bars[bar], static_cast<uint32_t>(phase & 1), abort_flag));
    };
    int stage = 0, lap = 0, b = 0, use = 0;   // operand stage and score buffer of tile k, and how often they came round
    for (int k = 0; k < n; ++k) {
      if (scores) {
        const bool starts = tc_seek(a, P, cur, k) || k == 0;
        ok = (!starts || wait(SM::kQFull, cur.index)) && wait(SM::kFull + stage, lap) && (FP8 || wait(SM::kCopied + stage, lap)) &&
             (use == 0 || wait(SM::kPvDone + b, use - 1));   // P(k - 3) lay where S(k) goes
        if (!ok) break;
        tc_fence_after();
        const uint64_t kk = dk + stage * (2 * SM::kTile >> 4);
        const uint32_t t_s = tmem + 64u * static_cast<uint32_t>(b), t_q = tmem + kTcQCol;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
          tc_mma_tmem_a(leader, t_s, t_q + 8u * ks, kk + ((ks >> 2) * SM::kHalf + (ks & 3) * 32) / 16, kIdescQK, ks > 0);
        tc_commit(leader, bar0 + 8 * (SM::kSFull + b));
      } else {
        const bool next = tc_seek(a, P, cur, k);
        ok = wait(SM::kPFull + b, use) && (!next || wait(SM::kOFree, cur.index - 1)) &&   // the last item's O has been read
             wait(SM::kFull + stage, lap) && (FP8 || wait(SM::kCopied + stage, lap));
        if (!ok) break;
        tc_fence_after();
        const uint64_t v = dv + stage * (2 * SM::kTile >> 4);
        const uint32_t more = k < cur.begin + 2 ? 0u : 1u;   // 0: a set's first tile of the item
#pragma unroll
        for (int ks = 0; ks < kTcRows / 16; ++ks)
          tc_mma_tmem_a(leader, tmem + kTcOCol + 128u * static_cast<uint32_t>(k & 1), tmem + 64u * static_cast<uint32_t>(b) + 8u * ks, v + ks * (2048 / 16), kIdescPV, more | ks);
        tc_commit(leader, bar0 + 8 * (SM::kEmpty + stage));
        tc_commit(leader, bar0 + 8 * (SM::kPvDone + b));
      }
      if (++stage == kSt) {
        stage = 0;
        ++lap;
      }
      if (++b == kTcScores) {
        b = 0;
        ++use;
      }
    }
    if (!ok && lane == 0) tw_fail(a.status, abort_flag);
  } else if (warp < kTcLoaderWarp && (warp & 3) < live_warps) {
    const int set = warp >> 2, r = tid & 127, tok = r >> 1;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    float2* set_ml = reinterpret_cast<float2*>(smem + SM::kMl);
    int k = 0;
    bool ok = true;
    auto wait = [&](int bar, int phase) {
      return __all_sync(0xffffffffu, tc_wait(&bars[bar], static_cast<uint32_t>(phase & 1), abort_flag));
    };
    // Row r of a seat's Q into TMEM, by the set that has the last scores of the seat before (so every one has been formed).
    auto write_q = [&](int seat) {
      const uint4* src = reinterpret_cast<const uint4*>(a.q + static_cast<long long>(seat) * a.q_seat + static_cast<long long>(tok) * a.q_tok +
                                                       (2 * h + (r & 1)) * kHeadDim);
      const bool mine = r < 2 * a.tokens;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (mine) v = __ldg(src + 8 * half + i);
          w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
        __syncwarp();
        tmem_st32u(tmem + kTcQCol + 32u * half + lane_base, w);
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[SM::kQFull]);
    };
    TcCursor nxt = cur;
    if (set == 0) write_q(cur.it.seat);
    while (k < n && ok) {
      tc_seek(a, P, cur, k);
      const int begin = cur.begin, end = cur.end;
      unsigned long long see = 0;
      if (tok < cur.it.drafts)
        see = static_cast<unsigned long long>(a.mask[static_cast<long long>(cur.it.seat) * a.mask_seat + tok]) &
              (~0ull >> (64 - cur.it.drafts));
      float m_run = -INFINITY, l_run = 0.f;
      const int k0 = begin + ((begin ^ set) & 1);                  // the set's first tile
      for (k = k0; k < end && ok; k += 2) {
        const int j = tc_chunk(cur, k), b = k % kTcScores, use = k / kTcScores;
        ok = wait(SM::kSFull + b, use);
        if (!ok) break;
        tc_fence_after();
        if (k == end - 1 && end < n) {
          tc_seek(a, P, nxt, end);
          write_q(nxt.it.seat);
        }
        const bool draft = j >= cur.it.nc;
        const int real = draft ? kTcRows : cur.it.len - j * kTcRows;
        const bool masked = draft || real < kTcRows;
        const unsigned long long keep = draft ? see : real < kTcRows ? (1ull << real) - 1 : ~0ull;   // real >= 1
        const uint32_t t_s = tmem + 64u * static_cast<uint32_t>(b) + lane_base;
        if (__builtin_expect(masked, 0)) {   // -inf where the row does not see the key
#pragma unroll 1
          for (int c = 0; c < kTcRows; c += 8) {
            float x[8];
            tmem_ld8(t_s + c, x);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = ((keep >> c >> i) & 1ull) ? x[i] : -INFINITY;
            tmem_st8(t_s + c, x);
          }
          tc_wait_st();
        }
        auto scores = [&](float (&x)[32], int half) {
          tmem_ld32(t_s + 32u * half, x);
          tc_wait_ld();
        };
        auto largest = [](const float (&x)[32]) {
          float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 32; ++i) m[i & 3] = fmaxf(m[i & 3], x[i]);
          return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
        };
        // e4m3: 96 registers hold one half of a row at a time, so its scores are read twice
        float sv[FP8 ? 1 : 2][32];
        float cmax;
        if constexpr (FP8) {
          cmax = -INFINITY;
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            scores(sv[0], half);
            cmax = fmaxf(cmax, largest(sv[0]));
          }
        } else {
          scores(sv[0], 0);
          scores(sv[1], 1);
          cmax = fmaxf(largest(sv[0]), largest(sv[1]));
        }
        cmax *= a.scale_log2;   // which is positive
        const bool grow = cmax > m_run + 8.f || (m_run == -INFINITY && cmax > -INFINITY);
        const float m_new = grow ? cmax : m_run;
        const float alpha = grow ? ex2_approx(m_run - m_new) : 1.f;
        const float mm = m_new == -INFINITY ? 0.f : m_new;
        const float2 sc2 = make_float2(a.scale_log2, a.scale_log2), nm2 = make_float2(-mm, -mm);
        float2 ls2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        m_run = m_new;
        // P(k) over S(k), columns 16 half .. + 15: the scores there have been read
#pragma unroll(FP8 ? 1 : 2)
        for (int half = 0; half < 2; ++half) {
          if constexpr (FP8) scores(sv[0], half);
          const float(&x)[32] = sv[FP8 ? 0 : half];
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 y = __ffma2_rn(make_float2(x[i], x[i + 1]), sc2, nm2);
            const float2 pp = make_float2(ex2_approx(y.x), ex2_approx(y.y));
            ls2[(i >> 1) & 1] = __fadd2_rn(ls2[(i >> 1) & 1], pp);
            pk[i / 2] = pack_bf16x2(pp.x, pp.y);
          }
          __syncwarp();
          tmem_st16u(t_s + 16u * half, pk);
        }
        const float2 ls = __fadd2_rn(ls2[0], ls2[1]);
        l_run = l_run * alpha + (ls.x + ls.y);
        if (__builtin_expect(k > k0 && __any_sync(0xffffffffu, alpha != 1.f), 0)) {   // a set's first tile of an item starts its O from zero
          ok = wait(SM::kPvDone + (k - 2) % kTcScores, (k - 2) / kTcScores);   // the set's last P V
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float ov[32];
            tmem_ld32(tmem + kTcOCol + 128u * set + lane_base + c * 32, ov);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] *= alpha;
            tmem_st32(tmem + kTcOCol + 128u * set + lane_base + c * 32, ov);
          }
          tc_wait_st();
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[SM::kPFull + b]);
      }
      k = end;
      if (!ok) break;
      // ---- the item's end: the sets exchange (maximum, sum) and wait for the last P V of both
      set_ml[((cur.index & 1) * 2 + set) * 128 + r] = make_float2(m_run, l_run);
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[SM::kSets + (warp & 3)]);
      ok = wait(SM::kSets + (warp & 3), cur.index) && wait(SM::kPvDone + (end - 1) % kTcScores, (end - 1) / kTcScores) &&
           (end - begin < 2 || wait(SM::kPvDone + (end - 2) % kTcScores, (end - 2) / kTcScores));
      if (!ok) break;
      tc_fence_after();
      const float2 other = set_ml[((cur.index & 1) * 2 + (set ^ 1)) * 128 + r];
      const float2 ml0 = set ? other : make_float2(m_run, l_run), ml1 = set ? make_float2(m_run, l_run) : other;
      const bool have0 = end - begin > 1 || (begin & 1) == 0, have1 = end - begin > 1 || (begin & 1) == 1;
      const float M = fmaxf(ml0.x, ml1.x), ref = M == -INFINITY ? 0.f : M;
      const float f0 = have0 ? exp2f(ml0.x - ref) : 0.f, f1 = have1 ? exp2f(ml1.x - ref) : 0.f;
      const float l = ml0.y * f0 + ml1.y * f1;   // an absent set's sum is 0
      // written when the item is complete here, else left as a partial (slot 2 share + 1: it starts here and goes on;
      // 2 share: it came in from the share before)
      const bool from_before = cur.first < P.c0, goes_on = cur.first + cur.it.n > P.c1;
      const int slot = from_before ? 2 * share : (goes_on ? 2 * share + 1 : -1);
      const bool mine = r < 2 * a.tokens;
      const bool none = l == 0.f || (a.draft_lens != nullptr && tok >= cur.it.drafts);
      const float inv = none ? 0.f : 1.f / l;
      const unsigned long long fix = !goes_on && odd[cur.index % kTcOddSlots] == cur.index + 1 ? see : 0ull;
      const long long col = (static_cast<long long>(max(slot, 0)) * kKvHeads + h) * (2 * a.tokens) + r;
      __nv_bfloat16* dst = a.out + static_cast<long long>(cur.it.seat) * a.out_seat +
                           static_cast<long long>(mine ? tok : 0) * a.out_tok + (2 * h + (r & 1)) * kHeadDim;
#pragma unroll 1
      for (int c = 2 * set; c < 2 * set + 2; ++c) {
        float ov[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) ov[i] = 0.f;
        if (have0) {
          tmem_ld32(tmem + kTcOCol + lane_base + c * 32, ov);
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) ov[i] *= f0;
        }
        if (have1) {
          float o1[32];
          tmem_ld32(tmem + kTcOCol + 128u + lane_base + c * 32, o1);
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) ov[i] = fmaf(o1[i], f1, ov[i]);
        }
        for (unsigned long long v = fix; v != 0; v &= v - 1) {   // infinities and NaN of drafted rows this row sees
          const __nv_bfloat16* src = a.v_new + static_cast<long long>(cur.it.seat) * a.kv_seat +
                                     static_cast<long long>(__ffsll(v) - 1) * a.kv_tok + h * kHeadDim + c * 32;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float x = __bfloat162float(src[i]);
            if (!(fabsf(x) < INFINITY)) ov[i] += x;
          }
        }
        if (mine && slot < 0) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 w;
            w.x = pack_bf16x2(ov[i] * inv, ov[i + 1] * inv);
            w.y = pack_bf16x2(ov[i + 2] * inv, ov[i + 3] * inv);
            w.z = pack_bf16x2(ov[i + 4] * inv, ov[i + 5] * inv);
            w.w = pack_bf16x2(ov[i + 6] * inv, ov[i + 7] * inv);
            *reinterpret_cast<uint4*>(dst + c * 32 + i) = none ? make_uint4(0, 0, 0, 0) : w;
          }
        } else if (mine) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(a.ws_o + col * kHeadDim + c * 32 + i) = make_float4(ov[i], ov[i + 1], ov[i + 2], ov[i + 3]);
        }
        __syncwarp();   // the TMEM loads are the whole warp's
      }
      if (slot >= 0 && mine && set == 0) *reinterpret_cast<float2*>(a.ws_ml + 2 * col) = make_float2(M, l);
      if (!from_before && h == 0 && tid == 0)
        tree_span(a, cur.w, share, goes_on ? tree_last_share(P, cur.first + cur.it.n - 1) : share);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[SM::kOFree]);
    }
    if (!ok && lane == 0) tw_fail(a.status, abort_flag);
  }

  // ------------------------------------------------------------------ teardown
  tc_fence_before();
  __syncthreads();
  if (*abort_flag && (warp == SM::kMmaWarp || warp == SM::kMmaWarp + 1) && tc_elect()) {   // let what is in flight finish (bounded)
    umma_commit(&bars[SM::kFinal + warp - SM::kMmaWarp]);
    mbar_wait_bounded(&bars[SM::kFinal + warp - SM::kMmaWarp], 0, 200000000ull);
    int top = 0;
    for (int i = 0; i < SM::kCopyWarps; ++i) top = max(top, issued[i]);
    for (int k = max(top - SM::kCopySlots - SM::kCopyWarps, 0); k < top; ++k)
      if (k < issued[k % SM::kCopyWarps])
        mbar_wait_bounded(&bars[SM::kCopied + k % SM::kCopySlots], (k / SM::kCopySlots) & 1, 200000000ull);
  }
  __syncthreads();
  tc_fence_after();
  if (warp == SM::kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTcTmemCols));
}

// A pool as rows of 1024 elements, read 128 bytes x box_rows rows at a time. bf16: 128-byte swizzle.
template <bool FP8>
bool make_pool_map(CUtensorMap* m, const void* base, long long rows, int box_rows) {
  const EncodeTiled enc = tensor_map_encoder();
  if (!enc || rows > (1ll << 31) - 1) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(kKvHeads * kHeadDim), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(FP8 ? kRowBytes / 2 : kRowBytes)};
  const cuuint32_t box[2] = {FP8 ? 128u : 64u, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1u, 1u};
  return enc(m, FP8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims,
             strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, FP8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
             FP8 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool FP8>
cudaError_t launch_tc(const TreeArgs& a, int grid, cudaStream_t stream) {
  auto kern = paged_tree_tc_kernel<FP8>;
  static thread_local int configured_device = -1;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (configured_device != dev) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, TcSmem<FP8>::kAlloc);
    if (e != cudaSuccess) return e;
    configured_device = dev;
  }
  TcParams p;
  memset(&p, 0, sizeof(p));
  p.a = a;
  const long long rows = static_cast<long long>(a.num_pages) * a.page_size;
  p.box_rows = a.page_size & -a.page_size;
  if (p.box_rows > kTcRows) p.box_rows = kTcRows;
  if (!make_pool_map<FP8>(&p.k, a.k_pool, rows, p.box_rows) || !make_pool_map<FP8>(&p.v, a.v_pool, rows, p.box_rows))
    return cudaErrorInvalidValue;
  kern<<<grid, TcSmem<FP8>::kThreads, TcSmem<FP8>::kAlloc, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_tree_tc(const TreeArgs& a, int shares, cudaStream_t stream) {
  return a.k_scale != nullptr ? launch_tc<true>(a, shares * kKvHeads, stream) : launch_tc<false>(a, shares * kKvHeads, stream);
}

}  // namespace q3
