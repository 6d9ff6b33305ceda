// Causal attention of many new tokens per request over the paged cache, on the fifth-generation
// matrix units (pd_prefill with maps = 1 or 2).
//
// Mathematics.  For one kv head the rows (token, head of its group) of a request are packed into
// tiles of 128; a tile walks the request's keys in blocks of 128 with the base-2 online softmax:
//   S = Q K^T,  m' = max(m, max S),  P = 2^(S - m'),  l = l 2^(m - m') + sum P,  O = O 2^(m - m') + P V.
// A CTA has two such tiles.  maps = 1: the two halves of 256 packed rows, against the same keys.
// maps = 2: the SAME 128 rows with their two queries against the two keys of the pair, and one V of
// 2 * head_dim columns; the epilogue subtracts, norms and stores.  A CTA holds at most 128 columns of
// V: for head_dim 128 the two halves belong to a cluster of two CTAs, which exchange the rows'
// sums of squares.
//
// Why so.  Per tile and block the matrix units take 128 * 128 * (D + DV) multiply-adds, 4096 a
// cycle, and the special function units 128 * 128 exponentials, 16 a cycle: 1024 cycles of each at
// D = DV = 128.  Neither may wait for the other, hence the two tiles: while one tile's softmax runs
// on its four warps, the matrix units work for the other.  A thread owns one row, so maximum and sum
// need no exchange.  S and O stay in tensor memory (2 * (128 + DV) columns), P replaces S there as
// 16-bit pairs and is read by the second product from tensor memory; shared memory holds Q and a
// ring of K and V tiles in the 128-byte swizzle.
//
// Three warps fill the ring, a lane for each TMA box of up to 128 tokens of a page and 64 columns.  What
// such boxes cost is their number: 32 of 16 tokens a block keep pace with the products only when the waits
// leave the SM alone and several warps issue (8192 tokens of 32/8 heads, head_dim 128, bf16, one set of inputs in a
// graph: 457 us at pages of 16 and of 128 alike, 1.2 PFLOP/s; one loader and polling waits: 649.  Calls over changing
// inputs under the power cap: 534, 1.03 PFLOP/s).  Pages that are no multiple of 16 tokens come by 16-byte asynchronous copies, row by row.  V's rows behind the last
// key are cleared behind the copy, because zero times the NaN that a page may hold would stay.
//
// P is rounded to the pages' 16-bit type for the product with V: relative to a result about what rounding
// the result itself costs (2.1e-4 of its norm in fp16, 1.7e-3 in bf16).  The difference of two maps that share
// V has sqrt((1 + lambda^2) / (1 + lambda^2 - 2 lambda r)) times as much, r their overlap: 3.2e-4 in all for
// fp16.  A second 16-bit term of the first map's P (products with V and stores of P half as many again) brought
// that to 2.3e-4 and cost 14 to 21 % (4096 new tokens of 16/4 heads, head_dim 128, fp16: 290 -> 350 us).
//
// The maximum that P refers to may lag behind the true one by kLag (2^3 or 2^8 at most): O is then not
// rescaled for every small rise.  It cancels in O / l; l and O are 32-bit.
//
// Few rows and long contexts: the key blocks are split over `splits` CTAs, each writes normalised
// 32-bit rows and their log-sum-exp, and a second kernel joins them.
//
// 8-bit pages: four more warps read the pages, widen the elements exactly and store them in the
// same swizzle; K's scales multiply S, V's scales multiply P (times 32, against fp16's subnormals),
// so nothing is rounded on the way but P itself; its sum l is that of the unrounded P, as P is rounded once for
// each value head, with that head's scales.  32 P times the scale keeps fp16's 11 bits
// down to 2^-14, below that it has a step of 2^-24.  Six chunks of 159 to 503 tokens behind 1.8 to 5.3 k of int8 keys (28/4 heads,
// head_dim 128): 201 us, 475 TFLOP/s; the scales' two multiplications a score on the softmax warps bound it.
//
// Two maps: one prompt of 4096 tokens, 16/4 pairs of head_dim 128, fp16: 292 us, 706 TFLOP/s, a third of the
// products more than counted because both CTAs of a cluster need S.  Drafts of 4 or 5 tokens behind 22 to 25 k
// (16/4 pairs of 64): 60 us, 3.3 TB/s, split 18 ways; the number of TMA boxes and the join bound it.
//
// Every wait is bounded; one that gives up raises PD_DEV_TIMEOUT and ends the CTA's loops.  Nobody
// skips a barrier on that way, tensor memory is freed, and copies and products in flight are
// awaited (bounded) first.
#pragma once

#include "pd_prefill.h"
#include "pd_stream_kernel.cuh"

namespace pd {

constexpr int kTcBlock = 128;      // keys of one block, rows of one tile
constexpr int kTcLeast = 4;        // key blocks a split has at least: what its start and end cost is about that
constexpr int kTcMetaRing = 16;    // blocks whose bad-page masks are kept
constexpr int kTcSmem = 227 * 1024;

template <int KV, int D, int MAPS, bool SCALED>
struct TcCfg {
  static constexpr bool WIDEN = !is_16bit(KV);             // 8-bit pages: four warps widen the tiles
  static constexpr bool BF16 = KV == PD_KV_BF16;
  static constexpr int DV = MAPS == 2 ? 128 : D;           // columns of V in one CTA
  static constexpr int SLICES = MAPS * D / DV;             // CTAs that share V's columns
  static constexpr int VH = DV / D > 1 ? DV / D : 1;       // V heads side by side in the slice
  static constexpr int NP = SCALED ? VH : 1;               // different P operands (one for each V head's scales)
  static constexpr int KT = MAPS;                          // K tiles of one block
  static constexpr int KH = D / 64, VC = DV / 64;          // 64-column pieces of a K and of a V row
  static constexpr int ROWS = MAPS == 2 ? 128 : 256;       // packed rows of one CTA
  static constexpr int QTILE = 128 * D * 2;
  static constexpr int SLOT = 128 * (D > DV ? D : DV) * 2;
  static constexpr int SCALE_FLOATS = SCALED ? (KT + VH) * 128 : 0;  // of one block
  static constexpr int SCALE_RING = 8;                     // more blocks than the ring of tiles can be ahead of the softmax
  static constexpr int MISC = 1024 + (MAPS == 2 ? 2560 : 0);
  static constexpr int RAW = WIDEN ? 128 * (D > DV ? D : DV) : 0;      // one 8-bit tile as it comes
  static constexpr int NRAW = 3;
  static constexpr int FIXED = 1024 + 2 * QTILE + SCALE_RING * SCALE_FLOATS * 4 + NRAW * RAW + MISC;
  static constexpr int FIT = (kTcSmem - FIXED) / SLOT;
  static constexpr int NSLOT = FIT > 8 ? 8 : FIT;
  static constexpr int SMEM = FIXED + NSLOT * SLOT;
  // softmax 0-3 and 4-7, matrix units 9, loaders 8, 10, 11; widening 12-15
  static constexpr int WARPS = WIDEN ? 16 : 12;
  // Registers.  A scheduler has a warp of each tile's softmax, one of the third group and, with 8-bit pages,
  // one that widens; what they hold adds up to the launch's 3 * 168 or 4 * 128.
  static constexpr int REGS_SOFTMAX = WIDEN ? 176 : 200, REGS_THIRD = WIDEN ? 80 : 104, REGS_WIDEN = 80;
  static_assert(WIDEN ? 2 * REGS_SOFTMAX + REGS_THIRD + REGS_WIDEN <= 4 * 128 : 2 * REGS_SOFTMAX + REGS_THIRD <= 3 * 168, "registers");
  static constexpr int THREADS = WARPS * 32;
  static constexpr int RING = WIDEN ? NRAW : NSLOT;        // what the loaders fill
  static_assert(NSLOT >= (WIDEN ? 3 : 4) && NRAW >= KT + 1 && SMEM <= kTcSmem, "shared memory; how far a loader's units are apart");
};

struct TcParams {
  PrefillParams a;
  int32_t tiles, heads, splits;  // grid: splits x tiles x heads (x slices)
  int32_t box_tokens;            // tokens of one TMA box
  int32_t target;                // CTAs to share the key blocks out over
  float* part_o;                 // splits > 1: [split][row][head, map][columns of V in all], log-sum-exps
  float* part_lse;
};

// ---- tcgen05 wrappers ----------------------------------------------------------------------------
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// The matrix units' warp runs its loops as one and lets a single lane (`mine`) issue: operands then
// live in the warp's uniform registers.  (Issued from inside a one-lane branch, an instruction took about
// 100 cycles, most of it moving operands there.)
__device__ __forceinline__ void tc_commit(uint32_t bar, uint32_t mine) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(bar), "r"(mine)
      : "memory");
}
// D (128 x N, f32, tensor memory) (+)= A (128 x 16) * B (16 x N); A and B by shared-memory descriptors
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate, uint32_t mine) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1 : 0), "r"(mine)
      : "memory");
}
// the same with A in tensor memory (16-bit pairs)
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate, uint32_t mine) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1 : 0), "r"(mine)
      : "memory");
}
#define PD_I8(x, i) "r"((x)[i]), "r"((x)[i + 1]), "r"((x)[i + 2]), "r"((x)[i + 3]), "r"((x)[i + 4]), \
                    "r"((x)[i + 5]), "r"((x)[i + 6]), "r"((x)[i + 7])
#define PD_F8(x, i) "=f"((x)[i]), "=f"((x)[i + 1]), "=f"((x)[i + 2]), "=f"((x)[i + 3]), "=f"((x)[i + 4]), \
                    "=f"((x)[i + 5]), "=f"((x)[i + 6]), "=f"((x)[i + 7])
#define PD_G8(x, i) "f"((x)[i]), "f"((x)[i + 1]), "f"((x)[i + 2]), "f"((x)[i + 3]), "f"((x)[i + 4]), \
                    "f"((x)[i + 5]), "f"((x)[i + 6]), "f"((x)[i + 7])
// 32 columns of the warp's 32 lanes: thread = lane, register = column
__device__ __forceinline__ void tc_ld32(uint32_t addr, float* x) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : PD_F8(x, 0), PD_F8(x, 8), PD_F8(x, 16), PD_F8(x, 24)
      : "r"(addr));
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const float* x) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(addr), PD_G8(x, 0), PD_G8(x, 8), PD_G8(x, 16), PD_G8(x, 24)
      : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t* x) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(addr), PD_I8(x, 0), PD_I8(x, 8)
      : "memory");
}

// Where row r, piece c (64 columns, 128 bytes) of a Q, K or V tile lies: one plane of 128 rows a piece.
__device__ __forceinline__ uint32_t tc_row(int r, int c) { return (uint32_t)(c * (128 * 128) + r * 128); }
// Shared-memory operand descriptor in the 128-byte swizzle: 8-row groups `stride` bytes apart.  K-major
// tiles have 64 elements of the inner dimension per row, the leading offset is not used; MN-major ones
// (V) have 64 columns per row and find the next 64 columns `lead` bytes on.
__device__ __forceinline__ uint64_t tc_desc(uint32_t addr, uint32_t stride, uint32_t lead) {
  return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)((lead >> 4) & 0x3fffu) << 16) |
         ((uint64_t)(stride >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// 16 bytes from global to shared memory (generic proxy); zeros when `live` is not set.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"((unsigned long long)src), "r"(live ? 16 : 0) : "memory");
}
// Instruction descriptor: f32 accumulators, f16 or bf16 operands, M = 128, N columns, B MN-major or K-major.
__host__ __device__ constexpr uint32_t tc_idesc(bool bf16, int n, bool b_mn) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

// A bounded wait for a barrier phase, by every lane of a warp; the answer is the warp's.  try_wait suspends
// the warp for up to kTcSuspendNs at a time, so a waiting warp costs the others next to nothing; after
// kTcTries of them (50 ms at the very least) it gives up, raises the CTA's abort flag and PD_DEV_TIMEOUT.
// Inline on purpose: a call keeps the softmax's 128 scores from staying in registers.
constexpr int kTcTries = 1 << 22;
constexpr unsigned kTcSuspendNs = 1000;
__device__ __forceinline__ bool tc_wait(uint32_t bar, uint32_t parity, uint32_t* status, volatile int* abort_flag) {
  bool ok = false;
  for (int i = 0; i < kTcTries; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity), "r"(kTcSuspendNs)
        : "memory");
    ok = done != 0;
    if (ok || *abort_flag) break;
  }
  if (__all_sync(0xffffffffu, ok)) return true;
  *abort_flag = 1;
  if (status) atomicOr(status, PD_DEV_TIMEOUT);
  return false;
}

// Gives what is still in flight a bounded chance to end (the abort flag is up).
__device__ __forceinline__ void tc_drain(uint32_t bar, uint32_t parity) {
  for (int i = 0; i < kTcTries && !mbar_try_wait(bar, parity); ++i) {
  }
}

// Two floats in one instruction, and the largest of three.
__device__ __forceinline__ void tc_fma2(float& x, float& y, float f, float g) {  // (x, y) = (x, y) * f + g
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\tmov.b64 c, {%3, %3};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(f), "f"(g));
}
__device__ __forceinline__ void tc_add2(float& x, float& y, float f, float g) {  // (x, y) += (f, g)
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
      "add.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(f), "f"(g));
}
__device__ __forceinline__ void tc_mul2(float& x, float& y, float f, float g) {  // (x, y) = (x * f, y * g)
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
      "mul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(f), "f"(g));
}
__device__ __forceinline__ float tc_max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

template <bool BF16>
__device__ __forceinline__ uint32_t tc_pack(float lo, float hi) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return pack_half2(lo, hi);
  }
}

// 128 rows of PIECES * 64 columns into a tile; row[i] of lane l is the offset of row 32 i + l's first column
// (-1: zeros).  Pieces beyond a head's D columns belong to the next head.
template <int PIECES, int D>
__device__ __forceinline__ void tc_copy_rows(uint32_t dst, const __half* cache, const int64_t (&row)[4], int64_t head_stride,
                                             int lane) {
  constexpr int CH = PIECES * 8;  // 16-byte chunks, and lanes, of a row
  constexpr int RPI = 32 / CH;    // rows of one warp-wide copy
  const int c = lane % CH, rr = lane / CH, piece = c / 8;
  const __half* mine = cache + (D == 64 && piece ? head_stride : 0) + (D == 64 ? c % 8 : c) * 8;
#pragma unroll
  for (int i = 0; i < 128 / RPI; ++i) {
    const int r = i * RPI + rr;
    const int64_t at = __shfl_sync(0xffffffffu, row[i * RPI / 32], r & 31);
    cp_async16(dst + tc_row(r, piece) + (((c & 7) ^ (r & 7)) << 4), at >= 0 ? mine + at : cache, at >= 0);
  }
}

// Offset of a token of the request in a cache tensor (kv head 0), and in the scales, or -1: no such key, or
// one in no page of the pool, which is noted in its block's mask.
__device__ __forceinline__ int64_t tc_place(const Params& p, int request, int token, int kv_end, unsigned* mask, unsigned bits,
                                            int64_t& scale_at) {
  scale_at = 0;
  if (token >= kv_end) return -1;
  const int page = token / p.page;
  const int id = __ldg(p.block_table + (int64_t)request * p.bt_stride + page);
  if ((unsigned)id < (unsigned)p.num_blocks) {
    scale_at = scale_offset(p, id, token - page * p.page, 0);
    return kv_row_offset(p, id, token - page * p.page, 0);
  }
  if (p.status) atomicOr(p.status, PD_DEV_BAD_BLOCK);
  if (mask) atomicOr(mask, bits);
  return -1;
}

// The 16-byte pieces of an 8-bit tile that thread `me` of 128 takes, from pages of odd sizes: piece c of the rows
// r0, r0 + 128 / P, ..  Bit i of the answer: piece i exists.  All addresses first, then all loads, and nothing
// that uses one: they are to be in flight together.
template <int P, int D, int PM>
__device__ __forceinline__ unsigned tc_fetch(const Params& p, int request, int j, int h, const void* cache, int kv_end,
                                             unsigned* mask, int me, uint4 (&x)[PM]) {
  const int c = me % P, r0 = me / P;
  const char* mine = (const char*)cache + (int64_t)(h + c * 16 / D) * p.kv_sh + c * 16 % D;
  const uint4* from[P];
  unsigned live = 0;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int r = r0 + i * (128 / P);
    int64_t unused;
    const int64_t at = tc_place(p, request, j * kTcBlock + r, kv_end, mask + r / 32, 1u << (r & 31), unused);
    live |= (at >= 0 ? 1u : 0u) << i;
    from[i] = reinterpret_cast<const uint4*>(mine + (at >= 0 ? at : 0));  // some row of the pool where there is none
  }
#pragma unroll
  for (int i = 0; i < P; ++i) x[i] = __ldg(from[i]);
  return live;
}
// The same pieces from a tile that has come by TMA; rows behind the last key (whatever their page holds) are left out.
template <int P, int D, int PM>
__device__ __forceinline__ unsigned tc_take(uint32_t raw, int keys, int me, uint4 (&x)[PM]) {
  const int c = me % P, r0 = me / P;
  unsigned live = 0;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int r = r0 + i * (128 / P);
    uint32_t w[4];
    lds128(raw + (c * 16 / D) * (128 * D) + r * D + c * 16 % D, w);
    x[i] = make_uint4(w[0], w[1], w[2], w[3]);
    live |= (r < keys ? 1u : 0u) << i;
  }
  return live;
}

// A warp's 32 result rows of CH 16-byte chunks, from a thread a row to whole rows at a time: the chunks go through
// 32 * CH * 16 bytes of shared memory (`area`), neighbouring lanes then store neighbouring chunks of a row.
// (Straight from the threads a store touched 32 rows.)  `off` of lane l: where row l begins in out, -1: nowhere.
template <int CH>
__device__ __forceinline__ void tc_put_chunk(uint32_t area, int lane, int c, const uint4& y) {
  sts128(area + lane * (CH * 16) + ((c ^ (lane & 7)) << 4), y);
}
template <int CH>
__device__ __forceinline__ void tc_store_rows(uint32_t area, int lane, __half* out, int64_t off) {
  __syncwarp();
  const int c = lane % CH;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int r = i * (32 / CH) + lane / CH;
    uint32_t w[4];
    lds128(area + r * (CH * 16) + ((c ^ (r & 7)) << 4), w);
    const int64_t at = __shfl_sync(0xffffffffu, off, r);
    if (at >= 0) *reinterpret_cast<uint4*>(out + at + c * 8) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// What a CTA works on.
struct TcTile {
  int request, row0, count;  // first packed row (within the request) and packed rows, at most ROWS
  int first_token;           // row of q of the request's first token
  int tokens, len;           // new tokens and cached tokens of the request
};

// The tile with number i: request b's tiles begin at floor(query_start[b] * group / ROWS) + b, which leaves
// room for ceil(tokens * group / ROWS) of them.  Found by one warp, 32 probes at a time.
__device__ __forceinline__ bool tc_find_tile(const PrefillParams& a, int rows_per_tile, int i, int lane, TcTile& t) {
  const Params& p = a.p;
  const int64_t group = p.group;
  int lo = 0, n = p.batch;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lane * step;
    const bool before = at < n && (int64_t)__ldg(a.starts + lo + at) * group / rows_per_tile + lo + at <= i;
    const int k = max(__popc(__ballot_sync(0xffffffffu, before)) - 1, 0);
    lo += k * step;
    n = min(step, n - k * step);
  }
  const int start = __ldg(a.starts + lo);
  const int tokens = __ldg(a.starts + lo + 1) - start;
  if (start < 0 || start >= a.rows || tokens <= 0) return false;
  const int held = min(tokens, a.rows - start);  // of them in q; those cut off still count for the others' positions
  const int64_t local = i - ((int64_t)start * group / rows_per_tile + lo);
  if (local < 0 || local * rows_per_tile >= (int64_t)held * group) return false;
  t.request = lo;
  t.row0 = (int)(local * rows_per_tile);
  t.count = (int)min((int64_t)rows_per_tile, (int64_t)held * group - t.row0);
  t.first_token = start;
  t.tokens = tokens;
  t.len = clamp_len(p, lo);
  return true;
}

// Unit `unit` of the loads: the first block's K tiles, then V of each block followed by the next one's K.
template <int KT>
__device__ __forceinline__ void tc_unit(int unit, int j0, int& j, int& k) {
  if (unit < KT) {
    j = j0;
    k = unit;
  } else {
    const int u = unit - KT;
    const int cyc = u / (KT + 1), in = u % (KT + 1);
    j = j0 + cyc + (in ? 1 : 0);
    k = in - 1;
  }
}

// Keys that packed row r of the request sees.
__device__ __forceinline__ int tc_limit(const TcTile& t, int r, int group) {
  const int n = t.len - t.tokens + r / group + 1;
  return n < 0 ? 0 : n;  // r is the request's: at most t.len
}

template <int KV, int D, int MAPS, bool SCALED>
__global__ void __launch_bounds__(TcCfg<KV, D, MAPS, SCALED>::THREADS, 1)
tc_prefill_kernel(const __grid_constant__ TcParams tp, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v) {
  using C = TcCfg<KV, D, MAPS, SCALED>;
  constexpr unsigned kFull = 0xffffffffu;
  constexpr float kLag = SCALED ? 3.f : 8.f;    // P is at most 2^kLag (times a V scale and 32: below fp16's range up to scales of 255)
  constexpr float kBoost = SCALED ? 32.f : 1.f;
  const PrefillParams& a = tp.a;
  const Params& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  // ring of tiles, Q, scales, 8-bit tiles, the rest
  const uint32_t ring0 = base, q0 = base + C::NSLOT * C::SLOT;
  const uint32_t raw0 = q0 + 2 * C::QTILE + C::SCALE_RING * C::SCALE_FLOATS * 4;
  float* scales = reinterpret_cast<float*>(smem + C::NSLOT * C::SLOT + 2 * C::QTILE);
  uint8_t* misc = smem + C::NSLOT * C::SLOT + 2 * C::QTILE + C::SCALE_RING * C::SCALE_FLOATS * 4 + C::NRAW * C::RAW;
  unsigned* meta = reinterpret_cast<unsigned*>(misc);  // [block mod 16][4]: its tokens whose page is not in the pool
  volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + 256);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(misc + 260);
  volatile int* have_tile = reinterpret_cast<volatile int*>(misc + 264);
  volatile int* share = reinterpret_cast<volatile int*>(misc + 268);  // key blocks of a piece
  TcTile* tile_sh = reinterpret_cast<TcTile*>(misc + 272);
  const uint32_t bars = smem_u32(misc) + 320;
  const uint32_t full0 = bars, empty0 = bars + 64, s_full = bars + 128, o_done = bars + 144, q_full = bars + 160,
                 drain_bar = bars + 168, tail_bar = bars + 208, raw_full = bars + 216, raw_empty = bars + 248, p_full = bars + 176;  // p_full: [tile][half of the keys]
  float* squares = reinterpret_cast<float*>(misc + 640);  // [tile][128] of this CTA's columns, then of the peer's
  float* weights = reinterpret_cast<float*>(misc + 640 + 2048);  // the norm's, of the slice
  static_assert(kTcMetaRing * 16 <= 256 && (MAPS == 1 ? 640 : 640 + 2048 + 512) <= C::MISC, "misc area");

  // ---- which tile ------------------------------------------------------------------------------
  const int slice = C::SLICES == 1 ? 0 : blockIdx.x % C::SLICES;
  int work = blockIdx.x / C::SLICES;
  const int head = work % tp.heads;  // kv head, or kv pair
  work /= tp.heads;
  const int tile_no = tp.tiles - 1 - work % tp.tiles;  // a prompt's last tiles are its longest: they go first
  const int split = work / tp.tiles;
  if (warp == 0) {
    if (lane < kTcMetaRing) *reinterpret_cast<uint4*>(meta + 4 * lane) = make_uint4(0, 0, 0, 0);
    TcTile t;
    const bool ok = tc_find_tile(a, C::ROWS, tile_no, lane, t);
    if (lane == 0) {
      *have_tile = ok ? 1 : 0;
      if (ok) *tile_sh = t;
      *abort_flag = 0;
    }
  }
  // With splits: the key blocks of all tiles shared out evenly over the CTAs that there are SMs for, so that a
  // long context is cut into more pieces than a short one (an even cut of each, nine pieces of contexts of
  // 16 to 32 k: the longest pieces were half as long again as the mean).
  if (warp == 1 && tp.splits > 1) {
    long long sum = 0;
    for (int b = lane; b < p.batch; b += 32) {
      const int tokens = __ldg(a.starts + b + 1) - __ldg(a.starts + b), len = __ldg(p.seq_lens + b);
      if (tokens > 0 && len > 0) {
        const long long tiles = ((long long)tokens * p.group + C::ROWS - 1) / C::ROWS;
        sum += tiles * ((min((long long)len, (long long)p.max_blocks * p.page) + kTcBlock - 1) / kTcBlock);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    if (lane == 0) *share = (int)min((sum * tp.heads * C::SLICES + tp.target - 1) / tp.target, (long long)INT32_MAX);
  }
  if (warp == 8 && lane == 0) {
    for (int s = 0; s < C::NSLOT; ++s) {
      mbar_init(full0 + 8 * s, C::WIDEN ? 128 : 32);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full + 8 * t, 1);
      mbar_init(p_full + 16 * t, 128);
      mbar_init(p_full + 16 * t + 8, 128);
      mbar_init(o_done + 8 * t, 1);
    }
    mbar_init(q_full, 256);
    mbar_init(drain_bar, 1);
    for (int s = 0; s < C::NRAW; ++s) {
      mbar_init(raw_full + 8 * s, 32);
      mbar_init(raw_empty + 8 * s, 128);
    }
    mbar_init(tail_bar, 1);
    fence_barrier_init();
    fence_proxy_async();
    asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&tm_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&tm_v) : "memory");
  }
  __syncthreads();
  if (!*have_tile) return;  // the whole cluster has the same tile: nobody waits for this CTA
  // the peer runs before anything is written to its shared memory
  if (C::SLICES == 2 && tp.splits == 1) tc_cluster_sync();
  if (MAPS == 2 && tid < 128) weights[tid] = a.weight ? __ldg(a.weight + slice * C::DV + tid) : 1.f;
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32((const void*)tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const TcTile tile = *tile_sh;

  // ---- the tiles' rows and key blocks ----------------------------------------------------------------
  // maps = 1: tile t has the packed rows 128 t ..; maps = 2: both tiles have the same rows
  int rows_of[2], begin[2], end[2];  // rows, first and last + 1 key block
  const int last_row = tile.row0 + tile.count - 1;
  const int blocks = (tc_limit(tile, last_row, p.group) + kTcBlock - 1) / kTcBlock;  // of the longest row
  int chunk = blocks;
  if (tp.splits > 1) chunk = max(max((blocks + tp.splits - 1) / tp.splits, *share), kTcLeast);
  const int j0 = min(split * chunk, blocks), j1 = min(j0 + chunk, blocks);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    rows_of[t] = MAPS == 2 ? tile.count : max(0, min(128, tile.count - 128 * t));
    const int top = rows_of[t] ? tc_limit(tile, tile.row0 + (MAPS == 2 ? 0 : 128 * t) + rows_of[t] - 1, p.group) : 0;
    begin[t] = j0;
    end[t] = max(j0, min(j1, (top + kTcBlock - 1) / kTcBlock));
  }
  const int jend = max(end[0], end[1]);
  const int kv_end = tc_limit(tile, last_row, p.group);  // keys from here on are zeros in shared memory

  // ================================ widening warps (8-bit pages) =======================================
  // Four warps; a thread takes the 16-byte pieces me, me + 128, .. of a tile's rows.  The tiles come by TMA (by
  // plain loads they came at 5 bytes a cycle, half the time of a block); the scales, two bytes a token, are
  // fetched a block ahead by the thread that owns the token.
  if (warp >= 12) {
    if constexpr (C::WIDEN) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_WIDEN));
      const int me = tid - 384;  // 0 .. 127
      constexpr int PK = D / 16, PV = C::DV / 16;        // 16-byte pieces of a K and of a V row = of a thread
      constexpr int PM = PK > PV ? PK : PV;
      constexpr int NS = SCALED ? C::KT + C::VH : 1;
      const int nb = jend - j0;
      const int units = nb > 0 ? nb * (C::KT + 1) : 0;
      const bool whole = p.page % 16 == 0;               // the loaders bring the tiles, and note pages outside the pool
      // the scales of token `me` of block j, K's and V's: the softmax needs V's ahead of V itself
      auto fetch_scales = [&](int j, __half (&sc)[NS]) {
        if constexpr (SCALED) {
          int64_t at;
          const bool live = j < jend && tc_place(p, tile.request, j * kTcBlock + me, kv_end, nullptr, 0, at) >= 0;
          at = (live ? at : 0) + head * MAPS;
#pragma unroll
          for (int z = 0; z < C::KT; ++z) sc[z] = __ldg(p.k_scale + at + z);
#pragma unroll
          for (int z = 0; z < C::VH; ++z) sc[C::KT + z] = __ldg(p.v_scale + at + (MAPS == 2 ? slice * C::DV / D + z : 0));
          return live;
        } else {
          return true;
        }
      };
      __half sc[NS];
      bool sc_live = units > 0 && fetch_scales(j0, sc);
      bool ok = true;
      for (int unit = 0; unit < units && ok; ++unit) {
        int j, k;
        tc_unit<C::KT>(unit, j0, j, k);
        unsigned* mask = meta + 4 * (j & (kTcMetaRing - 1));
        uint4 x[PM];
        unsigned live;
        if (whole) {
          const int rs = unit % C::NRAW;
          ok = tc_wait(raw_full + 8 * rs, (uint32_t)(unit / C::NRAW) & 1u, p.status, abort_flag);
          if (!ok) break;
          const uint32_t raw_tile = raw0 + rs * C::RAW;
          live = k < 0 ? tc_take<PV, D, PM>(raw_tile, kv_end - j * kTcBlock, me, x)
                       : tc_take<PK, D, PM>(raw_tile, kv_end - j * kTcBlock, me, x);
          mbar_arrive(raw_empty + 8 * rs);
        } else {
          // the mask of a block read long ago, of one far ahead
          if (k == 0 && me < 4) meta[4 * ((j + kTcMetaRing / 2) & (kTcMetaRing - 1)) + me] = 0;
          live = k < 0 ? tc_fetch<PV, D, PM>(p, tile.request, j, head * MAPS + slice * C::DV / D, p.v, kv_end, mask, me, x)
                       : tc_fetch<PK, D, PM>(p, tile.request, j, head * MAPS + k, p.k, kv_end, mask, me, x);
        }
        const int st = unit % C::NSLOT;
        const uint32_t dst = ring0 + st * C::SLOT;
        ok = tc_wait(empty0 + 8 * st, ((uint32_t)(unit / C::NSLOT) & 1u) ^ 1u, p.status, abort_flag);
        if (!ok) break;
        const int pieces = k < 0 ? PV : PK;
#pragma unroll
        for (int i = 0; i < PM; ++i) {
          if (i >= pieces) continue;
          const int n = me + i * 128, r = n / pieces, c = n % pieces;
          const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
          const uint32_t keep = (live >> i) & 1 ? 0xffffffffu : 0u;
          uint32_t h[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t y = KV == PD_KV_I8 ? (w[e] & keep) ^ 0x80808080u : w[e] & keep;
            h[2 * e] = cvt_pair<KV>(y, false);
            h[2 * e + 1] = cvt_pair<KV>(y, true);
          }
          const uint32_t row = dst + tc_row(r, c / 4);
          const int ch = (2 * c) & 7;
          // neighbours that share banks store their two halves in opposite order
          const int flip = (c >> 2) & 1;
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            const bool upper = (o ^ flip) != 0;
            const uint4 y = make_uint4(upper ? h[4] : h[0], upper ? h[5] : h[1], upper ? h[6] : h[2], upper ? h[7] : h[3]);
            sts128(row + (((ch + (upper ? 1 : 0)) ^ (r & 7)) << 4), y);
          }
        }
        if constexpr (SCALED) {
          if (k == 0) {
#pragma unroll
            for (int z = 0; z < NS; ++z)
              scales[(j % C::SCALE_RING) * C::SCALE_FLOATS + z * 128 + me] =
                  sc_live ? __half2float(sc[z]) * (z < C::KT ? 1.f : kBoost) : 0.f;
          }
        }
        fence_proxy_async();
        mbar_arrive(full0 + 8 * st);
        if (k == 0) sc_live = fetch_scales(j + 1, sc);
      }
    }
  }
  // ================================ the third group: loaders and the matrix units' warp =================
  else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_THIRD));
    // ================================ loaders ==============================================================
    // V's tiles: warp 8; K's: warps 10 and 11.  16-bit tiles go to the ring that the products read, 8-bit ones
    // to the one that the widening warps read (which fetch pages of odd sizes themselves).
    if (!C::WIDEN || p.page % 16 == 0) {
      if (warp != 9) {
        const int nb = jend - j0;
        const int units = nb > 0 ? nb * (C::KT + 1) : 0;
        const bool whole = p.page % 16 == 0;                 // 16 tokens lie in one page
        const int bt = tp.box_tokens, boxes = kTcBlock / bt;
        int issued = -1;
        bool tail_used = false;
        for (int unit = 0; unit < units; ++unit) {
          int j, k;  // block; K tile number or -1: V
          tc_unit<C::KT>(unit, j0, j, k);
          // Who takes it: V warp 8; two K tiles of a block warps 10 and 11, one K tile these two in turn.  Nobody may
          // skip more units than the ring has slots: a slot's barrier tells a phase only from the one before, and
          // a warp knows that the use before last is over by its own last unit.
          if (warp != (k < 0 ? 8 : 10 + (C::KT == 2 ? k : C::WIDEN ? 0 : (j - j0) & 1))) continue;
          const int st = unit % C::RING;
          const uint32_t dst = C::WIDEN ? raw0 + st * C::RAW : ring0 + st * C::SLOT;
          const uint32_t is_full = (C::WIDEN ? raw_full : full0) + 8 * st, is_empty = (C::WIDEN ? raw_empty : empty0) + 8 * st;
          const int head0 = head * MAPS + (k < 0 ? slice * C::DV / D : k);
          const int live = kv_end - j * kTcBlock;  // keys of the block that exist
          // One lane for each box, or for each of four times 32 tokens: where their rows are.
          int64_t row[4] = {-1, -1, -1, -1};
          unsigned bad[4] = {0, 0, 0, 0};
          int phys = p.num_blocks, off = 0;  // the block behind the last is out of the map: zeros
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (whole && i) break;
            const int in = whole ? lane * bt : 32 * i + lane;
            bool astray = false;
            if (in < kTcBlock && in < live) {
              const int token = j * kTcBlock + in, page = token / p.page;
              const int id = __ldg(p.block_table + (int64_t)tile.request * p.bt_stride + page);
              if ((unsigned)id < (unsigned)p.num_blocks) {
                phys = id;
                off = token - page * p.page;
                row[i] = kv_row_offset(p, id, off, head0);
              } else {
                if (p.status) atomicOr(p.status, PD_DEV_BAD_BLOCK);
                astray = true;
              }
            }
            bad[i] = __ballot_sync(kFull, astray);
          }
          if (whole && bad[0]) {  // a bit a box -> a bit a token
            const unsigned pieces = bad[0];
            for (int i = 0; i < 4; ++i) {
              bad[i] = 0;
              for (int e = 0; e < 32; ++e) bad[i] |= ((pieces >> ((32 * i + e) / bt)) & 1u) << e;
            }
          }
          if (!tc_wait(is_empty, ((uint32_t)(unit / C::RING) & 1u) ^ 1u, p.status, abort_flag)) break;
          if (k == 0 && lane == 0)  // ahead of the block's scores
            *reinterpret_cast<uint4*>(meta + 4 * (j & (kTcMetaRing - 1))) = make_uint4(bad[0], bad[1], bad[2], bad[3]);
          if constexpr (C::WIDEN) {
            if (lane == 0) mbar_arrive_expect_tx(is_full, 128 * (k < 0 ? C::DV : D));
            else mbar_arrive(is_full);
            __syncwarp();
            issued = unit;
            if (lane < boxes) {  // whole rows of a head: planes of 128 rows of D bytes
              if (k >= 0) {
                tma_load_4d(dst + lane * bt * D, &tm_k, is_full, 0, off, head0, phys);
              } else {
#pragma unroll
                for (int z = 0; z < C::VH; ++z) tma_load_4d(dst + z * (128 * D) + lane * bt * D, &tm_v, is_full, 0, off, head0 + z, phys);
              }
            }
            __syncwarp();
          } else if (whole) {
            const bool tail = k < 0 && live < kTcBlock && live % bt != 0;  // V rows behind the last key in its box
            const uint32_t bar = tail ? tail_bar : is_full;
            if (lane == 0) mbar_arrive_expect_tx(bar, 128 * 2 * (k < 0 ? C::DV : D));
            if (lane > 0 && !tail) mbar_arrive(bar);
            __syncwarp();
            issued = unit;
            if (lane < boxes) {
              const uint32_t at = dst + lane * bt * 128;
              if (k >= 0) {
#pragma unroll
                for (int c = 0; c < C::KH; ++c) tma_load_4d(at + c * (128 * 128), &tm_k, bar, c * 64, off, head0, phys);
              } else {
#pragma unroll
                for (int c = 0; c < C::VC; ++c)
                  tma_load_4d(at + c * (128 * 128), &tm_v, bar, D == 64 ? 0 : c * 64, off, D == 64 ? head0 + c : head0, phys);
              }
            }
            __syncwarp();
            if (tail) {
              tail_used = true;
              if (!tc_wait(tail_bar, 0, p.status, abort_flag)) break;  // the one tail of this CTA
              const int to = (live / bt + 1) * bt;
              for (int i = lane; i < (to - live) * C::VC * 8; i += 32) {
                const int r = live + i / 8 % (to - live), c = i / 8 / (to - live);
                sts128(dst + tc_row(r, c) + (i & 7) * 16, make_uint4(0, 0, 0, 0));
              }
              fence_proxy_async();
              mbar_arrive(is_full);
            }
          } else {
            if (k < 0) tc_copy_rows<C::VC, D>(dst, (const __half*)p.v, row, p.kv_sh, lane);
            else tc_copy_rows<C::KH, D>(dst, (const __half*)p.k, row, p.kv_sh, lane);
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_proxy_async();
            mbar_arrive(is_full);
          }
        }
        if (*abort_flag && issued >= 0) {  // boxes still in flight get a bounded chance to land
          for (int u = issued; u >= 0 && u > issued - C::RING; --u)
            tc_drain((C::WIDEN ? raw_full : full0) + 8 * (u % C::RING), (uint32_t)(u / C::RING) & 1u);
          if (tail_used) tc_drain(tail_bar, 0);
        }
      }
    }
  // ================================ matrix units ======================================================
    if (warp == 9) {
      constexpr uint32_t id_s = tc_idesc(C::BF16, 128, false);
      constexpr uint32_t id_o = tc_idesc(C::BF16, C::DV / C::NP, true);
      uint32_t mine;
      asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(mine));
      bool ok = true;
      auto wait_bar = [&](uint32_t bar, uint32_t parity) {
        return tc_wait(bar, parity, p.status, abort_flag);
      };
      auto scores = [&](int t, int kslot) {  // S_t = Q_t K^T
        const uint64_t qd = tc_desc(q0 + t * C::QTILE, 1024, 0), kd = tc_desc(ring0 + kslot * C::SLOT, 1024, 0);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          tc_mma_ss(tmem + t * 128, qd + (((ks / 4) * (128 * 128) + (ks % 4) * 32) >> 4),
                    kd + (((ks / 4) * (128 * 128) + (ks % 4) * 32) >> 4), id_s, ks > 0, mine);
        tc_commit(s_full + 8 * t, mine);
      };
      auto values = [&](int t, int vslot, bool first, int half) {  // O_t (+)= P_t V, 64 keys
        const uint64_t vd = tc_desc(ring0 + vslot * C::SLOT, 1024, 128 * 128);
#pragma unroll
        for (int z = 0; z < C::NP; ++z) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int ks = 4 * half + k;
            const uint32_t pa = C::NP == 1 ? 8 * ks : 32 * (ks / 2) + 16 * z + 8 * (ks % 2);
            tc_mma_ts(tmem + 256 + t * 128 + z * 64, tmem + t * 128 + pa, vd + ((z * (128 * 128) + ks * 2048) >> 4), id_o,
                      !first || ks > 0, mine);
          }
        }
      };
      if (jend > j0) {
        ok = wait_bar(q_full, 0);
        // unit u lives in slot u % NSLOT; slot and phase of the next unit are counted along
        int slot = 0;
        uint32_t phase = 0;
        auto step = [&] {
          if (++slot == C::NSLOT) {
            slot = 0;
            phase ^= 1;
          }
        };
        // the first block's scores
        if (ok) ok = wait_bar(full0, 0);
        if (ok) {
          tc_fence_after();
          if (end[0] > j0) scores(0, 0);
          step();
          if constexpr (MAPS == 2) {
            ok = wait_bar(full0 + 8, 0);
            if (ok) {
              tc_fence_after();
              scores(1, 1);
              tc_commit(empty0, mine);
              tc_commit(empty0 + 8, mine);
            }
            step();
          } else {
            if (end[1] > j0) scores(1, 0);
            tc_commit(empty0, mine);
          }
        }
        for (int j = j0; j < jend && ok; ++j) {
          const uint32_t par = (uint32_t)(j - j0) & 1u;
          const bool more = j + 1 < jend;
          const int vslot = slot;
          const uint32_t vphase = phase;
          int kslot[C::KT];
          uint32_t kphase[C::KT];
          step();
          if (more) {
#pragma unroll
            for (int k = 0; k < C::KT; ++k) {
              kslot[k] = slot;
              kphase[k] = phase;
              step();
            }
          }
          ok = wait_bar(full0 + 8 * vslot, vphase);
          if (more && C::KT == 1 && ok) ok = wait_bar(full0 + 8 * kslot[0], kphase[0]);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (j >= end[t] || !ok) continue;
            ok = wait_bar(p_full + 16 * t, par);
            if (!ok) break;
            tc_fence_after();
            values(t, vslot, j == j0, 0);
            ok = wait_bar(p_full + 16 * t + 8, par);
            if (!ok) break;
            tc_fence_after();
            values(t, vslot, j == j0, 1);
            if (j + 1 < end[t]) {
              if constexpr (C::KT == 2) {
                ok = wait_bar(full0 + 8 * kslot[t], kphase[t]);
                if (!ok) break;
                tc_fence_after();
              }
              scores(t, kslot[C::KT == 2 ? t : 0]);
            } else {
              tc_commit(o_done + 8 * t, mine);
            }
          }
          if (!ok) break;
          // both tiles' products with these tiles are issued: their slots are free when they are done
          tc_commit(empty0 + 8 * vslot, mine);
          if (more) {
#pragma unroll
            for (int k = 0; k < C::KT; ++k) tc_commit(empty0 + 8 * kslot[k], mine);
          }
        }
        if (!ok) {  // products in flight get a bounded chance to end before tensor memory is freed
          tc_commit(drain_bar, mine);
          tc_drain(drain_bar, 0);
        }
      }
      __syncwarp();
    }
  }
  // ================================ softmax ============================================================
  else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_SOFTMAX));
    const int t = warp >> 2;            // tile
    const int me = tid & 127;           // row of the tile
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 lanes of tensor memory
    const uint32_t s_at = tmem + t * 128 + lanes, o_at = tmem + 256 + t * 128 + lanes;
    const int first_row = tile.row0 + (MAPS == 2 ? 0 : 128 * t);  // packed row of the tile's row 0
    const int n_rows = rows_of[t];

    // ---- Q into shared memory, 16 bytes at a time, in the 128-byte swizzle --------------------------
    // Not for a tile whose rows all see nothing beside one that has keys: no product reads it, so nothing would
    // stand between these copies, which land all over the tile, and the zero results that pass through it.
    if (end[t] > j0) {
      constexpr int CH = D / 8;         // 16-byte chunks of a row
      constexpr int RPI = 128 / CH;     // rows of one round of the tile's threads
      const int c = me % CH, rr = me / CH;
      int tok = (first_row + rr) / p.group, g = (first_row + rr) - tok * p.group;
#pragma unroll
      for (int i = 0; i < 128 / RPI; ++i) {
        const int r = i * RPI + rr;
        const int64_t at = (int64_t)(tile.first_token + tok) * p.q_sb + (int64_t)(head * p.group + g) * p.q_sh +
                           (MAPS == 2 ? t * a.q_sm : 0) + c * 8;
        cp_async16(q0 + t * C::QTILE + tc_row(r, c / 8) + (((c & 7) ^ (r & 7)) << 4),
                   r < n_rows ? (const __half*)p.q + at : (const __half*)p.q, r < n_rows);
        g += RPI;
        while (g >= p.group) {
          g -= p.group;
          ++tok;
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_proxy_async();
    }
    if (jend > j0) mbar_arrive(q_full);

    const int limit = me < n_rows ? tc_limit(tile, first_row + me, p.group) : 0;
    const int least = n_rows ? tc_limit(tile, first_row, p.group) : 0;  // the tile's row that sees the fewest
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = j0; j < end[t]; ++j) {
      ok = tc_wait(s_full + 8 * t, (uint32_t)(j - j0) & 1u, p.status, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const volatile unsigned* bad = meta + 4 * (j & (kTcMetaRing - 1));
      const bool masked = (j + 1) * kTcBlock > least || (bad[0] | bad[1] | bad[2] | bad[3]);
      const int room = limit - j * kTcBlock;  // columns below this one are seen
      const float* ks = SCALED ? scales + (j % C::SCALE_RING) * C::SCALE_FLOATS + (MAPS == 2 ? t * 128 : 0) : nullptr;
      const float* vs = SCALED ? scales + (j % C::SCALE_RING) * C::SCALE_FLOATS + C::KT * 128 : nullptr;
      // 32 scores at a time: K's scales and the mask
      auto shape_scores = [&](float* x, int c0) {
        if constexpr (SCALED) {
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 f = *reinterpret_cast<const float4*>(ks + c0 + c);
            tc_mul2(x[c], x[c + 1], f.x, f.y);
            tc_mul2(x[c + 2], x[c + 3], f.z, f.w);
          }
        }
        if (masked) {
          const unsigned astray = bad[c0 / 32];
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (c0 + c >= room || ((astray >> c) & 1)) x[c] = -INFINITY;
        }
      };
      // the row's scores, in registers from here on, and their maximum
      float x[128];
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c0 = 0; c0 < 128; c0 += 32) tc_ld32(s_at + c0, x + c0);
      tc_wait_ld();
#pragma unroll
      for (int c0 = 0; c0 < 128; c0 += 32) {
        float* y = x + c0;
        shape_scores(y, c0);
#pragma unroll
        for (int c = 0; c < 32; c += 2) mx[(c >> 1) & 3] = tc_max3(mx[(c >> 1) & 3], y[c], y[c + 1]);
      }
      const float top = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2);
      if (j == j0) {
        m = top;
      } else if (__any_sync(kFull, top > m + kLag)) {
        // O is that of the blocks before: this block's scores were issued behind their products
        const float alpha = top == -INFINITY ? 1.f : fast_exp2(m - top);
#pragma unroll 1
        for (int c0 = 0; c0 < C::DV; c0 += 32) {
          float o[32];
          tc_ld32(o_at + c0, o);
          tc_wait_ld();
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] *= alpha;
          tc_st32(o_at + c0, o);
        }
        l *= alpha;
        m = top;
      }
      const float from = m == -INFINITY ? 0.f : m;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c0 = 0; c0 < 128; c0 += 32) {
        float* y = x + c0;
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          tc_fma2(y[c], y[c + 1], p.scale_log2, -from);
          y[c] = fast_exp2(y[c]);
          y[c + 1] = fast_exp2(y[c + 1]);
          if constexpr (SCALED || MAPS == 1) tc_add2(sum[c & 2], sum[(c & 2) + 1], y[c], y[c + 1]);
        }
        uint32_t pk[16];
#pragma unroll
        for (int z = 0; z < C::NP; ++z) {
          if constexpr (SCALED) {
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              float4 f = *reinterpret_cast<const float4*>(vs + z * 128 + c0 + c);
              tc_mul2(f.x, f.y, y[c], y[c + 1]);
              tc_mul2(f.z, f.w, y[c + 2], y[c + 3]);
              pk[c / 2] = tc_pack<C::BF16>(f.x, f.y);
              pk[c / 2 + 1] = tc_pack<C::BF16>(f.z, f.w);
            }
          } else {
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              pk[c / 2] = tc_pack<C::BF16>(y[c], y[c + 1]);
              // For a pair l is the sum of what the product with V reads, the rounded probabilities: what their
              // roundings have in common then cancels in O / l (700 new tokens, values with a mean of one standard
              // deviation, fp16: 2.28e-4 -> 2.21e-4 of the result; values without a mean: no difference).
              if constexpr (MAPS == 2) add_pair<C::BF16>(sum[c & 2], sum[(c & 2) + 1], pk[c / 2]);
            }
          }
          // columns below 16 (or 32) * (c0 / 32 + 1) hold scores that have been read
          tc_st16(s_at + (C::NP == 1 ? c0 / 2 : c0 + 16 * z), pk);
        }
        if (c0 & 32) {  // half of the keys: the product with V may begin on them
          tc_wait_st();
          tc_fence_before();
          mbar_arrive(p_full + 16 * t + 8 * (c0 / 64));
        }
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }

    // ---- results ----------------------------------------------------------------------------------------
    // (maps = 2: both tiles' products, of which the second tile's are the last: the ring is written below)
    if (ok && end[t] > j0) ok = tc_wait(o_done + 8 * (MAPS == 2 ? 1 : t), 0, p.status, abort_flag);
    tc_fence_after();
    const bool any = end[t] > j0;  // else tensor memory holds nothing of this tile
    const float inv = l > 0.f || l != l ? 1.f / (l * kBoost) : 0.f;
    const bool live = me < n_rows;
    const int pr = first_row + (live ? me : 0);
    const int tok = pr / p.group, g = pr - tok * p.group;
    const int64_t row = tile.first_token + tok;
    const int hq = head * p.group + g;  // query head, or pair
    // this warp's part of its tile's Q, which has been read: the results pass through it
    const uint32_t area = q0 + t * C::QTILE + (warp & 3) * (C::QTILE / 4);
    if (tp.splits > 1) {
      const int64_t at = (((int64_t)split * a.rows + row) * (p.hq / MAPS) + hq) * MAPS + (MAPS == 2 ? t : 0);
#pragma unroll 1
      for (int c0 = 0; c0 < C::DV; c0 += 32) {
        float o[32];
        if (any) {
          tc_ld32(o_at + c0, o);
          tc_wait_ld();
        }
        if (live && ok && any && inv != 0.f) {  // a row without keys is told by its log-sum-exp
          float4* dst = reinterpret_cast<float4*>(tp.part_o + at * (MAPS * D) + slice * C::DV + c0);
#pragma unroll
          for (int c = 0; c < 32; c += 4) dst[c / 4] = make_float4(o[c] * inv, o[c + 1] * inv, o[c + 2] * inv, o[c + 3] * inv);
        }
      }
      if (live && ok && slice == 0) tp.part_lse[at] = l > 0.f || l != l ? m + log2f(l) : -INFINITY;
    } else if constexpr (MAPS == 1) {
#pragma unroll 1
      for (int c0 = 0; c0 < C::DV; c0 += 32) {
        float o[32];
        if (any) {
          tc_ld32(o_at + c0, o);
          tc_wait_ld();
        }
        const bool some = any && inv != 0.f;
#pragma unroll
        for (int c = 0; c < 32; c += 8) {
          uint4 y = make_uint4(0, 0, 0, 0);
          if (some) {
            y.x = tc_pack<C::BF16>(o[c] * inv, o[c + 1] * inv);
            y.y = tc_pack<C::BF16>(o[c + 2] * inv, o[c + 3] * inv);
            y.z = tc_pack<C::BF16>(o[c + 4] * inv, o[c + 5] * inv);
            y.w = tc_pack<C::BF16>(o[c + 6] * inv, o[c + 7] * inv);
          }
          tc_put_chunk<D / 8>(area, lane, (c0 + c) / 8, y);
        }
      }
      tc_store_rows<D / 8>(area, lane, (__half*)p.out, live && ok ? row * p.o_sb + (int64_t)hq * p.o_sh : -1);
    } else {
      // A row's two maps are in two threads.  Through the ring (every tile in it has been read) the first map's
      // thread gets the second's columns 0..63 and gives its own 64..127, a column of 128 rows at a time:
      // neighbouring lanes, neighbouring words.  Each then has 64 columns of the difference in registers.
      float* pass = reinterpret_cast<float*>(smem) + t * (64 * 128);        // what this thread gives
      const float* take = reinterpret_cast<const float*>(smem) + (t ^ 1) * (64 * 128);
      static_assert(C::NSLOT * C::SLOT >= 128 * 128 * 4, "room for one tile of f32");
      const float mult = inv != 0.f && any ? (t == 0 ? inv : inv * a.lambda(row, hq)) : 0.f;
      float x[64];
#pragma unroll
      for (int c0 = 0; c0 < 128; c0 += 32) {
        float o[32];
        if (any) {
          tc_ld32(o_at + c0, o);
          tc_wait_ld();
        }
        const bool mine = (c0 < 64) == (t == 0);
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const float y = mult != 0.f ? o[c] * mult : 0.f;
          if (!mine) pass[((c0 & 32) + c) * 128 + me] = y;
          else x[(c0 & 32) + c] = y;
        }
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      float square = 0.f;
#pragma unroll
      for (int c = 0; c < 64; ++c) {
        const float y = take[c * 128 + me];
        x[c] = t == 0 ? x[c] - y : y - x[c];
        square = fmaf(x[c], x[c], square);
      }
      squares[t * 128 + me] = square;
      if constexpr (C::SLICES == 2) {  // the other half of V's columns is in the other CTA of the cluster
        uint32_t peer;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(smem_u32(squares + 256 + t * 128 + me)), "r"(slice ^ 1));
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(peer), "f"(square) : "memory");
        tc_cluster_sync();
      } else {
        asm volatile("bar.sync 1, 256;" ::: "memory");
      }
      {
        float total = squares[me] + squares[128 + me];
        if constexpr (C::SLICES == 2) total += squares[256 + me] + squares[384 + me];
        float factor = a.out_scale;
        if (a.norm) factor *= rsqrtf(total * (1.f / (MAPS * D)) + a.eps);
        const int col = slice * C::DV + t * 64;
        const float* wt = weights + t * 64;
#pragma unroll
        for (int c = 0; c < 64; c += 8) {
          const float4 w0 = *reinterpret_cast<const float4*>(wt + c), w1 = *reinterpret_cast<const float4*>(wt + c + 4);
          tc_put_chunk<8>(area, lane, c / 8,
                          make_uint4(tc_pack<C::BF16>(x[c] * factor * w0.x, x[c + 1] * factor * w0.y),
                                     tc_pack<C::BF16>(x[c + 2] * factor * w0.z, x[c + 3] * factor * w0.w),
                                     tc_pack<C::BF16>(x[c + 4] * factor * w1.x, x[c + 5] * factor * w1.y),
                                     tc_pack<C::BF16>(x[c + 6] * factor * w1.z, x[c + 7] * factor * w1.w)));
        }
        tc_store_rows<8>(area, lane, (__half*)p.out, live && ok ? row * p.o_sb + (int64_t)hq * p.o_sh + col : -1);
      }
    }
  }
  // the warps that are not part of the exchange of sums arrive for it here
  if (C::SLICES == 2 && tp.splits == 1 && warp >= 8) tc_cluster_sync();
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

}  // namespace pd
