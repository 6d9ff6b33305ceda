// Host side of the prefill kernel on the matrix units (pd_prefill_tc.cuh): which requests it serves, how
// they are split, launches, and the kernel that joins the splits.
#include <cstring>

#include "pd_prefill_tc.cuh"
#include "pd_prefill_tc.h"
#include "pd_stream.h"

namespace pd {

// ---------------------------------------------------------------------------------------------
// joining the splits
// ---------------------------------------------------------------------------------------------
// One warp per (row, head or pair).  The partials are normalised rows with base-2 log-sum-exps, so
// o = sum 2^(lse_s - M) o_s / sum 2^(lse_s - M); for maps = 2 then the difference and the norm.  A lane
// owns four neighbouring columns of every 128 (or two of 64).  Bound by its reads, splits * rows *
// heads * width * 4 bytes, which a call that splits keeps small (few rows).
template <int W, int MAPS>
__global__ void __launch_bounds__(128) tc_join_kernel(const TcParams tp, const int io_bf16) {
  constexpr int PER = W / 32;  // columns of a lane: 2, 4 or 8, in runs of up to 4
  constexpr int RUN = PER < 4 ? PER : 4;
  constexpr unsigned kFull = 0xffffffffu;
  const PrefillParams& a = tp.a;
  const Params& p = a.p;
  const int heads = p.hq / MAPS;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (item >= (int64_t)a.rows * heads) return;
  const int row = (int)(item / heads), hq = (int)(item % heads);
  if (request_of_row(a, row) < 0) return;
  float x[MAPS][PER];
#pragma unroll
  for (int i = 0; i < MAPS; ++i) {
    const int64_t first = ((int64_t)row * heads + hq) * MAPS + i, step = (int64_t)a.rows * heads * MAPS;
    // lane l has the weights of splits l and l + 32
    float w[2];
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int s = lane + 32 * k;
      w[k] = s < tp.splits ? __ldg(tp.part_lse + first + s * step) : -INFINITY;
      top = fmaxf(top, w[k]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
    const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int k = 0; k < 2; ++k) w[k] = exp2f(w[k] - from);
    float total = w[0] + w[1];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(kFull, total, o);
#pragma unroll
    for (int e = 0; e < PER; ++e) x[i][e] = 0.f;
    // four splits' rows in flight at a time (one after the other 18 splits took 12 us, most of it waiting)
    for (int s0 = 0; s0 < tp.splits; s0 += 4) {
      float y[4][PER], u[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int s = s0 + k;
        u[k] = __shfl_sync(kFull, s & 32 ? w[1] : w[0], s & 31);  // beyond the last split: lane 63's and so on, zero
        const float* src = tp.part_o + (first + s * step) * W;
#pragma unroll
        for (int e = 0; e < PER; e += RUN) {
          const float* at = src + (e / RUN) * 32 * RUN + lane * RUN;
#pragma unroll
          for (int q = 0; q < RUN; ++q) y[k][e + q] = 0.f;
          if (u[k] != 0.f) {  // an empty split wrote no row
            if constexpr (RUN == 4) {
              const float4 z = __ldg(reinterpret_cast<const float4*>(at));
              y[k][e] = z.x;
              y[k][e + 1] = z.y;
              y[k][e + 2] = z.z;
              y[k][e + 3] = z.w;
            } else {
              const float2 z = __ldg(reinterpret_cast<const float2*>(at));
              y[k][e] = z.x;
              y[k][e + 1] = z.y;
            }
          }
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < PER; ++e) x[i][e] = fmaf(u[k], y[k][e], x[i][e]);
    }
    const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) x[i][e] *= inv;
  }
  float factor = 1.f;
  if constexpr (MAPS == 2) {
    const float lam = a.lambda(row, hq);
    float square = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      x[0][e] -= lam * x[1][e];
      square = fmaf(x[0][e], x[0][e], square);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) square += __shfl_xor_sync(kFull, square, o);
    factor = a.out_scale;
    if (a.norm) factor *= rsqrtf(square * (1.f / W) + a.eps);
  }
  __half* dst = (__half*)p.out + (int64_t)row * p.o_sb + (int64_t)hq * p.o_sh;
#pragma unroll
  for (int e = 0; e < PER; e += 2) {
    const int col = (e / RUN) * 32 * RUN + lane * RUN + e % RUN;
    float y0 = x[0][e] * factor, y1 = x[0][e + 1] * factor;
    if (MAPS == 2 && a.weight) {
      y0 *= __ldg(a.weight + col);
      y1 *= __ldg(a.weight + col + 1);
    }
    *reinterpret_cast<uint32_t*>(dst + col) = io_bf16 ? tc_pack<true>(y0, y1) : tc_pack<false>(y0, y1);
  }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
constexpr int kTcMaxSplits = 64;
constexpr int kTcLong = 16;

struct TcPlan {
  int tiles, heads, splits, target;
  int64_t grid;
  uint64_t lse_off, bytes;
};

static TcPlan tc_plan(const PdPrefillArgs* a, int sm_count) {
  TcPlan t;
  const TcShape s = tc_shape(a->head_dim, a->maps);
  const int group = a->num_q_heads / a->num_kv_heads;
  t.tiles = (int)((int64_t)a->num_rows * group / s.rows + a->batch);
  t.heads = a->num_kv_heads / a->maps;
  // Split the keys where the tiles alone would leave SMs idle; the kernel cuts them into pieces of equal length.
  // Up to half a wave of tiles: pieces for one wave, of kTcLeast blocks and more, with room for twice as many
  // pieces of a context as of the mean one.  Up to two waves: pieces for three waves, of at least kTcLong blocks,
  // because contexts of a batch differ and the last tile to end is a long one; shorter pieces cost more in
  // starts and in the join than they even out (2048 tokens of 32/8 heads, 264 tiles: 47 us whole, 92 in two
  // pieces).  Beyond, the order of the tiles evens it out.
  // The lengths themselves are on the device.  What is known here is the room in the block table, or the
  // caller's max_seq_len where that is less: with a table wider than the contexts and no max_seq_len, contexts
  // too short for it are cut as well, into pieces of kTcLeast blocks and more, and all rows go through the join
  // (tables of 32768 tokens: 512 tokens of 32/8 heads 17 -> 29 us, the 2048 above 47 -> 92; with max_seq_len as exact).
  int64_t bound = (int64_t)a->max_blocks_per_seq * a->block_size;
  if (a->max_seq_len > 0 && a->max_seq_len < bound) bound = a->max_seq_len;
  const int64_t ctas = (int64_t)t.tiles * t.heads * s.slices;
  int64_t n = 1;
  if (ctas * 2 <= sm_count) {
    n = 2 * sm_count / (ctas > 0 ? ctas : 1);
    if (n > bound / kTcBlock / kTcLeast) n = bound / kTcBlock / kTcLeast;
  } else if (ctas < 2 * sm_count) {
    n = (3 * sm_count + ctas - 1) / ctas;
    if (n > bound / kTcBlock / kTcLong) n = bound / kTcBlock / kTcLong;
  }
  if (n > kTcMaxSplits) n = kTcMaxSplits;
  t.splits = n < 1 ? 1 : (int)n;
  t.target = ctas * 2 <= sm_count ? sm_count - (int)ctas : 3 * sm_count;  // one wave: every tile may end with a short piece
  t.grid = ctas * t.splits;
  t.lse_off = t.bytes = 0;
  if (t.splits > 1) {
    const uint64_t rows = (uint64_t)t.splits * a->num_rows * a->num_q_heads;  // maps counted
    t.lse_off = (rows * a->head_dim * a->maps * 4 + 255) / 256 * 256;
    t.bytes = t.lse_off + (rows * 4 + 255) / 256 * 256;
  }
  return t;
}

int tc_supports(const PdPrefillArgs* a) {
  if (!a->query_start) return PD_ERR_UNSUPPORTED;
  if (a->head_dim != 64 && a->head_dim != 128) return PD_ERR_UNSUPPORTED;
  if ((a->kv_dtype == PD_KV_BF16) != (a->io_dtype == PD_IO_BF16)) return PD_ERR_UNSUPPORTED;
  if (!(a->sm_scale > 0.f) || a->sm_scale > 1e30f) return PD_ERR_UNSUPPORTED;  // the maximum is taken ahead of the factor
  const int group = a->num_q_heads / a->num_kv_heads;
  if (group > 128) return PD_ERR_UNSUPPORTED;
  if ((uintptr_t)a->q % 16 || a->q_stride_t % 8 || a->q_stride_h % 8 || a->q_stride_m % 8) return PD_ERR_UNSUPPORTED;
  if ((uintptr_t)a->out % 16 || a->out_stride_t % 8 || a->out_stride_h % 8) return PD_ERR_UNSUPPORTED;
  const int64_t eb = a->kv_dtype <= PD_KV_BF16 ? 2 : 1;
  const int64_t strides[3] = {a->kv_stride_block, a->kv_stride_token, a->kv_stride_head};
  for (int64_t s : strides)
    if (s < 0 || s * eb >= (1ll << 40)) return PD_ERR_UNSUPPORTED;  // limits of the tensor maps
  if ((int64_t)a->num_rows * group / 128 + a->batch > (1 << 30)) return PD_ERR_UNSUPPORTED;
  const TcShape s = tc_shape(a->head_dim, a->maps);
  const int64_t grid = ((int64_t)a->num_rows * group / s.rows + a->batch) * (a->num_kv_heads / a->maps) * s.slices;
  return grid < (1ll << 31) ? PD_OK : PD_ERR_UNSUPPORTED;
}

uint64_t tc_workspace_bytes(const PdPrefillArgs* a, int sm_count) { return tc_plan(a, sm_count).bytes; }

int tc_run(const PdPrefillArgs* a, const PrefillParams& r, int sm_count) {
  const TcPlan t = tc_plan(a, sm_count);
  if (t.bytes && (!a->workspace || a->workspace_bytes < t.bytes)) return PD_ERR_WORKSPACE;
  TcParams tp;
  tp.a = r;
  tp.tiles = t.tiles;
  tp.heads = t.heads;
  tp.splits = t.splits;
  tp.target = t.target;
  tp.part_o = t.bytes ? (float*)a->workspace : nullptr;
  tp.part_lse = t.bytes ? (float*)((char*)a->workspace + t.lse_off) : nullptr;
  CUtensorMap mk, mv;
  memset(&mk, 0, sizeof(mk));
  memset(&mv, 0, sizeof(mv));
  tp.box_tokens = 16;  // the largest power of two up to a block that divides the page
  while (tp.box_tokens < kTcBlock && a->block_size % (2 * tp.box_tokens) == 0) tp.box_tokens *= 2;
  if (a->block_size % 16 == 0) {  // encoded for every call: nothing is kept by an address
    if (!encode_page_box(a, a->k_cache, tp.box_tokens, &mk) || !encode_page_box(a, a->v_cache, tp.box_tokens, &mv))
      return PD_ERR_CUDA;
  }
  const cudaStream_t st = (cudaStream_t)a->stream;
  auto* launch = a->kv_dtype == PD_KV_F16    ? tc_launch_f16
                 : a->kv_dtype == PD_KV_BF16 ? tc_launch_bf16
                 : a->kv_dtype == PD_KV_I8   ? tc_launch_i8
                 : a->k_scale                ? tc_launch_e5m2_scaled
                                             : tc_launch_e5m2;
  if (launch(a->head_dim, a->maps, tp, mk, mv, (unsigned)t.grid, st) != cudaSuccess) return PD_ERR_CUDA;
  if (t.splits > 1) {
    const int64_t items = (int64_t)a->num_rows * (a->num_q_heads / a->maps);
    const unsigned grid = (unsigned)((items + 3) / 4);
    const int bf = a->io_dtype == PD_IO_BF16;
    const int width = a->maps * a->head_dim;
    if (a->maps == 1) {
      if (width == 64) tc_join_kernel<64, 1><<<grid, 128, 0, st>>>(tp, bf);
      else tc_join_kernel<128, 1><<<grid, 128, 0, st>>>(tp, bf);
    } else {
      if (width == 128) tc_join_kernel<128, 2><<<grid, 128, 0, st>>>(tp, bf);
      else tc_join_kernel<256, 2><<<grid, 128, 0, st>>>(tp, bf);
    }
    if (cudaGetLastError() != cudaSuccess) return PD_ERR_CUDA;
  }
  return PD_OK;
}

}  // namespace pd
