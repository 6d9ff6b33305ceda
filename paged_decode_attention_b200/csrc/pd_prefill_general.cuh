// General kernel of pd_prefill and pd_diff_decode: one CTA per (row, query head or pair).
//
// CUDA cores only; any strides, every head_dim of {32, 64, 128, 256}, every page type, one or two
// maps.  Its four warps take the row's keys in turn, a lane owns head_dim / 32 elements of a key
// and of each value row; every warp runs a base-2 online softmax per map, and the four states are
// merged through shared memory.  It serves what the kernels on the matrix units do not and is the
// partner they are checked against; a key is read once for every query row and head, so it is no
// kernel for long prompts.  Everything is held in 32 bits up to the store.
#pragma once

#include "pd_prefill.h"

namespace pd {

constexpr int kGeneralWarps = 4;

// Stored elements as they are (pages of bf16 do not pass through fp16 here).
template <int KV, int N>
__device__ __forceinline__ void load_exact(const void* base, int64_t off, float (&dst)[N]) {
  if constexpr (KV == PD_KV_BF16) {
    const __nv_bfloat16* src = (const __nv_bfloat16*)base + off;
#pragma unroll
    for (int i = 0; i < N; ++i) dst[i] = __bfloat162float(src[i]);
  } else {
    load_elems<KV, N>(base, off, dst);
  }
}

template <int KV, int D, int MAPS, bool SCALED>
__global__ void __launch_bounds__(kGeneralWarps * 32) general_prefill_kernel(const PrefillParams a, const int io_bf16) {
  constexpr int EPL = D / 32, DV = MAPS * D;
  constexpr unsigned kFull = 0xffffffffu;
  const Params& p = a.p;
  const int t = blockIdx.x, head = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = request_of_row(a, t);
  if (b < 0) return;  // nobody's row: left as it was
  const int keys = keys_of_row(a, b, t, clamp_len(p, b));
  const int kvh = head / p.group * MAPS;  // first kv head of the head or pair

  float q[MAPS][EPL], m[MAPS], l[MAPS], acc[MAPS][MAPS * EPL];
#pragma unroll
  for (int i = 0; i < MAPS; ++i) {
    const int64_t at = (int64_t)t * p.q_sb + (int64_t)head * p.q_sh + i * a.q_sm + lane * EPL;
#pragma unroll
    for (int e = 0; e < EPL; ++e)
      q[i][e] = io_bf16 ? __bfloat162float(((const __nv_bfloat16*)p.q)[at + e]) : __half2float(((const __half*)p.q)[at + e]);
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int e = 0; e < MAPS * EPL; ++e) acc[i][e] = 0.f;
  }

  for (int k = warp; k < keys; k += kGeneralWarps) {
    const int blk = lookup_block(p, b, k / p.page);
    if (blk < 0) continue;
    const int slot = k % p.page;
    float v[MAPS * EPL];
    float s[MAPS];
#pragma unroll
    for (int i = 0; i < MAPS; ++i) {
      const int64_t row = kv_row_offset(p, blk, slot, kvh + i) + lane * EPL;
      float kf[EPL], vf[EPL];
      load_exact<KV, EPL>(p.k, row, kf);
      load_exact<KV, EPL>(p.v, row, vf);
      float ks = 1.f, vs = 1.f;
      if constexpr (SCALED) {
        const int64_t so = scale_offset(p, blk, slot, kvh + i);
        ks = __half2float(__ldg(p.k_scale + so));
        vs = __half2float(__ldg(p.v_scale + so));
      }
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        dot = fmaf(q[i][e], kf[e], dot);
        v[i * EPL + e] = vf[e] * vs;
      }
      s[i] = dot * ks;
    }
#pragma unroll
    for (int i = 0; i < MAPS; ++i) {
      float x = s[i];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(kFull, x, o);
      x *= p.scale_log2;
      const float top = fmaxf(m[i], x);
      const float from = top == -INFINITY ? 0.f : top;  // a score of -inf has weight zero, not NaN
      const float alpha = fast_exp2(m[i] - from), w = fast_exp2(x - from);
      l[i] = l[i] * alpha + w;
#pragma unroll
      for (int e = 0; e < MAPS * EPL; ++e) acc[i][e] = fmaf(acc[i][e], alpha, w * v[e]);
      m[i] = top;
    }
  }

  __shared__ float sm_m[kGeneralWarps][MAPS], sm_l[kGeneralWarps][MAPS], sm_acc[kGeneralWarps][MAPS][DV];
  __shared__ float sm_sq[kGeneralWarps];
#pragma unroll
  for (int i = 0; i < MAPS; ++i) {
    if (lane == 0) {
      sm_m[warp][i] = m[i];
      sm_l[warp][i] = l[i];
    }
#pragma unroll
    for (int j = 0; j < MAPS; ++j)
#pragma unroll
      for (int e = 0; e < EPL; ++e) sm_acc[warp][i][j * D + lane * EPL + e] = acc[i][j * EPL + e];
  }
  __syncthreads();

  constexpr int PER = (DV + kGeneralWarps * 32 - 1) / (kGeneralWarps * 32);
  float out[PER];
  float square = 0.f;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int d = threadIdx.x + j * kGeneralWarps * 32;
    out[j] = 0.f;
    if (d >= DV) continue;
#pragma unroll
    for (int i = 0; i < MAPS; ++i) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kGeneralWarps; ++w) top = fmaxf(top, sm_m[w][i]);
      const float from = top == -INFINITY ? 0.f : top;
      float total = 0.f, o = 0.f;
#pragma unroll
      for (int w = 0; w < kGeneralWarps; ++w) {
        const float f = fast_exp2(sm_m[w][i] - from);
        total += sm_l[w][i] * f;
        o += sm_acc[w][i][d] * f;
      }
      o = total > 0.f || total != total ? o / total : 0.f;
      out[j] = i == 0 ? o : out[j] - a.lambda(t, head) * o;
    }
    square = fmaf(out[j], out[j], square);
  }
  float factor = 1.f;
  if constexpr (MAPS == 2) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) square += __shfl_xor_sync(kFull, square, o);
    if (lane == 0) sm_sq[warp] = square;
    __syncthreads();
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < kGeneralWarps; ++w) total += sm_sq[w];
    factor = a.out_scale;
    if (a.norm) factor *= rsqrtf(total * (1.f / DV) + a.eps);
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int d = threadIdx.x + j * kGeneralWarps * 32;
    if (d >= DV) continue;
    float x = out[j] * factor;
    if (MAPS == 2 && a.weight) x *= __ldg(a.weight + d);
    const int64_t at = (int64_t)t * p.o_sb + (int64_t)head * p.o_sh + d;
    if (io_bf16) ((__nv_bfloat16*)p.out)[at] = __float2bfloat16_rn(x);
    else ((__half*)p.out)[at] = __float2half_rn(x);
  }
}

}  // namespace pd
