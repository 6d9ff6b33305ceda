// Dispatch of the prefill kernel on the matrix units from head_dim and maps to its instantiation.
#pragma once

#include "pd_prefill_tc.cuh"
#include "pd_prefill_tc.h"

namespace pd {

template <int KV, int D, int MAPS, bool SCALED>
static inline cudaError_t tc_launch_one(const TcParams& tp, const CUtensorMap& mk, const CUtensorMap& mv,
                                    unsigned grid, cudaStream_t st) {
  using C = TcCfg<KV, D, MAPS, SCALED>;
  auto* kern = tc_prefill_kernel<KV, D, MAPS, SCALED>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C::SLICES;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C::SLICES > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, tp, mk, mv);
}

template <int KV, bool SCALED>
static inline cudaError_t tc_launch(int head_dim, int maps, const TcParams& tp, const CUtensorMap& mk, const CUtensorMap& mv,
                                    unsigned grid, cudaStream_t st) {
  if (head_dim == 64)
    return maps == 2 ? tc_launch_one<KV, 64, 2, SCALED>(tp, mk, mv, grid, st) : tc_launch_one<KV, 64, 1, SCALED>(tp, mk, mv, grid, st);
  if (head_dim == 128)
    return maps == 2 ? tc_launch_one<KV, 128, 2, SCALED>(tp, mk, mv, grid, st) : tc_launch_one<KV, 128, 1, SCALED>(tp, mk, mv, grid, st);
  return cudaErrorInvalidValue;
}

}  // namespace pd
