// Host side of the prefill kernel on the matrix units: one translation unit per page element type holds
// its instantiations.
#pragma once

#include <cuda.h>

#include "pd_prefill.h"

namespace pd {

struct TcParams;

// What the host needs to know of an instantiation: packed rows and slices of V per tile.
struct TcShape {
  int rows, slices, dv;
};
__host__ inline TcShape tc_shape(int head_dim, int maps) {
  TcShape s;
  s.rows = maps == 2 ? 128 : 256;
  s.dv = maps == 2 ? 128 : head_dim;
  s.slices = maps * head_dim / s.dv;
  return s;
}

#define PD_TC_LAUNCHER(name) \
  cudaError_t name(int head_dim, int maps, const TcParams& tp, const CUtensorMap& mk, const CUtensorMap& mv, unsigned grid, cudaStream_t st)
PD_TC_LAUNCHER(tc_launch_f16);
PD_TC_LAUNCHER(tc_launch_bf16);
PD_TC_LAUNCHER(tc_launch_e5m2);
PD_TC_LAUNCHER(tc_launch_e5m2_scaled);
PD_TC_LAUNCHER(tc_launch_i8);

}  // namespace pd
