// Prefill kernel instantiations (matrix units) for int8 pages.
#include "pd_prefill_tc_launch.cuh"

namespace pd {

PD_TC_LAUNCHER(tc_launch_i8) { return tc_launch<PD_KV_I8, true>(head_dim, maps, tp, mk, mv, grid, st); }

}  // namespace pd
