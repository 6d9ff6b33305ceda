// Prefill kernel instantiations (matrix units) for fp8_e5m2 pages with scales.
#include "pd_prefill_tc_launch.cuh"

namespace pd {

PD_TC_LAUNCHER(tc_launch_e5m2_scaled) { return tc_launch<PD_KV_E5M2, true>(head_dim, maps, tp, mk, mv, grid, st); }

}  // namespace pd
