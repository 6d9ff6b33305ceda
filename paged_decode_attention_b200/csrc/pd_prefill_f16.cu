// Prefill kernel instantiations (matrix units) for fp16 pages.
#include "pd_prefill_tc_launch.cuh"

namespace pd {

PD_TC_LAUNCHER(tc_launch_f16) { return tc_launch<PD_KV_F16, false>(head_dim, maps, tp, mk, mv, grid, st); }

}  // namespace pd
