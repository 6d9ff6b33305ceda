// Prefill kernel instantiations (matrix units) for bf16 pages.
#include "pd_prefill_tc_launch.cuh"

namespace pd {

PD_TC_LAUNCHER(tc_launch_bf16) { return tc_launch<PD_KV_BF16, false>(head_dim, maps, tp, mk, mv, grid, st); }

}  // namespace pd
