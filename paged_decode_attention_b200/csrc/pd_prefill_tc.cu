// Placeholder until the kernel on the matrix units exists.
#include "pd_prefill.h"

namespace pd {
int tc_supports(const PdPrefillArgs*) { return PD_ERR_UNSUPPORTED; }
uint64_t tc_workspace_bytes(const PdPrefillArgs*, int) { return 0; }
int tc_run(const PdPrefillArgs*, const PrefillParams&, int) { return PD_ERR_UNSUPPORTED; }
}  // namespace pd
