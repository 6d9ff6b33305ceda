// Host interface between the entry points of pd_prefill / pd_diff_decode (pd_prefill.cu) and the
// kernel on the matrix units (pd_prefill_tc.cu).
#pragma once

#include "pd_common.cuh"

namespace pd {

// Device view of PdPrefillArgs.
struct PrefillParams {
  Params p;                 // q_sb and o_sb are the strides between rows
  const int32_t* starts;    // query_start, or NULL: row b is the one query of request b
  int32_t rows, maps;
  int64_t q_sm;
  const float* lam;
  int64_t lam_st, lam_sh;
  const float* weight;
  float lam_value, eps, out_scale;
  int32_t norm;
  __device__ __forceinline__ float lambda(int64_t row, int head) const {
    return lam ? __ldg(lam + row * lam_st + head * lam_sh) : lam_value;
  }
};

// The request that owns row t, or -1: the last b with starts[b] <= t (requests without rows share
// their start with the next one), if t lies before the end of all rows.
__device__ __forceinline__ int request_of_row(const PrefillParams& a, int t) {
  if (!a.starts) return t < a.p.batch ? t : -1;
  if (t < __ldg(a.starts) || t >= __ldg(a.starts + a.p.batch)) return -1;
  int lo = 0, hi = a.p.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(a.starts + mid) <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Keys that row t of request b attends to: all up to its own position, counted from the request's end.
__device__ __forceinline__ int keys_of_row(const PrefillParams& a, int b, int t, int len) {
  if (!a.starts) return len;
  const long long n = (long long)len - (__ldg(a.starts + b + 1) - 1 - t);
  return n < 0 ? 0 : n > len ? len : (int)n;
}

int tc_supports(const PdPrefillArgs* a);
uint64_t tc_workspace_bytes(const PdPrefillArgs* a, int sm_count);
int tc_run(const PdPrefillArgs* a, const PrefillParams& p, int sm_count);

}  // namespace pd
