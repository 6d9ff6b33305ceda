// Entry points of attention beyond plain decode (include/paged_decode.h: PdPrefillArgs): argument
// checks, kernel choice, and the general kernel's launches.
#include <cstring>

#include "pd_prefill_general.cuh"
#include "pd_stream.h"

namespace pd {

static bool aligned_to(const void* p, uintptr_t n) { return ((uintptr_t)p % n) == 0; }

// Checks everything that can be checked without touching the device.
static int validate_prefill(const PdPrefillArgs* a) {
  if (!a || !a->k_cache || !a->v_cache) return PD_ERR_INVALID_ARG;
  if (a->num_rows > 0 && (!a->q || !a->out)) return PD_ERR_INVALID_ARG;  // an empty tensor has no address
  if (a->batch > 0 && (!a->block_table || !a->seq_lens)) return PD_ERR_INVALID_ARG;
  if (a->num_rows < 0 || a->batch < 0 || a->num_q_heads <= 0 || a->num_kv_heads <= 0 || a->head_dim <= 0)
    return PD_ERR_INVALID_ARG;
  if (a->num_q_heads % a->num_kv_heads) return PD_ERR_INVALID_ARG;
  if (a->maps != 1 && a->maps != 2) return PD_ERR_INVALID_ARG;
  if (a->maps == 2 && a->num_kv_heads % 2) return PD_ERR_INVALID_ARG;  // heads come in pairs
  if (a->block_size <= 0 || a->num_blocks <= 0 || a->max_blocks_per_seq <= 0) return PD_ERR_INVALID_ARG;
  if (a->kv_dtype < PD_KV_F16 || a->kv_dtype > PD_KV_I8) return PD_ERR_INVALID_ARG;
  if (a->io_dtype != PD_IO_F16 && a->io_dtype != PD_IO_BF16) return PD_ERR_INVALID_ARG;
  if (a->kernel < PD_KERNEL_AUTO || a->kernel > PD_KERNEL_STREAM) return PD_ERR_INVALID_ARG;
  if (a->max_seq_len < 0 || a->sm_count < 0) return PD_ERR_INVALID_ARG;
  if (a->maps == 2 && a->norm && !(a->eps > 0.f)) return PD_ERR_INVALID_ARG;  // a row without keys is all zeros
  if ((a->k_scale == nullptr) != (a->v_scale == nullptr)) return PD_ERR_INVALID_ARG;
  if (a->kv_dtype == PD_KV_I8 && !a->k_scale) return PD_ERR_INVALID_ARG;
  if (a->kv_dtype <= PD_KV_BF16 && a->k_scale) return PD_ERR_INVALID_ARG;
  if (a->block_table_stride < a->max_blocks_per_seq) return PD_ERR_INVALID_ARG;
  if (!a->query_start && a->num_rows != a->batch) return PD_ERR_INVALID_ARG;
  if (a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) return PD_ERR_UNSUPPORTED;
  const int eb = a->kv_dtype <= PD_KV_BF16 ? 2 : 1;
  if ((a->kv_stride_block * eb) % 16 || (a->kv_stride_token * eb) % 16 || (a->kv_stride_head * eb) % 16)
    return PD_ERR_UNSUPPORTED;
  if (!aligned_to(a->k_cache, 16) || !aligned_to(a->v_cache, 16)) return PD_ERR_UNSUPPORTED;
  if (!aligned_to(a->q, 2) || !aligned_to(a->out, 2)) return PD_ERR_INVALID_ARG;
  if (a->workspace && !aligned_to(a->workspace, 256)) return PD_ERR_WORKSPACE;
  if (a->num_q_heads / a->maps > 65535) return PD_ERR_UNSUPPORTED;  // a grid dimension
  return PD_OK;
}

static int choose(const PdPrefillArgs* a) {
  if (a->kernel == PD_KERNEL_SIMPLE) return PD_KERNEL_SIMPLE;
  const int why = a->query_start ? tc_supports(a) : diff_stream_supports(a);
  if (why == PD_OK) return PD_KERNEL_STREAM;
  return a->kernel == PD_KERNEL_STREAM ? why : PD_KERNEL_SIMPLE;
}

static void fill(const PdPrefillArgs* a, PrefillParams& r) {
  Params& p = r.p;
  memset(&r, 0, sizeof(r));
  p.q = a->q;
  p.out = a->out;
  p.q_sb = a->q_stride_t;
  p.q_sh = a->q_stride_h;
  p.o_sb = a->out_stride_t;
  p.o_sh = a->out_stride_h;
  p.k = a->k_cache;
  p.v = a->v_cache;
  p.kv_sb = a->kv_stride_block;
  p.kv_st = a->kv_stride_token;
  p.kv_sh = a->kv_stride_head;
  p.k_scale = (const __half*)a->k_scale;
  p.v_scale = (const __half*)a->v_scale;
  p.sc_sb = a->scale_stride_block;
  p.sc_st = a->scale_stride_token;
  p.block_table = a->block_table;
  p.bt_stride = a->block_table_stride;
  p.seq_lens = a->seq_lens;
  p.batch = a->batch;
  p.hq = a->num_q_heads;
  p.hkv = a->num_kv_heads;
  p.d = a->head_dim;
  p.page = a->block_size;
  p.num_blocks = a->num_blocks;
  p.max_blocks = a->max_blocks_per_seq;
  p.group = a->num_q_heads / a->num_kv_heads;
  p.scale_log2 = a->sm_scale * kLog2e;
  p.status = a->status;
  r.starts = a->query_start;
  r.rows = a->num_rows;
  r.maps = a->maps;
  r.q_sm = a->q_stride_m;
  r.lam = a->lam;
  r.lam_st = a->lam_stride_t;
  r.lam_sh = a->lam_stride_h;
  r.lam_value = a->lam_value;
  r.weight = a->norm ? a->norm_weight : nullptr;  // the weight belongs to the norm
  r.eps = a->eps;
  r.out_scale = a->out_scale;
  r.norm = a->norm;
}

template <int KV, int D, bool SCALED>
static void launch_general_maps(const PrefillParams& r, int bf, dim3 grid, cudaStream_t st) {
  if (r.maps == 2) general_prefill_kernel<KV, D, 2, SCALED><<<grid, kGeneralWarps * 32, 0, st>>>(r, bf);
  else general_prefill_kernel<KV, D, 1, SCALED><<<grid, kGeneralWarps * 32, 0, st>>>(r, bf);
}

template <int KV, bool SCALED>
static void launch_general(const PrefillParams& r, int bf, dim3 grid, cudaStream_t st) {
  switch (r.p.d) {
    case 32: launch_general_maps<KV, 32, SCALED>(r, bf, grid, st); break;
    case 64: launch_general_maps<KV, 64, SCALED>(r, bf, grid, st); break;
    case 128: launch_general_maps<KV, 128, SCALED>(r, bf, grid, st); break;
    default: launch_general_maps<KV, 256, SCALED>(r, bf, grid, st); break;
  }
}

static int run(const PdPrefillArgs* a) {
  const int rc = validate_prefill(a);
  if (rc != PD_OK) return rc;
  const int kernel = choose(a);
  if (kernel < 0) return kernel;
  if (a->num_rows == 0 || a->batch == 0) return PD_OK;
  if (kernel == PD_KERNEL_STREAM) {
    PdDecodeArgs probe;
    memset(&probe, 0, sizeof(probe));
    probe.sm_count = a->sm_count;
    const int sms = resolve_sm_count(&probe);
    if (sms <= 0) return PD_ERR_CUDA;
    if (!a->query_start) return diff_stream_run(a, sms);
    PrefillParams r;
    fill(a, r);
    return tc_run(a, r, sms);
  }
  PrefillParams r;
  fill(a, r);
  const dim3 grid(a->num_rows, a->num_q_heads / a->maps);
  const cudaStream_t st = (cudaStream_t)a->stream;
  const int bf = a->io_dtype == PD_IO_BF16;
  switch (a->kv_dtype) {
    case PD_KV_F16: launch_general<PD_KV_F16, false>(r, bf, grid, st); break;
    case PD_KV_BF16: launch_general<PD_KV_BF16, false>(r, bf, grid, st); break;
    case PD_KV_E5M2:
      if (a->k_scale) launch_general<PD_KV_E5M2, true>(r, bf, grid, st);
      else launch_general<PD_KV_E5M2, false>(r, bf, grid, st);
      break;
    default: launch_general<PD_KV_I8, true>(r, bf, grid, st); break;
  }
  return cudaGetLastError() == cudaSuccess ? PD_OK : PD_ERR_CUDA;
}

}  // namespace pd

extern "C" {

PD_API int pd_prefill(const PdPrefillArgs* args) {
  if (!args || !args->query_start) return PD_ERR_INVALID_ARG;
  return pd::run(args);
}

PD_API int pd_diff_decode(const PdPrefillArgs* args) {
  if (!args || args->query_start || args->maps != 2) return PD_ERR_INVALID_ARG;
  return pd::run(args);
}

PD_API int pd_prefill_select_kernel(const PdPrefillArgs* args) {
  const int rc = pd::validate_prefill(args);
  return rc != PD_OK ? rc : pd::choose(args);
}

PD_API int pd_prefill_workspace_bytes(const PdPrefillArgs* args, uint64_t* bytes) {
  using namespace pd;
  if (!bytes) return PD_ERR_INVALID_ARG;
  *bytes = 0;
  const int kernel = pd_prefill_select_kernel(args);
  if (kernel < 0) return kernel;
  if (kernel == PD_KERNEL_SIMPLE || args->num_rows == 0 || args->batch == 0) return PD_OK;
  PdDecodeArgs probe;
  memset(&probe, 0, sizeof(probe));
  probe.sm_count = args->sm_count;
  const int sms = resolve_sm_count(&probe);
  if (sms <= 0) return PD_ERR_CUDA;
  *bytes = args->query_start ? tc_workspace_bytes(args, sms) : diff_stream_workspace_bytes(args, sms);
  return PD_OK;
}

}  // extern "C"
