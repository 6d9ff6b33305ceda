// Block tables, slot map, positions and lengths of one step, built on the GPU from request
// lengths (pd_plan_step).
//
// With context length c_b, n_b new tokens and page size P: need_b = ceil((c_b + n_b) / P) -
// ceil(c_b / P) pages, I_b = need_0 + .. + need_b.  A request is served when its pages fit its row
// and need_b = 0 or I_b <= num_free; page k of need_b comes from free_blocks[num_free - 1 -
// (I_b - need_b + k)].  A token's slot is table[b, pos / P] * P + pos % P.
//
// Bound by latency: a decode step of 256 requests moves 9 KB, a step of 64 requests with 10 k prompt tokens 172 KB.
// So it is one launch of one thread-block cluster (1 to 8 CTAs).  Every CTA makes the scans over
// the requests for itself in shared memory (a few microseconds' worth of nothing to exchange
// otherwise), then the CTAs share out the tokens and the table rows.  A token in a new page
// takes the block id from the free list itself, so nobody waits for the row being written.  The
// cluster barrier stands between the last read of the lengths and of num_free and their first
// write, which is what lets a caller update them in place without a counter in memory.
//
// 256 requests with a token each: 7.3 us a launch in a graph; 64 requests, 10479 tokens: 6.8 us; an empty launch
// takes 2 to 3.  The rest is the chain lengths -> scan -> block id -> store of dependent memory accesses.
#include "pd_common.cuh"

namespace pd {

constexpr int kPlanThreads = 512;
constexpr int kPlanMaxBatch = 8192;
constexpr int kPlanMaxCtas = 8;
// Consecutive tokens of one thread.  Up to a token for every thread there can be it is one: their block ids
// are then fetched side by side (256 requests with a token each: four a thread took 9.9 us, the chain of
// their four loads).  Above, four share a search and mostly a block id and are stored 16 bytes at a time.
constexpr int kPlanRunMany = 4;
constexpr int kPlanFewTokens = kPlanThreads * kPlanMaxCtas;

struct PlanParams {
  int32_t* table;
  int64_t table_stride;
  const int32_t* context;
  const int32_t* fresh;
  const int32_t* free_blocks;
  const int32_t* num_free;
  int64_t* slots;
  int64_t* positions;
  int32_t* starts;
  int32_t* lens;
  int32_t* num_free_out;
  int32_t batch, max_blocks, page, capacity, tokens, wide;
  uint32_t* status;
};

// One request in shared memory: first new token, context length, pages taken before it, and its own
// (-1: it is not served).
struct PlanRow {
  int start, context, before, need;
};

__device__ __forceinline__ int plan_pages(int64_t tokens, int page) { return (int)((tokens + page - 1) / page); }

template <int kPlanRun>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanParams p) {
  extern __shared__ PlanRow rows[];  // batch + 1: the last holds the totals
  __shared__ long long warp_sum[kPlanThreads / 32];
  __shared__ int taken_max;
  constexpr unsigned kFull = 0xffffffffu;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cta = blockIdx.x, ctas = gridDim.x;
  const int free_now = min(max(__ldg(p.num_free), 0), p.capacity);
  if (tid == 0) taken_max = 0;

  // ---- one scan of both counts (new tokens in the low word, pages in the high word) -----------
  const int per = (p.batch + kPlanThreads - 1) / kPlanThreads;
  const int first = min(tid * per, p.batch), last = min(first + per, p.batch);
  long long mine = 0;
  for (int b = first; b < last; ++b) {
    const int c = max(__ldg(p.context + b), 0), n = max(__ldg(p.fresh + b), 0);
    const int64_t want = ((int64_t)c + n + p.page - 1) / p.page;
    const int held = plan_pages(c, p.page);
    const bool fits = want <= p.max_blocks;
    rows[b].context = c;
    rows[b].start = n;
    rows[b].before = fits ? (int)want - held : -1;  // pages wanted, -1: no room in the row
    mine += (long long)(unsigned)n + ((long long)(fits ? want - held : 0) << 32);
  }
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(kFull, upto, o);
    if (lane >= o) upto += y;
  }
  if (lane == 31) warp_sum[warp] = upto;
  __syncthreads();
  if (warp == 0) {
    long long x = lane < kPlanThreads / 32 ? warp_sum[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(kFull, x, o);
      if (lane >= o) x += y;
    }
    if (lane < kPlanThreads / 32) warp_sum[lane] = x;
  }
  __syncthreads();
  long long run = upto - mine + (warp ? warp_sum[warp - 1] : 0);
  int refused = 0, most = 0;
  for (int b = first; b < last; ++b) {
    const int n = rows[b].start, need = rows[b].before;
    const int start = (int)(unsigned)(run & 0xffffffffll), before = (int)(run >> 32);
    const int end = before + max(need, 0);
    const bool served = need >= 0 && (need == 0 || (before >= 0 && end <= free_now));
    rows[b].start = start;
    rows[b].before = before;
    rows[b].need = served ? need : -1;
    if (served && need > 0) most = max(most, end);
    if (!served) refused = 1;
    run += (long long)(unsigned)n + ((long long)max(need, 0) << 32);
  }
  if (last == p.batch && (first < last || tid == 0)) rows[p.batch].start = (int)(unsigned)(run & 0xffffffffll);
  if (most) atomicMax(&taken_max, most);
  if (refused && cta == 0 && p.status) atomicOr(p.status, PD_DEV_NO_BLOCKS);
  __syncthreads();
  const int total = rows[p.batch].start;

  // ---- slots and positions: kPlanRun consecutive tokens a thread ----------------------------------
  const int64_t runs = ((int64_t)p.tokens + kPlanRun - 1) / kPlanRun;
  for (int64_t r = (int64_t)cta * kPlanThreads + tid; r < runs; r += (int64_t)ctas * kPlanThreads) {
    const int t0 = (int)(r * kPlanRun);
    int b = 0, hi = p.batch;  // the last b with start <= t0
    while (hi - b > 1) {
      const int mid = (b + hi) >> 1;
      if (rows[mid].start <= t0) b = mid;
      else hi = mid;
    }
    int64_t slot[kPlanRun], pos[kPlanRun];
    int held_page = -1, held_b = -1, block = -1;
#pragma unroll
    for (int k = 0; k < kPlanRun; ++k) {
      const int t = t0 + k;
      slot[k] = -1;
      pos[k] = 0;
      if (t < total && t < p.tokens) {
        while (b + 1 < p.batch && rows[b + 1].start <= t) ++b;
        const PlanRow row = rows[b];
        const int64_t at = (int64_t)row.context + (t - row.start);
        pos[k] = at;
        if (row.need >= 0) {
          const int page = (int)((uint32_t)at / (uint32_t)p.page);  // a served request fits its row: at < 2^31
          if (page != held_page || b != held_b) {
            // a page in use comes from the table, a new one from the free list
            const int held = plan_pages(row.context, p.page);
            block = -1;
            if (page < held) block = p.table[(int64_t)b * p.table_stride + page];
            else if (page - held < row.need) block = __ldg(p.free_blocks + (free_now - 1 - (row.before + page - held)));
            held_page = page;
            held_b = b;
          }
          if (block >= 0) slot[k] = (int64_t)block * p.page + ((int)at - page * p.page);
        }
      }
    }
    if (kPlanRun % 2 == 0 && p.wide && t0 + kPlanRun <= p.tokens) {
#pragma unroll
      for (int k = 0; k + 1 < kPlanRun; k += 2) {
        *reinterpret_cast<longlong2*>(p.slots + t0 + k) = make_longlong2(slot[k], slot[k + 1]);
        *reinterpret_cast<longlong2*>(p.positions + t0 + k) = make_longlong2(pos[k], pos[k + 1]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kPlanRun; ++k) {
        if (t0 + k < p.tokens) {
          p.slots[t0 + k] = slot[k];
          p.positions[t0 + k] = pos[k];
        }
      }
    }
  }

  // ---- new table entries: a warp per request -----------------------------------------------------
  for (int b = cta * (kPlanThreads / 32) + warp; b < p.batch; b += ctas * (kPlanThreads / 32)) {
    const PlanRow row = rows[b];
    const int held = plan_pages(row.context, p.page);
    for (int k = lane; k < row.need; k += 32)
      p.table[(int64_t)b * p.table_stride + held + k] = __ldg(p.free_blocks + (free_now - 1 - (row.before + k)));
  }

  // ---- lengths and the free count: behind everybody's last read of their old values --------------
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  for (int b = cta * kPlanThreads + tid; b <= p.batch; b += ctas * kPlanThreads) {
    const PlanRow row = rows[b];
    p.starts[b] = row.start;
    if (b < p.batch) p.lens[b] = row.context + (row.need >= 0 ? max(__ldg(p.fresh + b), 0) : 0);
  }
  if (cta == 0 && tid == 0) *p.num_free_out = free_now - taken_max;
}

}  // namespace pd

extern "C" PD_API int pd_plan_step(const PdPlanArgs* a) {
  using namespace pd;
  if (!a || !a->num_free || !a->query_start || !a->num_free_out) return PD_ERR_INVALID_ARG;
  if (a->batch < 0 || a->max_blocks_per_seq <= 0 || a->block_size <= 0 || a->free_capacity < 0 || a->num_tokens < 0)
    return PD_ERR_INVALID_ARG;
  if (a->batch > 0 && (!a->block_table || !a->context_lens || !a->new_tokens || !a->seq_lens)) return PD_ERR_INVALID_ARG;
  if (a->batch > 1 && a->block_table_stride < a->max_blocks_per_seq) return PD_ERR_INVALID_ARG;
  if (a->free_capacity > 0 && !a->free_blocks) return PD_ERR_INVALID_ARG;
  if (a->num_tokens > 0 && (!a->slot_mapping || !a->positions)) return PD_ERR_INVALID_ARG;
  // the scan holds both counts in 32 bits each
  if (a->batch > kPlanMaxBatch || (int64_t)a->batch * a->max_blocks_per_seq > INT32_MAX ||
      (int64_t)a->max_blocks_per_seq * a->block_size > INT32_MAX)
    return PD_ERR_UNSUPPORTED;
  PlanParams p;
  p.table = a->block_table;
  p.table_stride = a->block_table_stride;
  p.context = a->context_lens;
  p.fresh = a->new_tokens;
  p.free_blocks = a->free_blocks;
  p.num_free = a->num_free;
  p.slots = a->slot_mapping;
  p.positions = a->positions;
  p.starts = a->query_start;
  p.lens = a->seq_lens;
  p.num_free_out = a->num_free_out;
  p.batch = a->batch;
  p.max_blocks = a->max_blocks_per_seq;
  p.page = a->block_size;
  p.capacity = a->free_capacity;
  p.tokens = a->num_tokens;
  p.wide = ((uintptr_t)a->slot_mapping % 16 == 0 && (uintptr_t)a->positions % 16 == 0) ? 1 : 0;
  p.status = a->status;
  const bool few = a->num_tokens <= kPlanFewTokens;
  auto* kern = few ? plan_kernel<1> : plan_kernel<kPlanRunMany>;
  // as many CTAs as give every thread its run, up to the cluster's eight
  int ctas = 1;
  while (ctas < kPlanMaxCtas && (int64_t)ctas * kPlanThreads * (few ? 1 : kPlanRunMany) < a->num_tokens) ctas <<= 1;
  const size_t smem = (size_t)(a->batch + 1) * sizeof(PlanRow);
  // 48 KB are granted unasked, to the rows here and the kernel's static arrays (some 150 bytes) together
  if (smem > 47 * 1024 &&
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (int)((kPlanMaxBatch + 1) * sizeof(PlanRow))) != cudaSuccess)
    return PD_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)a->stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? PD_OK : PD_ERR_CUDA;
}
