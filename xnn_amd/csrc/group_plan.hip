// The plan of rows by group (gfx950, wave64): a stable counting sort of the rows' group numbers, and for every
// tile size the prefix sums of the groups' tiles. Nothing is read on the host.
//
// A wave counts a run of rows in LDS; one block turns the runs' counts into places; each wave then writes its rows
// in their order, 64 at a time: a row's place among the 64 is the number of lower lanes of its group (ballots over
// the bits of the group number), so the order is that of the rows and the same at every call. Bound by the latency
// of three short dependent launches: 8, 6 and 10 us for 72,000 rows of 9 groups, 2, 4 and 2 for 21.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "dense.h"

namespace xnn {

constexpr int kPlanRun = 1024;     // rows of a wave

// the bucket of row t: its group, or n_groups where that is none
__device__ __forceinline__ int bucket_of(const int64_t* __restrict__ ids, int64_t t, int n_groups) {
  const int64_t g = ids[t];
  return g >= 0 && g < n_groups ? (int)g : n_groups;
}

// counts[run][bucket]
__global__ __launch_bounds__(kWave) void group_count_kernel(const int64_t* __restrict__ ids, int n, int n_groups,
                                                            int32_t* __restrict__ counts) {
  __shared__ int32_t c[kMaxGroups + 1];
  for (int b = threadIdx.x; b <= n_groups; b += kWave) c[b] = 0;
  wave_sync();
  const int begin = blockIdx.x * kPlanRun, end = min(n, begin + kPlanRun);
  for (int t = begin + threadIdx.x; t < end; t += kWave) atomicAdd(&c[bucket_of(ids, t, n_groups)], 1);
  wave_sync();
  for (int b = threadIdx.x; b <= n_groups; b += kWave)
    counts[(int64_t)blockIdx.x * (n_groups + 1) + b] = c[b];
}

// Counts become the place of each run's first row of the bucket; row_ptr and the levels' tile_ptr. A bucket's counts go
// to 2^k threads, each a stretch of the runs; then a wave a list adds up the buckets, 64 at a time.
__global__ __launch_bounds__(1024) void group_place_kernel(int32_t* __restrict__ counts, int runs, int n_groups,
                                                           int lanes, int32_t* __restrict__ row_ptr) {
  __shared__ int32_t total[kMaxGroups + 1];
  __shared__ int32_t part[1024];
  const int tid = threadIdx.x, buckets = n_groups + 1;
  const int per = 1024 / lanes, lane = tid / per, each = (runs + lanes - 1) / lanes;
  const int r0 = min(runs, lane * each), r1 = min(runs, r0 + each);
  for (int b0 = 0; b0 < buckets; b0 += per) {
    const int b = b0 + tid % per;
    int32_t s = 0;
    if (b < buckets)
#pragma unroll 8
      for (int r = r0; r < r1; ++r) s += counts[(int64_t)r * buckets + b];
    part[tid] = s;
    __syncthreads();
    if (b < buckets) {
      int32_t at = 0;
      for (int l = 0; l < lane; ++l) at += part[l * per + tid % per];
      if (lane == lanes - 1) total[b] = at + s;
      for (int r = r0; r < r1; ++r) {
        int32_t* p = counts + (int64_t)r * buckets + b;
        const int32_t v = *p;
        *p = at;
        at += v;
      }
    }
    __syncthreads();
  }
  for (int list = tid / kWave; list <= kGroupLevels; list += 1024 / kWave) {
    int32_t* out = row_ptr + (int64_t)list * (n_groups + 2);
    const int size = list == 0 ? 1 : level_rows(list - 1);
    int32_t before = 0;
    for (int b0 = 0; b0 < buckets; b0 += kWave) {
      const int b = b0 + tid % kWave;
      const int32_t own = b < buckets ? (int32_t)(((int64_t)total[b] + size - 1) / size) : 0;
      int32_t sum = own;                                   // inclusive
#pragma unroll
      for (int o = 1; o < kWave; o *= 2) {
        const int32_t v = __shfl_up(sum, o, kWave);
        if (tid % kWave >= o) sum += v;
      }
      if (b < buckets) out[b] = before + sum - own;
      before += __shfl(sum, kWave - 1, kWave);
    }
    if (tid % kWave == 0) out[buckets] = before;
  }
}

__global__ __launch_bounds__(kWave) void group_scatter_kernel(const int64_t* __restrict__ ids, int n, int n_groups,
                                                              int bits, const int32_t* __restrict__ counts,
                                                              const int32_t* __restrict__ row_ptr,
                                                              int32_t* __restrict__ order) {
  __shared__ int32_t place[kMaxGroups + 1];
  for (int b = threadIdx.x; b <= n_groups; b += kWave)
    place[b] = row_ptr[b] + counts[(int64_t)blockIdx.x * (n_groups + 1) + b];
  wave_sync();
  const int lane = threadIdx.x;
  const int begin = blockIdx.x * kPlanRun, end = min(n, begin + kPlanRun);
  for (int t0 = begin; t0 < end; t0 += kWave) {
    const int t = t0 + lane;
    const bool live = t < end;
    const int b = live ? bucket_of(ids, t, n_groups) : 0;
    uint64_t same = __ballot(live);
    for (int i = 0; i < bits; ++i) {
      const uint64_t set = __ballot((b >> i) & 1);
      same &= (b >> i) & 1 ? set : ~set;
    }
    const uint64_t below = same & ((1ull << lane) - 1);
    const int at = live ? place[b] : 0;
    wave_sync();
    if (live) {
      order[at + __popcll(below)] = t;
      if ((same >> lane) >> 1 == 0) place[b] = at + __popcll(same);   // the last lane of its group
    }
    wave_sync();
  }
}

}  // namespace xnn

using namespace xnn;

extern "C" {

int xnn_group_plan_size(int64_t n, int32_t n_groups, size_t* plan_bytes, size_t* work_bytes) {
  XNN_REQUIRE(n >= 0 && n < ((int64_t)1 << 30), "n must be in [0, 2^30)");
  XNN_REQUIRE(n_groups >= 1 && n_groups <= kMaxGroups, "n_groups must be in [1, %d]", kMaxGroups);
  XNN_REQUIRE(plan_bytes && work_bytes, "NULL size");
  *plan_bytes = (size_t)group_plan_ints(n, n_groups) * sizeof(int32_t);
  *work_bytes = (size_t)((n + kPlanRun - 1) / kPlanRun) * (n_groups + 1) * sizeof(int32_t);
  return XNN_OK;
}

int xnn_group_plan(const int64_t* ids, int64_t n, int32_t n_groups, int32_t* plan, void* work,
                   size_t work_bytes, xnn_stream_t stream) {
  size_t need_plan = 0, need = 0;
  const int status = xnn_group_plan_size(n, n_groups, &need_plan, &need);
  if (status != XNN_OK) return status;
  XNN_REQUIRE(plan, "NULL plan");
  XNN_REQUIRE(n == 0 || ids, "NULL ids");
  XNN_REQUIRE(need == 0 || (work && work_bytes >= need), "work too small");
  hipStream_t s = as_hip(stream);
  const int runs = (int)((n + kPlanRun - 1) / kPlanRun);
  int32_t *counts = (int32_t*)work, *row_ptr = plan + n;
  int bits = 1;
  while ((1 << bits) <= n_groups) ++bits;
  if (runs > 0)
    hipLaunchKernelGGL(group_count_kernel, dim3(runs), dim3(kWave), 0, s, ids, (int)n, n_groups, counts);
  int lanes = 1;                   // threads of a bucket's counts
  while (lanes < runs && lanes * 2 * (n_groups + 1) <= 1024) lanes *= 2;
  hipLaunchKernelGGL(group_place_kernel, dim3(1), dim3(1024), 0, s, counts, runs, n_groups, lanes, row_ptr);
  if (runs > 0)
    hipLaunchKernelGGL(group_scatter_kernel, dim3(runs), dim3(kWave), 0, s, ids, (int)n, n_groups, bits, counts,
                       row_ptr, plan);
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

}  // extern "C"
