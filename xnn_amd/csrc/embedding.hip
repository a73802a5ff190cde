// Rows of a table by index with a scale, and the table's gradient by sorted indices
// (gfx950, wave64).
//
//   out[t]    = scale table[ids[t]]                       (xnn_embedding)
//   grad[v]   = scale sum_{t: ids[t] = v} g[t]            (xnn_embedding_grad)
//
// Both are streams: the rows are moved 16 bytes a lane. The gradient sorts the (id, t) pairs and sums
// the runs of one id in the order of t, so that no sum is an atomic one and every call gives the same
// bits; sums are held in float32 and rounded once. Three ways by size:
//
//   small tables (at most 255 rows, species): each block sorts its own tokens by counting, sums their
//     runs and leaves a row for each id it has seen; a block a row of the table adds those in order
//     (72,000 x 128 in float32, forward and backward call: 51 us, by the ways below 86; 21 tokens 50 and 53)
//   up to 32,768 tokens: chunks of 1,024 sorted in LDS while other blocks clear the table, merged by
//     rank (16,384 ids: 10 us in place of 30 in the LDS of one block and 26 by the passes below); then
//     runs of the sorted order are summed in chunks, and those that cross chunks joined
//   beyond: the same with a radix sort of three launches a pass (both passes of 128 channels from 50,000
//     rows, merged and radix: 32,768 tokens 59 and 76 us, 49,152 86 and 84, 131,072 391 and 198)
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.h"
#include "device.h"
#include "storage.h"

namespace xnn {

constexpr int kBins = 256;         // digits of a sort pass, ids of a small table
constexpr int kSortTile = 1024;    // ids a block of a sort pass takes, at least
constexpr int kSortBlocks = 512;   // blocks of a sort pass, at most
constexpr int kSortMerge = 32768;  // ids sorted in chunks of 1,024 that are merged, at most
constexpr int kChunk = 32;         // sorted positions a group of lanes sums
constexpr int kOwnTokens = 4096;   // tokens a block sorts for a small table, at most

static int64_t round64(int64_t b) { return (b + 63) / 64 * 64; }

struct EmbeddingWork {
  bool small, merge;
  int passes;
  int64_t blocks, per, chunks;                             // of the sort, of the sums
  int64_t key[2], perm[2], hist, part, seen, bytes;        // offsets
};

static EmbeddingWork embedding_work(int64_t n, int64_t n_rows, int64_t C) {
  EmbeddingWork w = {};
  w.small = n_rows < kBins;
  int64_t o = 0;
  if (w.small) {
    // as many blocks as fill the chip, with tokens enough that a block's rows are few beside them
    w.per = 256;
    while (w.per < kOwnTokens && n > w.per * 512) w.per *= 2;
    w.chunks = (n + w.per - 1) / w.per;
    w.seen = o;
    o += round64(w.chunks * (kBins / 8));
    w.part = o;
    o += 4 * w.chunks * n_rows * C;
    w.bytes = o;
    return w;
  }
  int bits = 1;
  while (bits < 31 && (n_rows >> bits) != 0) ++bits;       // n_rows itself is the invalid id
  w.passes = (bits + 7) / 8;
  w.merge = n <= kSortMerge;
  w.per = std::max<int64_t>(kSortTile,
                            (n + (int64_t)kSortBlocks * kSortTile - 1) / ((int64_t)kSortBlocks * kSortTile) *
                                kSortTile);
  w.blocks = (n + w.per - 1) / w.per;
  w.chunks = (n + kChunk - 1) / kChunk;
  for (int i = 0; i < 2; ++i) {
    w.key[i] = o;
    o += round64(4 * n);
    w.perm[i] = o;
    o += round64(4 * n);
  }
  w.hist = o;
  if (!w.merge) o += round64(4 * kBins * w.blocks);
  w.part = o;
  o += 8 * w.chunks * C;
  w.bytes = o;
  return w;
}

// ---------------------------------------------------------------- lookup
// A thread 16 bytes of a row. Narrow rows are bound by the 64-bit division that finds a thread's row: 72,000 rows
// of 128 in float32 10.8 us, 3.4 TB/s, the vector unit busy 55 % of the time; wide ones by the rows read and
// written: 16,384 rows of 1,024 in bfloat16 from 50,000 10.6 us, 6.3 TB/s (part of it in the last-level cache).
template <typename T, int N>
__global__ __launch_bounds__(256) void embedding_kernel(const int64_t* __restrict__ ids, int64_t n,
                                                        const T* __restrict__ table,
                                                        int64_t n_rows, int64_t C, float scale,
                                                        T* __restrict__ out) {
  const int64_t per = C / N, total = n * per;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t t = i / per, c = (i - t * per) * N;
    const int64_t z = ids[t];
    float v[N];
    if (z >= 0 && z < n_rows) {
      load_pack<T, N>(table + z * C + c, v);
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] *= scale;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = __builtin_nanf("");
    }
    store_pack<T, N>(out + t * C + c, v);
  }
}

// ---------------------------------------------------------------- sort
// the sort key of position i: in the first pass the id itself, n_rows for one outside the table
__device__ __forceinline__ uint32_t sort_key(const int64_t* ids, const uint32_t* key, int64_t i,
                                             int64_t n_rows) {
  if (key != nullptr) return key[i];
  const int64_t z = ids[i];
  return (uint32_t)(z >= 0 && z < n_rows ? z : n_rows);
}

__global__ __launch_bounds__(256) void sort_count_kernel(const int64_t* __restrict__ ids,
                                                         const uint32_t* __restrict__ key,
                                                         int64_t n, int64_t n_rows, int64_t per,
                                                         int shift, uint32_t* __restrict__ hist) {
  __shared__ uint32_t count[kBins];
  count[threadIdx.x] = 0;
  __syncthreads();
  const int64_t end = min(n, ((int64_t)blockIdx.x + 1) * per);
  for (int64_t i = (int64_t)blockIdx.x * per + threadIdx.x; i < end; i += 256)
    atomicAdd(&count[(sort_key(ids, key, i, n_rows) >> shift) & (kBins - 1)], 1u);
  __syncthreads();
  hist[(int64_t)threadIdx.x * gridDim.x + blockIdx.x] = count[threadIdx.x];
}

// exclusive scan of `m` counts in place, one block
__global__ __launch_bounds__(1024) void sort_scan_kernel(uint32_t* __restrict__ a, int64_t m) {
  __shared__ uint32_t sums[16];
  const int lane = threadIdx.x & (kWave - 1), wave = wave_in_block();
  const int64_t per = (m + 1023) / 1024;
  const int64_t i0 = min(m, threadIdx.x * per), i1 = min(m, i0 + per);
  uint32_t s = 0;
  for (int64_t i = i0; i < i1; ++i) s += a[i];
  uint32_t x = s;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint32_t y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  if (lane == kWave - 1) sums[wave] = x;
  __syncthreads();
  uint32_t before = x - s;
  for (int w = 0; w < wave; ++w) before += sums[w];
  for (int64_t i = i0; i < i1; ++i) {
    const uint32_t c = a[i];
    a[i] = before;
    before += c;
  }
}

__global__ __launch_bounds__(256) void sort_scatter_kernel(
    const int64_t* __restrict__ ids, const uint32_t* __restrict__ key,
    const uint32_t* __restrict__ perm, int64_t n, int64_t n_rows, int64_t per, int shift,
    const uint32_t* __restrict__ hist, uint32_t* __restrict__ key_out,
    uint32_t* __restrict__ perm_out) {
  __shared__ uint32_t base[kBins];
  __shared__ uint32_t count[4][kBins];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = wave_in_block();
  base[tid] = hist[(int64_t)tid * gridDim.x + blockIdx.x];
#pragma unroll
  for (int w = 0; w < 4; ++w) count[w][tid] = 0;
  __syncthreads();
  const int64_t begin = (int64_t)blockIdx.x * per, end = min(n, begin + per);
  for (int64_t i0 = begin; i0 < end; i0 += 256) {
    const int64_t i = i0 + tid;
    const bool live = i < end;
    const uint32_t k = live ? sort_key(ids, key, i, n_rows) : 0u;
    const uint32_t d = (k >> shift) & (kBins - 1);
    // the lanes of this wave with the same digit
    uint64_t same = __ballot(live);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const uint64_t set = __ballot((d >> b) & 1);
      same &= ((d >> b) & 1) ? set : ~set;
    }
    const uint32_t rank = __popcll(same & ((1ull << lane) - 1));
    if (live && rank == 0) count[wave][d] = __popcll(same);
    __syncthreads();
    if (live) {
      uint32_t to = base[d] + rank;
      for (int w = 0; w < wave; ++w) to += count[w][d];
      key_out[to] = k;
      perm_out[to] = perm != nullptr ? perm[i] : (uint32_t)i;
    }
    __syncthreads();
    uint32_t add = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      add += count[w][tid];
      count[w][tid] = 0;
    }
    base[tid] += add;
    __syncthreads();
  }
}

// Stable ranks of a block's keys by one digit: wave w holds rounds * 64 consecutive keys, lane l the
// l-th of each round. count[w][d] (zero before) becomes the wave's keys of digit d; rank[r] the key's
// place among them.
template <int ROUNDS>
__device__ __forceinline__ void wave_ranks(const uint32_t (&digit)[ROUNDS], int rounds, int live_rounds_end,
                                           uint32_t* count, uint32_t (&rank)[ROUNDS]) {
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    if (r < rounds) {
      const bool live = r * kWave + lane < live_rounds_end;
      const uint32_t d = digit[r];
      uint64_t same = __ballot(live);                      // the lanes with the same digit
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        const uint64_t set = __ballot((d >> b) & 1);
        same &= ((d >> b) & 1) ? set : ~set;
      }
      const uint32_t below = __popcll(same & ((1ull << lane) - 1));
      const uint32_t before = live ? count[d] : 0;
      rank[r] = before + below;
      wave_sync();
      if (live && below == 0) count[d] = before + __popcll(same);
      wave_sync();
    }
  }
}

// 16 bytes of zeros a thread and turn
__device__ __forceinline__ void clear16(char* p, int64_t bytes, int64_t thread, int64_t threads) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const int64_t whole = (uintptr_t)p % 16 == 0 ? bytes / 16 : 0;
  for (int64_t i = thread; i < whole; i += threads) reinterpret_cast<u32x4*>(p)[i] = u32x4{0, 0, 0, 0};
  for (int64_t i = whole * 16 + thread; i < bytes; i += threads) p[i] = 0;
}

__global__ __launch_bounds__(256) void clear_kernel(char* __restrict__ p, int64_t bytes) {
  clear16(p, bytes, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}

// Blocks below `chunks` sort 1,024 ids each in LDS, one a thread; the others clear the gradient, whose
// writes bound it where the table is large (50,000 rows of 1,024 in bfloat16: 15.6 us, 6.6 TB/s with the
// last-level cache; the sort of 16,384 ids alone 7).
__global__ __launch_bounds__(1024) void sort_chunk_kernel(const int64_t* __restrict__ ids, int n,
                                                          int64_t n_rows, int passes, int chunks,
                                                          uint32_t* __restrict__ key_out,
                                                          uint32_t* __restrict__ perm_out,
                                                          char* __restrict__ grad, int64_t bytes) {
  if ((int)blockIdx.x >= chunks) {
    clear16(grad, bytes, ((int64_t)blockIdx.x - chunks) * 1024 + threadIdx.x,
            ((int64_t)gridDim.x - chunks) * 1024);
    return;
  }
  __shared__ uint32_t keys[1024];
  __shared__ uint16_t perms[1024];
  __shared__ uint32_t count[16][kBins];
  __shared__ uint32_t sums[4];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = wave_in_block();
  const int begin = blockIdx.x * 1024, m = min(1024, n - begin);
  const int mine = min(max(m - wave * kWave, 0), kWave);
  const bool live = tid < m;
  uint32_t key = live ? sort_key(ids, nullptr, begin + tid, n_rows) : 0u;
  uint32_t perm = tid, digit[1], rank[1];
  for (int p = 0; p < passes; ++p) {
    for (int i = tid; i < 16 * kBins; i += 1024) (&count[0][0])[i] = 0;
    digit[0] = (key >> (8 * p)) & (kBins - 1);
    __syncthreads();
    wave_ranks(digit, 1, mine, count[wave], rank);
    __syncthreads();
    // keys of smaller digits, then those of the same digit in earlier waves
    uint32_t total = 0, x = 0;
    if (tid < kBins) {
#pragma unroll
      for (int w = 0; w < 16; ++w) total += count[w][tid];
      x = total;
#pragma unroll
      for (int o = 1; o < kWave; o <<= 1) {
        const uint32_t y = __shfl_up(x, o);
        if (lane >= o) x += y;
      }
      if (lane == kWave - 1) sums[wave] = x;
    }
    __syncthreads();
    if (tid < kBins) {
      uint32_t at = x - total;
      for (int w = 0; w < wave; ++w) at += sums[w];
#pragma unroll
      for (int w = 0; w < 16; ++w) {
        const uint32_t c = count[w][tid];
        count[w][tid] = at;
        at += c;
      }
    }
    __syncthreads();
    if (live) {
      const uint32_t to = count[wave][digit[0]] + rank[0];
      keys[to] = key;
      perms[to] = (uint16_t)perm;
    }
    __syncthreads();
    if (live) {
      key = keys[tid];
      perm = perms[tid];
    }
    __syncthreads();
  }
  if (live) {
    key_out[begin + tid] = key;
    perm_out[begin + tid] = begin + perm;
  }
}

// The place of every element of the sorted chunks among all: in its own chunk, plus the elements of each
// other chunk that come before it (equal ones of earlier chunks do), by bisection, `lanes` lanes an
// element. 6.3 us for 16,384 ids: sixteen bisections of ten dependent loads, in parallel lanes.
__global__ __launch_bounds__(256) void sort_merge_kernel(const uint32_t* __restrict__ key,
                                                         const uint32_t* __restrict__ perm, int n,
                                                         int chunks, int lanes,
                                                         uint32_t* __restrict__ key_out,
                                                         uint32_t* __restrict__ perm_out) {
  const int i = (int)(((int64_t)blockIdx.x * 256 + threadIdx.x) / lanes);
  const bool live = i < n;
  const uint32_t k = live ? key[i] : 0u;
  const int own = i / 1024;
  int before = 0;
  for (int c = threadIdx.x % lanes; live && c < chunks; c += lanes) {
    if (c == own) continue;
    const uint32_t* a = key + c * 1024;
    int lo = 0, hi = min(1024, n - c * 1024);
    while (lo < hi) {                                      // the first element not before this one
      const int mid = (lo + hi) / 2;
      const bool earlier = c < own ? a[mid] <= k : a[mid] < k;
      lo = earlier ? mid + 1 : lo;
      hi = earlier ? hi : mid;
    }
    before += lo;
  }
  for (int o = 1; o < lanes; o <<= 1) before += __shfl_xor(before, o);
  if (live && threadIdx.x % lanes == 0) {
    const int to = i % 1024 + before;
    key_out[to] = k;
    perm_out[to] = perm[i];
  }
}

// ---------------------------------------------------------------- small tables
// A block's `per` tokens sorted by id (counting, at most sixteen rounds of its four waves), then their
// runs summed by groups of `lanes` lanes over consecutive sorted positions, N channels a lane. A run
// within one group's positions goes to part[block][id]; of a run that crosses groups each leaves its
// sum in LDS and the group where it begins adds them in order. Bounded by latency: 72,000 rows of 128 in float32,
// two ids, 13.8 us, 2.7 TB/s, in 282 blocks, about one wave a SIMD, which asks for no cotangent before its
// ids are sorted.
template <typename T, int N>
__global__ __launch_bounds__(256) void own_sum_kernel(const int64_t* __restrict__ ids, int64_t n,
                                                      int n_rows, int64_t C, int64_t per, int lanes,
                                                      const T* __restrict__ g,
                                                      uint32_t* __restrict__ seen,
                                                      float* __restrict__ part) {
  __shared__ uint32_t count[4][kBins];
  __shared__ uint32_t sums[4];
  __shared__ uint16_t order[kOwnTokens];
  __shared__ uint8_t sorted[kOwnTokens];
  __shared__ float head[256 * N], tail[256 * N];           // of each group: its first run, its last
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = wave_in_block();
  const int64_t begin = (int64_t)blockIdx.x * per;
  const int m = (int)min(per, n - begin), rounds = (int)(per / 256);
  const int first = wave * rounds * kWave, mine = min(max(m - first, 0), rounds * kWave);
#pragma unroll
  for (int w = 0; w < 4; ++w) count[w][tid] = 0;
  uint32_t digit[16], rank[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    digit[r] = 0;
    const int i = r * kWave + lane;
    if (r < rounds && i < mine) digit[r] = sort_key(ids, nullptr, begin + first + i, n_rows);
  }
  __syncthreads();
  wave_ranks(digit, rounds, mine, count[wave], rank);
  __syncthreads();
  uint32_t total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) total += count[w][tid];
  uint32_t x = total;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint32_t y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  if (lane == kWave - 1) sums[wave] = x;
  const uint64_t present = __ballot(total > 0 && tid < n_rows);
  if (lane < 2 && blockIdx.y == 0)
    seen[(int64_t)blockIdx.x * (kBins / 32) + 2 * wave + lane] = (uint32_t)(present >> (32 * lane));
  __syncthreads();
  uint32_t at = x - total;
  for (int w = 0; w < wave; ++w) at += sums[w];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t c = count[w][tid];
    count[w][tid] = at;
    at += c;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (r < rounds && r * kWave + lane < mine) {
      const uint32_t to = count[wave][digit[r]] + rank[r];
      order[to] = (uint16_t)(first + r * kWave + lane);
      sorted[to] = (uint8_t)digit[r];
    }
  __syncthreads();

  const int groups = 256 / lanes, group = tid / lanes;
  const int64_t c = ((int64_t)blockIdx.y * lanes + tid % lanes) * N;
  const int each = (m + groups - 1) / groups;
  const int p0 = min(m, group * each), p1 = min(m, p0 + each);
  float* row = part + (int64_t)blockIdx.x * n_rows * C + c;
  bool crosses = false;                                    // the last run goes on in the next group
  if (c < C && p0 < p1) {
    const bool from_before = p0 > 0 && sorted[p0 - 1] == sorted[p0];
    crosses = p1 < m && sorted[p1] == sorted[p1 - 1];
    float sum[N] = {};
    int began = p0;
    constexpr int kAhead = 8;                              // rows in flight
    for (int p = p0; p < p1; p += kAhead) {
      float v[kAhead][N];
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        load_pack<T, N>(g + (begin + order[min(p + j, p1 - 1)]) * C + c, v[j]);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int i = p + j;
        if (i < p1) {
#pragma unroll
          for (int e = 0; e < N; ++e) sum[e] += v[j][e];
          const int k = sorted[i];
          if (i + 1 == p1 || sorted[i + 1] != k) {
            if (began == p0 && from_before)
              store_pack<float, N>(head + tid * N, sum);
            else if (i + 1 == p1 && crosses)
              store_pack<float, N>(tail + tid * N, sum);
            else if (k < n_rows)
              store_pack<float, N>(row + (int64_t)k * C, sum);
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] = 0.0f;
            began = i + 1;
          }
        }
      }
    }
    // a run that covers the group from end to end began before and belongs to an earlier group
    crosses = crosses && !(from_before && sorted[p0] == sorted[p1 - 1]);
  }
  __syncthreads();
  if (crosses && sorted[p1 - 1] < n_rows) {
    const int k = sorted[p1 - 1];
    float sum[N];
    load_pack<float, N>(tail + tid * N, sum);
    for (int q = group + 1; q < groups && q * each < m && sorted[q * each] == k; ++q) {
      float v[N];
      load_pack<float, N>(head + (tid + (q - group) * lanes) * N, v);
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] += v[e];
    }
    store_pack<float, N>(row + (int64_t)k * C, sum);
  }
}

// A block a row and 64 channels: the sums of the blocks that have seen it, sixteen waves in turn, and
// theirs in order; zero where none has. 7.6 us for 119 rows of 128 from 282 blocks, bound by the latency
// of those loads one after the other.
template <typename T>
__global__ __launch_bounds__(1024) void own_join_kernel(const uint32_t* __restrict__ seen,
                                                        const float* __restrict__ part, int64_t chunks,
                                                        int n_rows, int64_t C, float scale,
                                                        T* __restrict__ out) {
  __shared__ float s[16][kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = wave_in_block(), k = blockIdx.x;
  const int64_t c = (int64_t)blockIdx.y * kWave + lane;
  float sum = 0.0f;
  constexpr int kAhead = 8;
  for (int64_t q0 = wave; q0 < chunks; q0 += 16 * kAhead) {
    float v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int64_t q = q0 + 16 * j;
      v[j] = 0.0f;
      if (q < chunks && c < C && (seen[q * (kBins / 32) + k / 32] >> (k % 32)) & 1)
        v[j] = part[(q * n_rows + k) * C + c];
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) sum += v[j];
  }
  s[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && c < C) {
    float r = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) r += s[w][lane];
    out[k * C + c] = (T)(r * scale);
  }
}

// ---------------------------------------------------------------- sums
// A group of `lanes` lanes sums chunk positions of the sorted order, N channels a lane. A run that
// lies within the chunk goes to its row; one that goes on in the next chunk leaves its sum in
// part[chunk][1], one that came from the chunk before in part[chunk][0]. Bounded by rows gathered in
// sorted order: 16,384 rows of 1,024 in bfloat16 13.6 us, 2.5 TB/s read.
template <typename T, int N>
__global__ __launch_bounds__(256) void run_sum_kernel(
    const uint32_t* __restrict__ key, const uint32_t* __restrict__ perm, int64_t n, int64_t n_rows,
    int64_t C, int lanes, const T* __restrict__ g, float scale, float* __restrict__ part,
    T* __restrict__ out) {
  const int64_t chunk = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
  const int64_t c = ((int64_t)blockIdx.y * lanes + threadIdx.x % lanes) * N;
  const int64_t begin = chunk * kChunk, end = min(n, begin + kChunk);
  if (begin >= n || c >= C) return;
  const bool from_before = begin > 0 && key[begin - 1] == key[begin];
  const bool goes_on = end < n && key[end] == key[end - 1];
  float sum[N] = {};
  int64_t first = begin;
  constexpr int kAhead = 8;                                // rows in flight
  for (int64_t i0 = begin; i0 < end; i0 += kAhead) {
    float v[kAhead][N];
    uint32_t k[kAhead + 1];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int64_t i = min(i0 + j, end - 1);
      k[j] = key[i];
      load_pack<T, N>(g + (int64_t)perm[i] * C + c, v[j]);
    }
    k[kAhead] = i0 + kAhead < end ? key[i0 + kAhead] : 0;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int64_t i = i0 + j;
      if (i >= end) break;
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] += v[j][e];
      const bool last = i + 1 == end;
      if (!last && k[j + 1] == k[j]) continue;
      if (k[j] < n_rows) {
        if (first == begin && from_before) {
          store_pack<float, N>(part + 2 * chunk * C + c, sum);
        } else if (last && goes_on) {
          store_pack<float, N>(part + (2 * chunk + 1) * C + c, sum);
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) sum[e] *= scale;
          store_pack<T, N>(out + (int64_t)k[j] * C + c, sum);
        }
      }
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] = 0.0f;
      first = i + 1;
    }
  }
}

// The rows whose runs cross chunks: the block of the chunk where a run begins adds what the
// following chunks left, its four waves in turn, and their sums in order. N channels a lane. 7.6 us for
// 512 chunks of 1,024 channels, the longest run 18 % of the tokens; bound by that run: where one id of 300 holds
// 1,048,576 tokens of 128 in float32 the gradient takes 1.4 ms (of 200 ids, summed by blocks, 0.14).
template <typename T, int N>
__global__ __launch_bounds__(256) void run_join_kernel(const uint32_t* __restrict__ key, int64_t n,
                                                       int64_t n_rows, int64_t C, float scale,
                                                       const float* __restrict__ part,
                                                       T* __restrict__ out) {
  __shared__ float s[4][kWave * N];
  const int64_t chunk = blockIdx.x, begin = chunk * kChunk, end = min(n, begin + kChunk);
  if (end >= n) return;
  const uint32_t k = key[end - 1];
  if (k >= n_rows || key[end] != k) return;
  if (key[begin] == k && begin > 0 && key[begin - 1] == k) return;   // began before
  // the first position beyond the run
  int64_t lo = end, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (key[mid] == k)
      lo = mid + 1;
    else
      hi = mid;
  }
  const int64_t last = (lo - 1) / kChunk;                  // the chunk of its last position
  const int lane = threadIdx.x & (kWave - 1), wave = wave_in_block();
  const int64_t c = ((int64_t)blockIdx.y * kWave + lane) * N;
  float sum[N] = {};
  if (c < C) {
    if (wave == 0) load_pack<float, N>(part + (2 * chunk + 1) * C + c, sum);
#pragma unroll 4
    for (int64_t q = chunk + 1 + wave; q <= last; q += 4) {
      float v[N];
      load_pack<float, N>(part + 2 * q * C + c, v);
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] += v[e];
    }
  }
  store_pack<float, N>(&s[wave][lane * N], sum);
  __syncthreads();
  if (wave == 0 && c < C) {
#pragma unroll
    for (int e = 0; e < N; ++e)
      sum[e] = (((s[0][lane * N + e] + s[1][lane * N + e]) + s[2][lane * N + e]) + s[3][lane * N + e]) * scale;
    store_pack<T, N>(out + (int64_t)k * C + c, sum);
  }
}

template <typename T>
static int embedding(const int64_t* ids, int64_t n, const void* table, int64_t n_rows, int64_t C,
                     float scale, void* out, hipStream_t s) {
  constexpr int kN = 16 / sizeof(T);
  const bool vec = ((uintptr_t)table | (uintptr_t)out) % 16 == 0 && C % kN == 0;
  const int64_t total = n * (vec ? C / kN : C);
  const dim3 grid((unsigned)std::min<int64_t>((total + 255) / 256, 1 << 20)), block(256);
  const T* t = static_cast<const T*>(table);
  T* o = static_cast<T*>(out);
  if (vec)
    hipLaunchKernelGGL((embedding_kernel<T, kN>), grid, block, 0, s, ids, n, t, n_rows, C, scale, o);
  else
    hipLaunchKernelGGL((embedding_kernel<T, 1>), grid, block, 0, s, ids, n, t, n_rows, C, scale, o);
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

// lanes of a group that share a row, N channels each
static int row_lanes(int64_t C, int N, int most) {
  int lanes = 1;
  while (lanes < most && lanes * N < C) lanes *= 2;
  return lanes;
}

template <typename T, int N>
static void own_sums(const int64_t* ids, int64_t n, int64_t n_rows, int64_t C, const EmbeddingWork& w,
                     const T* g, float scale, uint32_t* seen, float* part, T* out, hipStream_t s) {
  const int lanes = row_lanes(C, N, 64);
  hipLaunchKernelGGL((own_sum_kernel<T, N>),
                     dim3((unsigned)w.chunks, (unsigned)((C + lanes * N - 1) / (lanes * N))), dim3(256),
                     0, s, ids, n, (int)n_rows, C, w.per, lanes, g, seen, part);
  hipLaunchKernelGGL(own_join_kernel<T>, dim3((unsigned)n_rows, (unsigned)((C + kWave - 1) / kWave)),
                     dim3(1024), 0, s, seen, part, w.chunks, (int)n_rows, C, scale, out);
}

template <typename T, int N>
static void run_sums(const uint32_t* key, const uint32_t* perm, int64_t n, int64_t n_rows, int64_t C,
                     const EmbeddingWork& w, const T* g, float scale, float* part, T* out,
                     hipStream_t s) {
  const int lanes = row_lanes(C, N, 256);
  const int64_t groups = 256 / lanes;
  const dim3 grid((unsigned)((w.chunks + groups - 1) / groups),
                  (unsigned)((C + lanes * N - 1) / (lanes * N)));
  hipLaunchKernelGGL((run_sum_kernel<T, N>), grid, dim3(256), 0, s, key, perm, n, n_rows, C, lanes,
                     g, scale, part, out);
  constexpr int kJoin = N == 1 ? 1 : 4;
  hipLaunchKernelGGL((run_join_kernel<T, kJoin>),
                     dim3((unsigned)w.chunks, (unsigned)((C + kWave * kJoin - 1) / (kWave * kJoin))),
                     dim3(256), 0, s, key, n, n_rows, C, scale, part, out);
}

template <typename T>
static int embedding_grad(const int64_t* ids, int64_t n, const void* g, int64_t n_rows, int64_t C,
                          float scale, void* out, char* work, hipStream_t s) {
  constexpr int kN = 16 / sizeof(T);
  const T* gt = static_cast<const T*>(g);
  T* o = static_cast<T*>(out);
  char* grad = static_cast<char*>(out);
  const bool vec = ((uintptr_t)g | (uintptr_t)out) % 16 == 0 && C % kN == 0;
  const int64_t bytes = n_rows * C * (int64_t)sizeof(T);
  const EmbeddingWork w = embedding_work(n, n_rows, C);
  float* part = (float*)(work + w.part);
  if (n == 0) {
    hipLaunchKernelGGL(clear_kernel, dim3((unsigned)std::min<int64_t>(bytes / 4096 + 1, 4096)),
                       dim3(256), 0, s, grad, bytes);
  } else if (w.small) {
    uint32_t* seen = (uint32_t*)(work + w.seen);
    if (vec)
      own_sums<T, kN>(ids, n, n_rows, C, w, gt, scale, seen, part, o, s);
    else
      own_sums<T, 1>(ids, n, n_rows, C, w, gt, scale, seen, part, o, s);
  } else {
    uint32_t *key[2], *perm[2], *hist = (uint32_t*)(work + w.hist);
    for (int i = 0; i < 2; ++i) {
      key[i] = (uint32_t*)(work + w.key[i]);
      perm[i] = (uint32_t*)(work + w.perm[i]);
    }
    int from = 0;
    if (w.merge) {
      const int chunks = (int)((n + 1023) / 1024);
      const int64_t clear = std::min<int64_t>(bytes / 16384 + 1, 2048);
      from = chunks > 1 ? 1 : 0;
      hipLaunchKernelGGL(sort_chunk_kernel, dim3((unsigned)(chunks + clear)), dim3(1024), 0, s, ids, (int)n,
                         n_rows, w.passes, chunks, key[0], perm[0], grad, bytes);
      if (chunks > 1) {
        const int lanes = row_lanes(chunks, 1, 64);
        hipLaunchKernelGGL(sort_merge_kernel, dim3((unsigned)((n * lanes + 255) / 256)), dim3(256), 0, s,
                           key[0], perm[0], (int)n, chunks, lanes, key[1], perm[1]);
      }
    } else {
      hipLaunchKernelGGL(clear_kernel, dim3((unsigned)std::min<int64_t>(bytes / 4096 + 1, 8192)),
                         dim3(256), 0, s, grad, bytes);
      const dim3 grid((unsigned)w.blocks);
      from = 1;
      for (int p = 0; p < w.passes; ++p) {
        const uint32_t* k = p == 0 ? nullptr : key[from];
        const uint32_t* q = p == 0 ? nullptr : perm[from];
        hipLaunchKernelGGL(sort_count_kernel, grid, dim3(256), 0, s, ids, k, n, n_rows, w.per, 8 * p,
                           hist);
        hipLaunchKernelGGL(sort_scan_kernel, dim3(1), dim3(1024), 0, s, hist, kBins * w.blocks);
        hipLaunchKernelGGL(sort_scatter_kernel, grid, dim3(256), 0, s, ids, k, q, n, n_rows, w.per,
                           8 * p, hist, key[1 - from], perm[1 - from]);
        from = 1 - from;
      }
    }
    if (vec)
      run_sums<T, kN>(key[from], perm[from], n, n_rows, C, w, gt, scale, part, o, s);
    else
      run_sums<T, 1>(key[from], perm[from], n, n_rows, C, w, gt, scale, part, o, s);
  }
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

}  // namespace xnn

using namespace xnn;

extern "C" {

int xnn_embedding(int dtype, const int64_t* ids, int64_t n, const void* table, int64_t n_rows,
                  int64_t n_channels, float scale, void* out, xnn_stream_t stream) {
  XNN_REQUIRE(is_storage(dtype), "dtype must be XNN_F32, XNN_BF16 or XNN_F16");
  XNN_REQUIRE(n >= 0 && n_rows >= 0 && n_channels >= 0, "negative size");
  if (n == 0 || n_channels == 0) return XNN_OK;
  XNN_REQUIRE(ids && out && (n_rows == 0 || table), "NULL input or output");
  XNN_STORAGE_DISPATCH(dtype, T,
                       return embedding<T>(ids, n, table, n_rows, n_channels, scale, out,
                                           as_hip(stream)));
}

int xnn_embedding_grad_work_size(int64_t n, int64_t n_rows, int64_t n_channels, size_t* bytes) {
  XNN_REQUIRE(n >= 0 && n_rows >= 0 && n_channels >= 0, "negative size");
  XNN_REQUIRE(n < ((int64_t)1 << 31) && n_rows < ((int64_t)1 << 31) - 1, "too many ids or rows");
  XNN_REQUIRE(bytes != nullptr, "NULL size");
  *bytes = (size_t)embedding_work(n, n_rows, n_channels).bytes;
  return XNN_OK;
}

int xnn_embedding_grad(int dtype, const int64_t* ids, int64_t n, const void* grad_out,
                       int64_t n_rows, int64_t n_channels, float scale, void* grad_table,
                       void* work, size_t work_bytes, xnn_stream_t stream) {
  XNN_REQUIRE(is_storage(dtype), "dtype must be XNN_F32, XNN_BF16 or XNN_F16");
  XNN_REQUIRE(n >= 0 && n_rows >= 0 && n_channels >= 0, "negative size");
  XNN_REQUIRE(n < ((int64_t)1 << 31) && n_rows < ((int64_t)1 << 31) - 1, "too many ids or rows");
  XNN_REQUIRE(n_channels <= 65535 * (int64_t)kWave, "too many channels");
  if (n_rows == 0 || n_channels == 0) return XNN_OK;
  XNN_REQUIRE(grad_table && (n == 0 || (ids && grad_out && work)), "NULL input, output or work");
  XNN_REQUIRE(work_bytes >= (size_t)embedding_work(n, n_rows, n_channels).bytes, "work too small");
  XNN_REQUIRE((uintptr_t)work % 16 == 0, "work must be aligned to 16 bytes");
  XNN_STORAGE_DISPATCH(dtype, T,
                       return embedding_grad<T>(ids, n, grad_out, n_rows, n_channels, scale,
                                                grad_table, (char*)work, as_hip(stream)));
}

}  // extern "C"
