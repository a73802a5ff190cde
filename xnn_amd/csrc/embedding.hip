// Rows of a table by index with a scale, and the table's gradient by sorted indices
// (gfx950, wave64).
//
//   out[t]    = scale table[ids[t]]                       (xnn_embedding)
//   grad[v]   = scale sum_{t: ids[t] = v} g[t]            (xnn_embedding_grad)
//
// Both are streams: the rows are moved 16 bytes a lane. The gradient sorts the (id, t) pairs by a
// stable least-significant-digit radix sort (8 bits a pass, as many passes as the number of rows
// has bits), sums chunks of kChunk sorted positions a group of lanes each, in the order of t, and
// joins the runs that cross chunks afterwards in a fixed order: no atomics on floats, the
// same bits at every call. Sums are held in float32 and rounded once.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.h"
#include "device.h"
#include "storage.h"

namespace xnn {

constexpr int kBins = 256;        // digits of a sort pass
constexpr int kSortTile = 1024;   // ids a block of a sort pass takes, at least
constexpr int kSortBlocks = 512;  // blocks of a sort pass, at most
constexpr int kChunk = 32;        // sorted positions a group of lanes sums

static int64_t round64(int64_t b) { return (b + 63) / 64 * 64; }

struct EmbeddingWork {
  int passes;
  int64_t blocks, per, chunks;                             // of the sort, of the sums
  int64_t key[2], perm[2], hist, part, bytes;              // offsets
};

static EmbeddingWork embedding_work(int64_t n, int64_t n_rows, int64_t C) {
  EmbeddingWork w;
  int bits = 1;
  while (bits < 31 && (n_rows >> bits) != 0) ++bits;       // n_rows itself is the invalid id
  w.passes = (bits + 7) / 8;
  w.per = std::max<int64_t>(kSortTile,
                            (n + (int64_t)kSortBlocks * kSortTile - 1) / ((int64_t)kSortBlocks * kSortTile) *
                                kSortTile);
  w.blocks = (n + w.per - 1) / w.per;
  w.chunks = (n + kChunk - 1) / kChunk;
  int64_t o = 0;
  for (int i = 0; i < 2; ++i) {
    w.key[i] = o;
    o += round64(4 * n);
    w.perm[i] = o;
    o += round64(4 * n);
  }
  w.hist = o;
  o += round64(4 * kBins * w.blocks);
  w.part = o;
  o += 8 * w.chunks * C;
  w.bytes = o;
  return w;
}

// ---------------------------------------------------------------- lookup
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

// ---------------------------------------------------------------- sums
template <typename T>
__global__ __launch_bounds__(256) void fill_zero_kernel(T* __restrict__ out, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x)
    out[i] = (T)0.0f;
}

// A group of `lanes` lanes sums chunk positions of the sorted order, N channels a lane. A run that
// lies within the chunk goes to its row; one that goes on in the next chunk leaves its sum in
// part[chunk][1], one that came from the chunk before in part[chunk][0].
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
  float sum[N];
#pragma unroll
  for (int j = 0; j < N; ++j) sum[j] = 0.0f;
  int64_t first = begin;
  for (int64_t i = begin; i < end; ++i) {
    const uint32_t k = key[i];
    float v[N];
    load_pack<T, N>(g + (int64_t)perm[i] * C + c, v);
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] += v[j];
    const bool last = i + 1 == end;
    if (!last && key[i + 1] == k) continue;
    if (k < n_rows) {
      if (first == begin && from_before) {
        store_pack<float, N>(part + 2 * chunk * C + c, sum);
      } else if (last && goes_on) {
        store_pack<float, N>(part + (2 * chunk + 1) * C + c, sum);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] *= scale;
        store_pack<T, N>(out + (int64_t)k * C + c, sum);
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] = 0.0f;
    first = i + 1;
  }
}

// The rows whose runs cross chunks: the block of the chunk where a run begins adds what the
// following chunks left, sixteen waves in turn, and their sums in order.
template <typename T>
__global__ __launch_bounds__(1024) void run_join_kernel(const uint32_t* __restrict__ key, int64_t n,
                                                        int64_t n_rows, int64_t C, float scale,
                                                        const float* __restrict__ part,
                                                        T* __restrict__ out) {
  __shared__ float s[16][kWave];
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
  const int64_t c = (int64_t)blockIdx.y * kWave + lane;
  float sum = 0.0f;
  if (c < C) {
    if (wave == 0) sum = part[(2 * chunk + 1) * C + c];
#pragma unroll 4
    for (int64_t q = chunk + 1 + wave; q <= last; q += 16) sum += part[2 * q * C + c];
  }
  s[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && c < C) {
    float r = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) r += s[w][lane];
    out[(int64_t)k * C + c] = (T)(r * scale);
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

template <typename T, int N>
static void run_sums(const uint32_t* key, const uint32_t* perm, int64_t n, int64_t n_rows, int64_t C,
                     const EmbeddingWork& w, const T* g, float scale, float* part, T* out,
                     hipStream_t s) {
  int lanes = 1;
  while (lanes < 256 && lanes * N < C) lanes *= 2;
  const int64_t groups = 256 / lanes;
  const dim3 grid((unsigned)((w.chunks + groups - 1) / groups),
                  (unsigned)((C + lanes * N - 1) / (lanes * N)));
  hipLaunchKernelGGL((run_sum_kernel<T, N>), grid, dim3(256), 0, s, key, perm, n, n_rows, C, lanes,
                     g, scale, part, out);
}

template <typename T>
static int embedding_grad(const int64_t* ids, int64_t n, const void* g, int64_t n_rows, int64_t C,
                          float scale, void* out, char* work, hipStream_t s) {
  constexpr int kN = 16 / sizeof(T);
  T* o = static_cast<T*>(out);
  const int64_t cells = n_rows * C;
  const bool words = (uintptr_t)out % 16 == 0 && cells % kN == 0;
  const int64_t fill = words ? cells / kN * 4 : cells;
  const dim3 fill_grid((unsigned)std::min<int64_t>((fill + 255) / 256, 8192));
  if (words)
    hipLaunchKernelGGL(fill_zero_kernel<float>, fill_grid, dim3(256), 0, s, (float*)out, fill);
  else
    hipLaunchKernelGGL(fill_zero_kernel<T>, fill_grid, dim3(256), 0, s, o, fill);
  if (n > 0) {
    const EmbeddingWork w = embedding_work(n, n_rows, C);
    uint32_t *key[2], *perm[2], *hist = (uint32_t*)(work + w.hist);
    for (int i = 0; i < 2; ++i) {
      key[i] = (uint32_t*)(work + w.key[i]);
      perm[i] = (uint32_t*)(work + w.perm[i]);
    }
    float* part = (float*)(work + w.part);
    const dim3 grid((unsigned)w.blocks);
    int from = 1;
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
    const T* gt = static_cast<const T*>(g);
    if (((uintptr_t)g | (uintptr_t)out) % 16 == 0 && C % kN == 0)
      run_sums<T, kN>(key[from], perm[from], n, n_rows, C, w, gt, scale, part, o, s);
    else
      run_sums<T, 1>(key[from], perm[from], n, n_rows, C, w, gt, scale, part, o, s);
    hipLaunchKernelGGL(run_join_kernel<T>, dim3((unsigned)w.chunks, (unsigned)((C + 63) / 64)),
                       dim3(1024), 0, s, key[from], n, n_rows, C, scale, part, o);
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
