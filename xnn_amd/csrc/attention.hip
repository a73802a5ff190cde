// Attention within the structures of a batch (gfx950, wave64): the plan of its tiles and the
// forward pass.
//
//   out_i = sum_j p_ij v_j,  p_ij = exp(scale q_i . k_j - L_i),  L_i = log sum_j exp(scale q_i . k_j)
//
// over the atoms j of i's structure that the mask keeps; a row with none is zero (L = -inf). One
// pass over the keys with the running maximum and sum of each row, in base 2: the scores are never
// in memory. Heads of keys and values are shared by heads / kv_heads query heads each.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "attention.h"
#include "common.h"

namespace xnn {

// ---------------------------------------------------------------- plan
constexpr int kLengths = 1024;     // classes of lengths, 32 rows each (the last: all longer ones)

__device__ __forceinline__ int64_t atoms_of(const int64_t* n_atoms, int64_t b, int64_t n_tokens,
                                            bool& wrong) {
  const int64_t n = n_atoms[b];
  const bool bad = n < 0 || n > n_tokens;
  wrong |= bad;
  return bad ? 0 : n;
}

// exclusive sum over the block's 1,024 threads, and the total
__device__ __forceinline__ int64_t block_before(int64_t x, int64_t* sums, int64_t& total) {
  const int lane = threadIdx.x & (kWave - 1), wave = wave_in_block();
  int64_t y = x;
  for (int o = 1; o < kWave; o <<= 1) {
    const int64_t z = __shfl_up(y, o);
    if (lane >= o) y += z;
  }
  __syncthreads();
  if (lane == kWave - 1) sums[wave] = y;
  __syncthreads();
  int64_t before = y - x;
  total = 0;
  for (int w = 0; w < 16; ++w) {
    if (w < wave) before += sums[w];
    total += sums[w];
  }
  return before;
}

// One block: where each structure's rows begin (ptr), the structures by falling length (order; those
// of one class in any order, which moves no result: every tile has an owner), the tiles of 32 and of
// 128 rows before each of them (tile_ptr), info: tiles of each list, longest structure, status, rows
// in all. Once a batch, not a call: 11 us for 1,024 structures, bound by its scans' barriers.
__global__ __launch_bounds__(1024) void attention_plan_count_kernel(
    const int64_t* __restrict__ n_atoms, int64_t n_structures, int64_t n_tokens,
    int64_t* __restrict__ ptr, int64_t* __restrict__ tile_ptr, int64_t* order,
    int64_t* __restrict__ info) {
  __shared__ int64_t sums[16];
  __shared__ int count[kLengths], wrong_any;
  __shared__ unsigned long long longest;
  const int tid = threadIdx.x;
  const int64_t per = (n_structures + 1023) / 1024;
  const int64_t b0 = min(n_structures, tid * per), b1 = min(n_structures, b0 + per);
  count[tid] = 0;
  if (tid == 0) {
    wrong_any = 0;
    longest = 0;
  }
  __syncthreads();
  const auto class_of = [](int64_t n) { return (int)(kLengths - 1 - min((n + 31) / 32, (int64_t)kLengths - 1)); };
  int64_t s = 0, most = 0;
  bool wrong = false;
  for (int64_t b = b0; b < b1; ++b) {
    const int64_t n = atoms_of(n_atoms, b, n_tokens, wrong);
    s += n;
    most = max(most, n);
    atomicAdd(&count[class_of(n)], 1);
  }
  if (wrong) atomicOr(&wrong_any, 1);
  atomicMax(&longest, (unsigned long long)most);
  int64_t rows;
  int64_t at = block_before(s, sums, rows);
  for (int64_t b = b0; b < b1; ++b) {
    ptr[b] = at;
    at += atoms_of(n_atoms, b, n_tokens, wrong);
  }
  int64_t all;
  const int before = (int)block_before(count[tid], sums, all);
  count[tid] = before;
  __syncthreads();
  for (int64_t b = b0; b < b1; ++b)
    order[atomicAdd(&count[class_of(atoms_of(n_atoms, b, n_tokens, wrong))], 1)] = b;
  __threadfence_block();
  __syncthreads();
  int64_t tiles[2];
  for (int list = 0; list < 2; ++list) {
    const int64_t size = list == 0 ? 32 : 128;
    s = 0;
    for (int64_t i = b0; i < b1; ++i) s += (atoms_of(n_atoms, order[i], n_tokens, wrong) + size - 1) / size;
    at = block_before(s, sums, tiles[list]);
    int64_t* out = tile_ptr + list * (n_structures + 1);
    for (int64_t i = b0; i < b1; ++i) {
      out[i] = at;
      at += (atoms_of(n_atoms, order[i], n_tokens, wrong) + size - 1) / size;
    }
    if (tid == 0) out[n_structures] = tiles[list];
  }
  if (tid == 0) {
    ptr[n_structures] = rows;
    info[0] = tiles[0];
    info[1] = tiles[1];
    info[2] = (int64_t)longest;
    info[3] = wrong_any ? 1 : rows != n_tokens ? 2 : 0;
    info[4] = rows;
  }
}

// one thread a tile: (first row, end of its structure, begin of its structure)
__global__ __launch_bounds__(256) void attention_plan_fill_kernel(
    const int64_t* __restrict__ ptr, const int64_t* __restrict__ tile_ptr,
    const int64_t* __restrict__ order, int64_t n_structures, const int64_t* __restrict__ info,
    int64_t capacity32, int64_t capacity128, int32_t* __restrict__ tiles32,
    int32_t* __restrict__ tiles128) {
  if (info[3] != 0) return;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int list = t < capacity32 ? 0 : 1;
  const int64_t i = list == 0 ? t : t - capacity32;
  if (i >= (list == 0 ? capacity32 : capacity128) || i >= info[list]) return;
  const int64_t* p = tile_ptr + list * (n_structures + 1);
  int64_t lo = 0, hi = n_structures;                        // p[lo] <= i < p[hi]
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (p[mid] <= i)
      lo = mid;
    else
      hi = mid;
  }
  const int64_t b = order[lo];
  int32_t* out = (list == 0 ? tiles32 : tiles128) + 3 * i;
  out[0] = (int32_t)(ptr[b] + (i - p[lo]) * (list == 0 ? 32 : 128));
  out[1] = (int32_t)ptr[b + 1];
  out[2] = (int32_t)ptr[b];
}

// ---------------------------------------------------------------- forward
// Two products, n^2 D multiplications each a head, and between them about eight vector instructions a
// score: a SIMD's vector unit and its matrix core take turns within a wave and overlap only between the
// two waves that share it. Bounded by their sum (vector 41-64 %, matrix 38-59 % of the cycles), not by
// memory: a block of four waves reads each staged row for 128 query rows.
//   24,000 rows, 4 heads of 64, bfloat16: 751 us, 785 TFLOP/s (large library product: 1,202)
//   9,000 rows, 4 heads of 32, float32: 262 us and 8 of the join, 158 TFLOP/s (154)
//   1,024 structures of 10-60 rows, 4 heads of 16, float32: 18 us, bounded by latency: a block of one wave
//     has one or two tiles to walk
// The next tile is asked for before this one is used and waits in registers. No gain came from two LDS
// buffers and one barrier a tile, from raised wave priority around the products, or from products of the
// next tile between the exponentials of this one (24,000 rows in bfloat16, both passes:
// 3,020-3,117 us against 3,040).
template <typename T, int DP, int WAVES, int TILE, bool VEC, int WP>
__global__ __launch_bounds__(WAVES* kWave, (Head<T, DP>::kForward)) void attention_kernel(AttentionArgs a) {
  typedef Head<T, DP, TILE> S;
  constexpr int kParts = S::kTile / 32;                    // 32-row products of a tile
  __shared__ __align__(16) char k_tile[S::kBytes];
  __shared__ __align__(16) char v_tile[S::kBytes];
  Tile t;
  block_tile(a, a.heads, t);
  const int lane = threadIdx.x & (kWave - 1), half = lane / 32;
  const int64_t row = t.first + kOwn * wave_in_block() + lane % 32;
  const bool live = row < t.end;
  const bool busy = t.first + kOwn * wave_in_block() < t.end;   // the wave has rows
  const int64_t kv = t.head / (a.heads / a.kv_heads);
  const T* k = (const T*)a.k + kv * a.k_head;
  const T* v = (const T*)a.v + kv * a.v_head;
  const float scale = a.scale * kLog2e;
  int64_t from, to;
  walk_part((t.end - t.begin + S::kTile - 1) / S::kTile, a, t.split, from, to);
  from = t.begin + from * S::kTile;
  to = min(t.end, t.begin + to * S::kTile);
  Stage<T, S, WAVES * kWave, VEC> next_k, next_v;
  uint8_t next_keep = 0;
  next_k.init(a.k_token, a.D);
  next_v.init(a.v_token, a.D);
  const auto fetch = [&](int64_t j0) {
    next_keep = row_byte<S::kTile>(j0, to, a.mask, lane);
    next_k.fetch(k + j0 * a.k_token, a.k_token, to - j0, a.D);
    next_v.fetch(v + j0 * a.v_token, a.v_token, to - j0, a.D);
  };
  if (from < to) fetch(from);
  Operand<T> q[S::kSteps];
  load_own<T, DP, VEC>((const T*)a.q + t.head * a.q_head, a.q_token, row, live, a.D, half, scale, q);
  f32x16 o[S::kBlocks] = {};
  float top = -INFINITY, sum = 0.0f;                       // the sum over this lane's keys only
  for (int64_t j0 = from; j0 < to; j0 += S::kTile) {
    __syncthreads();
    const uint64_t keep = __ballot(next_keep != 0);
    next_k.commit(k_tile, a.D, keep);
    next_v.commit(v_tile, a.D, keep);
    __syncthreads();
    if (j0 + S::kTile < to) fetch(j0 + S::kTile);
    if (!busy || keep == 0) continue;
    f32x16 p[kParts] = {};
#pragma unroll
    for (int c = 0; c < S::kSteps; ++c)
#pragma unroll
      for (int b = 0; b < kParts; ++b)
        mma<T>(natural_operand<T, S>(k_tile, 32 * b + lane % 32, c, half), q[c], p[b]);
    if (keep != (~0ull >> (64 - S::kTile))) {
#pragma unroll
      for (int b = 0; b < kParts; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          p[b][r] = has_row((uint32_t)(keep >> (32 * b)), r) ? p[b][r] : -INFINITY;
    }
    float m = p[0][0];
#pragma unroll
    for (int b = 0; b < kParts; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) m = fmaxf(m, p[b][r]);
    m = score<T>(max_xor32(m), scale);
    const float next = fmaxf(top, m);
    const float base = next == -INFINITY ? 0.0f : next;    // nothing kept so far
    if (__any(next != top)) {                              // rare once the walk is under way
      const float shrink = __builtin_amdgcn_exp2f(top - base);
      sum *= shrink;
#pragma unroll
      for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= shrink;
      top = next;
    }
#pragma unroll
    for (int b = 0; b < kParts; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[b][r] = weight<T>(p[b][r], scale, base);
        sum += p[b][r];
      }
#pragma unroll
    for (int b = 0; b < kParts; ++b)
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const auto w = weight_operand<T, WP>(p[b], f);
#pragma unroll
        for (int d = 0; d < S::kBlocks; ++d)
          mma<T>(transposed_operand<T, S>(v_tile, 32 * b, d, f, lane), w, o[d]);
      }
  }
  sum = add_xor32(sum);
  if (!live) return;
  const bool empty = sum == 0.0f;
  const float factor = empty ? 0.0f : 1.0f / sum;
  const float lse = empty ? -INFINITY : top + __builtin_amdgcn_logf(sum);
  const int64_t at = row * a.heads + t.head;
  if (a.splits > 1) {
    const int64_t part = (int64_t)t.split * a.n_tokens * a.heads + at;
    store_own(a.part + part * a.D, o, factor, a.D, a.D % 4 == 0, half);
    if (half == 0) a.part_lse[part] = lse;
  } else {
    store_own((T*)a.result + at * a.D, o, factor, a.D, a.vec_out, half);
    if (a.lse != nullptr && half == 0) a.lse[(int64_t)t.head * a.n_tokens + row] = lse;
  }
}

// The parts of a row joined: out = sum_s 2^(L_s - L) out_s, L = log2 sum_s 2^L_s. A thread takes N
// elements of a row of one head. A stream: 9,000 rows of 4 x 32 in five parts 7.6 us, 3.6 TB/s.
template <typename T, int N>
__global__ __launch_bounds__(256) void attention_join_kernel(AttentionArgs a) {
  const int64_t per = (a.D + N - 1) / N, n = a.n_tokens * a.heads;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n * per) return;
  const int64_t at = i / per, d = (i - at * per) * N;
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_lse[s * n + at]);
  const float base = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f, acc[N] = {};
  for (int s = 0; s < a.splits; ++s) {
    const float w = __builtin_amdgcn_exp2f(a.part_lse[s * n + at] - base);
    float x[N];
    load_pack<float, N>(a.part + (s * n + at) * a.D + d, x);
    sum += w;
    // a part of weight zero is not read into the sum: what it holds may not be finite
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] += w == 0.0f ? 0.0f : w * x[j];
  }
  const float factor = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] *= factor;
  store_pack<T, N>((T*)a.result + at * a.D + d, acc);
  if (a.lse != nullptr && d == 0)
    a.lse[at % a.heads * a.n_tokens + at / a.heads] =
        sum == 0.0f ? -INFINITY : top + __builtin_amdgcn_logf(sum);
}

template <typename T, int DP>
static void attention_launch(const AttentionArgs& a, int rows, bool fine, hipStream_t s) {
  const dim3 grid((unsigned)(a.n_tiles * a.heads * a.splits));
  XNN_ATTENTION_LAUNCH(attention_kernel, grid, fine);
  if (a.splits == 1) return;
  const int64_t n = a.n_tokens * a.heads;
  if (a.vec_out)
    hipLaunchKernelGGL((attention_join_kernel<T, 4>), dim3((unsigned)((n * (a.D / 4) + 255) / 256)),
                       dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((attention_join_kernel<T, 1>), dim3((unsigned)((n * a.D + 255) / 256)),
                       dim3(256), 0, s, a);
}

// parts of a launch: short structures, whose blocks are of one wave, are walked whole
static int part_count(const xnn_attention_tiles* plan, int heads, int dtype, int D) {
  return attention_rows(plan, storage_bytes(dtype), D) == 32
             ? 1
             : forward_splits(attention_blocks(plan, heads), plan->max_atoms, split_rows(dtype, D));
}

static size_t forward_bytes(int64_t n_tokens, int heads, int D, int splits) {
  return splits == 1 ? 0 : sizeof(float) * (size_t)splits * n_tokens * heads * (D + 1);
}

}  // namespace xnn

using namespace xnn;

extern "C" {

int xnn_attention_plan(const int64_t* n_atoms, int64_t n_structures, int64_t n_tokens, int64_t* ptr,
                       int64_t* tile_ptr, int64_t* order, int32_t* tiles32, int64_t capacity32,
                       int32_t* tiles128, int64_t capacity128, int64_t* info, xnn_stream_t stream) {
  XNN_REQUIRE(n_structures >= 0 && n_tokens >= 0, "negative size");
  XNN_REQUIRE(n_tokens < ((int64_t)1 << 31) - 128 && n_structures < (int64_t)1 << 31,
              "too many tokens or structures");
  XNN_REQUIRE(ptr && tile_ptr && info && (n_structures == 0 || (n_atoms && order)),
              "NULL input or output");
  XNN_REQUIRE(capacity32 >= n_tokens / 32 + n_structures &&
                  capacity128 >= n_tokens / 128 + n_structures,
              "a tile list is too small");
  XNN_REQUIRE((capacity32 == 0 || tiles32) && (capacity128 == 0 || tiles128), "NULL tile list");
  hipStream_t s = as_hip(stream);
  hipLaunchKernelGGL(attention_plan_count_kernel, dim3(1), dim3(1024), 0, s, n_atoms, n_structures,
                     n_tokens, ptr, tile_ptr, order, info);
  const int64_t all = capacity32 + capacity128;
  if (all > 0)
    hipLaunchKernelGGL(attention_plan_fill_kernel, dim3((unsigned)((all + 255) / 256)), dim3(256), 0,
                       s, ptr, tile_ptr, order, n_structures, info, capacity32, capacity128, tiles32,
                       tiles128);
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

int xnn_attention_work_size(int dtype, int64_t n_tokens, int32_t n_heads, int32_t head_dim,
                            const xnn_attention_tiles* plan, size_t* bytes) {
  XNN_REQUIRE(is_storage(dtype), "dtype must be XNN_F32, XNN_BF16 or XNN_F16");
  XNN_REQUIRE(plan && bytes, "NULL plan or size");
  XNN_REQUIRE(n_tokens >= 0 && n_heads >= 1 && head_dim >= 1, "sizes out of range");
  const int splits = part_count(plan, n_heads, dtype, head_dim);
  *bytes = forward_bytes(n_tokens, n_heads, head_dim, splits);
  return XNN_OK;
}

int xnn_attention(int dtype, const xnn_heads* q, const xnn_heads* k, const xnn_heads* v,
                  int64_t n_tokens, int32_t head_dim, const xnn_attention_tiles* plan,
                  const uint8_t* mask, float scale, void* out, float* lse, void* work,
                  size_t work_bytes, xnn_stream_t stream) {
  AttentionArgs a;
  const int status = attention_args(a, dtype, q, k, v, n_tokens, head_dim, plan, mask, scale);
  if (status != XNN_OK || n_tokens == 0) return status;
  XNN_REQUIRE(out != nullptr, "NULL output");
  a.splits = part_count(plan, a.heads, dtype, head_dim);
  if (a.splits > 1) {
    XNN_REQUIRE(work && work_bytes >= forward_bytes(n_tokens, a.heads, head_dim, a.splits),
                "work too small");
    XNN_REQUIRE((uintptr_t)work % 16 == 0, "work must be aligned to 16 bytes");
  }
  a.result = out;
  a.lse = lse;
  a.part = (float*)work;
  a.part_lse = a.part + (size_t)a.splits * n_tokens * a.heads * head_dim;
  a.vec_out = head_dim % 4 == 0 && (uintptr_t)out % 16 == 0;
  const int rows = attention_pick(a, plan, dtype);
  const bool fine = fine_weights(a, plan);
  hipStream_t s = as_hip(stream);
  XNN_STORAGE_DISPATCH(dtype, T, {
    if (head_dim <= 16)
      attention_launch<T, 16>(a, rows, fine, s);
    else if (head_dim <= 32)
      attention_launch<T, 32>(a, rows, fine, s);
    else if (head_dim <= 64)
      attention_launch<T, 64>(a, rows, fine, s);
    else if (head_dim <= 96)
      attention_launch<T, 96>(a, rows, fine, s);
    else
      attention_launch<T, 128>(a, rows, fine, s);
  });
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

}  // extern "C"
