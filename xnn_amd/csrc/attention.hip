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
// tile counts of lists of 64 and 128 rows; info: tiles of each list, longest structure, status
__global__ __launch_bounds__(1024) void attention_plan_count_kernel(
    const int64_t* __restrict__ n_atoms, int64_t n_structures, int64_t n_tokens,
    int64_t* __restrict__ ptr, int64_t* __restrict__ tile_ptr, int64_t* __restrict__ info) {
  __shared__ int64_t sums[3][16];
  __shared__ int64_t top[16];
  __shared__ int bad[16];
  const int lane = threadIdx.x & (kWave - 1), wave = wave_in_block();
  const int64_t per = (n_structures + 1023) / 1024;
  const int64_t b0 = min(n_structures, threadIdx.x * per), b1 = min(n_structures, b0 + per);
  int64_t s[3] = {0, 0, 0}, most = 0;
  bool wrong = false;
  for (int64_t b = b0; b < b1; ++b) {
    int64_t n = n_atoms[b];
    wrong |= n < 0 || n > n_tokens;
    n = n < 0 || n > n_tokens ? 0 : n;
    s[0] += n;
    s[1] += (n + 63) / 64;
    s[2] += (n + 127) / 128;
    most = max(most, n);
  }
  int64_t x[3];
  for (int q = 0; q < 3; ++q) {
    x[q] = s[q];
    for (int o = 1; o < kWave; o <<= 1) {
      const int64_t y = __shfl_up(x[q], o);
      if (lane >= o) x[q] += y;
    }
    if (lane == kWave - 1) sums[q][wave] = x[q];
  }
  for (int o = 1; o < kWave; o <<= 1) most = max(most, (int64_t)__shfl_xor(most, o));
  wrong = __any(wrong);
  if (lane == 0) {
    top[wave] = most;
    bad[wave] = wrong;
  }
  __syncthreads();
  int64_t at[3];
  for (int q = 0; q < 3; ++q) {
    at[q] = x[q] - s[q];
    for (int w = 0; w < wave; ++w) at[q] += sums[q][w];
  }
  for (int64_t b = b0; b < b1; ++b) {
    int64_t n = n_atoms[b];
    n = n < 0 || n > n_tokens ? 0 : n;
    ptr[b] = at[0];
    tile_ptr[b] = at[1];
    tile_ptr[n_structures + 1 + b] = at[2];
    at[0] += n;
    at[1] += (n + 63) / 64;
    at[2] += (n + 127) / 128;
  }
  if (threadIdx.x == 0) {
    int64_t total[3] = {0, 0, 0}, longest = 0;
    bool any = false;
    for (int w = 0; w < 16; ++w) {
      for (int q = 0; q < 3; ++q) total[q] += sums[q][w];
      longest = max(longest, top[w]);
      any |= bad[w] != 0;
    }
    ptr[n_structures] = total[0];
    tile_ptr[n_structures] = total[1];
    tile_ptr[2 * n_structures + 1] = total[2];
    info[0] = total[1];
    info[1] = total[2];
    info[2] = longest;
    info[3] = any ? 1 : total[0] != n_tokens ? 2 : 0;
    info[4] = total[0];
  }
}

// one thread a tile: (first row, end of its structure, begin of its structure)
__global__ __launch_bounds__(256) void attention_plan_fill_kernel(
    const int64_t* __restrict__ ptr, const int64_t* __restrict__ tile_ptr, int64_t n_structures,
    const int64_t* __restrict__ info, int64_t capacity64, int64_t capacity128,
    int32_t* __restrict__ tiles64, int32_t* __restrict__ tiles128) {
  if (info[3] != 0) return;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int list = t < capacity64 ? 0 : 1;
  const int64_t i = list == 0 ? t : t - capacity64;
  if (i >= (list == 0 ? capacity64 : capacity128) || i >= info[list]) return;
  const int64_t* p = tile_ptr + list * (n_structures + 1);
  int64_t lo = 0, hi = n_structures;                        // p[lo] <= i < p[hi]
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (p[mid] <= i)
      lo = mid;
    else
      hi = mid;
  }
  int32_t* out = (list == 0 ? tiles64 : tiles128) + 3 * i;
  out[0] = (int32_t)(ptr[lo] + (i - p[lo]) * (list == 0 ? 64 : 128));
  out[1] = (int32_t)ptr[lo + 1];
  out[2] = (int32_t)ptr[lo];
}

// ---------------------------------------------------------------- forward
template <typename T, int DP, int WAVES>
__global__ __launch_bounds__(WAVES* kWave, (Head<T, DP>::kOccupancy)) void attention_kernel(AttentionArgs a) {
  typedef Head<T, DP> S;
  constexpr int kParts = S::kTile / 32;                    // 32-row products of a tile
  __shared__ __align__(16) char k_tile[S::kBytes];
  __shared__ __align__(16) char v_tile[S::kBytes];
  Tile t;
  if (!block_tile(a, a.heads, t)) return;
  const int lane = threadIdx.x & (kWave - 1), half = lane / 32;
  const int64_t row = t.first + kOwn * wave_in_block() + lane % 32;
  const bool live = row < t.end;
  const int64_t kv = t.head / (a.heads / a.kv_heads);
  const T* k = (const T*)a.k + kv * a.k_head;
  const T* v = (const T*)a.v + kv * a.v_head;
  const float scale = a.scale * kLog2e;
  int64_t from, to;
  walk_part((t.end - t.begin + S::kTile - 1) / S::kTile, a, t.split, from, to);
  from = t.begin + from * S::kTile;
  to = min(t.end, t.begin + to * S::kTile);
  Stage<T, DP, WAVES * kWave> next_k, next_v;
  uint64_t next_keep = 0;
  if (from < to) {
    next_k.fetch(k, a.k_token, from, to, a.D, a.vec, a.mask);
    next_v.fetch(v, a.v_token, from, to, a.D, a.vec, a.mask);
    next_keep = live_rows<S::kTile>(from, to, a.mask, lane);
  }
  Operand<T> q[S::kSteps];
  load_own<T, DP>((const T*)a.q + t.head * a.q_head, a.q_token, row, live, a.D, a.vec, half, scale, q);
  f32x16 o[S::kBlocks] = {};
  float top = -INFINITY, sum = 0.0f;                       // the sum over this lane's keys only
  for (int64_t j0 = from; j0 < to; j0 += S::kTile) {
    __syncthreads();
    next_k.commit(k_tile);
    next_v.commit(v_tile);
    const uint64_t keep = next_keep;
    __syncthreads();
    if (j0 + S::kTile < to) {
      next_k.fetch(k, a.k_token, j0 + S::kTile, to, a.D, a.vec, a.mask);
      next_v.fetch(v, a.v_token, j0 + S::kTile, to, a.D, a.vec, a.mask);
      next_keep = live_rows<S::kTile>(j0 + S::kTile, to, a.mask, lane);
    }
    f32x16 p[kParts] = {};
#pragma unroll
    for (int c = 0; c < S::kSteps; ++c)
#pragma unroll
      for (int b = 0; b < kParts; ++b)
        mma<T>(natural_operand<T, DP>(k_tile, 32 * b + lane % 32, c, half), q[c], p[b]);
    if (keep != (~0ull >> (64 - S::kTile))) {
      const uint64_t mine = keep >> (4 * half);
#pragma unroll
      for (int b = 0; b < kParts; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          p[b][r] = (mine >> (32 * b + tile_row(r, 0))) & 1 ? p[b][r] : -INFINITY;
    }
    float m = p[0][0];
#pragma unroll
    for (int b = 0; b < kParts; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) m = fmaxf(m, p[b][r]);
    m = score<T>(fmaxf(m, __shfl_xor(m, 32)), scale);
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
        const Operand<T> w = weight_operand<T, Store<T>::kPlanes>(p[b], f);
#pragma unroll
        for (int d = 0; d < S::kBlocks; ++d)
          mma<T>(transposed_operand<T, DP>(v_tile, 32 * b, d, f, lane), w, o[d]);
      }
  }
  sum += __shfl_xor(sum, 32);
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
// elements of a row of one head.
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
static void attention_launch(const AttentionArgs& a, int rows, hipStream_t s) {
  const dim3 grid((unsigned)xcd_blocks(a.n_tiles * a.heads * a.splits));
  if (rows == 64)
    hipLaunchKernelGGL((attention_kernel<T, DP, 2>), grid, dim3(128), 0, s, a);
  else
    hipLaunchKernelGGL((attention_kernel<T, DP, 4>), grid, dim3(256), 0, s, a);
  if (a.splits == 1) return;
  const int64_t n = a.n_tokens * a.heads;
  if (a.vec_out)
    hipLaunchKernelGGL((attention_join_kernel<T, 4>), dim3((unsigned)((n * (a.D / 4) + 255) / 256)),
                       dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((attention_join_kernel<T, 1>), dim3((unsigned)((n * a.D + 255) / 256)),
                       dim3(256), 0, s, a);
}

static size_t forward_bytes(int64_t n_tokens, int heads, int D, int splits) {
  return splits == 1 ? 0 : sizeof(float) * (size_t)splits * n_tokens * heads * (D + 1);
}

}  // namespace xnn

using namespace xnn;

extern "C" {

int xnn_attention_plan(const int64_t* n_atoms, int64_t n_structures, int64_t n_tokens, int64_t* ptr,
                       int64_t* tile_ptr, int32_t* tiles64, int64_t capacity64, int32_t* tiles128,
                       int64_t capacity128, int64_t* info, xnn_stream_t stream) {
  XNN_REQUIRE(n_structures >= 0 && n_tokens >= 0, "negative size");
  XNN_REQUIRE(n_tokens < ((int64_t)1 << 31) - 128, "too many tokens");
  XNN_REQUIRE(ptr && tile_ptr && info && (n_structures == 0 || n_atoms), "NULL input or output");
  XNN_REQUIRE(capacity64 >= n_tokens / 64 + n_structures &&
                  capacity128 >= n_tokens / 128 + n_structures,
              "a tile list is too small");
  XNN_REQUIRE((capacity64 == 0 || tiles64) && (capacity128 == 0 || tiles128), "NULL tile list");
  hipStream_t s = as_hip(stream);
  hipLaunchKernelGGL(attention_plan_count_kernel, dim3(1), dim3(1024), 0, s, n_atoms, n_structures,
                     n_tokens, ptr, tile_ptr, info);
  const int64_t all = capacity64 + capacity128;
  if (all > 0)
    hipLaunchKernelGGL(attention_plan_fill_kernel, dim3((unsigned)((all + 255) / 256)), dim3(256), 0,
                       s, ptr, tile_ptr, n_structures, info, capacity64, capacity128, tiles64,
                       tiles128);
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

int xnn_attention_work_size(int64_t n_tokens, int32_t n_heads, int32_t head_dim,
                            const xnn_attention_tiles* plan, size_t* bytes) {
  XNN_REQUIRE(plan && bytes, "NULL plan or size");
  XNN_REQUIRE(n_tokens >= 0 && n_heads >= 1 && head_dim >= 1, "sizes out of range");
  const int splits = attention_splits(attention_blocks(plan, n_heads), plan->max_atoms);
  *bytes = forward_bytes(n_tokens, n_heads, head_dim, splits);
  return XNN_OK;
}

int xnn_attention(int dtype, const xnn_heads* q, const xnn_heads* k, const xnn_heads* v,
                  int64_t n_tokens, int32_t head_dim, const xnn_attention_tiles* plan,
                  const uint8_t* mask, float scale, void* out, float* lse, void* work,
                  size_t work_bytes, xnn_stream_t stream) {
  AttentionArgs a;
  int rows = 0;
  const int status = attention_args(a, dtype, q, k, v, n_tokens, head_dim, plan, mask, scale, rows);
  if (status != XNN_OK || n_tokens == 0) return status;
  XNN_REQUIRE(out != nullptr, "NULL output");
  a.splits = attention_splits(attention_blocks(plan, a.heads), plan->max_atoms);
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
  hipStream_t s = as_hip(stream);
  XNN_STORAGE_DISPATCH(dtype, T, {
    if (head_dim <= 16)
      attention_launch<T, 16>(a, rows, s);
    else if (head_dim <= 32)
      attention_launch<T, 32>(a, rows, s);
    else if (head_dim <= 64)
      attention_launch<T, 64>(a, rows, s);
    else
      attention_launch<T, 128>(a, rows, s);
  });
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

}  // extern "C"
