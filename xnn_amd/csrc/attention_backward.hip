// The backward pass of attention within structures (gfx950, wave64): the probabilities are formed
// again from the scores and the rows' base-2 logarithms L that the forward pass left.
//
//   p_ij = exp2(scale log2(e) q_i . k_j - L_i),  ds_ij = p_ij (g_i . v_j - d_i),  d_i = g_i . out_i
//   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i,   dv_j = sum_i p_ij g_i
//
// Two kernels, no atomics: one owns query rows and walks the keys (d_i and dq), one owns
// keys and walks the query rows of every head that shares them (dk and dv). The second formation of
// the scores costs two of seven products; in exchange every sum has one owner and a fixed order.
// A masked key gets zeros, a row without keys gives zeros, whatever such rows hold.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "attention.h"
#include "common.h"

namespace xnn {

// Queries' gradients: three products, with q, g and dq of the wave's rows in registers. Bounded as the
// forward pass is, by vector and matrix instructions in turn.
//   24,000 rows, 4 heads of 64, bfloat16: 984 us, 900 TFLOP/s, and 10 us of the sum over two parts
//   9,000 rows, 4 heads of 32, float32: 354 us and 5, 176 TFLOP/s
//   1,024 structures of 10-60 rows, 4 heads of 16, float32: 26 us
template <typename T, int DP, int WAVES, int TILE, bool VEC, int WP>
__global__ __launch_bounds__(WAVES* kWave, (Head<T, DP>::kOccupancy)) void attention_dq_kernel(AttentionArgs a) {
  typedef Head<T, DP, TILE> S;
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
  Operand<T> q[S::kSteps], g[S::kSteps];
  const int64_t out_stride = (int64_t)a.heads * a.D, at_head = (int64_t)t.head * a.D;
  load_own<T, DP, VEC>((const T*)a.q + t.head * a.q_head, a.q_token, row, live, a.D, half, scale, q);
  load_own<T, DP, VEC>((const T*)a.grad + at_head, out_stride, row, live, a.D, half, 1.0f, g);
  // d_i by the products that form g_i . v_j, out_i in the place of v_j: where one key has all the
  // weight the two are the same bits and its gradient is exactly zero. The wave's 32 x 32 tile of
  // out . g holds the rows' own products on its diagonal.
  float delta = 0.0f;
  {
    Operand<T> o[S::kSteps];
    load_own<T, DP, VEC>((const T*)a.out + at_head, out_stride, row, live, a.D, half, 1.0f, o);
    f32x16 all = {};
#pragma unroll
    for (int c = 0; c < S::kSteps; ++c) mma<T>(o[c], g[c], all);
#pragma unroll
    for (int r = 0; r < 16; ++r) delta = tile_row(r, half) == lane % 32 ? all[r] : delta;
    const float other = __shfl_xor(delta, 32);
    delta = ((lane >> 2) & 1) == half ? delta : other;
  }
  float lse = live ? a.lse[(int64_t)t.head * a.n_tokens + row] : -INFINITY;
  const bool empty = lse == -INFINITY;
  const int carry = carried<T>(t.end - t.begin);
  const float factor = ldexpf(a.scale, -carry);
  lse -= (float)carry;
  if (empty) lse = INFINITY;                               // every probability of the row is zero
  // Where the row's keys are one product, d_i = sum_j p_ij g_i . v_j from the registers: what the stored out
  // lost in its rounding, much beside the differences of two or three keys, is not in it.
  const bool single = t.end - t.begin <= 32;
  f32x16 dq[S::kBlocks] = {};
  GradientRange<T> range;
  for (int64_t j0 = from; j0 < to; j0 += S::kTile) {
    __syncthreads();
    const uint64_t keep = __ballot(next_keep != 0);
    next_k.commit(k_tile, a.D, keep);
    next_v.commit(v_tile, a.D, keep);
    __syncthreads();
    if (j0 + S::kTile < to) fetch(j0 + S::kTile);
    if (!busy || keep == 0) continue;
#pragma unroll
    for (int b = 0; b < S::kTile / 32; ++b) {
      f32x16 p = {}, dp = {};
#pragma unroll
      for (int c = 0; c < S::kSteps; ++c) {
        mma<T>(natural_operand<T, S>(k_tile, 32 * b + lane % 32, c, half), q[c], p);
        mma<T>(natural_operand<T, S>(v_tile, 32 * b + lane % 32, c, half), g[c], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) p[r] = weight<T>(p[r], scale, lse);
      if (keep != (~0ull >> (64 - S::kTile))) {            // the left out keys' g . v is zero
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] = has_row((uint32_t)(keep >> (32 * b)), r) ? p[r] : 0.0f;
      }
      if (single && b == 0) {
        delta = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) delta = fmaf(p[r], dp[r], delta);
        delta = add_xor32(delta);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) p[r] *= dp[r] - delta;
      range.hold(p, dq);
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const auto w = weight_operand<T, WP>(p, f);
#pragma unroll
        for (int d = 0; d < S::kBlocks; ++d)
          mma<T>(transposed_operand<T, S>(k_tile, 32 * b, d, f, lane), w, dq[d]);
      }
    }
  }
  if (!live) return;
  if (half == 0 && (single ? from < to : t.split == 0)) a.delta[(int64_t)t.head * a.n_tokens + row] = delta;
  if (empty) {
#pragma unroll
    for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) dq[d][r] = 0.0f;
  }
  const int64_t at = (row * a.heads + t.head) * a.D;
  if (a.splits > 1)
    store_own(a.part + (int64_t)t.split * a.n_tokens * a.heads * a.D + at, dq, factor * range.back(), a.D,
              a.D % 4 == 0, half);
  else
    store_own((T*)a.dq + at, dq, factor * range.back(), a.D, a.vec_out, half);
}

// Keys' and values' gradients: four products, with k, v, dk and dv of the wave's rows in registers.
// Bounded as the forward pass is; float32 heads of 97 to 128 also by 260 bytes a lane that do not fit
// the registers of one wave a SIMD.
//   24,000 rows, 4 heads of 64, bfloat16: 1,283 us, 920 TFLOP/s, and 18 us of the sums over two parts
//   9,000 rows, 4 heads of 32, float32: 464 us and 10, 179 TFLOP/s
//   1,024 structures of 10-60 rows, 4 heads of 16, float32: 27 us
template <typename T, int DP, int WAVES, int TILE, bool VEC, int WP>
__global__ __launch_bounds__(WAVES* kWave, (Head<T, DP>::kOccupancy)) void attention_dkv_kernel(AttentionArgs a) {
  typedef Head<T, DP, TILE> S;
  __shared__ __align__(16) char q_tile[S::kBytes];
  __shared__ __align__(16) char g_tile[S::kBytes];
  __shared__ __align__(16) float lse_tile[S::kTile], delta_tile[S::kTile];
  Tile t;
  block_tile(a, a.kv_heads, t);
  const int lane = threadIdx.x & (kWave - 1), half = lane / 32;
  const int64_t key = t.first + kOwn * wave_in_block() + lane % 32;
  const bool live = key < t.end;
  const bool busy = t.first + kOwn * wave_in_block() < t.end;   // the wave has keys
  const bool kept = live && (a.mask == nullptr || a.mask[key] != 0);
  const float scale = a.scale * kLog2e;
  const int group = a.heads / a.kv_heads;
  const int64_t out_stride = (int64_t)a.heads * a.D;
  const int carry = carried<T>(t.end - t.begin);
  // the walk: the rows of every head that shares these keys
  const int64_t per = (t.end - t.begin + S::kTile - 1) / S::kTile;
  int64_t from, to;
  walk_part(per * group, a, t.split, from, to);
  Stage<T, S, WAVES * kWave, VEC> next_q, next_g;
  float next_lse = 0.0f, next_delta = 0.0f;
  uint64_t next_keep = 0;
  next_q.init(a.q_token, a.D);
  next_g.init(out_stride, a.D);
  const auto fetch = [&](int64_t n) {
    const int h = t.head * group + (int)(n / per);
    const int64_t i0 = t.begin + n % per * S::kTile;
    next_keep = rows_before<S::kTile>(t.end - i0);
    next_q.fetch((const T*)a.q + h * a.q_head + i0 * a.q_token, a.q_token, t.end - i0, a.D);
    next_g.fetch((const T*)a.grad + (int64_t)h * a.D + i0 * out_stride, out_stride, t.end - i0, a.D);
    const int64_t i = i0 + threadIdx.x;
    if (threadIdx.x < S::kTile) {
      next_lse = i < t.end ? a.lse[(int64_t)h * a.n_tokens + i] : -INFINITY;
      next_delta = i < t.end ? a.delta[(int64_t)h * a.n_tokens + i] : 0.0f;
    }
  };
  if (from < to) fetch(from);
  Operand<T> k[S::kSteps], v[S::kSteps];
  load_own<T, DP, VEC>((const T*)a.k + t.head * a.k_head, a.k_token, key, kept, a.D, half, scale, k);
  load_own<T, DP, VEC>((const T*)a.v + t.head * a.v_head, a.v_token, key, kept, a.D, half, 1.0f, v);
  f32x16 dk[S::kBlocks] = {}, dv[S::kBlocks] = {};
  GradientRange<T> range;
  for (int64_t n = from; n < to; ++n) {
    __syncthreads();
    next_q.commit(q_tile, a.D, next_keep);
    next_g.commit(g_tile, a.D, next_keep);
    if (threadIdx.x < S::kTile) {
      // a row beyond the structure or without keys: every probability is zero
      lse_tile[threadIdx.x] = next_lse == -INFINITY ? INFINITY : next_lse - (float)carry;
      delta_tile[threadIdx.x] = next_delta;
    }
    __syncthreads();
    if (n + 1 < to) fetch(n + 1);
    if (!busy) continue;
#pragma unroll
    for (int b = 0; b < S::kTile / 32; ++b) {
      f32x16 p = {}, dp = {};
#pragma unroll
      for (int c = 0; c < S::kSteps; ++c) {
        mma<T>(natural_operand<T, S>(q_tile, 32 * b + lane % 32, c, half), k[c], p);
        mma<T>(natural_operand<T, S>(g_tile, 32 * b + lane % 32, c, half), v[c], dp);
      }
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const f32x4 l = *(const f32x4*)(lse_tile + 32 * b + 8 * q4 + 4 * half);
        const f32x4 d = *(const f32x4*)(delta_tile + 32 * b + 8 * q4 + 4 * half);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 4 * q4 + j;
          p[r] = weight<T>(p[r], scale, l[j]);
          dp[r] = p[r] * (dp[r] - d[j]);
        }
      }
      range.hold(dp, dk);
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const auto w = weight_operand<T, WP>(p, f);
        const auto dw = weight_operand<T, WP>(dp, f);
#pragma unroll
        for (int d = 0; d < S::kBlocks; ++d) {
          mma<T>(transposed_operand<T, S>(g_tile, 32 * b, d, f, lane), w, dv[d]);
          mma<T>(transposed_operand<T, S>(q_tile, 32 * b, d, f, lane), dw, dk[d]);
        }
      }
    }
  }
  if (!live) return;
  if (!kept) {
#pragma unroll
    for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) dk[d][r] = dv[d][r] = 0.0f;
  }
  const int64_t at = (key * a.kv_heads + t.head) * a.D;
  const float k_factor = ldexpf(a.scale, -carry) * range.back(), v_factor = ldexpf(1.0f, -carry);
  if (a.splits > 1) {
    const int64_t one = a.n_tokens * a.kv_heads * a.D;
    store_own(a.part + t.split * one + at, dk, k_factor, a.D, a.D % 4 == 0, half);
    store_own(a.part + (a.splits + t.split) * one + at, dv, v_factor, a.D, a.D % 4 == 0, half);
  } else {
    store_own((T*)a.dk + at, dk, k_factor, a.D, a.vec_out, half);
    store_own((T*)a.dv + at, dv, v_factor, a.D, a.vec_out, half);
  }
}

// out[i] = sum over the parts in order, N elements a thread; blockIdx.y: the first or the second of
// two gradients, whose parts follow each other. A stream: 24,000 x 256 in two parts 10 us a gradient, 6 TB/s
// (part of it from the last-level cache).
template <typename T, int N>
__global__ __launch_bounds__(256) void attention_sum_kernel(const float* __restrict__ part, int64_t n,
                                                            int splits, T* __restrict__ a,
                                                            T* __restrict__ b) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * N;
  if (i >= n) return;
  part += (int64_t)blockIdx.y * splits * n;
  float sum[N] = {};
  for (int s = 0; s < splits; ++s) {
    float x[N];
    load_pack<float, N>(part + s * n + i, x);
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] += x[j];
  }
  store_pack<T, N>((blockIdx.y == 0 ? a : b) + i, sum);
}

template <typename T>
static void attention_sum(const AttentionArgs& a, int64_t n, void* x, void* y, hipStream_t s) {
  const unsigned both = y == nullptr ? 1 : 2;
  if (a.vec_out)
    hipLaunchKernelGGL((attention_sum_kernel<T, 4>), dim3((unsigned)((n / 4 + 255) / 256), both),
                       dim3(256), 0, s, a.part, n, a.splits, (T*)x, (T*)y);
  else
    hipLaunchKernelGGL((attention_sum_kernel<T, 1>), dim3((unsigned)((n + 255) / 256), both),
                       dim3(256), 0, s, a.part, n, a.splits, (T*)x, (T*)y);
}

template <typename T, int DP>
static void attention_backward_launch(AttentionArgs a, int rows, bool fine_query, bool fine, int q_splits,
                                      int k_splits, hipStream_t s) {
  const dim3 q_grid((unsigned)(a.n_tiles * a.heads * q_splits));
  const dim3 k_grid((unsigned)(a.n_tiles * a.kv_heads * k_splits));
  a.splits = q_splits;
  XNN_ATTENTION_LAUNCH(attention_dq_kernel, q_grid, fine_query);
  if (q_splits > 1) attention_sum<T>(a, a.n_tokens * a.heads * a.D, a.dq, nullptr, s);
  a.splits = k_splits;
  XNN_ATTENTION_LAUNCH(attention_dkv_kernel, k_grid, fine);
  if (k_splits > 1) attention_sum<T>(a, a.n_tokens * a.kv_heads * a.D, a.dk, a.dv, s);
}

// parts of the queries' gradient, which walks keys, and of the keys' and values', which walks the rows of
// every head that shares them; short structures, whose blocks are of one wave, are walked whole
static void part_counts(const xnn_attention_tiles* plan, int heads, int kv_heads, int dtype, int D, int& q,
                        int& k) {
  q = k = 1;
  if (attention_rows(plan, storage_bytes(dtype), D) == 32) return;
  const int64_t rows = split_rows(dtype, D);
  q = backward_splits(attention_blocks(plan, heads), plan->max_atoms, rows);
  k = backward_splits(attention_blocks(plan, kv_heads), plan->max_atoms * (heads / kv_heads), rows);
}

// the rows' dot products, then the parts of the queries' gradients and after those the parts of the
// keys' and values' (one after the other in the same place)
static int64_t delta_floats(int64_t n_tokens, int heads) { return (n_tokens * heads + 3) / 4 * 4; }

static size_t backward_bytes(int64_t n_tokens, int heads, int kv_heads, int D, int q_splits,
                             int k_splits) {
  const int64_t q = q_splits == 1 ? 0 : (int64_t)q_splits * heads;
  const int64_t k = k_splits == 1 ? 0 : (int64_t)2 * k_splits * kv_heads;
  return sizeof(float) * (size_t)(delta_floats(n_tokens, heads) + std::max(q, k) * n_tokens * D);
}

}  // namespace xnn

using namespace xnn;

extern "C" {

int xnn_attention_backward_work_size(int dtype, int64_t n_tokens, int32_t n_heads,
                                     int32_t n_kv_heads, int32_t head_dim, const xnn_attention_tiles* plan,
                                     size_t* bytes) {
  XNN_REQUIRE(is_storage(dtype), "dtype must be XNN_F32, XNN_BF16 or XNN_F16");
  XNN_REQUIRE(plan && bytes, "NULL plan or size");
  XNN_REQUIRE(n_tokens >= 0 && n_heads >= 1 && n_kv_heads >= 1 && n_heads % n_kv_heads == 0 &&
                  head_dim >= 1,
              "sizes out of range");
  int q, k;
  part_counts(plan, n_heads, n_kv_heads, dtype, head_dim, q, k);
  *bytes = backward_bytes(n_tokens, n_heads, n_kv_heads, head_dim, q, k);
  return XNN_OK;
}

int xnn_attention_backward(int dtype, const xnn_heads* q, const xnn_heads* k, const xnn_heads* v,
                           int64_t n_tokens, int32_t head_dim, const xnn_attention_tiles* plan,
                           const uint8_t* mask, float scale, const void* out, const float* lse,
                           const void* grad, void* dq, void* dk, void* dv, void* work,
                           size_t work_bytes, xnn_stream_t stream) {
  AttentionArgs a;
  const int status = attention_args(a, dtype, q, k, v, n_tokens, head_dim, plan, mask, scale);
  if (status != XNN_OK || n_tokens == 0) return status;
  XNN_REQUIRE(out && lse && grad && dq && dk && dv && work, "NULL input, output or work");
  int q_splits, k_splits;
  part_counts(plan, a.heads, a.kv_heads, dtype, head_dim, q_splits, k_splits);
  XNN_REQUIRE(work_bytes >= backward_bytes(n_tokens, a.heads, a.kv_heads, head_dim, q_splits, k_splits),
              "work too small");
  XNN_REQUIRE((uintptr_t)work % 16 == 0, "work must be aligned to 16 bytes");
  a.out = out;
  a.lse = const_cast<float*>(lse);
  a.grad = grad;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.delta = (float*)work;
  a.part = a.delta + delta_floats(n_tokens, a.heads);
  a.vec_out = head_dim % (16 / storage_bytes(dtype)) == 0 &&
              ((uintptr_t)out | (uintptr_t)grad | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) % 16 == 0;
  a.vec = a.vec && a.vec_out;
  const int rows = attention_pick(a, plan, dtype);
  const bool fine = fine_weights(a, plan), fine_query = fine_query_gradient(a, plan);
  hipStream_t s = as_hip(stream);
  XNN_STORAGE_DISPATCH(dtype, T, {
    if (head_dim <= 16)
      attention_backward_launch<T, 16>(a, rows, fine_query, fine, q_splits, k_splits, s);
    else if (head_dim <= 32)
      attention_backward_launch<T, 32>(a, rows, fine_query, fine, q_splits, k_splits, s);
    else if (head_dim <= 64)
      attention_backward_launch<T, 64>(a, rows, fine_query, fine, q_splits, k_splits, s);
    else if (head_dim <= 96)
      attention_backward_launch<T, 96>(a, rows, fine_query, fine, q_splits, k_splits, s);
    else
      attention_backward_launch<T, 128>(a, rows, fine_query, fine, q_splits, k_splits, s);
  });
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

}  // extern "C"
