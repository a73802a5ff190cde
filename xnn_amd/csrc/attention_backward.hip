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

template <typename T, int DP, int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void attention_dq_kernel(AttentionArgs a) {
  typedef Head<T, DP> S;
  constexpr int kTile = 64;
  __shared__ __align__(16) char k_tile[kTile * S::kRow];
  __shared__ __align__(16) char v_tile[kTile * S::kRow];
  Tile t;
  if (!block_tile(a, a.heads, t)) return;
  const int lane = threadIdx.x & (kWave - 1), half = lane / 32;
  const int64_t row = t.first + kOwn * wave_in_block() + lane % 32;
  const bool live = row < t.end;
  const int64_t kv = t.head / (a.heads / a.kv_heads);
  const T* k = (const T*)a.k + kv * a.k_head;
  const T* v = (const T*)a.v + kv * a.v_head;
  typename Mma<T>::Frag q[S::kSteps], g[S::kSteps];
  load_own<T, DP>((const T*)a.q + t.head * a.q_head, a.q_token, row, live, a.D, a.vec, half, q);
  const int64_t out_stride = (int64_t)a.heads * a.D;
  load_own<T, DP>((const T*)a.grad + (int64_t)t.head * a.D, out_stride, row, live, a.D, a.vec_out, half, g);
  // d_i by the products that form g_i . v_j, out_i in the place of v_j: where one key has all the
  // weight the two are the same bits and its gradient is exactly zero. The wave's 32 x 32 tile of
  // out . g holds the rows' own products on its diagonal.
  float delta = 0.0f;
  {
    typename Mma<T>::Frag o[S::kSteps];
    load_own<T, DP>((const T*)a.out + (int64_t)t.head * a.D, out_stride, row, live, a.D, a.vec_out, half, o);
    f32x16 all = {};
#pragma unroll
    for (int c = 0; c < S::kSteps; ++c) Mma<T>::mma(o[c], g[c], all);
#pragma unroll
    for (int r = 0; r < 16; ++r) delta = tile_row(r, half) == lane % 32 ? all[r] : delta;
    const float other = __shfl_xor(delta, 32);
    delta = ((lane >> 2) & 1) == half ? delta : other;
  }
  float lse = live ? a.lse[(int64_t)t.head * a.n_tokens + row] : -INFINITY;
  const bool empty = lse == -INFINITY;
  if (empty) lse = INFINITY;                               // every probability of the row is zero
  if (live && half == 0) a.delta[(int64_t)t.head * a.n_tokens + row] = delta;
  f32x16 dq[S::kBlocks] = {};
  const float scale = a.scale * kLog2e;
  scale_own<T, DP>(scale, q);
  for (int64_t j0 = t.begin; j0 < t.end; j0 += kTile) {
    __syncthreads();
    stage<T, DP, kTile, WAVES * kWave>(k, a.k_token, j0, t.end, a.D, a.vec, a.mask, k_tile);
    stage<T, DP, kTile, WAVES * kWave>(v, a.v_token, j0, t.end, a.D, a.vec, a.mask, v_tile);
    const uint64_t keep = live_rows(j0, t.end, a.mask, lane);
    __syncthreads();
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      f32x16 p = {}, dp = {};
#pragma unroll
      for (int c = 0; c < S::kSteps; ++c) {
        Mma<T>::mma(natural_frag<T, DP>(k_tile, 32 * b + lane % 32, c, half), q[c], p);
        Mma<T>::mma(natural_frag<T, DP>(v_tile, 32 * b + lane % 32, c, half), g[c], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r)
        p[r] = weight<T>(p[r], scale, lse) * (dp[r] - delta);
      if (keep != ~0ull) {
        const uint64_t mine = keep >> (32 * b + 4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] = (mine >> tile_row(r, 0)) & 1 ? p[r] : 0.0f;
      }
#pragma unroll
      for (int f = 0; f < S::kFrags; ++f) {
        const typename Mma<T>::Frag w = weight_frag<T>(p, f);
#pragma unroll
        for (int d = 0; d < S::kBlocks; ++d)
          Mma<T>::mma(transposed_frag<T, DP>(k_tile, 32 * b, d, f, lane), w, dq[d]);
      }
    }
  }
  if (!live) return;
  if (empty) {
#pragma unroll
    for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) dq[d][r] = 0.0f;
  }
  store_own<T, DP>((T*)a.dq + (row * a.heads + t.head) * a.D, dq, a.scale, a.D, a.vec_out, half);
}

template <typename T, int DP, int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void attention_dkv_kernel(AttentionArgs a) {
  typedef Head<T, DP> S;
  constexpr int kTile = 64;                                // query rows of a staged tile
  __shared__ __align__(16) char q_tile[kTile * S::kRow];
  __shared__ __align__(16) char g_tile[kTile * S::kRow];
  __shared__ __align__(16) float lse_tile[kTile], delta_tile[kTile];
  Tile t;
  if (!block_tile(a, a.kv_heads, t)) return;
  const int lane = threadIdx.x & (kWave - 1), half = lane / 32;
  const int64_t key = t.first + kOwn * wave_in_block() + lane % 32;
  const bool live = key < t.end;
  const bool kept = live && (a.mask == nullptr || a.mask[key] != 0);
  typename Mma<T>::Frag k[S::kSteps], v[S::kSteps];
  load_own<T, DP>((const T*)a.k + t.head * a.k_head, a.k_token, key, kept, a.D, a.vec, half, k);
  load_own<T, DP>((const T*)a.v + t.head * a.v_head, a.v_token, key, kept, a.D, a.vec, half, v);
  f32x16 dk[S::kBlocks] = {}, dv[S::kBlocks] = {};
  const float scale = a.scale * kLog2e;
  scale_own<T, DP>(scale, k);
  const int group = a.heads / a.kv_heads;
  const int64_t out_stride = (int64_t)a.heads * a.D;
  for (int h = t.head * group; h < (t.head + 1) * group; ++h) {
    const T* q = (const T*)a.q + h * a.q_head;
    const T* g = (const T*)a.grad + (int64_t)h * a.D;
    for (int64_t i0 = t.begin; i0 < t.end; i0 += kTile) {
      __syncthreads();
      stage<T, DP, kTile, WAVES * kWave>(q, a.q_token, i0, t.end, a.D, a.vec, nullptr, q_tile);
      stage<T, DP, kTile, WAVES * kWave>(g, out_stride, i0, t.end, a.D, a.vec_out, nullptr, g_tile);
      if (threadIdx.x < kTile) {
        const int64_t i = i0 + threadIdx.x;
        const float l = i < t.end ? a.lse[(int64_t)h * a.n_tokens + i] : -INFINITY;
        lse_tile[threadIdx.x] = l == -INFINITY ? INFINITY : l;
        delta_tile[threadIdx.x] = i < t.end ? a.delta[(int64_t)h * a.n_tokens + i] : 0.0f;
      }
      __syncthreads();
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        f32x16 p = {}, dp = {};
#pragma unroll
        for (int c = 0; c < S::kSteps; ++c) {
          Mma<T>::mma(natural_frag<T, DP>(q_tile, 32 * b + lane % 32, c, half), k[c], p);
          Mma<T>::mma(natural_frag<T, DP>(g_tile, 32 * b + lane % 32, c, half), v[c], dp);
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
#pragma unroll
        for (int f = 0; f < S::kFrags; ++f) {
          const typename Mma<T>::Frag w = weight_frag<T>(p, f), dw = weight_frag<T>(dp, f);
#pragma unroll
          for (int d = 0; d < S::kBlocks; ++d) {
            Mma<T>::mma(transposed_frag<T, DP>(g_tile, 32 * b, d, f, lane), w, dv[d]);
            Mma<T>::mma(transposed_frag<T, DP>(q_tile, 32 * b, d, f, lane), dw, dk[d]);
          }
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
  store_own<T, DP>((T*)a.dk + at, dk, a.scale, a.D, a.vec_out, half);
  store_own<T, DP>((T*)a.dv + at, dv, 1.0f, a.D, a.vec_out, half);
}

template <typename T, int DP>
static void attention_backward_launch(const AttentionArgs& a, int rows, hipStream_t s) {
  const dim3 q_grid((unsigned)xcd_blocks(a.n_tiles * a.heads));
  const dim3 k_grid((unsigned)xcd_blocks(a.n_tiles * a.kv_heads));
  if (rows == 64) {
    hipLaunchKernelGGL((attention_dq_kernel<T, DP, 2>), q_grid, dim3(128), 0, s, a);
    hipLaunchKernelGGL((attention_dkv_kernel<T, DP, 2>), k_grid, dim3(128), 0, s, a);
  } else {
    hipLaunchKernelGGL((attention_dq_kernel<T, DP, 4>), q_grid, dim3(256), 0, s, a);
    hipLaunchKernelGGL((attention_dkv_kernel<T, DP, 4>), k_grid, dim3(256), 0, s, a);
  }
}

}  // namespace xnn

using namespace xnn;

extern "C" {

int xnn_attention_backward_work_size(int64_t n_tokens, int32_t n_heads, size_t* bytes) {
  XNN_REQUIRE(n_tokens >= 0 && n_heads >= 1, "sizes out of range");
  XNN_REQUIRE(bytes != nullptr, "NULL size");
  *bytes = sizeof(float) * (size_t)n_tokens * (size_t)n_heads;
  return XNN_OK;
}

int xnn_attention_backward(int dtype, const xnn_heads* q, const xnn_heads* k, const xnn_heads* v,
                           int64_t n_tokens, int32_t head_dim, const xnn_attention_tiles* plan,
                           const uint8_t* mask, float scale, const void* out, const float* lse,
                           const void* grad, void* dq, void* dk, void* dv, void* work,
                           size_t work_bytes, xnn_stream_t stream) {
  AttentionArgs a;
  int rows = 0;
  const int status = attention_args(a, dtype, q, k, v, n_tokens, head_dim, plan, mask, scale, rows);
  if (status != XNN_OK || n_tokens == 0) return status;
  XNN_REQUIRE(out && lse && grad && dq && dk && dv && work, "NULL input, output or work");
  XNN_REQUIRE(work_bytes >= sizeof(float) * (size_t)n_tokens * (size_t)q->n_heads, "work too small");
  a.out = out;
  a.lse = const_cast<float*>(lse);
  a.grad = grad;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.delta = (float*)work;
  a.vec_out = head_dim % (16 / storage_bytes(dtype)) == 0 &&
              ((uintptr_t)out | (uintptr_t)grad | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) % 16 == 0;
  hipStream_t s = as_hip(stream);
  XNN_STORAGE_DISPATCH(dtype, T, {
    if (head_dim <= 16)
      attention_backward_launch<T, 16>(a, rows, s);
    else if (head_dim <= 32)
      attention_backward_launch<T, 32>(a, rows, s);
    else if (head_dim <= 64)
      attention_backward_launch<T, 64>(a, rows, s);
    else
      attention_backward_launch<T, 128>(a, rows, s);
  });
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

}  // extern "C"
