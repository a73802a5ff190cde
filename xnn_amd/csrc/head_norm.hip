// Norms of queries and keys for each head with the rotation in the same pass, and the backward
// pass (gfx950, wave64).
//
//   n = x / sqrt(mean_d x^2 + eps),  u = w n,  (a, b) -> (a c - b s, a s + b c)
//
// over the D elements of one head of one token; the first R elements form R / 2 pairs (i, i + R/2)
// or (2 i, 2 i + 1) turned by the angle whose cosine and sine are row `positions[t]` (or t) of the
// tables, the other elements are not turned. Backward, with g the cotangent turned back:
//
//   dx = r (w g - n mean_d(w g n)),  dw = sum_{t, heads} g n,
//   dc = sum_heads (ga a + gb b),    ds = sum_heads (gb a - ga b)
//
// A stream over queries and keys in one launch: a head lies in the registers of G lanes, 2 N
// elements a lane in two accesses of N (both members of a pair in one lane), so the sums over
// d are exchanges within G lanes and the sums over heads exchanges across the lanes of the token.
// All arithmetic is float32 and every sum has a fixed order.
//
// Measured, 24,000 tokens of 16 + 4 heads of 128 in bfloat16: forward 44 us for the
// 246 MB it reads and writes, the rate of a large copy, which bounds it; backward 80 us for 369 MB, 4.6 TB/s,
// where loads wait on the two sums of a head before the next head's are issued (asking for the next head's
// loads first: 196 us against 100, for the registers). 9,000 tokens of 4 + 4 heads of 32 in float32: 5.9
// and 10.4 us, the launch and two loads in a row, the tables' and the heads'.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.h"
#include "device.h"
#include "storage.h"

namespace xnn {

constexpr int kNormBlocks = 1280;  // blocks of the backward pass, at most: five a CU, as many as it holds

struct HeadArgs {
  const void *q, *k, *gq, *gk, *wq, *wk;
  int64_t q_token, q_head, k_token, k_head;
  int64_t n_tokens, n_rows;
  const int64_t* positions;
  const float *cos, *sin;
  int heads, kv_heads, D, R;
  int lanes, parallel;             // lanes of a head, heads a token has in flight
  float eps, inv_d;
  void *q_out, *k_out;
  float *d_cos, *d_sin, *part;
};

template <int N>
struct Unit {                      // the 2 N elements of one lane
  float a[N], b[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_unit(const T* p, int o0, int o1, int D, Unit<N>& x) {
  load_pack<T, N>(p + o0, x.a);
  if (o1 < D) {
    load_pack<T, N>(p + o1, x.b);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) x.b[j] = 0.0f;
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_unit(T* p, int o0, int o1, int D, const Unit<N>& x) {
  store_pack<T, N>(p + o0, x.a);
  if (o1 < D) store_pack<T, N>(p + o1, x.b);
}

// member `m` of pair `p` of a unit's elements
template <int N, bool INTER>
__device__ __forceinline__ float& member(Unit<N>& x, int p, int m) {
  if (!INTER || N == 1) return m == 0 ? x.a[p] : x.b[p];
  const int e = 2 * p + m;
  return e < N ? x.a[e] : x.b[e - N];
}

// the sum over the `lanes` (a power of two) lanes of a head, every lane getting it: within a row of sixteen by
// lane permutes of the vector unit, which leave the LDS unit to the weights (24,000 x 20 heads of 128: the
// backward pass 101 us with shuffles, 94 so)
__device__ __forceinline__ float lanes_sum(float x, int lanes) {
  if (lanes > 1) x += dpp_move<0xB1>(x);                   // neighbours
  if (lanes > 2) x += dpp_move<0x4E>(x);                   // pairs
  if (lanes > 4) x += dpp_move<0x141>(x);                  // the half row mirrored
  if (lanes > 8) x += dpp_move<0x140>(x);                  // the row mirrored
  if (lanes > 16) x = add_xor16(x);
  if (lanes > 32) x = add_xor32(x);
  return x;
}

// x[j] += x[j] of lane ^ o for o = from, 2 from, ... below `to` (powers of two), in the vector unit:
// the backward pass of 9,000 tokens 10.4 us, by shuffles through the LDS unit 12.3
template <int N>
__device__ __forceinline__ void add_lanes(float (&x)[N], int from, int to) {
#define XNN_ADD_LANES(O, SUM)                   \
  if (from <= O && O < to) {                    \
    _Pragma("unroll") for (int j = 0; j < N; ++j) x[j] = SUM; \
  }
  XNN_ADD_LANES(1, x[j] + dpp_move<0xB1>(x[j]))
  XNN_ADD_LANES(2, x[j] + dpp_move<0x4E>(x[j]))
  XNN_ADD_LANES(4, x[j] + dpp_move<0x1B>(dpp_move<0x141>(x[j])))   // the half row mirrored, its quads turned back
  XNN_ADD_LANES(8, x[j] + dpp_move<0x128>(x[j]))                   // the row turned by half
  XNN_ADD_LANES(16, add_xor16(x[j]))
  XNN_ADD_LANES(32, add_xor32(x[j]))
#undef XNN_ADD_LANES
}

template <typename T, int N, bool INTER, bool BACK>
__global__ __launch_bounds__(256, BACK ? 5 : 4) void head_norm_kernel(HeadArgs h) {
  const int lane = threadIdx.x & (kWave - 1), wave = wave_in_block();
  const int per_token = h.lanes * h.parallel, tokens = kWave / per_token;
  const int u = lane % h.lanes, slot = (lane / h.lanes) % h.parallel;
  const int all = h.heads + h.kv_heads, D = h.D;
  const int o0 = INTER || 2 * u * N >= h.R ? 2 * u * N : u * N;
  const int o1 = INTER || 2 * u * N >= h.R ? o0 + N : h.R / 2 + u * N;
  const bool mine = 2 * u * N < D, turned = 2 * u * N < h.R;
  // the weights lie in LDS: a wave more a SIMD than with them in registers
  __shared__ __align__(16) float weights[2][128];
  for (int i = threadIdx.x; i < 2 * 128; i += 256) {
    const int d = i % 128;
    weights[i / 128][d] = d < D ? (float)((const T*)(i < 128 ? h.wq : h.wk))[d] : 0.0f;
  }
  __syncthreads();
  Unit<N> dwq, dwk;
#pragma unroll
  for (int j = 0; j < N; ++j) dwq.a[j] = dwq.b[j] = dwk.a[j] = dwk.b[j] = 0.0f;
  const int w0 = mine ? o0 : 0, w1 = mine && o1 < D ? o1 : 0;
  const int64_t step = (int64_t)gridDim.x * 4 * tokens;
  for (int64_t t0 = ((int64_t)blockIdx.x * 4 + wave) * tokens; t0 < h.n_tokens; t0 += step) {
    const int64_t t = t0 + lane / per_token;
    const bool live = mine && t < h.n_tokens;
    float c[N], s[N], dc[N], ds[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      c[j] = 1.0f;
      s[j] = dc[j] = ds[j] = 0.0f;
    }
    if (live && turned) {
      const int64_t row = h.positions != nullptr ? h.positions[t] : t;
      if (row >= 0 && row < h.n_rows) {
        load_pack<float, N>(h.cos + row * (h.R / 2) + u * N, c);
        load_pack<float, N>(h.sin + row * (h.R / 2) + u * N, s);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) c[j] = s[j] = __builtin_nanf("");
      }
    }
    // the token's queries and keys, in and out: 64-bit products once a token
    const T *q_in = (const T*)h.q + t * h.q_token, *k_in = (const T*)h.k + t * h.k_token;
    const int64_t q_at = t * h.heads * D, k_at = t * h.kv_heads * D;
    for (int i0 = 0; i0 < all; i0 += h.parallel) {
      const int i = i0 + slot;
      const bool on = live && i < all, is_q = i < h.heads;
      const int head = is_q ? i : i - h.heads;
      const int64_t at = (is_q ? q_at : k_at) + (int64_t)head * D;
      Unit<N> x;
#pragma unroll
      for (int j = 0; j < N; ++j) x.a[j] = x.b[j] = 0.0f;
      if (on)
        load_unit<T, N>(is_q ? q_in + head * h.q_head : k_in + head * h.k_head, o0, o1, D, x);
      Unit<N> g = x;
      if (BACK && on) load_unit<T, N>((const T*)(is_q ? h.gq : h.gk) + at, o0, o1, D, g);
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < N; ++j) sum += x.a[j] * x.a[j] + x.b[j] * x.b[j];
      const float r = rsqrtf(fmaf(lanes_sum(sum, h.lanes), h.inv_d, h.eps));
      Unit<N> w;
      load_pack<float, N>(weights[is_q ? 0 : 1] + w0, w.a);
      load_pack<float, N>(weights[is_q ? 0 : 1] + w1, w.b);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        x.a[j] *= r;                                       // x is n from here
        x.b[j] *= r;
      }
      if (!BACK) {
        Unit<N> y = x;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          y.a[j] *= w.a[j];
          y.b[j] *= w.b[j];
        }
        if (turned) {
#pragma unroll
          for (int p = 0; p < N; ++p) {
            const float a = member<N, INTER>(y, p, 0), b = member<N, INTER>(y, p, 1);
            member<N, INTER>(y, p, 0) = a * c[p] - b * s[p];
            member<N, INTER>(y, p, 1) = a * s[p] + b * c[p];
          }
        }
        if (on) store_unit<T, N>((T*)(is_q ? h.q_out : h.k_out) + at, o0, o1, D, y);
        continue;
      }
      if (turned && on) {
#pragma unroll
        for (int p = 0; p < N; ++p) {
          const float ga = member<N, INTER>(g, p, 0), gb = member<N, INTER>(g, p, 1);
          const float a = member<N, INTER>(x, p, 0) * member<N, INTER>(w, p, 0);
          const float b = member<N, INTER>(x, p, 1) * member<N, INTER>(w, p, 1);
          dc[p] += ga * a + gb * b;
          ds[p] += gb * a - ga * b;
          member<N, INTER>(g, p, 0) = ga * c[p] + gb * s[p];
          member<N, INTER>(g, p, 1) = gb * c[p] - ga * s[p];
        }
      }
      float dot = 0.0f;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float na = on ? g.a[j] * x.a[j] : 0.0f, nb = on ? g.b[j] * x.b[j] : 0.0f;
        dwq.a[j] += is_q ? na : 0.0f;
        dwq.b[j] += is_q ? nb : 0.0f;
        dwk.a[j] += is_q ? 0.0f : na;
        dwk.b[j] += is_q ? 0.0f : nb;
        dot += na * w.a[j] + nb * w.b[j];
      }
      dot = lanes_sum(dot, h.lanes) * h.inv_d;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        x.a[j] = r * (g.a[j] * w.a[j] - x.a[j] * dot);
        x.b[j] = r * (g.b[j] * w.b[j] - x.b[j] * dot);
      }
      if (on) store_unit<T, N>((T*)(is_q ? h.q_out : h.k_out) + at, o0, o1, D, x);
    }
    if (BACK && h.d_cos != nullptr) {
      add_lanes(dc, h.lanes, per_token);
      add_lanes(ds, h.lanes, per_token);
      if (live && turned && slot == 0) {
        store_pack<float, N>(h.d_cos + t * (h.R / 2) + u * N, dc);
        store_pack<float, N>(h.d_sin + t * (h.R / 2) + u * N, ds);
      }
    }
  }
  if (BACK && h.part != nullptr) {
    // the block's sums over tokens and heads: across the lanes of a wave, then its waves in order
    __shared__ float sums[4][2][128];
    add_lanes(dwq.a, h.lanes, kWave);
    add_lanes(dwq.b, h.lanes, kWave);
    add_lanes(dwk.a, h.lanes, kWave);
    add_lanes(dwk.b, h.lanes, kWave);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (mine && lane < h.lanes) {
        sums[wave][0][o0 + j] = dwq.a[j];
        sums[wave][1][o0 + j] = dwk.a[j];
        if (o1 < D) {
          sums[wave][0][o1 + j] = dwq.b[j];
          sums[wave][1][o1 + j] = dwk.b[j];
        }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += 256) {
      const int m = i / D, d = i - m * D;
      h.part[(int64_t)blockIdx.x * 2 * D + i] =
          (sums[0][m][d] + sums[1][m][d]) + (sums[2][m][d] + sums[3][m][d]);
    }
  }
}

// the blocks' weight sums added in float64: sixty-four of them at a time, then those in order; 5 us for
// 1,280 blocks of 2 x 128, bound by the latency of twenty loads in a row
template <typename T>
__global__ __launch_bounds__(1024) void head_weight_kernel(const float* __restrict__ part, int blocks,
                                                           int D, T* __restrict__ dwq,
                                                           T* __restrict__ dwk) {
  __shared__ double s[64][17];
  const int x = threadIdx.x % 16, y = threadIdx.x / 16;
  const int i = blockIdx.x * 16 + x;
  double v = 0.0;
  if (i < 2 * D)
#pragma unroll 4
    for (int b = y; b < blocks; b += 64) v += part[(int64_t)b * 2 * D + i];
  s[y][x] = v;
  __syncthreads();
  if (y == 0 && i < 2 * D) {
    double r = 0.0;
#pragma unroll
    for (int q = 0; q < 64; ++q) r += s[q][x];
    if (i < D)
      dwq[i] = (T)(float)r;
    else
      dwk[i - D] = (T)(float)r;
  }
}

static int pow2_at_least(int n) {
  int p = 1;
  while (p < n) p *= 2;
  return p;
}

// The widest access that the addresses, strides and pair layout allow, in the backward pass at most four
// elements (24,000 x 20 heads of 128 in bfloat16: 125 us with eight, whose registers leave two waves a
// SIMD, 85 with four and five waves); fills in the lanes.
template <typename T>
static int head_width(HeadArgs& h, bool back) {
  const uintptr_t at = (uintptr_t)h.q | (uintptr_t)h.k | (uintptr_t)h.wq | (uintptr_t)h.wk |
                       (uintptr_t)h.q_out | (uintptr_t)h.k_out |
                       (back ? (uintptr_t)h.gq | (uintptr_t)h.gk : 0);
  const uintptr_t tables = (uintptr_t)h.cos | (uintptr_t)h.sin | (uintptr_t)h.d_cos | (uintptr_t)h.d_sin;
  const int64_t strides = h.q_token | h.q_head | h.k_token | h.k_head;
  int n = back ? 4 : 16 / sizeof(T);
  while (n > 1 && (at % (n * sizeof(T)) != 0 || tables % 16 != 0 || strides % n != 0 ||
                   h.D % (2 * n) != 0 || h.R % (2 * n) != 0))
    n /= 2;
  h.lanes = pow2_at_least((h.D + 2 * n - 1) / (2 * n));
  h.parallel = std::min(kWave / h.lanes, pow2_at_least(h.heads + h.kv_heads));
  return n;
}

static int norm_blocks(const HeadArgs& h, int64_t most) {
  const int64_t per = 4 * (kWave / (h.lanes * h.parallel));
  return (int)std::min<int64_t>((h.n_tokens + per - 1) / per, most);
}

template <typename T, bool BACK>
static void head_norm_launch(const HeadArgs& h, int n, int inter, int blocks, hipStream_t s) {
#define XNN_HEAD_LAUNCH(N)                                                                         \
  do {                                                                                             \
    if (inter)                                                                                     \
      hipLaunchKernelGGL((head_norm_kernel<T, N, true, BACK>), dim3(blocks), dim3(256), 0, s, h);  \
    else                                                                                           \
      hipLaunchKernelGGL((head_norm_kernel<T, N, false, BACK>), dim3(blocks), dim3(256), 0, s, h); \
  } while (0)
  if constexpr (sizeof(T) == 2 && !BACK) {
    if (n == 8) {
      XNN_HEAD_LAUNCH(8);
      return;
    }
  }
  if (n == 4)
    XNN_HEAD_LAUNCH(4);
  else if (n == 2)
    XNN_HEAD_LAUNCH(2);
  else
    XNN_HEAD_LAUNCH(1);
#undef XNN_HEAD_LAUNCH
}

static size_t norm_work_bytes(int D) { return (size_t)kNormBlocks * 2 * D * sizeof(float); }

static int head_args(HeadArgs& h, const xnn_heads* q, const xnn_heads* k, int64_t n_tokens,
                     int32_t head_dim, int32_t rotated, const void* q_weight, const void* k_weight,
                     const float* cos, const float* sin, int64_t n_rows, const int64_t* positions,
                     float eps) {
  XNN_REQUIRE(q && k, "NULL heads");
  XNN_REQUIRE(n_tokens >= 0 && n_rows >= 0, "negative size");
  XNN_REQUIRE(q->n_heads >= 1 && k->n_heads >= 1, "no heads");
  XNN_REQUIRE(head_dim >= 1 && head_dim <= 128, "head_dim must be in [1, 128]");
  XNN_REQUIRE(rotated >= 0 && rotated <= head_dim && rotated % 2 == 0,
              "rotated must be even and at most head_dim");
  if (n_tokens > 0) {
    XNN_REQUIRE(positions != nullptr || rotated == 0 || n_rows == n_tokens,
                "without positions the tables have a row a token");
    XNN_REQUIRE(q->data && k->data && q_weight && k_weight, "NULL input");
    XNN_REQUIRE(rotated == 0 || n_rows == 0 || (cos && sin), "NULL table");
  }
  h = HeadArgs{};
  h.q = q->data;
  h.k = k->data;
  h.q_token = q->token_stride;
  h.q_head = q->head_stride;
  h.k_token = k->token_stride;
  h.k_head = k->head_stride;
  h.heads = q->n_heads;
  h.kv_heads = k->n_heads;
  h.n_tokens = n_tokens;
  h.n_rows = n_rows;
  h.positions = positions;
  h.cos = cos;
  h.sin = sin;
  h.D = head_dim;
  h.inv_d = 1.0f / (float)head_dim;
  h.R = rotated;
  h.wq = q_weight;
  h.wk = k_weight;
  h.eps = eps;
  return XNN_OK;
}

}  // namespace xnn

using namespace xnn;

extern "C" {

int xnn_head_norm_rotate(int dtype, const xnn_heads* q, const xnn_heads* k, int64_t n_tokens,
                         int32_t head_dim, int32_t rotated, const void* q_weight,
                         const void* k_weight, const float* cos, const float* sin, int64_t n_rows,
                         const int64_t* positions, float eps, int32_t interleaved, void* q_out,
                         void* k_out, xnn_stream_t stream) {
  XNN_REQUIRE(is_storage(dtype), "dtype must be XNN_F32, XNN_BF16 or XNN_F16");
  HeadArgs h;
  const int status = head_args(h, q, k, n_tokens, head_dim, rotated, q_weight, k_weight, cos, sin,
                               n_rows, positions, eps);
  if (status != XNN_OK || n_tokens == 0) return status;
  XNN_REQUIRE(q_out && k_out, "NULL output");
  h.q_out = q_out;
  h.k_out = k_out;
  XNN_STORAGE_DISPATCH(dtype, T, {
    const int n = head_width<T>(h, false);
    head_norm_launch<T, false>(h, n, interleaved, norm_blocks(h, 1 << 20), as_hip(stream));
  });
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

int xnn_head_norm_rotate_backward_work_size(int32_t head_dim, size_t* bytes) {
  XNN_REQUIRE(head_dim >= 1 && head_dim <= 128, "head_dim must be in [1, 128]");
  XNN_REQUIRE(bytes != nullptr, "NULL size");
  *bytes = norm_work_bytes(head_dim);
  return XNN_OK;
}

int xnn_head_norm_rotate_backward(int dtype, const xnn_heads* q, const xnn_heads* k,
                                  int64_t n_tokens, int32_t head_dim, int32_t rotated,
                                  const void* q_weight, const void* k_weight, const float* cos,
                                  const float* sin, int64_t n_rows, const int64_t* positions,
                                  float eps, int32_t interleaved, const void* grad_q,
                                  const void* grad_k, void* d_q, void* d_k, void* d_q_weight,
                                  void* d_k_weight, float* d_cos, float* d_sin, void* work,
                                  size_t work_bytes, xnn_stream_t stream) {
  XNN_REQUIRE(is_storage(dtype), "dtype must be XNN_F32, XNN_BF16 or XNN_F16");
  HeadArgs h;
  const int status = head_args(h, q, k, n_tokens, head_dim, rotated, q_weight, k_weight, cos, sin,
                               n_rows, positions, eps);
  if (status != XNN_OK) return status;
  XNN_REQUIRE((d_q_weight == nullptr) == (d_k_weight == nullptr),
              "the weights' gradients go together");
  XNN_REQUIRE((d_cos == nullptr) == (d_sin == nullptr), "the tables' gradients go together");
  XNN_REQUIRE(d_cos == nullptr || positions == nullptr,
              "tables read by position have no gradient here");
  XNN_REQUIRE(n_tokens == 0 || (grad_q && grad_k && d_q && d_k), "NULL cotangent or gradient");
  if (d_q_weight != nullptr)
    XNN_REQUIRE(work && work_bytes >= norm_work_bytes(head_dim), "work too small");
  h.gq = grad_q;
  h.gk = grad_k;
  h.q_out = d_q;
  h.k_out = d_k;
  h.d_cos = d_cos;
  h.d_sin = d_sin;
  h.part = d_q_weight != nullptr ? (float*)work : nullptr;
  hipStream_t s = as_hip(stream);
  XNN_STORAGE_DISPATCH(dtype, T, {
    int blocks = 0;
    if (n_tokens > 0) {
      const int n = head_width<T>(h, true);
      blocks = norm_blocks(h, kNormBlocks);
      head_norm_launch<T, true>(h, n, interleaved, blocks, s);
    }
    if (d_q_weight != nullptr)
      hipLaunchKernelGGL(head_weight_kernel<T>, dim3((2 * head_dim + 15) / 16), dim3(1024), 0, s,
                         (const float*)work, blocks, head_dim, (T*)d_q_weight, (T*)d_k_weight);
  });
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

}  // extern "C"
