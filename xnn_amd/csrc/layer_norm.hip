// Layer norm of rows and its backward pass with the sums of the weight's and the bias's gradients
// (gfx950, wave64).
//
//   n = (x - mean x) r,  r = 1 / sqrt(mean (x - mean x)^2 + eps),  y = w n + b
//   dx = r (g w - mean(g w) - n mean(g w n)),   dw = sum_rows g n,   db = sum_rows g
//
// A stream: a row lies in the registers of 2^k threads, U pieces of 16 bytes a thread, so that the
// squares are of the centered values and nothing is read twice. Sums over a row are exchanges within a wave and,
// for rows of more than a wave, through LDS. A thread keeps its columns from row to row and adds up
// their gradients in registers; the blocks' sums are added in their order. Arithmetic is float32.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "dense.h"

namespace xnn {

constexpr int kNormThreads = 1024;
constexpr int kNormWaves = kNormThreads / kWave;
constexpr int kNormParts = 512;    // blocks of the backward pass, at most: two a CU
constexpr int kMaxNormWidth = 16384;

struct LayerNormArgs {
  const void *x, *w, *b, *g;
  void *out;                       // the output, or x's gradient
  float* stats;                    // (rows, 2): mean and r
  float* part;                     // (blocks, 2, width)
  void *dw, *db;
  int64_t x_stride, n_rows;
  int width, lanes;                // lanes: threads of a row, a power of two
  float eps, inv;
};

// The sums of N values over the `lanes` threads of each row, every thread getting them; `s` (two in turn) for rows
// of more than a wave, where all threads of the block call it.
template <int N>
__device__ __forceinline__ void row_sums(float (&v)[N], int lanes, float (*s)[kNormWaves][2], int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (lanes > 1) v[i] += dpp_move<0xB1>(v[i]);
    if (lanes > 2) v[i] += dpp_move<0x4E>(v[i]);
    if (lanes > 4) v[i] += dpp_move<0x141>(v[i]);
    if (lanes > 8) v[i] += dpp_move<0x140>(v[i]);
    if (lanes > 16) v[i] = add_xor16(v[i]);
    if (lanes > 32) v[i] = add_xor32(v[i]);
  }
  if (lanes <= kWave) return;
  const int wave = wave_in_block(), waves = lanes / kWave;
  if (threadIdx.x % kWave == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) s[turn][wave][i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.0f;
  for (int w = wave / waves * waves; w < (wave / waves + 1) * waves; ++w)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += s[turn][w][i];
  turn ^= 1;
}

// piece `at` of a row: zeros beyond its width
template <typename T, int N>
__device__ __forceinline__ void norm_piece(const T* row, int at, int width, bool edge, float (&out)[N]) {
  const Pack<T, N> x = load_piece<T, N>(row, at, width, edge);
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = at + i < width ? (float)x.v[i] : 0.0f;
}

template <typename T, int U, bool BACK>
__global__ __launch_bounds__(kNormThreads) void layer_norm_kernel(LayerNormArgs p) {
  constexpr int N = 16 / sizeof(T);
  __shared__ float sums[2][kNormWaves][2];
  __shared__ __align__(16) float columns[BACK ? kNormThreads * N : 4];
  int turn = 0;
  const int rows = kNormThreads / p.lanes, slot = threadIdx.x / p.lanes, lane = threadIdx.x % p.lanes;
  float w[U][N], b[U][N], dw[BACK ? U : 1][N], db[BACK ? U : 1][N];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = (u * p.lanes + lane) * N;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      w[u][i] = 1.0f;
      b[u][i] = 0.0f;
      if constexpr (BACK) dw[u][i] = db[u][i] = 0.0f;
    }
    if (p.w != nullptr) norm_piece<T, N>((const T*)p.w, at, p.width, true, w[u]);
    if (!BACK && p.b != nullptr) norm_piece<T, N>((const T*)p.b, at, p.width, true, b[u]);
  }
  const bool small = p.x_stride < N;
  for (int64_t r0 = (int64_t)blockIdx.x * rows; r0 < p.n_rows; r0 += (int64_t)gridDim.x * rows) {
    // threads without a row go through the sums with the last one's
    const bool live = r0 + slot < p.n_rows;
    const int64_t r = live ? r0 + slot : p.n_rows - 1;
    const bool edge = r == p.n_rows - 1;
    const T* row = (const T*)p.x + r * p.x_stride;
    float x[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u)
      norm_piece<T, N>(row, (u * p.lanes + lane) * N, p.width, edge || small, x[u]);
    if constexpr (!BACK) {
      float s[1] = {0.0f};
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) s[0] += x[u][i];
      row_sums<1>(s, p.lanes, sums, turn);
      const float mean = s[0] * p.inv;
      s[0] = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          x[u][i] = (u * p.lanes + lane) * N + i < p.width ? x[u][i] - mean : 0.0f;
          s[0] = fmaf(x[u][i], x[u][i], s[0]);
        }
      row_sums<1>(s, p.lanes, sums, turn);
      const float rstd = rsqrtf(fmaf(s[0], p.inv, p.eps));
      if (!live) continue;
      if (p.stats != nullptr && lane == 0) {
        p.stats[2 * r] = mean;
        p.stats[2 * r + 1] = rstd;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = (u * p.lanes + lane) * N;
        if (at >= p.width) break;
        float y[N];
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = fmaf(x[u][i] * rstd, w[u][i], b[u][i]);
        store_row_part<T, N>((T*)p.out + r * p.width, at, p.width, y);
      }
    } else {
      const bool g_edge = edge || p.width < N;
      const float mean = p.stats[2 * r], rstd = p.stats[2 * r + 1];
      float g[U][N], s[2] = {0.0f, 0.0f};
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = (u * p.lanes + lane) * N;
        norm_piece<T, N>((const T*)p.g + r * p.width, at, p.width, g_edge, g[u]);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          x[u][i] = at + i < p.width ? (x[u][i] - mean) * rstd : 0.0f;
          if (live) {
            dw[u][i] = fmaf(g[u][i], x[u][i], dw[u][i]);
            db[u][i] += g[u][i];
          }
          g[u][i] *= w[u][i];
          s[0] += g[u][i];
          s[1] = fmaf(g[u][i], x[u][i], s[1]);
        }
      }
      row_sums<2>(s, p.lanes, sums, turn);
      if (!live || p.out == nullptr) continue;
      const float mg = s[0] * p.inv, mgn = s[1] * p.inv;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = (u * p.lanes + lane) * N;
        if (at >= p.width) break;
        float y[N];
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = rstd * (g[u][i] - fmaf(x[u][i], mgn, mg));
        store_row_part<T, N>((T*)p.out + r * p.width, at, p.width, y);
      }
    }
  }
  if constexpr (BACK) {
    if (p.dw == nullptr && p.db == nullptr) return;
    // the block's rows' sums of each column, in order: a block alone writes the gradients
    const int span = p.lanes * N;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        __syncthreads();
        store_pack<float, N>(columns + (size_t)threadIdx.x * N, m == 0 ? dw[u] : db[u]);
        __syncthreads();
        for (int i = threadIdx.x; i < span; i += kNormThreads) {
          const int c = u * span + i;
          if (c >= p.width) continue;
          float v = 0.0f;
          for (int q = 0; q < rows; ++q) v += columns[q * span + i];
          if (gridDim.x > 1)
            p.part[((int64_t)blockIdx.x * 2 + m) * p.width + c] = v;
          else if ((m == 0 ? p.dw : p.db) != nullptr)
            ((T*)(m == 0 ? p.dw : p.db))[c] = (T)v;
        }
      }
  }
}

// the blocks' sums added in float64: sixty-four of them at a time, then those in order
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_join_kernel(const float* __restrict__ part, int blocks, int width,
                                                               T* __restrict__ dw, T* __restrict__ db) {
  __shared__ double s[64][17];
  const int x = threadIdx.x % 16, y = threadIdx.x / 16;
  const int64_t i = (int64_t)blockIdx.x * 16 + x;
  double v = 0.0;
  if (i < 2 * width)
#pragma unroll 4
    for (int b = y; b < blocks; b += 64) v += part[(int64_t)b * 2 * width + i];
  s[y][x] = v;
  __syncthreads();
  if (y == 0 && i < 2 * width) {
    double r = 0.0;
#pragma unroll
    for (int q = 0; q < 64; ++q) r += s[q][x];
    T* out = i < width ? dw : db;
    if (out != nullptr) out[i < width ? i : i - width] = (T)(float)r;
  }
}

// pieces a thread; fills in the threads of a row
template <typename T>
static int norm_pieces(LayerNormArgs& p) {
  constexpr int N = 16 / sizeof(T);
  const int pieces = (p.width + N - 1) / N;
  int u = 1;
  while (u * kNormThreads < pieces) u *= 2;
  p.lanes = 1;
  while (u * p.lanes < pieces) p.lanes *= 2;
  return u;
}

template <typename T, bool BACK>
static void layer_norm_launch(LayerNormArgs p, int blocks, int u, hipStream_t s) {
  if (u == 1)
    hipLaunchKernelGGL((layer_norm_kernel<T, 1, BACK>), dim3(blocks), dim3(kNormThreads), 0, s, p);
  else if (u == 2)
    hipLaunchKernelGGL((layer_norm_kernel<T, 2, BACK>), dim3(blocks), dim3(kNormThreads), 0, s, p);
  else if constexpr (sizeof(T) == 4)
    hipLaunchKernelGGL((layer_norm_kernel<T, 4, BACK>), dim3(blocks), dim3(kNormThreads), 0, s, p);
}

static int layer_norm_sizes(int dtype, int64_t n_rows, int32_t width) {
  XNN_REQUIRE(is_storage(dtype), "dtype must be XNN_F32, XNN_BF16 or XNN_F16");
  XNN_REQUIRE(n_rows >= 0 && n_rows < ((int64_t)1 << 31), "n_rows must be in [0, 2^31)");
  XNN_REQUIRE(width >= 1 && width <= kMaxNormWidth, "width must be in [1, %d]", kMaxNormWidth);
  return XNN_OK;
}

static size_t norm_part_bytes(int32_t width) { return (size_t)kNormParts * 2 * width * sizeof(float); }

}  // namespace xnn

using namespace xnn;

extern "C" {

int xnn_layer_norm(int dtype, const void* x, int64_t x_stride, int64_t n_rows, int32_t width, const void* weight,
                   const void* bias, float eps, void* out, float* stats, xnn_stream_t stream) {
  const int status = layer_norm_sizes(dtype, n_rows, width);
  if (status != XNN_OK || n_rows == 0) return status;
  XNN_REQUIRE(x && out, "NULL input or output");
  XNN_REQUIRE(x_stride >= width, "rows of x overlap");
  LayerNormArgs p{};
  p.x = x;
  p.w = weight;
  p.b = bias;
  p.out = out;
  p.stats = stats;
  p.x_stride = x_stride;
  p.n_rows = n_rows;
  p.width = width;
  p.eps = eps;
  p.inv = 1.0f / (float)width;
  XNN_STORAGE_DISPATCH(dtype, T, {
    const int u = norm_pieces<T>(p);
    const int64_t rows = kNormThreads / p.lanes;
    layer_norm_launch<T, false>(p, (int)std::min<int64_t>((n_rows + rows - 1) / rows, 1 << 20), u,
                                as_hip(stream));
  });
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

int xnn_layer_norm_backward_work_size(int32_t width, size_t* bytes) {
  XNN_REQUIRE(width >= 1 && width <= kMaxNormWidth, "width must be in [1, %d]", kMaxNormWidth);
  XNN_REQUIRE(bytes != nullptr, "NULL size");
  *bytes = norm_part_bytes(width);
  return XNN_OK;
}

int xnn_layer_norm_backward(int dtype, const void* grad, const void* x, int64_t x_stride, int64_t n_rows,
                            int32_t width, const void* weight, const float* stats, void* dx, void* dweight,
                            void* dbias, void* work, size_t work_bytes, xnn_stream_t stream) {
  const int status = layer_norm_sizes(dtype, n_rows, width);
  if (status != XNN_OK) return status;
  const bool weights = dweight != nullptr || dbias != nullptr;
  XNN_REQUIRE(n_rows == 0 || (grad && x && stats), "NULL input");
  XNN_REQUIRE(n_rows == 0 || x_stride >= width, "rows of x overlap");
  XNN_REQUIRE(!weights || (work && work_bytes >= norm_part_bytes(width)), "work too small");
  if (!weights && (n_rows == 0 || dx == nullptr)) return XNN_OK;
  LayerNormArgs p{};
  p.x = x;
  p.w = weight;
  p.g = grad;
  p.out = dx;
  p.stats = const_cast<float*>(stats);
  p.part = (float*)work;
  p.dw = dweight;
  p.db = dbias;
  p.x_stride = x_stride;
  p.n_rows = n_rows;
  p.width = width;
  p.inv = 1.0f / (float)width;
  hipStream_t s = as_hip(stream);
  XNN_STORAGE_DISPATCH(dtype, T, {
    int blocks = 0;
    if (n_rows > 0) {
      const int u = norm_pieces<T>(p);
      const int64_t rows = kNormThreads / p.lanes;
      blocks = (int)std::min<int64_t>((n_rows + rows - 1) / rows, kNormParts);
      layer_norm_launch<T, true>(p, blocks, u, s);
    }
    if (weights && blocks != 1)
      hipLaunchKernelGGL(layer_norm_join_kernel<T>, dim3((2 * width + 15) / 16), dim3(1024), 0, s,
                         (const float*)work, blocks, width, (T*)dweight, (T*)dbias);
  });
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

}  // extern "C"
