// Layer norm of rows and its backward pass with the sums of the weight's and the bias's gradients
// (gfx950, wave64).
//
//   n = (x - mean x) r,  r = 1 / sqrt(mean (x - mean x)^2 + eps),  y = w n + b
//   dx = r (g w - mean(g w) - n mean(g w n)),   dw = sum_rows g n,   db = sum_rows g
//
// A stream: a row lies in the registers of 2^k threads, U pieces of 16 bytes a thread, so that the squares are of
// the centered values and nothing is read twice. A wave has a row of its own up to four pieces a lane: its sums are
// exchanges in the vector unit and wait for no other wave (24,000 rows of 2,048 in bfloat16, a piece a thread and
// four waves a row: forward 81 us, so 38, the rate of a large copy). Longer rows add their waves' sums through LDS.
// A thread keeps its columns from row to row and adds up their gradients in registers; the blocks' sums are added
// in their order. Arithmetic is float32. The backward pass of those rows takes 64 us (4.6 TB/s) and the join 5.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "dense.h"

namespace xnn {

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
template <int N, int WAVES>
__device__ __forceinline__ void row_sums(float (&v)[N], int lanes, float (*s)[WAVES][2], int& turn) {
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

// piece `at` of a row as it is in memory, zeros beyond its width
template <typename T>
__device__ __forceinline__ u32x4 norm_piece(const T* row, int at, int width, bool last) {
  const int left = width - at;
  u32x4 x = load_raw<T>(reinterpret_cast<const char*>(row + at), left, last);
  if (left < (int)(16 / sizeof(T))) x = piece_head<T>(x, left);
  return x;
}
template <typename T>
__device__ __forceinline__ void piece_values(u32x4 x, float (&v)[16 / sizeof(T)]) {
  constexpr int N = 16 / sizeof(T);
  const Pack<T, N> p = __builtin_bit_cast(Pack<T, N>, x);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = (float)p.v[i];
}

template <typename T, int THREADS, int U, bool BACK>
__global__ __launch_bounds__(THREADS) void layer_norm_kernel(LayerNormArgs p) {
  constexpr int N = 16 / sizeof(T), WAVES = THREADS / kWave;
  __shared__ float sums[2][WAVES][2];
  __shared__ __align__(16) float columns[BACK ? THREADS * N : 4];
  int turn = 0;
  const int rows = THREADS / p.lanes, slot = threadIdx.x / p.lanes, lane = threadIdx.x % p.lanes;
  // values stay as they are in memory, two to a register in 16 bits, and are taken apart where they are used: the
  // backward pass of rows of 2,048 in bfloat16 has three waves a SIMD so, one (and 178 us) with them apart
  const auto place = [&](int u) { return (u * p.lanes + lane) * N; };
  u32x4 w[U], b[U];
  float dw[BACK ? U : 1][N], db[BACK ? U : 1][N];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (p.w != nullptr) w[u] = norm_piece<T>((const T*)p.w, place(u), p.width, true);
    if (!BACK && p.b != nullptr) b[u] = norm_piece<T>((const T*)p.b, place(u), p.width, true);
    if constexpr (BACK)
#pragma unroll
      for (int i = 0; i < N; ++i) dw[u][i] = db[u][i] = 0.0f;
  }
  const bool small = p.x_stride < N;
  for (int64_t r0 = (int64_t)blockIdx.x * rows; r0 < p.n_rows; r0 += (int64_t)gridDim.x * rows) {
    // threads without a row go through the sums with the last one's
    const bool live = r0 + slot < p.n_rows;
    const int64_t r = live ? r0 + slot : p.n_rows - 1;
    const bool last = r == p.n_rows - 1;
    const T* row = (const T*)p.x + r * p.x_stride;
    T* out = (T*)p.out + r * p.width;
    u32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = norm_piece<T>(row, place(u), p.width, last || small);
    if constexpr (!BACK) {
      float s[1] = {0.0f};
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[N];
        piece_values<T>(x[u], v);
#pragma unroll
        for (int i = 0; i < N; ++i) s[0] += v[i];
      }
      row_sums<1, WAVES>(s, p.lanes, sums, turn);
      const float mean = s[0] * p.inv;
      s[0] = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[N];
        piece_values<T>(x[u], v);
        if (place(u) + N <= p.width) {
#pragma unroll
          for (int i = 0; i < N; ++i) s[0] = fmaf(v[i] - mean, v[i] - mean, s[0]);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) s[0] = place(u) + i < p.width ? fmaf(v[i] - mean, v[i] - mean, s[0]) : s[0];
        }
      }
      row_sums<1, WAVES>(s, p.lanes, sums, turn);
      const float rstd = rsqrtf(fmaf(s[0], p.inv, p.eps));
      if (!live) continue;
      if (p.stats != nullptr && lane == 0) {
        p.stats[2 * r] = mean;
        p.stats[2 * r + 1] = rstd;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (place(u) >= p.width) break;
        float v[N], f[N];
        piece_values<T>(x[u], v);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (v[i] - mean) * rstd;
        if (p.w != nullptr) {
          piece_values<T>(w[u], f);
#pragma unroll
          for (int i = 0; i < N; ++i) v[i] *= f[i];
        }
        if (p.b != nullptr) {
          piece_values<T>(b[u], f);
#pragma unroll
          for (int i = 0; i < N; ++i) v[i] += f[i];
        }
        store_row_part<T, N>(out, place(u), p.width, v);
      }
    } else {
      const T* cotangent = (const T*)p.g + r * p.width;
      const float mean = p.stats[2 * r], rstd = p.stats[2 * r + 1];
      u32x4 g[U];
      float s[2] = {0.0f, 0.0f};
#pragma unroll
      for (int u = 0; u < U; ++u) g[u] = norm_piece<T>(cotangent, place(u), p.width, last || p.width < N);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float n[N], v[N], f[N];
        piece_values<T>(x[u], n);
        piece_values<T>(g[u], v);
        if (p.w != nullptr) piece_values<T>(w[u], f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          n[i] = (n[i] - mean) * rstd;                     // beyond the width g is zero
          if (live) {
            dw[u][i] = fmaf(v[i], n[i], dw[u][i]);
            db[u][i] += v[i];
          }
          if (p.w != nullptr) v[i] *= f[i];
          s[0] += v[i];
          s[1] = fmaf(v[i], n[i], s[1]);
        }
      }
      row_sums<2, WAVES>(s, p.lanes, sums, turn);
      if (!live || p.out == nullptr) continue;
      const float mg = s[0] * p.inv, mgn = s[1] * p.inv;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (place(u) >= p.width) break;
        float n[N], v[N], f[N];
        piece_values<T>(x[u], n);
        piece_values<T>(g[u], v);
        if (p.w != nullptr) {
          piece_values<T>(w[u], f);
#pragma unroll
          for (int i = 0; i < N; ++i) v[i] *= f[i];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = rstd * (v[i] - fmaf((n[i] - mean) * rstd, mgn, mg));
        store_row_part<T, N>(out, place(u), p.width, v);
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
        for (int i = threadIdx.x; i < span; i += THREADS) {
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

// Threads of a block, pieces a thread; fills in the threads of a row: a wave at most where four pieces a lane do
struct NormShape {
  int threads, pieces;
  int64_t rows;                    // of a block
};
template <typename T>
static NormShape norm_shape(LayerNormArgs& p) {
  constexpr int N = 16 / sizeof(T);
  const int pieces = (p.width + N - 1) / N;
  NormShape n{pieces > 4 * 256 ? 1024 : 256, 1, 0};
  const int most = n.threads == 1024 ? 1024 : kWave;
  while (n.pieces < 4 && n.pieces * most < pieces) n.pieces *= 2;
  p.lanes = 1;
  while (n.pieces * p.lanes < pieces) p.lanes *= 2;
  n.rows = n.threads / p.lanes;
  return n;
}

template <typename T, bool BACK>
static void layer_norm_launch(LayerNormArgs p, int blocks, const NormShape& n, hipStream_t s) {
#define XNN_NORM_LAUNCH(THREADS, U)                                                                        \
  hipLaunchKernelGGL((layer_norm_kernel<T, THREADS, U, BACK>), dim3(blocks), dim3(THREADS), 0, s, p)
  if (n.threads == 1024) {
    if constexpr (sizeof(T) == 4) {
      if (n.pieces == 4) {
        XNN_NORM_LAUNCH(1024, 4);
        return;
      }
    }
    XNN_NORM_LAUNCH(1024, 2);
  } else if (n.pieces == 1) {
    XNN_NORM_LAUNCH(256, 1);
  } else if (n.pieces == 2) {
    XNN_NORM_LAUNCH(256, 2);
  } else {
    XNN_NORM_LAUNCH(256, 4);
  }
#undef XNN_NORM_LAUNCH
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
    const NormShape n = norm_shape<T>(p);
    // eight blocks a CU go over the rows: their weights are read once
    layer_norm_launch<T, false>(p, (int)std::min<int64_t>((n_rows + n.rows - 1) / n.rows, 2048), n, as_hip(stream));
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
      const NormShape n = norm_shape<T>(p);
      blocks = (int)std::min<int64_t>((n_rows + n.rows - 1) / n.rows, kNormParts);
      layer_norm_launch<T, true>(p, blocks, n, s);
    }
    if (weights && blocks != 1)
      hipLaunchKernelGGL(layer_norm_join_kernel<T>, dim3((2 * width + 15) / 16), dim3(1024), 0, s,
                         (const float*)work, blocks, width, (T*)dweight, (T*)dbias);
  });
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

}  // extern "C"
