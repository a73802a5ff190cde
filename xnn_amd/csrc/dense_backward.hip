// Dense layers, backward (gfx950, wave64): with d = g f'(z), the slope f'(z) kept by the forward pass,
//
//   dx = d W^T,   dW = x^T d,   db = sum of d over the rows
//
// of one weight or of each row's group. d is formed once, with db's sums, by a pass that reads g and the slope;
// without an activation d is g, which that pass reads for db alone. A weight's reduction runs over all rows of
// its group: it is cut into parts, one a block, which are added in their order where there is more than one.
// (d formed where each product stages it: 24,000 rows of 1,024 -> 4,096 in bfloat16, both products 843 us, for the
// registers, against 529 and 110 for the pass.)
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "dense.h"

namespace xnn {

struct BackwardArgs {
  const void *g, *slope, *x, *w;   // g: d where there is a slope (the products')
  void *d, *dx, *dw, *db;
  float *part, *part_bias;         // the parts' sums
  int64_t x_stride, tiles;
  GroupView groups, bias_groups;
  int n_rows, n_in, n_out, tiles_m, tiles_n;
  int rows, bias_rows;             // of a part of the weight's sums, of the bias's
};

// Where the sums of the part of sorted rows from `begin` on stand: parts of one weight follow each other; among
// groups of more than one part, their first parts begin at least `rows` apart, and so do their others.
__device__ __forceinline__ int64_t part_slot(const GroupView& v, int begin, int rows, bool first) {
  return v.n_groups == 0 ? begin / rows : 2 * (int64_t)(begin / rows) + (first ? 1 : 0);
}
// whether part `t` of rows is its group's only one, which writes the gradient itself
__device__ __forceinline__ bool part_alone(const GroupView& v, int n_rows, int rows, int group) {
  return n_rows <= rows || (v.n_groups > 0 && v.tile_ptr[group + 1] - v.tile_ptr[group] == 1);
}

// ---------------------------------------------------------------- d and db
// A block takes a part of the rows and, by pieces of 16 bytes, 2^k of the columns' pieces: a stream, with the
// columns' sums in registers
template <typename T>
__global__ __launch_bounds__(256) void dense_cotangent_kernel(BackwardArgs p, int lanes) {
  constexpr int N = 16 / sizeof(T);
  typedef typename Slope<T>::type S;
  __shared__ __align__(16) float sums[256 * N];
  const int slots = 256 / lanes, lane = threadIdx.x % lanes, slot = threadIdx.x / lanes;
  const int part = blockIdx.x / p.tiles_n, c = ((blockIdx.x % p.tiles_n) * lanes + lane) * N;
  // rows of no group are in no sum, and their d in no product
  const RowTile t = row_tile(p.bias_groups, p.bias_groups.n_groups, p.n_rows, part, p.bias_rows);
  if (t.group < 0) return;
  float sum[N];
#pragma unroll
  for (int i = 0; i < N; ++i) sum[i] = 0.0f;
  if (c < p.n_out)
#pragma unroll 2
    for (int r = t.begin + slot; r < t.end; r += slots) {
      const int64_t row = group_row(p.bias_groups, r);
      if (row < 0 || row >= p.n_rows) continue;
      const bool edge = row == p.n_rows - 1 || p.n_out < N;
      const Pack<T, N> g = load_piece<T, N>((const T*)p.g + row * p.n_out, c, p.n_out, edge);
      float v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = (float)g.v[i];
      if (p.slope != nullptr) {
        const Pack<S, N> s = load_piece<S, N>((const S*)p.slope + row * p.n_out, c, p.n_out, edge);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= slope_value<T>(s.v[i]);
        store_row_part<T, N>((T*)p.d + row * p.n_out, c, p.n_out, v);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) sum[i] += v[i];
    }
  if (p.db == nullptr) return;
  store_pack<float, N>(sums + threadIdx.x * N, sum);
  __syncthreads();
  const bool only = part_alone(p.bias_groups, p.n_rows, p.bias_rows, t.group);
  const int64_t at = part_slot(p.bias_groups, t.begin, p.bias_rows,
                               p.bias_groups.n_groups > 0 && part == p.bias_groups.tile_ptr[t.group]);
  const int c0 = (blockIdx.x % p.tiles_n) * lanes * N;
  for (int i = threadIdx.x; i < lanes * N && c0 + i < p.n_out; i += 256) {
    float v = 0.0f;
    for (int q = 0; q < slots; ++q) v += sums[q * lanes * N + i];
    if (only)
      ((T*)p.db)[(int64_t)t.group * p.n_out + c0 + i] = (T)v;
    else
      p.part_bias[at * p.n_out + c0 + i] = v;
  }
}

// ---------------------------------------------------------------- the products
template <typename T, typename L>
__global__ __launch_bounds__(kDenseThreads) void dense_input_kernel(BackwardArgs p) {
  typedef DenseLds<L, T, true, true> S;
  __shared__ __align__(16) char lds[S::kBytes];
  const int64_t slot = xcd_slot();
  if (slot >= p.tiles) return;
  const int n0 = (int)(slot % p.tiles_n) * L::BN;
  const RowTile t = row_tile(p.groups, p.groups.n_groups + 1, p.n_rows, (int)(slot / p.tiles_n), L::BM);
  if (t.group < 0) return;
  if (p.groups.n_groups > 0 && t.group == p.groups.n_groups) {   // rows of no group
    fill_rows<T, L::BN>(p.groups, t, p.n_rows, (T*)p.dx, n0, p.n_in, (T)0.0f);
    return;
  }
  Operator<T, L::BM, true> a;
  Operator<T, L::BN, true> b;
  a.init(p.g, p.groups.order, p.n_out, p.n_rows, p.n_out, t.begin, t.end, 0);
  b.init((const T*)p.w + (int64_t)t.group * p.n_in * p.n_out, nullptr, p.n_out, p.n_in, p.n_out, n0,
         min(n0 + L::BN, p.n_in), 0);
  f32x16 acc[L::MT][L::NT];
  dense_product<T, L, true, true>(a, b, p.n_out, lds, acc);
  int c;
  dense_rows<L>(
      lds, acc, [&](int n) { c = n0 + n; },
      [&](int m, float(&v)[8]) {
        const int r = t.begin + m;
        if (r >= t.end || c >= p.n_in) return;
        const int64_t row = group_row(p.groups, r);
        if (row < 0 || row >= p.n_rows) return;
        store_row_part<T, 8>((T*)p.dx + row * p.n_in, c, p.n_in, v);
      });
}

template <typename T, typename L>
__global__ __launch_bounds__(kDenseThreads) void dense_weight_kernel(BackwardArgs p) {
  typedef DenseLds<L, T, false, false> S;
  __shared__ __align__(16) char lds[S::kBytes];
  const int64_t slot = xcd_slot();
  if (slot >= p.tiles) return;
  const int tile = (int)(slot % (p.tiles_m * p.tiles_n));
  const int m0 = tile / p.tiles_n * L::BM, n0 = tile % p.tiles_n * L::BN;
  const int part = (int)(slot / (p.tiles_m * p.tiles_n));
  const RowTile t = row_tile(p.groups, p.groups.n_groups, p.n_rows, part, p.rows);
  if (t.group < 0) return;
  Operator<T, L::BM, false> a;
  Operator<T, L::BN, false> b;
  a.init(p.x, p.groups.order, p.x_stride, p.n_rows, p.n_in, t.begin, t.end, m0);
  b.init(p.g, p.groups.order, p.n_out, p.n_rows, p.n_out, t.begin, t.end, n0);
  f32x16 acc[L::MT][L::NT];
  dense_product<T, L, false, false>(a, b, t.end - t.begin, lds, acc);
  const bool only = part_alone(p.groups, p.n_rows, p.rows, t.group);
  const int64_t at =
      part_slot(p.groups, t.begin, p.rows, p.groups.n_groups > 0 && part == p.groups.tile_ptr[t.group]);
  T* dw = (T*)p.dw + (int64_t)t.group * p.n_in * p.n_out;
  float* sum = p.part + at * p.n_in * p.n_out;
  int c;
  dense_rows<L>(
      lds, acc, [&](int n) { c = n0 + n; },
      [&](int m, float(&v)[8]) {
        const int r = m0 + m;
        if (r >= p.n_in || c >= p.n_out) return;
        if (only)
          store_row_part<T, 8>(dw + (int64_t)r * p.n_out, c, p.n_out, v);
        else
          store_row_part<float, 8>(sum + (int64_t)r * p.n_out, c, p.n_out, v);
      });
}

// ---------------------------------------------------------------- the parts
// the sum over the parts of a group of element k of `size` (4 of them in a row), in the parts' order; false where the
// group's only part has written it
template <int N>
__device__ __forceinline__ bool part_sum(const GroupView& v, int n_rows, int rows, int group, const float* part,
                                         int64_t size, int64_t k, float (&out)[N]) {
  int begin = 0, parts = (n_rows + rows - 1) / rows;
  if (v.n_groups > 0) {
    begin = min(max(v.row_ptr[group], 0), n_rows);
    parts = min(v.tile_ptr[group + 1] - v.tile_ptr[group], (n_rows - begin + rows - 1) / rows);
  }
  if (parts == 1) return false;
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = 0.0f;
#pragma unroll 4
  for (int n = 0; n < parts; ++n) {
    const float* p = part + part_slot(v, begin + n * rows, rows, n == 0) * size + k;
    float x[N];
    if constexpr (N == 1)
      x[0] = *p;
    else
      load_row_part<float, N>(p, 0, N, x);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] += x[i];
  }
  return true;
}

// The parts of a weight and of its bias added in their order, zeros where there is none
template <typename T>
__global__ __launch_bounds__(256) void dense_join_kernel(BackwardArgs p, int blocks) {
  const int g = blockIdx.x / blocks, block = blockIdx.x % blocks;
  const int64_t size = (int64_t)p.n_in * p.n_out;
  T* dw = (T*)p.dw + g * size;
  for (int64_t k = ((int64_t)block * 256 + threadIdx.x) * 4; p.dw != nullptr && k < size; k += (int64_t)blocks * 1024) {
    float v[4];
    if (k + 4 <= size) {
      if (!part_sum<4>(p.groups, p.n_rows, p.rows, g, p.part, size, k, v)) break;
      store_row_part<T, 4>(dw + k, 0, 4, v);
    } else {
      for (int64_t e = k; e < size; ++e) {
        float one[1];
        if (!part_sum<1>(p.groups, p.n_rows, p.rows, g, p.part, size, e, one)) break;
        dw[e] = (T)one[0];
      }
    }
  }
  if (p.db == nullptr) return;
  for (int c = block * 256 + threadIdx.x; c < p.n_out; c += blocks * 256) {
    float one[1];
    if (!part_sum<1>(p.bias_groups, p.n_rows, p.bias_rows, g, p.part_bias, p.n_out, c, one)) break;
    ((T*)p.db)[(int64_t)g * p.n_out + c] = (T)one[0];
  }
}

// ---------------------------------------------------------------- host side
struct Parts {
  int rows;
  int64_t slots;                   // parts that have sums of their own
};
// Parts of at least `least` rows, about `want` of them; in groups of a power of two rows (the plan has their tiles)
static Parts parts_of(int64_t n_rows, bool grouped, int64_t want, int64_t least) {
  int64_t rows = std::max<int64_t>(least, (n_rows + want - 1) / std::max<int64_t>(want, 1));
  Parts w;
  if (grouped) {
    rows = (int64_t)32 << std::min(group_level(rows), kGroupLevels - 1);
    w.slots = n_rows <= rows ? 0 : 2 * (n_rows / rows + 1);
  } else {
    rows = (rows + 63) / 64 * 64;
    w.slots = n_rows <= rows ? 0 : (n_rows + rows - 1) / rows;
  }
  w.rows = (int)std::min<int64_t>(rows, 1 << 30);
  return w;
}

struct BackwardPlan {
  int side;                        // of the weight's tiles
  Parts weight, bias;
  size_t d, bytes;                 // of d, of all: the weight's parts, the bias's, d
  size_t bias_at, d_at;
};
static BackwardPlan backward_plan(int dtype, int64_t n_rows, int32_t n_in, int32_t n_out, bool grouped, bool slope,
                                  bool weight, bool bias) {
  BackwardPlan b{};
  const int64_t size = storage_bytes(dtype);
  const auto tiles = [&](int64_t s) { return ((n_in + s - 1) / s) * ((n_out + s - 1) / s); };
  // parts times tiles: two blocks a CU of 128 x 128 tiles and smaller, one of the larger
  b.side = n_in > 64 && n_out > 64 ? 128 : 64;
  if (size == 2 && n_in >= 192 && n_out >= 192 && n_rows * tiles(256) >= 256 * 512) b.side = 256;
  if (weight)
    b.weight = parts_of(n_rows, grouped, std::max<int64_t>(1, (b.side == 256 ? 256 : 512) / tiles(b.side)), 256);
  if (bias || slope) b.bias = parts_of(n_rows, grouped, 512, 64);
  const auto room = [](size_t n) { return (n + 255) / 256 * 256; };
  b.d = slope ? (size_t)n_rows * n_out * size : 0;
  b.bias_at = room((size_t)b.weight.slots * n_in * n_out * sizeof(float));
  b.d_at = b.bias_at + (bias ? room((size_t)b.bias.slots * n_out * sizeof(float)) : 0);
  b.bytes = b.d_at + b.d;
  return b;
}

template <typename T>
static void cotangent_launch(BackwardArgs p, const int32_t* plan, int n_groups, hipStream_t s) {
  constexpr int N = 16 / sizeof(T);
  int lanes = 1;
  while (lanes < 32 && lanes * N < p.n_out) lanes *= 2;
  p.tiles_n = (p.n_out + lanes * N - 1) / (lanes * N);
  const int64_t blocks = row_tiles(p.n_rows, n_groups, plan != nullptr, p.bias_rows) * p.tiles_n;
  hipLaunchKernelGGL(dense_cotangent_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, s, p, lanes);
}

template <typename T, typename L>
static void input_launch(BackwardArgs p, const int32_t* plan, int n_groups, hipStream_t s) {
  p.groups = group_view(plan, p.n_rows, n_groups, group_level(L::BM));
  p.tiles_n = (p.n_in + L::BN - 1) / L::BN;
  p.tiles = row_tiles(p.n_rows, n_groups, plan != nullptr, L::BM) * p.tiles_n;
  hipLaunchKernelGGL((dense_input_kernel<T, L>), dim3((unsigned)xcd_blocks(p.tiles)), dim3(kDenseThreads), 0, s, p);
}

template <typename T, typename L>
static void weight_launch(BackwardArgs p, const int32_t* plan, int n_groups, hipStream_t s) {
  p.tiles_m = (p.n_in + L::BM - 1) / L::BM;
  p.tiles_n = (p.n_out + L::BN - 1) / L::BN;
  p.tiles = row_tiles(p.n_rows, n_groups, plan != nullptr, p.rows) * p.tiles_m * p.tiles_n;
  hipLaunchKernelGGL((dense_weight_kernel<T, L>), dim3((unsigned)xcd_blocks(p.tiles)), dim3(kDenseThreads), 0, s, p);
}

}  // namespace xnn

using namespace xnn;

extern "C" {

int xnn_linear_backward_work_size(int dtype, int64_t n_rows, int32_t n_in, int32_t n_out, int32_t n_groups,
                                  int32_t grouped, int32_t slope, int32_t weight, int32_t bias, size_t* bytes) {
  static const int32_t some = 0;
  const int status = dense_sizes(dtype, n_rows, n_in, n_out, &some, n_groups);
  if (status != XNN_OK) return status;
  XNN_REQUIRE(bytes != nullptr, "NULL size");
  *bytes = backward_plan(dtype, n_rows, n_in, n_out, grouped != 0, slope != 0, weight != 0, bias != 0).bytes;
  return XNN_OK;
}

int xnn_linear_backward(int dtype, const void* grad, const void* slope, const void* x, int64_t x_stride,
                        int64_t n_rows, int32_t n_in, int32_t n_out, const void* weight, const int32_t* plan,
                        int32_t n_groups, void* dx, void* dweight, void* dbias, void* work,
                        size_t work_bytes, xnn_stream_t stream) {
  const int status = dense_sizes(dtype, n_rows, n_in, n_out, plan, n_groups);
  if (status != XNN_OK) return status;
  XNN_REQUIRE(n_rows == 0 || grad, "NULL cotangent");
  XNN_REQUIRE(n_rows == 0 || dx == nullptr || weight, "NULL weight");
  XNN_REQUIRE(dweight == nullptr || n_rows == 0 || x, "NULL input");
  XNN_REQUIRE(dweight == nullptr || n_rows == 0 || x_stride >= n_in, "rows of x overlap");
  if (dx == nullptr && dweight == nullptr && dbias == nullptr) return XNN_OK;
  if (n_rows == 0 && dweight == nullptr && dbias == nullptr) return XNN_OK;
  const bool grouped = plan != nullptr && n_rows > 0;
  const BackwardPlan b = backward_plan(dtype, n_rows, n_in, n_out, grouped, slope != nullptr, dweight != nullptr,
                                       dbias != nullptr);
  XNN_REQUIRE(b.bytes == 0 || (work && work_bytes >= b.bytes), "work too small");
  XNN_REQUIRE((uintptr_t)work % 16 == 0, "work must be aligned to 16 bytes");
  BackwardArgs p{};
  p.g = grad;
  p.slope = slope;
  p.x = x;
  p.w = weight;
  p.dx = dx;
  p.dw = dweight;
  p.db = dbias;
  p.part = (float*)work;
  p.part_bias = (float*)((char*)work + b.bias_at);
  p.d = (char*)work + b.d_at;
  p.x_stride = x_stride;
  p.n_rows = (int)n_rows;
  p.n_in = n_in;
  p.n_out = n_out;
  p.rows = std::max(b.weight.rows, 1);
  p.bias_rows = std::max(b.bias.rows, 1);
  const int32_t* order = grouped ? plan : nullptr;
  p.groups = group_view(order, n_rows, n_groups, grouped ? group_level(p.rows) : 0);
  p.bias_groups = group_view(order, n_rows, n_groups, grouped ? group_level(p.bias_rows) : 0);
  hipStream_t s = as_hip(stream);
  const int side = dense_tile(storage_bytes(dtype), n_rows, n_in);
  XNN_STORAGE_DISPATCH(dtype, T, {
    if (n_rows > 0 && (slope != nullptr || dbias != nullptr)) cotangent_launch<T>(p, order, n_groups, s);
    if (slope != nullptr) p.g = p.d;
    if (n_rows > 0 && dx != nullptr) XNN_TILE_DISPATCH(side, T, L, input_launch<T, L>(p, order, n_groups, s));
    if (n_rows > 0 && dweight != nullptr)
      XNN_TILE_DISPATCH(b.side, T, L, weight_launch<T, L>(p, order, n_groups, s));
    // groups without rows have zeros, parts have sums
    if ((dweight != nullptr && (grouped || b.weight.slots > 0 || n_rows == 0)) ||
        (dbias != nullptr && (grouped || b.bias.slots > 0 || n_rows == 0))) {
      const int64_t all = dweight != nullptr ? (int64_t)n_in * n_out : n_out;
      const int blocks = (int)std::max<int64_t>(1, std::min<int64_t>((all + 1023) / 1024, 65536 / n_groups));
      hipLaunchKernelGGL(dense_join_kernel<T>, dim3((unsigned)(blocks * n_groups)), dim3(256), 0, s, p, blocks);
    }
  });
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

}  // extern "C"
