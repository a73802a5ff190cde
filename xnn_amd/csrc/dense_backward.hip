// Dense layers, backward (gfx950, wave64): with d = g f'(z), the slope f'(z) kept by the forward pass,
//
//   dx = d W^T,   dW = x^T d,   db = sum of d over the rows
//
// of one weight or of each row's group. d is formed where it is staged and never stored; db adds up the
// values that the weight's product stages. A weight's reduction runs over all rows of its group: it is
// cut into parts of whole steps, one a block, which are added in their order where there is more than one.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "dense.h"

namespace xnn {

struct BackwardArgs {
  const void *g, *slope, *x, *w;
  void *dx, *dw, *db;
  float *part, *part_bias;         // the parts' sums
  int64_t x_stride, tiles;
  GroupView groups;
  int n_rows, n_in, n_out, tiles_m, tiles_n, rows;   // rows: of a part
};

template <typename T, typename L, bool TIMES>
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
  Operator<T, L::BM, true, TIMES> a;
  Operator<T, L::BN, true, false> b;
  a.init(p.g, p.slope, p.groups.order, p.n_out, p.n_rows, p.n_out, t.begin, t.end, 0);
  b.init((const T*)p.w + (int64_t)t.group * p.n_in * p.n_out, nullptr, nullptr, p.n_out, p.n_in, p.n_out, n0,
         min(n0 + L::BN, p.n_in), 0);
  f32x16 acc[L::MT][L::NT];
  dense_product<T, L, true, true, false>(a, b, 0, p.n_out, p.n_out, lds, acc);
  dense_rows<L>(lds, acc, [&](int m, int n, float (&v)[8]) {
    const int r = t.begin + m, c = n0 + n;
    if (r >= t.end || c >= p.n_in) return;
    const int64_t row = group_row(p.groups, r);
    if (row < 0 || row >= p.n_rows) return;
    store_row_part<T, 8>((T*)p.dx + row * p.n_in, c, p.n_in, v);
  });
}

// Where the sums of the part of sorted rows from `begin` on stand: parts of one weight follow each other; among
// groups of more than one part, their first parts begin at least `rows` apart, and so do their others.
__device__ __forceinline__ int64_t part_slot(const GroupView& v, int begin, int rows, bool first) {
  return v.n_groups == 0 ? begin / rows : 2 * (int64_t)(begin / rows) + (first ? 1 : 0);
}

template <typename T, typename L, bool TIMES>
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
  Operator<T, L::BM, false, false> a;
  Operator<T, L::BN, false, TIMES> b;
  typedef Operator<T, L::BN, false, TIMES> B;
  a.init(p.x, nullptr, p.groups.order, p.x_stride, p.n_rows, p.n_in, t.begin, t.end, m0);
  b.init(p.g, p.slope, p.groups.order, p.n_out, p.n_rows, p.n_out, t.begin, t.end, n0);
  f32x16 acc[L::MT][L::NT];
  float sums[B::kPer];
#pragma unroll
  for (int i = 0; i < B::kPer; ++i) sums[i] = 0.0f;
  const int length = t.end - t.begin;
  dense_product<T, L, false, false, true>(a, b, 0, length, length, lds, acc, sums);
  // one part: the gradient itself
  bool only = p.n_rows <= p.rows;                           // then there is no room for parts
  int64_t at = part_slot(p.groups, t.begin, p.rows, false);
  if (p.groups.n_groups > 0) {
    only = only || p.groups.tile_ptr[t.group + 1] - p.groups.tile_ptr[t.group] == 1;
    at = part_slot(p.groups, t.begin, p.rows, part == p.groups.tile_ptr[t.group]);
  }
  if (p.db != nullptr && m0 == 0) {
    float* s = reinterpret_cast<float*>(lds);                // (kStep, BN)
    store_pack<float, B::kPer>(s + b.row * L::BN + threadIdx.x % B::kChunks * B::kPer, sums);
    __syncthreads();
    for (int i = threadIdx.x; i < L::BN; i += kDenseThreads) {
      float v = 0.0f;
#pragma unroll
      for (int r = 0; r < B::kStep; ++r) v += s[r * L::BN + i];
      if (n0 + i < p.n_out) {
        if (only)
          ((T*)p.db)[(int64_t)t.group * p.n_out + n0 + i] = (T)v;
        else
          p.part_bias[at * p.n_out + n0 + i] = v;
      }
    }
    __syncthreads();
  }
  T* dw = (T*)p.dw + (int64_t)t.group * p.n_in * p.n_out;
  float* sum = p.part + at * p.n_in * p.n_out;
  dense_rows<L>(lds, acc, [&](int m, int n, float (&v)[8]) {
    const int r = m0 + m, c = n0 + n;
    if (r >= p.n_in || c >= p.n_out) return;
    if (only)
      store_row_part<T, 8>(dw + (int64_t)r * p.n_out, c, p.n_out, v);
    else
      store_row_part<float, 8>(sum + (int64_t)r * p.n_out, c, p.n_out, v);
  });
}

// The parts of a weight and of its bias added in their order, zeros where there is none; those of one part are
// done.
template <typename T>
__global__ __launch_bounds__(256) void dense_join_kernel(BackwardArgs p, int blocks) {
  const int g = blockIdx.x / blocks;
  const int64_t size = (int64_t)p.n_in * p.n_out;
  int begin = 0, parts = (p.n_rows + p.rows - 1) / p.rows;
  if (p.groups.n_groups > 0) {
    begin = min(max(p.groups.row_ptr[g], 0), p.n_rows);
    parts = min(p.groups.tile_ptr[g + 1] - p.groups.tile_ptr[g], (p.n_rows - begin + p.rows - 1) / p.rows);
  }
  if (parts == 1) return;
  const int64_t all = size + (p.db != nullptr ? p.n_out : 0);
  for (int64_t i = ((int64_t)(blockIdx.x % blocks) * 256 + threadIdx.x) * 4; i < all; i += (int64_t)blocks * 1024) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t k = i + e;
      if (k >= all) break;
      const bool weight = k < size;
      const float* s = weight ? p.part + k : p.part_bias + (k - size);
      const int64_t step = weight ? size : p.n_out;
      float v = 0.0f;
      for (int n = 0; n < parts; ++n) v += s[part_slot(p.groups, begin + n * p.rows, p.rows, n == 0) * step];
      if (weight)
        ((T*)p.dw)[g * size + k] = (T)v;
      else
        ((T*)p.db)[(int64_t)g * p.n_out + (k - size)] = (T)v;
    }
  }
}

// ---------------------------------------------------------------- host side
// Rows of a part: whole steps, in groups a power of two (the plan has their tiles), so that the parts times the
// tiles of the weight fill the card twice.
struct Parts {
  int tile, rows;
  int64_t slots;                   // parts that have sums of their own
};
static Parts weight_parts(size_t size, int64_t n_rows, int32_t n_in, int32_t n_out, bool grouped) {
  Parts w;
  w.tile = n_in > 64 && n_out > 64 ? 1 : 0;
  const int64_t b = w.tile == 1 ? 128 : 64;
  const int64_t tiles = ((n_in + b - 1) / b) * ((n_out + b - 1) / b);
  const int64_t want = std::max<int64_t>(1, 512 / tiles);
  int64_t rows = std::max<int64_t>(256, (n_rows + want - 1) / want);
  if (grouped) {
    const int level = std::min(group_level(rows), kGroupLevels - 1);
    rows = (int64_t)32 << level;
    w.slots = n_rows <= rows ? 0 : 2 * (n_rows / rows + 1);
  } else {
    rows = (rows + 63) / 64 * 64;
    w.slots = n_rows <= rows ? 0 : (n_rows + rows - 1) / rows;
  }
  w.rows = (int)std::min<int64_t>(rows, 1 << 30);
  return w;
}

template <typename T, typename L>
static void input_launch(BackwardArgs p, const int32_t* plan, int n_groups, hipStream_t s) {
  p.groups = group_view(plan, p.n_rows, n_groups, group_level(L::BM));
  p.tiles_n = (p.n_in + L::BN - 1) / L::BN;
  p.tiles = row_tiles(p.n_rows, n_groups, plan != nullptr, L::BM) * p.tiles_n;
  const dim3 grid((unsigned)xcd_blocks(p.tiles));
  if (p.slope != nullptr)
    hipLaunchKernelGGL((dense_input_kernel<T, L, true>), grid, dim3(kDenseThreads), 0, s, p);
  else
    hipLaunchKernelGGL((dense_input_kernel<T, L, false>), grid, dim3(kDenseThreads), 0, s, p);
}

template <typename T, typename L>
static void weight_launch(BackwardArgs p, const int32_t* plan, int n_groups, hipStream_t s) {
  p.groups = group_view(plan, p.n_rows, n_groups, plan == nullptr ? 0 : group_level(p.rows));
  p.tiles_m = (p.n_in + L::BM - 1) / L::BM;
  p.tiles_n = (p.n_out + L::BN - 1) / L::BN;
  p.tiles = row_tiles(p.n_rows, n_groups, plan != nullptr, p.rows) * p.tiles_m * p.tiles_n;
  const dim3 grid((unsigned)xcd_blocks(p.tiles));
  if (p.slope != nullptr)
    hipLaunchKernelGGL((dense_weight_kernel<T, L, true>), grid, dim3(kDenseThreads), 0, s, p);
  else
    hipLaunchKernelGGL((dense_weight_kernel<T, L, false>), grid, dim3(kDenseThreads), 0, s, p);
}

}  // namespace xnn

using namespace xnn;

extern "C" {

int xnn_linear_backward_work_size(int dtype, int64_t n_rows, int32_t n_in, int32_t n_out, int32_t n_groups,
                                  int32_t grouped, size_t* bytes) {
  static const int32_t some = 0;
  const int status = dense_sizes(dtype, n_rows, n_in, n_out, &some, n_groups);
  if (status != XNN_OK) return status;
  XNN_REQUIRE(bytes != nullptr, "NULL size");
  const Parts w = weight_parts(storage_bytes(dtype), n_rows, n_in, n_out, grouped != 0);
  *bytes = (size_t)w.slots * ((size_t)n_in + 1) * n_out * sizeof(float);
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
  XNN_REQUIRE(dbias == nullptr || dweight != nullptr, "the bias's gradient goes with the weight's");
  XNN_REQUIRE(dweight == nullptr || x_stride >= n_in, "rows of x overlap");
  BackwardArgs p{};
  p.g = grad;
  p.slope = slope;
  p.x = x;
  p.w = weight;
  p.dx = dx;
  p.dw = dweight;
  p.db = dbias;
  p.x_stride = x_stride;
  p.n_rows = (int)n_rows;
  p.n_in = n_in;
  p.n_out = n_out;
  hipStream_t s = as_hip(stream);
  if (dx != nullptr && n_rows > 0) {
    XNN_STORAGE_DISPATCH(dtype, T, {
      switch (dense_tile(sizeof(T), n_rows, n_in)) {
        case 0: input_launch<T, Small<T>>(p, plan, n_groups, s); break;
        case 1: input_launch<T, Middle<T>>(p, plan, n_groups, s); break;
        default: input_launch<T, Large<T>>(p, plan, n_groups, s);
      }
    });
    XNN_LAUNCH_CHECK();
  }
  if (dweight == nullptr) return XNN_OK;
  const Parts w = weight_parts(storage_bytes(dtype), n_rows, n_in, n_out, plan != nullptr);
  const size_t need = (size_t)w.slots * ((size_t)n_in + 1) * n_out * sizeof(float);
  XNN_REQUIRE(need == 0 || (work && work_bytes >= need), "work too small");
  XNN_REQUIRE((uintptr_t)work % 16 == 0, "work must be aligned to 16 bytes");
  p.part = (float*)work;
  p.part_bias = p.part == nullptr ? nullptr : p.part + w.slots * (int64_t)n_in * n_out;
  p.rows = w.rows;
  XNN_STORAGE_DISPATCH(dtype, T, {
    if (n_rows > 0) {
      if (w.tile == 1)
        weight_launch<T, Middle<T>>(p, plan, n_groups, s);
      else
        weight_launch<T, Small<T>>(p, plan, n_groups, s);
    }
    if (plan != nullptr || w.slots > 0 || n_rows == 0) {
      const bool grouped = plan != nullptr && n_rows > 0;
      p.groups = group_view(grouped ? plan : nullptr, n_rows, n_groups, grouped ? group_level(p.rows) : 0);
      const int64_t all = ((int64_t)n_in + 1) * n_out;
      const int blocks = (int)std::max<int64_t>(1, std::min<int64_t>((all + 1023) / 1024, 65536 / n_groups));
      hipLaunchKernelGGL(dense_join_kernel<T>, dim3((unsigned)(blocks * n_groups)), dim3(256), 0, s, p, blocks);
    }
  });
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

}  // extern "C"
