// Dense layers, forward: out = residual + f(x W + b), with one weight or with that of each row's group
// (gfx950, wave64). The products are dense.h's; bias, activation, its slope for the backward pass and the
// residual are applied to the sums as they leave, so what is written is the result.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "dense.h"

namespace xnn {

struct ForwardArgs {
  const void *x, *w;
  int64_t x_stride, tiles;
  int n_in, tiles_n, parts, steps; // parts of the reduction, of so many steps
  Output o;
};

template <typename T, typename L>
__global__ __launch_bounds__(kDenseThreads) void dense_forward_kernel(ForwardArgs p) {
  typedef DenseLds<L, T, true, false> S;
  __shared__ __align__(16) char lds[S::kBytes];
  __shared__ int32_t rows[L::BM];
  const Output& o = p.o;
  const int64_t slot = xcd_slot();
  if (slot >= p.tiles * p.parts) return;
  const int part = (int)(slot / p.tiles), tile = (int)(slot % p.tiles);
  const RowTile t = row_tile(o.groups, o.groups.n_groups + 1, o.n_rows, tile / p.tiles_n, L::BM);
  if (t.group < 0) return;
  const int n0 = tile % p.tiles_n * L::BN;
  if (o.groups.n_groups > 0 && t.group == o.groups.n_groups) {   // rows of no group
    if (part == 0) fill_rows<T, L::BN>(o.groups, t, o.n_rows, (T*)o.out, n0, o.width, (T)o.none);
    return;
  }
  const int k0 = part * p.steps * L::BK, k1 = min(p.n_in, k0 + p.steps * L::BK);
  note_rows(o.groups, t, o.n_rows, rows);
  Operator<T, L::BM, L::BK, true> a;
  Operator<T, L::BN, L::BK, false> b;
  a.init(p.x, o.groups.order, p.x_stride, o.n_rows, p.n_in, t.begin, t.end, k0);
  b.init((const T*)p.w + (int64_t)t.group * p.n_in * o.width, nullptr, o.width, p.n_in, o.width, k0, k1, n0);
  f32x16 acc[L::MT][L::NT];
  dense_product<T, L, true, false>(a, b, k1 - k0, lds, acc, [](int) {});
  put_tile<T, L>(lds, acc, o, p.parts, part, t.group, rows, n0);
}

template <typename T, typename L>
static void forward_launch(ForwardArgs p, const int32_t* plan, int n_groups, hipStream_t s) {
  p.o.groups = group_view(plan, p.o.n_rows, n_groups, group_level(L::BM));
  p.tiles_n = (p.o.width + L::BN - 1) / L::BN;
  p.tiles = row_tiles(p.o.n_rows, n_groups, plan != nullptr, L::BM) * p.tiles_n;
  if (p.parts == 1) p.steps = (p.n_in + L::BK - 1) / L::BK;
  hipLaunchKernelGGL((dense_forward_kernel<T, L>), dim3((unsigned)xcd_blocks(p.tiles * p.parts)), dim3(kDenseThreads),
                     0, s, p);
  if (p.parts > 1) parts_launch<T>(p.o, plan, n_groups, p.parts, s);
}

}  // namespace xnn

using namespace xnn;

extern "C" {

int xnn_linear_work_size(int dtype, int64_t n_rows, int32_t n_in, int32_t n_out, int32_t n_groups, int32_t grouped,
                         size_t* bytes) {
  static const int32_t some = 0;
  const int status = dense_sizes(dtype, n_rows, n_in, n_out, &some, n_groups);
  if (status != XNN_OK) return status;
  XNN_REQUIRE(bytes != nullptr, "NULL size");
  const size_t size = storage_bytes(dtype);
  *bytes = dense_split(size, dense_tile(size, n_rows, n_out, grouped ? n_groups : 0), n_rows, n_out, n_in).bytes;
  return XNN_OK;
}

int xnn_linear(int dtype, const void* x, int64_t x_stride, int64_t n_rows, int32_t n_in, int32_t n_out,
               const void* weight, const void* bias, int32_t activation, const void* residual,
               const int32_t* plan, int32_t n_groups, void* out, void* slope, void* work, size_t work_bytes,
               xnn_stream_t stream) {
  const int status = dense_sizes(dtype, n_rows, n_in, n_out, plan, n_groups);
  if (status != XNN_OK) return status;
  XNN_REQUIRE(activation >= XNN_NO_ACTIVATION && activation <= XNN_TANH, "unknown activation");
  XNN_REQUIRE(slope == nullptr || activation != XNN_NO_ACTIVATION, "no activation has no slope");
  if (n_rows == 0) return XNN_OK;
  XNN_REQUIRE(x && weight && out, "NULL input or output");
  XNN_REQUIRE(x_stride >= n_in, "rows of x overlap");
  const size_t size = storage_bytes(dtype);
  const int kind = dense_tile(size, n_rows, n_out, plan != nullptr ? n_groups : 0);
  const Split split = dense_split(size, kind, n_rows, n_out, n_in);
  XNN_REQUIRE(split.bytes == 0 || (work && work_bytes >= split.bytes), "work too small");
  XNN_REQUIRE((uintptr_t)work % 16 == 0, "work must be aligned to 16 bytes");
  ForwardArgs p{};
  p.x = x;
  p.w = weight;
  p.x_stride = x_stride;
  p.n_in = n_in;
  p.parts = split.parts;
  p.steps = split.steps;
  p.o = Output{bias,       residual, out, slope, (float*)work, GroupView{}, (int)n_rows, n_out,
               activation, __builtin_nanf("")};
  hipStream_t s = as_hip(stream);
  XNN_STORAGE_DISPATCH(dtype, T, XNN_TILE_DISPATCH(kind, T, L, forward_launch<T, L>(p, plan, n_groups, s)));
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

}  // extern "C"
