// Dense layers, forward: out = residual + f(x W + b), with one weight or with that of each row's group
// (gfx950, wave64). The products are dense.h's; bias, activation, its slope for the backward pass and the
// residual are applied to the sums as they leave, so what is written is the result.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "dense.h"

namespace xnn {

struct ForwardArgs {
  const void *x, *w, *bias, *residual;
  void *out, *slope;
  int64_t x_stride, tiles;
  GroupView groups;
  int n_rows, n_in, n_out, activation, tiles_n;
};

template <typename T, typename L>
__global__ __launch_bounds__(kDenseThreads) void dense_forward_kernel(ForwardArgs p) {
  typedef DenseLds<L, T, true, false> S;
  __shared__ __align__(16) char lds[S::kBytes];
  __shared__ int32_t rows[L::BM];
  const int64_t slot = xcd_slot();
  if (slot >= p.tiles) return;
  const int tn = (int)(slot % p.tiles_n);
  const RowTile t = row_tile(p.groups, p.groups.n_groups + 1, p.n_rows, (int)(slot / p.tiles_n), L::BM);
  if (t.group < 0) return;
  const int n0 = tn * L::BN;
  if (p.groups.n_groups > 0 && t.group == p.groups.n_groups) {   // rows of no group
    fill_rows<T, L::BN>(p.groups, t, p.n_rows, (T*)p.out, n0, p.n_out, (T)__builtin_nanf(""));
    return;
  }
  note_rows(p.groups, t, p.n_rows, rows);
  Operator<T, L::BM, L::BK, true> a;
  Operator<T, L::BN, L::BK, false> b;
  a.init(p.x, p.groups.order, p.x_stride, p.n_rows, p.n_in, t.begin, t.end, 0);
  b.init((const T*)p.w + (int64_t)t.group * p.n_in * p.n_out, nullptr, p.n_out, p.n_in, p.n_out, 0, p.n_in, n0);
  f32x16 acc[L::MT][L::NT];
  dense_product<T, L, true, false>(a, b, p.n_in, lds, acc, [](int) {});
  typedef typename Slope<T>::type SlopeType;
  constexpr int N = 16 / sizeof(T);
  int c;
  float bias[N];
  dense_rows<L, N>(
      lds, acc,
      [&](int n) {
        c = n0 + n;
#pragma unroll
        for (int i = 0; i < N; ++i) bias[i] = 0.0f;
        if (p.bias != nullptr && c < p.n_out)
          load_row_part<T, N>((const T*)p.bias + (int64_t)t.group * p.n_out, c, p.n_out, bias);
      },
      [&](int m, float(&v)[N]) {
        const int64_t row = rows[m];
        if (row < 0 || c >= p.n_out) return;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += bias[i];
        if (p.activation != kNone) {
          SlopeType slope[N];
#pragma unroll
          for (int i = 0; i < N; ++i) {
            float s;
            activate(p.activation, v[i], v[i], s);
            slope[i] = slope_stored<T>(s);
          }
          if (p.slope != nullptr)
            store_row_part<SlopeType, N>((SlopeType*)p.slope + row * p.n_out, c, p.n_out, slope);
        }
        if (p.residual != nullptr) {
          float z[N];
          load_row_part<T, N>((const T*)p.residual + row * p.n_out, c, p.n_out, z);
#pragma unroll
          for (int i = 0; i < N; ++i) v[i] += z[i];
        }
        store_row_part<T, N>((T*)p.out + row * p.n_out, c, p.n_out, v);
      });
}

template <typename T, typename L>
static void forward_launch(ForwardArgs p, const int32_t* plan, int n_groups, hipStream_t s) {
  p.groups = group_view(plan, p.n_rows, n_groups, group_level(L::BM));
  p.tiles_n = (p.n_out + L::BN - 1) / L::BN;
  p.tiles = row_tiles(p.n_rows, n_groups, plan != nullptr, L::BM) * p.tiles_n;
  hipLaunchKernelGGL((dense_forward_kernel<T, L>), dim3((unsigned)xcd_blocks(p.tiles)), dim3(kDenseThreads), 0,
                     s, p);
}

}  // namespace xnn

using namespace xnn;

extern "C" {

int xnn_linear(int dtype, const void* x, int64_t x_stride, int64_t n_rows, int32_t n_in, int32_t n_out,
               const void* weight, const void* bias, int32_t activation, const void* residual,
               const int32_t* plan, int32_t n_groups, void* out, void* slope, xnn_stream_t stream) {
  const int status = dense_sizes(dtype, n_rows, n_in, n_out, plan, n_groups);
  if (status != XNN_OK) return status;
  XNN_REQUIRE(activation >= XNN_NO_ACTIVATION && activation <= XNN_TANH, "unknown activation");
  XNN_REQUIRE(slope == nullptr || activation != XNN_NO_ACTIVATION, "no activation has no slope");
  if (n_rows == 0) return XNN_OK;
  XNN_REQUIRE(x && weight && out, "NULL input or output");
  XNN_REQUIRE(x_stride >= n_in, "rows of x overlap");
  ForwardArgs p{};
  p.x = x;
  p.w = weight;
  p.bias = bias;
  p.residual = residual;
  p.out = out;
  p.slope = slope;
  p.x_stride = x_stride;
  p.n_rows = (int)n_rows;
  p.n_in = n_in;
  p.n_out = n_out;
  p.activation = activation;
  hipStream_t s = as_hip(stream);
  const int kind = dense_tile(storage_bytes(dtype), n_rows, n_out, plan != nullptr ? n_groups : 0);
  XNN_STORAGE_DISPATCH(dtype, T, XNN_TILE_DISPATCH(kind, T, L, forward_launch<T, L>(p, plan, n_groups, s)));
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

}  // extern "C"
