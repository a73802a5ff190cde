// Dense layers, forward: out = residual + f(x W + b), with one weight or with that of each row's group
// (gfx950, wave64). The products are dense.h's; bias, activation, its slope for the backward pass and the
// residual are applied to the sums as they leave, so what is written is the result.
//
// Large products are bound by the matrix cores' feed: 8,192^3 in bfloat16 1,005 to 1,020 TFLOP/s, float32 of 8,192
// x 4,096 x 4,096 194 (as six products 1,160). What leaves costs beside them: 24,000 x 1,024 -> 4,096 in bfloat16
// 275 us, with gelu and its slope 376 to 388 (31 vector instructions an element, two of them of four times the
// cycles; 375 MB written). Short reductions are bound by it: 72,000 x 128 -> 512 in float32 with silu and its slope
// 120 to 137 us, 281 MB written.
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
__global__ __launch_bounds__(kDenseThreads, 2) void dense_forward_kernel(ForwardArgs p) {
  typedef DenseLds<L, T, true, false> S;
  __shared__ __align__(16) char lds[S::kBytes];
  __shared__ int32_t rows[L::BM];
  const Output& o = p.o;
  int64_t tiles;
  const int64_t slot = tile_slot(o.groups, p.tiles, p.tiles_n, p.parts, tiles);
  if (slot < 0) return;
  const int part = (int)(slot / tiles), tile = (int)(slot % tiles);
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

// ---------------------------------------------------------------- few rows
// One or two rows (in groups each by itself): a stream of the weight, which bounds it. A block takes a strip of `lanes`
// 16-byte pieces of the columns and the whole reduction, its 512 threads each every 512 / lanes-th row of the
// weight, sixteen of them in flight before the first is used; x lies in LDS as float32. The sums of
// the threads of a column are added across lanes and then waves, in a fixed order. float32 products are float32's
// own here.
constexpr int kFewThreads = 512;

// x[j] += x[j] of the lanes at distances from, 2 from, ... 32
template <int N>
__device__ __forceinline__ void add_lanes_from(float (&x)[N], int from) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (from <= 2) x[j] += dpp_move<0x4E>(x[j]);
    if (from <= 4) x[j] += dpp_move<0x1B>(dpp_move<0x141>(x[j]));   // the half row mirrored, its quads turned back
    if (from <= 8) x[j] += dpp_move<0x128>(x[j]);
    x[j] = add_xor32(add_xor16(x[j]));
  }
}

template <typename T, int MR>
__global__ __launch_bounds__(kFewThreads) void dense_few_kernel(ForwardArgs p, int lanes) {
  constexpr int N = 16 / sizeof(T), LOADS = 16, WAVES = kFewThreads / kWave;
  constexpr int kRound = kFewThreads / 2 * LOADS;          // rows of the weight a round, for the fewest lanes
  __shared__ float xs[MR][kRound];
  __shared__ float sums[WAVES][8][MR * N];
  const Output& o = p.o;
  const int tid = threadIdx.x, lane = tid % lanes, slice = tid / lanes, slices = kFewThreads / lanes;
  const int c = (blockIdx.x * lanes + lane) * N;
  // the block's rows: all, or in groups the blockIdx.y-th in their order
  int group = 0;
  int64_t row0 = 0;
  int rows = o.n_rows;
  if (o.groups.n_groups > 0) {
    const int g = find_group(o.groups.row_ptr, o.groups.n_groups + 1, blockIdx.y);
    row0 = group_row(o.groups, blockIdx.y);
    rows = 1;
    if (row0 < 0 || row0 >= o.n_rows) return;
    if (g == o.groups.n_groups) {
      if (slice == 0)
        for (int i = 0; i < N && c + i < o.width; ++i) ((T*)o.out)[row0 * o.width + c + i] = (T)o.none;
      return;
    }
    group = g;
  }
  const T* x = (const T*)p.x + row0 * p.x_stride;
  const T* w = (const T*)p.w + (int64_t)group * p.n_in * o.width;
  float acc[MR * N];
#pragma unroll
  for (int i = 0; i < MR * N; ++i) acc[i] = 0.0f;
  const int round = min(kRound, slices * LOADS);
  for (int k0 = 0; k0 < p.n_in; k0 += round) {
    u32x4 piece[LOADS];
    const int length = min(round, p.n_in - k0);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int k = slice + i * slices;
      piece[i] = u32x4{0, 0, 0, 0};
      if (k < length && c < o.width)
        piece[i] = load_raw<T>(reinterpret_cast<const char*>(w + (int64_t)(k0 + k) * o.width + c), o.width - c,
                               k0 + k == p.n_in - 1 || o.width < N);
    }
    if (k0 > 0) __syncthreads();
#pragma unroll
    for (int m = 0; m < MR; ++m)
      for (int k = tid; k < length; k += kFewThreads)
        xs[m][k] = m < rows ? (float)x[m * p.x_stride + k0 + k] : 0.0f;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      if (i * slices >= length) break;
      const int k = slice + i * slices;
      const bool in = k < length;                          // else the piece is zero, and so is x, whatever it holds
      const Pack<T, N> v = __builtin_bit_cast(Pack<T, N>, piece[i]);
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        const float f = in ? xs[m][min(k, length - 1)] : 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) acc[m * N + j] = fmaf(f, (float)v.v[j], acc[m * N + j]);
      }
    }
  }
  add_lanes_from<MR * N>(acc, lanes);
  if (tid % kWave < lanes)
#pragma unroll
    for (int i = 0; i < MR * N; ++i) sums[tid / kWave][lane][i] = acc[i];
  __syncthreads();
  const int m = tid / lanes;
  if (m >= rows || m >= MR || c >= o.width) return;
  float v[N], bias[N];
  load_bias<T>(o, group, c, bias);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.0f;
#pragma unroll 4
  for (int q = 0; q < WAVES; ++q)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += sums[q][lane][m * N + i];
  put_row<T>(o, row0 + m, c, v, bias);
}

template <typename T>
static void few_launch(ForwardArgs p, const int32_t* plan, int n_groups, hipStream_t s) {
  constexpr int N = 16 / sizeof(T);
  const int rows = p.o.n_rows;
  p.o.groups = group_view(plan, rows, n_groups, 0);
  // strips of 128 bytes, a line each, where they make 64 blocks; else narrower ones
  int lanes = 8;
  while (lanes > 2 && (p.o.width + lanes * N - 1) / (lanes * N) < 64) lanes /= 2;
  const dim3 grid((p.o.width + lanes * N - 1) / (lanes * N), plan != nullptr ? rows : 1);
#define XNN_FEW_LAUNCH(MR) \
  hipLaunchKernelGGL((dense_few_kernel<T, MR>), grid, dim3(kFewThreads), 0, s, p, lanes)
  if (rows == 1 || plan != nullptr)
    XNN_FEW_LAUNCH(1);
  else
    XNN_FEW_LAUNCH(2);
#undef XNN_FEW_LAUNCH
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
  *bytes = 0;
  if (!few_rows(n_rows, n_in))
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
  const bool few = few_rows(n_rows, n_in);
  const int kind = dense_tile(size, n_rows, n_out, plan != nullptr ? n_groups : 0);
  const Split split = few ? Split{1, 0, 0} : dense_split(size, kind, n_rows, n_out, n_in);
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
               activation, __builtin_nanf(""), past_caches(n_rows, n_out, size)};
  hipStream_t s = as_hip(stream);
  XNN_STORAGE_DISPATCH(dtype, T, {
    if (few)
      few_launch<T>(p, plan, n_groups, s);
    else
      XNN_TILE_DISPATCH(kind, T, L, forward_launch<T, L>(p, plan, n_groups, s));
  });
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

}  // extern "C"
