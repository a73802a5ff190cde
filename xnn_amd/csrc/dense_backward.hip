// Dense layers, backward (gfx950, wave64): with d = g f'(z), the slope f'(z) kept by the forward pass,
//
//   dx = d W^T,   dW = x^T d,   db = sum of d over the rows
//
// of one weight or of each row's group. Where both products need d once (a width of 128 at most in x), they form it
// as they stage it; else a pass over g and the slope does, with db's sums. (Formed in the staging of 24,000 rows of
// 1,024 -> 4,096 in bfloat16, both products 843 us, for the registers, against 529 and 110 for the pass; 72,000
// rows of 128 -> 512 in float32: 217 us, and 189 with 94 for the pass.) A weight's reduction runs over all rows of
// its group: it is cut into parts, one a block, which are added in their order where there is more than one.
// Without the pass db's sums are the weight's product's, taken from what it stages.
//
// Bounds: of large products the matrix cores' feed (8,192^3 in bfloat16 dx 955 to 970, dW 1,040 to 1,090 TFLOP/s:
// dW reads both operands across their rows, by the transposing read, with a tenth of the LDS conflicts), of the
// pass memory (24,000 x 4,096 in bfloat16, 590 MB in 137 us: 4.3 TB/s), of short reductions what is around the
// products (72,000 rows of 128 -> 512 in float32, two species: dx 97 to 116 us, dW 77 to 86, join 10). Weights of
// 64 uneven groups (16,384 rows, 1,024 x 1,024 in bfloat16): with the join 98 to 106 back to back, 115 to 124 within a step, whose
// other kernels have the caches; 134 MB of gradients, and the parts' sums.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "dense.h"

namespace xnn {

struct BackwardArgs {
  const void *g, *slope, *x, *w;   // g: d where there is a slope (the products')
  void *d, *dx, *dw, *db;
  float *part, *part_bias;         // the parts' sums
  int64_t x_stride, tiles, parts;  // parts: of the weight's sums, at most
  GroupView groups, bias_groups;
  int n_rows, n_in, n_out, tiles_m, tiles_n;
  int rows, bias_rows;             // of a part of the weight's sums, of the bias's
  int spread;                      // parts of different lengths: to the XCDs in turn (1), or a part's tiles, so many
  int sums;                        // the weight's product adds up db
  int stream;                      // dw is larger than the caches of the dies
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
// (g, the slope and d once through: 24,000 x 4,096 in bfloat16 132 to 137 us.)
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
#pragma unroll 4
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
template <typename T, typename L, bool TIMES>
__global__ __launch_bounds__(kDenseThreads, 2) void dense_input_kernel(BackwardArgs p, Output o, int parts, int steps) {
  typedef DenseLds<L, T, true, true> S;
  __shared__ __align__(16) char lds[S::kBytes];
  __shared__ int32_t rows[L::BM];
  int64_t tiles;
  const int64_t slot = tile_slot(o.groups, p.tiles, p.tiles_n, parts, tiles);
  if (slot < 0) return;
  const int part = (int)(slot / tiles), tile = (int)(slot % tiles);
  const RowTile t = row_tile(o.groups, o.groups.n_groups + 1, o.n_rows, tile / p.tiles_n, L::BM);
  if (t.group < 0) return;
  const int n0 = tile % p.tiles_n * L::BN;
  if (o.groups.n_groups > 0 && t.group == o.groups.n_groups) {   // rows of no group
    if (part == 0) fill_rows<T, L::BN>(o.groups, t, o.n_rows, (T*)o.out, n0, o.width, (T)o.none);
    return;
  }
  const int k0 = part * steps * L::BK, k1 = min(p.n_out, k0 + steps * L::BK);
  note_rows(o.groups, t, o.n_rows, rows);
  Operator<T, L::BM, L::BK, true, TIMES> a;
  Operator<T, L::BN, L::BK, true> b;
  a.init(p.g, o.groups.order, p.n_out, o.n_rows, p.n_out, t.begin, t.end, k0, p.slope);
  b.init((const T*)p.w + (int64_t)t.group * p.n_in * p.n_out, nullptr, p.n_out, p.n_in, p.n_out, n0,
         min(n0 + L::BN, p.n_in), k0);
  f32x16 acc[L::MT][L::NT];
  dense_product<T, L, true, true>(a, b, k1 - k0, lds, acc, [](int) {});
  put_tile<T, L>(lds, acc, o, parts, part, t.group, rows, n0);
}

// the parts go to the XCDs in turn, a part's tiles to one
__device__ __forceinline__ int64_t slot_of_xcd(int64_t tiles, int64_t& tile) {
  const int64_t i = blockIdx.x / kXcds;
  tile = i % tiles;
  return i / tiles * kXcds + blockIdx.x % kXcds;
}

template <typename T, typename L, bool TIMES, bool ORDERED>
__global__ __launch_bounds__(kDenseThreads, 2) void dense_weight_kernel(BackwardArgs p) {
  typedef DenseLds<L, T, false, false> S;
  __shared__ __align__(16) char lds[S::kBytes];
  const int64_t slot = xcd_slot();
  int64_t part, tile;
  if (p.spread > 1) {
    const int each = p.spread / kXcds, i = (int)(blockIdx.x / kXcds);
    part = i / each;
    tile = (int)(blockIdx.x % kXcds) * each + i % each;
  } else if (p.spread) {
    part = slot_of_xcd(p.tiles_m * p.tiles_n, tile);
  } else {
    part = slot / (p.tiles_m * p.tiles_n);
    tile = slot % (p.tiles_m * p.tiles_n);
  }
  if (part >= p.parts) return;
  const int m0 = (int)(tile / p.tiles_n) * L::BM, n0 = (int)(tile % p.tiles_n) * L::BN;
  const RowTile t = row_tile(p.groups, p.groups.n_groups, p.n_rows, (int)part, p.rows);
  if (t.group < 0) return;
  typedef Operator<T, L::BN, L::BK, false, TIMES, ORDERED> B;
  Operator<T, L::BM, L::BK, false, false, ORDERED> a;
  B b;
  a.init(p.x, p.groups.order, p.x_stride, p.n_rows, p.n_in, t.begin, t.end, m0);
  b.init(p.g, p.groups.order, p.n_out, p.n_rows, p.n_out, t.begin, t.end, n0, p.slope);
  f32x16 acc[L::MT][L::NT];
  const bool bias = p.sums && m0 == 0;
  const int length = t.end - t.begin;
  float sums[B::kPer];
#pragma unroll
  for (int i = 0; i < B::kPer; ++i) sums[i] = 0.0f;
  // two loops: a branch in one would part its loads from its products (TIMES: of one row of tiles, one loop)
  if (TIMES || bias)
    dense_product<T, L, false, false>(a, b, length, lds, acc, [&](int k) { b.add_rows(k, length, sums); });
  else
    dense_product<T, L, false, false>(a, b, length, lds, acc, [](int) {});
  const bool only = part_alone(p.groups, p.n_rows, p.rows, t.group);
  const int64_t at =
      part_slot(p.groups, t.begin, p.rows, p.groups.n_groups > 0 && part == p.groups.tile_ptr[t.group]);
  if (bias) {
    float* s = reinterpret_cast<float*>(lds);                // (kStep, BN)
    store_pack<float, B::kPer>(s + b.row * L::BN + threadIdx.x % B::kChunks * B::kPer, sums);
    __syncthreads();
    for (int i = threadIdx.x; i < L::BN && n0 + i < p.n_out; i += kDenseThreads) {
      float v = 0.0f;
#pragma unroll
      for (int r = 0; r < B::kStep; ++r) v += s[r * L::BN + i];
      if (only)
        ((T*)p.db)[(int64_t)t.group * p.n_out + n0 + i] = (T)v;
      else
        p.part_bias[at * p.n_out + n0 + i] = v;
    }
    __syncthreads();
  }
  T* dw = (T*)p.dw + (int64_t)t.group * p.n_in * p.n_out;
  float* sum = p.part + at * p.n_in * p.n_out;
  int c;
  if (only) {
    constexpr int N = 16 / sizeof(T);
    dense_rows<L, N>(
        lds, acc, [&](int n) { c = n0 + n; },
        [&](int m, float(&v)[N]) {
          if (m0 + m >= p.n_in || c >= p.n_out) return;
          if (p.stream)
            store_row_part<T, N, true>(dw + (int64_t)(m0 + m) * p.n_out, c, p.n_out, v);
          else
            store_row_part<T, N>(dw + (int64_t)(m0 + m) * p.n_out, c, p.n_out, v);
        });
  } else {
    dense_rows<L, 4>(
        lds, acc, [&](int n) { c = n0 + n; },
        [&](int m, float(&v)[4]) {
          if (m0 + m < p.n_in && c < p.n_out)
            store_row_part<float, 4>(sum + (int64_t)(m0 + m) * p.n_out, c, p.n_out, v);
        });
  }
}

// ---------------------------------------------------------------- the parts
// the parts of a group, and where its sorted rows begin
__device__ __forceinline__ int group_parts(const GroupView& v, int n_rows, int rows, int group, int& begin) {
  begin = 0;
  if (v.n_groups == 0) return (n_rows + rows - 1) / rows;
  begin = min(max(v.row_ptr[group], 0), n_rows);
  return min((int)((uint32_t)v.tile_ptr[group + 1] - (uint32_t)v.tile_ptr[group]), (n_rows - begin + rows - 1) / rows);
}

// part n of the group whose sorted rows begin at `begin`: as part_slot(begin + n rows)
struct PartSlots {
  int64_t first, next, step;
  __device__ __forceinline__ PartSlots(const GroupView& v, int begin, int rows)
      : first(part_slot(v, begin, rows, true)), next(part_slot(v, begin, rows, false)), step(v.n_groups == 0 ? 1 : 2) {}
  __device__ __forceinline__ int64_t operator()(int n) const { return n == 0 ? first : next + n * step; }
};

// call(group, its parts, its first sorted row) for those groups set, set + sets, ... whose gradients no part has
// written by itself, 64 looked at at a time; all threads of a block go the same way
template <typename F>
__device__ __forceinline__ void unfinished_groups(const GroupView& v, int n_rows, int rows, int n_groups, int set,
                                                  int sets, F&& call) {
  for (int g0 = set; g0 < n_groups; g0 += sets * kWave) {
    const int g = g0 + (int)(threadIdx.x % kWave) * sets;
    int begin = 0, parts = 1;
    if (g < n_groups) parts = group_parts(v, n_rows, rows, g, begin);
    for (uint64_t todo = __ballot(parts != 1); todo != 0; todo &= todo - 1) {
      const int lane = __builtin_ctzll(todo);
      call(g0 + lane * sets, __builtin_amdgcn_readlane(parts, lane), __builtin_amdgcn_readlane(begin, lane));
    }
  }
}

// The parts of a weight and of its bias added in their order, zeros where there is none; a group's only part is done.
// The blocks of a weight, then those of its bias, sixteen columns each, whose parts may be many: sixteen of them at
// a time, then those sums in order. A block looks through a set of the groups: one for each group cost 38 us with
// 64 groups of 1,024 x 1,024 in bfloat16, most of them done; 11 so.
template <typename T>
__global__ __launch_bounds__(256) void dense_join_kernel(BackwardArgs p, int n_groups, int weight_blocks,
                                                         int weight_sets, int bias_blocks, int bias_sets) {
  const int weights = weight_blocks * weight_sets;
  if ((int)blockIdx.x >= weights) {
    __shared__ float s[16][17];
    const int block = (blockIdx.x - weights) % bias_blocks, set = (blockIdx.x - weights) / bias_blocks;
    const int x = threadIdx.x % 16, y = threadIdx.x / 16, c = block * 16 + x;
    unfinished_groups(p.bias_groups, p.n_rows, p.bias_rows, n_groups, set, bias_sets, [&](int g, int parts, int begin) {
      const PartSlots slot(p.bias_groups, begin, p.bias_rows);
      float v = 0.0f;
      if (c < p.n_out)
#pragma unroll 4
        for (int n = y; n < parts; n += 16) v += p.part_bias[slot(n) * p.n_out + c];
      s[y][x] = v;
      __syncthreads();
      if (y == 0 && c < p.n_out) {
        v = 0.0f;
#pragma unroll
        for (int q = 0; q < 16; ++q) v += s[q][x];
        ((T*)p.db)[(int64_t)g * p.n_out + c] = (T)v;
      }
      __syncthreads();
    });
    return;
  }
  const int block = blockIdx.x % weight_blocks, set = blockIdx.x / weight_blocks;
  const int64_t size = (int64_t)p.n_in * p.n_out;
  unfinished_groups(p.groups, p.n_rows, p.rows, n_groups, set, weight_sets, [&](int g, int parts, int begin) {
    T* dw = (T*)p.dw + g * size;
    const PartSlots slot(p.groups, begin, p.rows);
    for (int64_t k = ((int64_t)block * 256 + threadIdx.x) * 4; k < size; k += (int64_t)weight_blocks * 1024) {
      const int count = (int)min((int64_t)4, size - k);
      const float* from = p.part + k;
      float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      const auto add = [&](int n) {
        const Pack<float, 4> x = load_piece<float, 4>(from + slot(n) * size);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += x.v[i];
      };
      if (count == 4) {            // eight loads in flight
        if (parts > 0) add(0);
        int n = 1;
        for (; n + 8 <= parts; n += 8) {
#pragma unroll
          for (int i = 0; i < 8; ++i) add(n + i);
        }
        for (; n < parts; ++n) add(n);
      } else {
        for (int n = 0; n < parts; ++n)
          for (int i = 0; i < 4; ++i) v[i] += i < count ? from[slot(n) * size + i] : 0.0f;
      }
      store_row_part<T, 4>(dw + k, 0, count, v);
    }
  });
}

// ---------------------------------------------------------------- host side
struct Parts {
  int rows;
  int64_t slots;                   // parts that have sums of their own
};
// Parts of at least `least` rows, about `want` of them; in groups of a level's rows (the plan has their tiles)
static Parts parts_of(int64_t n_rows, bool grouped, int64_t want, int64_t least) {
  int64_t rows = std::max<int64_t>(least, (n_rows + want - 1) / std::max<int64_t>(want, 1));
  Parts w;
  if (grouped) {
    rows = level_rows(group_level(rows));
    w.slots = n_rows <= rows ? 0 : 2 * (n_rows / rows + 1);
  } else {
    rows = (rows + 63) / 64 * 64;
    w.slots = n_rows <= rows ? 0 : (n_rows + rows - 1) / rows;
  }
  w.rows = (int)std::min<int64_t>(rows, 1 << 30);
  return w;
}

// the width of x up to which the products form d themselves: a tile of both
constexpr int kFormInProducts = 128;

struct BackwardPlan {
  int input_kind, kind;            // of the input's tiles, of the weight's
  Split split;                     // of the input's reduction, whose sums are gone before the weight's are there
  Parts weight, bias;
  bool pass;                       // forms d
  size_t bytes;                    // of the weight's parts, the bias's, d
  size_t bias_at, d_at;
  int64_t blocks;                  // of the largest launch, at most
};
static BackwardPlan backward_plan(int dtype, int64_t n_rows, int32_t n_in, int32_t n_out, int64_t n_groups,
                                  bool grouped, bool slope, bool input, bool weight, bool bias) {
  BackwardPlan b{};
  const int64_t size = storage_bytes(dtype);
  const auto tiles = [&](int64_t bm, int64_t bn) { return ((n_in + bm - 1) / bm) * ((n_out + bn - 1) / bn); };
  if (weight) {
    // The tiles and the number of parts with the least time, estimated from the rates of large products (kinds 0,
    // 1, 2: microseconds of 64 rows of a tile with all of a CU's blocks at work, and those blocks) and the parts'
    // sums, written and read at 4 TB/s. Parts of one length come in rounds; those of groups, of any, fill the card
    // but for about one long one's time and a half at its end. Weights of groups take tiles of up to 128 x 128 (256 x 128
    // cost 14 % at 64 uneven groups, 30 % at four even ones). 64 x 64 tiles of groups cost a third more than of one
    // weight, for each looks up its rows: bfloat16, with the join, 64 x 64 and 128 x 128 (chosen: *) of 5,000 rows of
    // four species, 256 -> 128 10.8* and 13.7 us, 256 -> 512 20.7 and 19.5*; 72,000 of two, 256 -> 128 33 and 27*, 512 ->
    // 512 120 and 78*; 16,384 of 64 uneven groups 128 -> 128 12.8* and 14.9, 256 -> 128 18.6* and 17.3, 1,024 -> 1,024
    // 147 and 98*. Of one weight 40 sizes from 21 x 128 -> 128 to 72,000 x 2,048 -> 2,048 take the better kind or one within
    // 4 %. (In 16 bits a third block of 128 x 128 fits a CU; the step counted is that of two, which it does not change.)
    static const double step16[] = {0.9, 1.4, 2.2}, step32[] = {2.9, 5.4, 0.0}, grouped16 = 1.2;
    static const int per_cu[] = {3, 2, 2}, bm[] = {64, 128, 256}, bn[] = {64, 128, 128};
    const double sums = (double)n_in * n_out * 8 / 4e6;
    double best = 0.0;
    for (int kind = 0; kind < (size == 2 && !grouped && !(slope && n_in <= kFormInProducts) ? 3 : 2); ++kind) {
      const double t = (double)tiles(bm[kind], bn[kind]), blocks = 256.0 * per_cu[kind];
      const double step = size == 4 ? step32[kind] : grouped && kind == kTile64 ? grouped16 : step16[kind];
      for (int64_t want = 1; want <= 1024; want += std::max<int64_t>(1, want / 4)) {
        const Parts parts = parts_of(n_rows, grouped, want, 256);
        const double n = (double)row_tiles(n_rows, 0, false, parts.rows), all = n + (grouped ? n_groups / 2 : 0);
        const double steps = (double)std::min<int64_t>(parts.rows, n_rows) / 64 + 2;   // and two for what is around
        double time = std::max(1.0, std::ceil(all * t / blocks)) * steps * step;
        if (grouped && all * t > blocks)
          time = ((double)n_rows / 64 + 2 * all) * t / blocks * step + 1.4 * steps * step;
        if (parts.slots > 0) time += 5.0 + sums * n;
        if (best == 0.0 || time < best) {
          best = time;
          b.kind = kind;
          b.weight = parts;
        }
        if (parts.slots > 0 && parts.rows <= 256) break;
      }
    }
  }
  b.pass = slope && n_in > kFormInProducts;
  b.input_kind = dense_tile(size, n_rows, n_in, grouped ? n_groups : 0);
  if (slope && !b.pass) b.input_kind = std::min<int>(b.input_kind, kTile128);
  b.split = dense_split(size, b.input_kind, n_rows, n_in, n_out);
  b.bias = b.weight;
  // sixteen blocks a CU of 512 bytes of the columns each
  if (b.pass) b.bias = parts_of(n_rows, grouped, std::max<int64_t>(1, 4096 / ((n_out * size + 511) / 512)), 64);
  if (weight)
    b.blocks = (row_tiles(n_rows, n_groups, grouped, b.weight.rows) + kXcds) *
               (b.kind == kTile64 ? tiles(64, 64) : b.kind == kTile128 ? tiles(128, 128) : tiles(256, 128));
  if (b.pass)
    b.blocks = std::max(b.blocks, row_tiles(n_rows, n_groups, grouped, b.bias.rows) * ((n_out * size + 511) / 512));
  const auto room = [](size_t n) { return (n + 255) / 256 * 256; };
  b.bias_at = std::max(room((size_t)b.weight.slots * n_in * n_out * sizeof(float)), input ? room(b.split.bytes) : 0);
  b.d_at = b.bias_at + (bias ? room((size_t)b.bias.slots * n_out * sizeof(float)) : 0);
  b.bytes = b.d_at + (b.pass ? (size_t)n_rows * n_out * size : 0);
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
static void input_launch(BackwardArgs p, const Split& split, const int32_t* plan, int n_groups, hipStream_t s) {
  Output o{nullptr, nullptr, p.dx, nullptr, p.part, GroupView{}, p.n_rows, p.n_in, kNone, 0.0f,
           past_caches(p.n_rows, p.n_in, sizeof(T))};
  o.groups = group_view(plan, p.n_rows, n_groups, group_level(L::BM));
  p.tiles_n = (p.n_in + L::BN - 1) / L::BN;
  p.tiles = row_tiles(p.n_rows, n_groups, plan != nullptr, L::BM) * p.tiles_n;
  const int steps = split.parts > 1 ? split.steps : (p.n_out + L::BK - 1) / L::BK;
  const dim3 grid((unsigned)xcd_blocks(p.tiles * split.parts));
  if (p.slope == nullptr)
    hipLaunchKernelGGL((dense_input_kernel<T, L, false>), grid, dim3(kDenseThreads), 0, s, p, o, split.parts, steps);
  else if constexpr (L::BM <= 128)
    hipLaunchKernelGGL((dense_input_kernel<T, L, true>), grid, dim3(kDenseThreads), 0, s, p, o, split.parts, steps);
  if (split.parts > 1) parts_launch<T>(o, plan, n_groups, split.parts, s);
}

// Groups of different sizes have parts of different lengths, the long ones next to each other: spread over the XCDs
// where there are enough of them (16,384 rows in 64 uneven groups, 1,024 x 1,024 in bfloat16: 212 us, in turn 161), and
// where a weight's tiles are a multiple of eight each part's over all XCDs, whose work is then the same (those in turn had
// up to 1.7 times the mean: with the join 134 us, so 117; even groups 79 and 83, for x and d read by each XCD).
template <typename T, typename L>
static void weight_launch(BackwardArgs p, const int32_t* plan, int n_groups, hipStream_t s) {
  p.tiles_m = (p.n_in + L::BM - 1) / L::BM;
  p.tiles_n = (p.n_out + L::BN - 1) / L::BN;
  p.parts = row_tiles(p.n_rows, n_groups, plan != nullptr, p.rows);
  p.spread = plan != nullptr && p.parts >= 4 * kXcds;
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  if (p.spread && tiles % kXcds == 0) p.spread = (int)tiles;
  const int64_t blocks = p.spread == 1 ? xcd_blocks(p.parts) * tiles : xcd_blocks(p.parts * tiles);
  const dim3 grid((unsigned)blocks), threads(kDenseThreads);
  // 256 x 128 tiles are of one weight, and of a d that is there
  if (plan == nullptr && p.slope == nullptr) {
    hipLaunchKernelGGL((dense_weight_kernel<T, L, false, false>), grid, threads, 0, s, p);
  } else if constexpr (L::BM <= 128) {
    if (plan == nullptr)
      hipLaunchKernelGGL((dense_weight_kernel<T, L, true, false>), grid, threads, 0, s, p);
    else if (p.slope == nullptr)
      hipLaunchKernelGGL((dense_weight_kernel<T, L, false, true>), grid, threads, 0, s, p);
    else
      hipLaunchKernelGGL((dense_weight_kernel<T, L, true, true>), grid, threads, 0, s, p);
  }
}

}  // namespace xnn

using namespace xnn;

extern "C" {

int xnn_linear_backward_work_size(int dtype, int64_t n_rows, int32_t n_in, int32_t n_out, int32_t n_groups,
                                  int32_t grouped, int32_t slope, int32_t input, int32_t weight, int32_t bias,
                                  size_t* bytes) {
  static const int32_t some = 0;
  const int status = dense_sizes(dtype, n_rows, n_in, n_out, &some, n_groups);
  if (status != XNN_OK) return status;
  XNN_REQUIRE(bytes != nullptr, "NULL size");
  const BackwardPlan b = backward_plan(dtype, n_rows, n_in, n_out, n_groups, grouped != 0, slope != 0, input != 0,
                                       weight != 0, bias != 0);
  XNN_REQUIRE(b.blocks < kMaxBlocks, "too many tiles");
  *bytes = b.bytes;
  return XNN_OK;
}

int xnn_linear_variants(int dtype, int64_t n_rows, int32_t n_in, int32_t n_out, int32_t n_groups, int32_t grouped,
                        int32_t slope, xnn_linear_variant* out) {
  static const int32_t some = 0;
  const int status = dense_sizes(dtype, n_rows, n_in, n_out, &some, n_groups);
  if (status != XNN_OK) return status;
  XNN_REQUIRE(n_rows > 0, "no rows");
  XNN_REQUIRE(out != nullptr, "NULL variant");
  const size_t size = storage_bytes(dtype);
  const bool few = few_rows(n_rows, n_in);
  const int kind = dense_tile(size, n_rows, n_out, grouped ? n_groups : 0);
  const BackwardPlan b =
      backward_plan(dtype, n_rows, n_in, n_out, n_groups, grouped != 0, slope != 0, true, true, true);
  *out = xnn_linear_variant{few ? 0 : 64 << kind, few ? 1 : dense_split(size, kind, n_rows, n_out, n_in).parts,
                            64 << b.input_kind, b.split.parts, 64 << b.kind,
                            (int32_t)row_tiles(n_rows, n_groups, grouped != 0, b.weight.rows), b.weight.rows, b.pass};
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
  XNN_REQUIRE(dbias == nullptr || dweight != nullptr, "the bias's gradient goes with the weight's");
  if (dweight == nullptr && (dx == nullptr || n_rows == 0)) return XNN_OK;
  const bool grouped = plan != nullptr && n_rows > 0;
  const BackwardPlan b = backward_plan(dtype, n_rows, n_in, n_out, n_groups, grouped, slope != nullptr, dx != nullptr,
                                       dweight != nullptr, dbias != nullptr);
  XNN_REQUIRE(b.blocks < kMaxBlocks, "too many tiles");
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
  p.sums = dbias != nullptr && !b.pass;
  p.stream = past_caches((int64_t)n_groups * n_in, n_out, storage_bytes(dtype));
  XNN_STORAGE_DISPATCH(dtype, T, {
    if (b.pass && n_rows > 0) {
      cotangent_launch<T>(p, order, n_groups, s);
      p.g = p.d;
      p.slope = nullptr;
    }
    if (n_rows > 0 && dx != nullptr) XNN_TILE_DISPATCH(b.input_kind, T, L, input_launch<T, L>(p, b.split, order, n_groups, s));
    if (n_rows > 0 && dweight != nullptr)
      XNN_TILE_DISPATCH(b.kind, T, L, weight_launch<T, L>(p, order, n_groups, s));
    // groups without rows have zeros, parts have sums
    if (dweight != nullptr &&
        (grouped || b.weight.slots > 0 || n_rows == 0 || (dbias != nullptr && b.bias.slots > 0))) {
      const int blocks = (int)std::min<int64_t>(((int64_t)n_in * n_out + 1023) / 1024, 4096);
      const int bias_blocks = dbias != nullptr ? (n_out + 15) / 16 : 0;
      const auto sets = [&](int of) { return std::max(1, std::min(n_groups, 4096 / std::max(of, 1))); };
      hipLaunchKernelGGL(dense_join_kernel<T>, dim3(blocks * sets(blocks) + bias_blocks * sets(bias_blocks)),
                         dim3(256), 0, s, p, n_groups, blocks, sets(blocks), bias_blocks, sets(bias_blocks));
    }
  });
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

}  // extern "C"
