// Matrix products of a dense layer on tiles, shared by its forward and backward kernels (gfx950, wave64).
//
//   forward   out = residual + f(x W + b)    rows of x (reduction along them)    x  W read across its rows
//   input     dx  = d W^T,  d = g f'(z)      rows of g                           x  rows of W
//   weight    dW  = x^T d                    x read across its rows              x  d read across its rows
//
// A block owns a tile of the output and walks the reduction in steps that all its threads stage in LDS,
// every operand as it lies in memory: rows along the reduction are read back 16 bytes a lane, rows
// across it by the transposing LDS read, and both give a lane the same eight reduction indices. The
// global loads of the next step are in registers while the matrix cores work on this one.
// v_mfma_f32_32x32x16 with float32 sums. float32 operands are taken apart into three bfloat16 planes as they
// are staged, each the rounded rest of those before: x = h + m + l with |m| <= 2^-8 |x| and |l| <= 2^-16 |x|.
// Of the nine products of planes the six of order 2^-16 and larger are formed (mma in attention.h); those left
// out are below 2^-23 of |x w| together, about a float32 rounding of it. An operand that is not finite, or
// rounds to infinity in bfloat16 (above 3.39e38), makes the outputs it enters NaN.
//
// Rows of groups (the species of an atom, its expert) are gathered as they are staged and scattered as they
// are stored: no copy in sorted order is made. Rows and columns beyond an output's edge are loaded from
// places that exist and never stored; indices beyond the reduction become zeros in both operands.
#pragma once
#include <hip/hip_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "attention.h"
#include "common.h"
#include "device.h"
#include "storage.h"

namespace xnn {

constexpr int kDenseThreads = 256;
constexpr int kDenseWaves = kDenseThreads / kWave;

// ---------------------------------------------------------------- groups
// What xnn_group_plan leaves, in int32: `order`, the rows by group (stable); row_ptr (n_groups + 2), where a
// group's rows begin, the last bucket holding the rows of no group; for each level s the prefix sums of the
// groups' tiles of 32 << s rows.
constexpr int kGroupLevels = 16;
constexpr int kMaxGroups = 4096;

struct GroupView {
  const int32_t *order, *row_ptr, *tile_ptr;   // tile_ptr of the level in use
  int n_groups;                                // 0: one weight, rows in their order
};

inline GroupView group_view(const int32_t* plan, int64_t n_rows, int n_groups, int level) {
  GroupView v{};
  if (plan == nullptr) return v;
  v.order = plan;
  v.row_ptr = plan + n_rows;
  v.tile_ptr = v.row_ptr + (int64_t)(level + 1) * (n_groups + 2);
  v.n_groups = n_groups;
  return v;
}
inline int64_t group_plan_ints(int64_t n_rows, int64_t n_groups) {
  return n_rows + (kGroupLevels + 1) * (n_groups + 2);
}

// the g with p[g] <= t < p[g + 1] among n; all lanes of the wave look at 64 places at once
__device__ __forceinline__ int find_group(const int32_t* __restrict__ p, int n, int t) {
  const int lane = threadIdx.x % kWave;
  int lo = 0, len = n;
  while (len > 1) {
    const int step = (len + kWave - 1) / kWave, at = lane * step;
    const int v = at < len ? p[lo + at] : INT_MAX;
    const int k = __popcll(__ballot(v <= t)) - 1;
    lo += k * step;
    len = min(step, len - k * step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// Rows of one tile: sorted positions [begin, end) of group g (g < 0: no such tile). A plan is taken as it is
// given: one that is not of these rows gives wrong results, and reaches nothing outside them.
struct RowTile {
  int begin, end, group;
};
__device__ __forceinline__ RowTile row_tile(const GroupView& v, int n_buckets, int n_rows, int t, int size) {
  if (v.n_groups == 0) {
    const int begin = t * size;
    return RowTile{begin, min(n_rows, begin + size), 0};
  }
  if (t >= v.tile_ptr[n_buckets]) return RowTile{0, 0, -1};
  const int g = find_group(v.tile_ptr, n_buckets, t);
  const int begin = max(0, v.row_ptr[g] + (t - v.tile_ptr[g]) * size);
  const int end = min(min(v.row_ptr[g + 1], n_rows), begin + size);
  return RowTile{begin, end, begin < end ? g : -1};
}

__device__ __forceinline__ int64_t group_row(const GroupView& v, int r) {
  return v.order == nullptr ? r : v.order[r];
}

// the tile's columns [n0, n0 + BN) of the tile's rows, all of one value
template <typename T, int BN>
__device__ __forceinline__ void fill_rows(const GroupView& v, const RowTile& t, int n_rows, T* out, int n0,
                                          int width, T value) {
  for (int i = threadIdx.x; i < (t.end - t.begin) * BN; i += blockDim.x) {
    const int c = n0 + i % BN;
    const int64_t row = group_row(v, t.begin + i / BN);
    if (c < width && row >= 0 && row < n_rows) out[row * width + c] = value;
  }
}

// ---------------------------------------------------------------- activations
enum Activation : int { kNone = 0, kSilu = 1, kGelu = 2, kTanh = 3 };

// f(z) and f'(z)
__device__ __forceinline__ void activate(int kind, float z, float& y, float& slope) {
  if (kind == kSilu) {
    // the exponential's error is |z| 2^-24 of it, p (1 - p) |z| < 1/4 of that in p
    const float p = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * z));
    y = z * p;
    slope = p * fmaf(z, 1.0f - p, 1.0f);
  } else if (kind == kGelu) {
    const float c = fmaf(0.5f, erff(0.70710678118654752f * z), 0.5f);
    y = z * c;
    slope = fmaf(z * 0.39894228040143268f, __builtin_amdgcn_exp2f(-0.5f * kLog2e * z * z), c);
  } else if (kind == kTanh) {
    y = tanhf(z);
    slope = fmaf(-y, y, 1.0f);
  } else {
    y = z;
    slope = 1.0f;
  }
}

// ---------------------------------------------------------------- sizes
// BK: 64 elements of the reduction a step in 16 bits, 32 in float32 (eight 16-byte pieces of a row each)
template <typename T, int BM_, int BN_, int WM_, int WN_>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, kWavesM = WM_, kWavesN = WN_;
  static constexpr int MT = BM / WM_ / 32, NT = BN / WN_ / 32;   // 32 x 32 products of a wave
  static constexpr int BK = 128 / sizeof(T);
  static constexpr int kPer = 16 / sizeof(T);
  static constexpr int kPlanes = Store<T>::kPlanes;
  static_assert(WM_ * WN_ == kDenseWaves, "");
};

// an operand in LDS: ROWS outer indices
template <typename T, int ROWS, bool ALONG>
struct Place;
template <typename T, int ROWS>
struct Place<T, ROWS, true> {      // rows along the reduction; 16 bytes more spread the banks
  static constexpr int BK = 128 / sizeof(T);
  static constexpr int kRow = BK * 2 + 16, kPlane = ROWS * kRow;
  static constexpr int kBytes = kPlane * Store<T>::kPlanes;
};
template <typename T, int ROWS>
struct Place<T, ROWS, false> {     // rows across it; 64 more: four rows of a transposing read on other banks
  static constexpr int BK = 128 / sizeof(T);
  static constexpr int kRow = ROWS * 2 + 64, kPlane = BK * kRow;
  static constexpr int kBytes = kPlane * Store<T>::kPlanes;
};

// ---------------------------------------------------------------- staging
// the planes of two float32: 11 instructions
__device__ __forceinline__ void rounded_planes(float a, float b, uint32_t (&out)[3]) {
  typedef bf16_t Two __attribute__((ext_vector_type(2)));
  f32x2 x = {a, b};
#pragma unroll
  for (int n = 0; n < 3; ++n) {
    out[n] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, Two));
    x[0] -= __uint_as_float(out[n] << 16);
    x[1] -= __uint_as_float(out[n] & 0xFFFF0000u);
  }
}

// One 16-byte piece to LDS: as it is, or in three planes of half the bytes
template <typename T, int N>
__device__ __forceinline__ void put_piece(char* at, int plane, const Pack<T, N>& x) {
  if constexpr (sizeof(T) == 4) {
    uint32_t a[3], b[3];
    rounded_planes(x.v[0], x.v[1], a);
    rounded_planes(x.v[2], x.v[3], b);
#pragma unroll
    for (int n = 0; n < 3; ++n) *reinterpret_cast<u32x2*>(at + n * plane) = u32x2{a[n], b[n]};
  } else {
    *reinterpret_cast<Pack<T, N>*>(at) = x;
  }
}

// Pieces need no alignment (the loads are unaligned ones, at full rate where the address happens to be aligned).
// One that reaches beyond its row's `width` elements is within the tensor where another row follows; the last
// row's is taken element by element.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_piece(const T* p) {
  Pack<T, N> x;
  __builtin_memcpy(&x, p, sizeof(x));
  return x;
}
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_piece(const T* row, int at, int width, bool last) {
  if (at + N <= width || (at < width && !last)) return load_piece<T, N>(row + at);
  Pack<T, N> x;
#pragma unroll
  for (int i = 0; i < N; ++i) x.v[i] = at + i < width ? row[at + i] : (T)0.0f;
  return x;
}

// One operand on its way: a matrix of `tensor_rows` rows of `width` elements, row r at data + r stride (and
// the factor of d beside it, of the same layout), of which LEN rows or columns are this tile's. ALONG: the
// tile's rows, along which the reduction runs; else its columns, and the reduction runs over the rows. Row r of
// the tile, or of the reduction, is order[first + r], or first + r without an order.
template <typename T, int LEN, bool ALONG, bool TIMES>
struct Operator {
  static constexpr int BK = 128 / sizeof(T), kPer = 16 / sizeof(T);
  static constexpr int kRows = ALONG ? LEN : BK, kCols = ALONG ? BK : LEN;   // of a staged step
  static constexpr int kChunks = kCols / kPer;
  static constexpr int kStep = kDenseThreads / kChunks;
  static constexpr int kCount = kRows / kStep;
  static_assert(kDenseThreads % kChunks == 0 && kRows % kStep == 0, "");
  typedef Pack<T, kPer> Piece;
  typedef Place<T, LEN, ALONG> At;

  const T *data, *factor;
  const int32_t* order;
  int64_t stride;
  int width, row, at, first, end, last;   // last: the tensor's last row
  bool whole;                      // no piece reaches beyond its row
  int32_t index[kCount];           // rows of the next step (ALONG: of all)
  Piece x[kCount], y[TIMES ? kCount : 1];

  // rows [first_row, end_row), columns from first_col on
  __device__ __forceinline__ void init(const void* data_, const void* factor_, const int32_t* order_,
                                       int64_t stride_, int tensor_rows, int width_, int first_row,
                                       int end_row, int first_col) {
    data = (const T*)data_;
    factor = (const T*)factor_;
    order = order_;
    stride = stride_;
    last = tensor_rows - 1;
    width = width_;
    row = threadIdx.x / kChunks;
    at = first_col + threadIdx.x % kChunks * kPer;
    if (!ALONG && at >= width) at = 0;                     // columns beyond the edge: any that exist
    first = first_row;
    end = end_row - first_row;
    whole = width % kPer == 0;
    look(0);
  }
  // the rows that the step from reduction index k0 on reads
  __device__ __forceinline__ void look(int k0) {
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const int r = first + min((ALONG ? 0 : k0) + row + n * kStep, end - 1);
      index[n] = order == nullptr ? r : min(max(order[r], 0), last);
    }
  }
  // the step from reduction index k0 on (across the rows: that of the last look)
  __device__ __forceinline__ void fetch(int k0) {
    const int col = ALONG ? at + k0 : at;
    if (whole && (!ALONG || k0 + BK <= width)) {
#pragma unroll
      for (int n = 0; n < kCount; ++n) {
        const int64_t i = index[n] * stride + col;
        x[n] = load_piece<T, kPer>(data + i);
        if constexpr (TIMES) y[n] = load_piece<T, kPer>(factor + i);
      }
    } else {
#pragma unroll
      for (int n = 0; n < kCount; ++n) {
        const int64_t i = index[n] * stride;
        const bool edge = index[n] == last || stride < kPer;
        x[n] = load_piece<T, kPer>(data + i, col, width, edge);
        if constexpr (TIMES) y[n] = load_piece<T, kPer>(factor + i, col, width, edge);
      }
    }
    if (!ALONG) look(k0 + BK);
  }
  // to LDS, zeros beyond the reduction's `length`; sums: of each of the thread's columns, added to
  template <bool SUMS = false>
  __device__ __forceinline__ void commit(char* lds, int k0, int length, float* sums = nullptr) {
    const bool tail = k0 + BK > length;
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const int r = row + n * kStep, c = threadIdx.x % kChunks * kPer;
      float v[kPer];
      Piece out;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        out.v[i] = x[n].v[i];
        if constexpr (TIMES) out.v[i] = (T)(v[i] = (float)x[n].v[i] * (float)y[n].v[i]);
      }
      if (tail) {
        const int left = ALONG ? length - k0 - c : k0 + r < length ? kPer : 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (i >= left) {
            out.v[i] = (T)0.0f;
            v[i] = 0.0f;
          }
      }
      if constexpr (SUMS)
#pragma unroll
        for (int i = 0; i < kPer; ++i) sums[i] += TIMES ? v[i] : (float)out.v[i];
      put_piece<T, kPer>(lds + r * At::kRow + c * 2, At::kPlane, out);
    }
  }
};

// operand `step` of 16 reduction indices for the 32 outer indices from `outer` on
template <typename T, int LEN, bool ALONG>
__device__ __forceinline__ Operand<T> dense_operand(const char* lds, int outer, int step) {
  typedef Place<T, LEN, ALONG> At;
  const int lane = threadIdx.x % kWave, half = lane / 32;
  Operand<T> out;
  if constexpr (ALONG) {
    const char* p = lds + (outer + lane % 32) * At::kRow + 32 * step + 16 * half;
#pragma unroll
    for (int n = 0; n < Store<T>::kPlanes; ++n)
      out.p[n] = *reinterpret_cast<const Frag<T>*>(p + n * At::kPlane);
  } else {
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    const int l = lane % 16;
    const char* p = lds + (16 * step + 8 * half + l / 4) * At::kRow +
                    (outer + 16 * ((lane / 16) & 1) + 4 * (l % 4)) * 2;
#pragma unroll
    for (int n = 0; n < Store<T>::kPlanes; ++n) {
      const char* q = p + n * At::kPlane;
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)q);
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(q + 4 * At::kRow));
      out.p[n] = __builtin_bit_cast(Frag<T>, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
  return out;
}

// ---------------------------------------------------------------- the product
// LDS of a block: one stage of both operands, and the waves' rows on their way out
template <typename L, typename T, bool ALONG_A, bool ALONG_B>
struct DenseLds {
  static constexpr int kA = Place<T, L::BM, ALONG_A>::kBytes, kB = Place<T, L::BN, ALONG_B>::kBytes;
  static constexpr int kOutRow = L::NT * 32 + 4;                         // floats
  static constexpr int kOut = kDenseWaves * 32 * kOutRow * 4;
  static constexpr int kStages = 2 * (kA + kB) <= 150 * 1024 && sizeof(T) == 2 ? 2 : 1;
  static constexpr int kBytes = kStages * (kA + kB) > kOut ? kStages * (kA + kB) : kOut;
};

// acc = the reduction over [k_begin, k_end) of `length` indices; SUMS: b's columns added up in `sums`
template <typename T, typename L, bool ALONG_A, bool ALONG_B, bool SUMS, typename A, typename B>
__device__ __forceinline__ void dense_product(A& a, B& b, int k_begin, int k_end, int length, char* lds,
                                              f32x16 (&acc)[L::MT][L::NT], float* sums = nullptr) {
  typedef DenseLds<L, T, ALONG_A, ALONG_B> S;
  constexpr int BK = L::BK;
  const int wave = wave_in_block();
  const int m0 = wave / L::kWavesN * L::MT * 32, n0 = wave % L::kWavesN * L::NT * 32;
#pragma unroll
  for (int i = 0; i < L::MT; ++i)
#pragma unroll
    for (int j = 0; j < L::NT; ++j) acc[i][j] = f32x16{};
  if (k_begin >= k_end) return;
  const auto compute = [&](const char* s) {
#pragma unroll
    for (int step = 0; step < BK / 16; ++step) {
      Operand<T> fa[L::MT], fb[L::NT];
#pragma unroll
      for (int i = 0; i < L::MT; ++i) fa[i] = dense_operand<T, L::BM, ALONG_A>(s, m0 + 32 * i, step);
#pragma unroll
      for (int j = 0; j < L::NT; ++j) fb[j] = dense_operand<T, L::BN, ALONG_B>(s + S::kA, n0 + 32 * j, step);
#pragma unroll
      for (int i = 0; i < L::MT; ++i)
#pragma unroll
        for (int j = 0; j < L::NT; ++j) mma<T>(fa[i], fb[j], acc[i][j]);
    }
  };
  const auto commit = [&](char* s, int k) {
    a.commit(s, k, length);
    b.template commit<SUMS>(s + S::kA, k, length, sums);
  };
  const auto fetch = [&](int k) {
    a.fetch(k);
    b.fetch(k);
  };
  fetch(k_begin);
  if constexpr (S::kStages == 2) {
    commit(lds, k_begin);
    if (k_begin + BK < k_end) fetch(k_begin + BK);
    __syncthreads();
    int stage = 0;
    for (int k = k_begin; k < k_end; k += BK, stage ^= 1) {
      if (k + BK < k_end) commit(lds + (stage ^ 1) * (S::kA + S::kB), k + BK);
      if (k + 2 * BK < k_end) fetch(k + 2 * BK);
      compute(lds + stage * (S::kA + S::kB));
      __syncthreads();
    }
  } else {
    for (int k = k_begin; k < k_end; k += BK) {
      commit(lds, k);
      __syncthreads();
      if (k + BK < k_end) fetch(k + BK);
      compute(lds);
      __syncthreads();
    }
  }
}

// The wave's sums by rows of the output: 8 columns a lane at a time, through its own part of the LDS.
// put(row of the tile, column of the tile, its 8 sums)
template <typename L, typename F>
__device__ __forceinline__ void dense_rows(char* lds, const f32x16 (&acc)[L::MT][L::NT], F&& put) {
  constexpr int kRow = L::NT * 32 + 4, kLanes = L::NT * 4, kRows = kWave / kLanes;
  const int wave = wave_in_block(), lane = threadIdx.x % kWave;
  const int m0 = wave / L::kWavesN * L::MT * 32, n0 = wave % L::kWavesN * L::NT * 32;
  float* s = reinterpret_cast<float*>(lds) + wave * 32 * kRow;
#pragma unroll
  for (int i = 0; i < L::MT; ++i) {
#pragma unroll
    for (int j = 0; j < L::NT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[tile_row(r, lane / 32) * kRow + 32 * j + lane % 32] = acc[i][j][r];
    wave_sync();
#pragma unroll 4
    for (int r = lane / kLanes; r < 32; r += kRows) {
      const int c = lane % kLanes * 8;
      float v[8];
      load_pack<float, 4>(s + r * kRow + c, v);
      load_pack<float, 4>(s + r * kRow + c + 4, v + 4);
      put(m0 + 32 * i + r, n0 + c, v);
    }
    wave_sync();
  }
}

// N elements from `at` on of a row of `width`: as one unaligned access where they are all inside
template <typename T, int N>
__device__ __forceinline__ void load_row_part(const T* row, int at, int width, float* out) {
  if (at + N <= width) {
    const Pack<T, N> x = load_piece<T, N>(row + at);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = (float)x.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = at + i < width ? (float)row[at + i] : 0.0f;
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_row_part(T* row, int at, int width, const float* in) {
  if (at + N <= width) {
    Pack<T, N> x;
#pragma unroll
    for (int i = 0; i < N; ++i) x.v[i] = (T)in[i];
    __builtin_memcpy(row + at, &x, sizeof(x));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (at + i < width) row[at + i] = (T)in[i];
  }
}

// ---------------------------------------------------------------- host side
template <typename T>
using Small = Shape<T, 64, 64, 2, 2>;
template <typename T>
using Middle = Shape<T, 128, 128, 2, 2>;
template <typename T>
using Large = Shape<T, sizeof(T) == 4 ? 128 : 256, 256, 2, 2>;

// the tile of an output of m x n: 0, 1, 2
inline int dense_tile(size_t size, int64_t m, int64_t n) {
  const auto tiles = [&](int64_t bm, int64_t bn) { return ((m + bm - 1) / bm) * ((n + bn - 1) / bn); };
  if (n >= 256 && tiles(size == 4 ? 128 : 256, 256) >= 256) return 2;
  return tiles(128, 128) >= 256 ? 1 : 0;
}

inline int group_level(int64_t rows) {
  int s = 0;
  while ((32 << s) < rows) ++s;
  return s;
}

// an upper bound of the tiles of `size` rows
inline int64_t row_tiles(int64_t n_rows, int64_t n_groups, bool grouped, int64_t size) {
  return grouped ? n_rows / size + std::min<int64_t>(n_groups + 1, n_rows) : (n_rows + size - 1) / size;
}

inline int dense_sizes(int dtype, int64_t n_rows, int32_t n_in, int32_t n_out, const int32_t* plan,
                       int32_t n_groups) {
  XNN_REQUIRE(is_storage(dtype), "dtype must be XNN_F32, XNN_BF16 or XNN_F16");
  XNN_REQUIRE(n_rows >= 0 && n_rows < ((int64_t)1 << 30), "n_rows must be in [0, 2^30)");
  XNN_REQUIRE(n_in >= 1 && n_in < (1 << 20) && n_out >= 1 && n_out < (1 << 20), "widths must be in [1, 2^20)");
  XNN_REQUIRE(n_groups >= 1 && n_groups <= kMaxGroups, "n_groups must be in [1, %d]", kMaxGroups);
  XNN_REQUIRE(plan != nullptr || n_groups == 1 || n_rows == 0, "groups need a plan");
  XNN_REQUIRE(((n_rows >> 6) + n_groups + 2) * ((std::max(n_in, n_out) >> 6) + 1) < ((int64_t)1 << 31) - 8,
              "too many tiles");
  return XNN_OK;
}

}  // namespace xnn
