// Matrix products of a dense layer on tiles, shared by its forward and backward kernels (gfx950, wave64).
//
//   forward   out = residual + f(x W + b)    rows of x (reduction along them)    x  W read across its rows
//   input     dx  = d W^T,  d = g f'(z)      rows of d                           x  rows of W
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

constexpr int kDenseThreads = 256;     // and two blocks a CU: two waves of at most 256 registers a SIMD
constexpr int kDenseWaves = kDenseThreads / kWave;

// ---------------------------------------------------------------- groups
// What xnn_group_plan leaves, in int32: `order`, the rows by group (stable); row_ptr (n_groups + 2), where a
// group's rows begin, the last bucket holding the rows of no group; for each level the prefix sums of the groups'
// tiles of its rows: 32, 64, 128, 256, then four levels an octave, so that a weight's parts fill whole rounds of
// blocks nearly as well as parts of any size do.
constexpr int kGroupLevels = 52;
constexpr int kMaxGroups = 4096;

__host__ __device__ constexpr int level_rows(int level) {
  return level < 4 ? 32 << level : (256 << ((level - 4) / 4)) / 4 * (5 + (level - 4) % 4);
}
static_assert(level_rows(4) == 320 && level_rows(7) == 512 && level_rows(kGroupLevels - 1) == 1 << 20, "");

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
    const int below = __popcll(__ballot(v <= t)), k = max(below - 1, 0);   // a list of other numbers: within it, too
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
  int g, before, from, to;         // tiles before the group's, its rows
  if (n_buckets < kWave) {         // both lists in one load each
    const int lane = min((int)(threadIdx.x % kWave), n_buckets);
    const int tiles = v.tile_ptr[lane], rows = v.row_ptr[lane];
    if (t >= __builtin_amdgcn_readlane(tiles, n_buckets)) return RowTile{0, 0, -1};
    g = __builtin_amdgcn_readfirstlane(__popcll(__ballot(threadIdx.x % kWave < n_buckets && tiles <= t)) - 1);
    g = max(g, 0);
    before = __builtin_amdgcn_readlane(tiles, g);
    from = __builtin_amdgcn_readlane(rows, g);
    to = __builtin_amdgcn_readlane(rows, g + 1);
  } else {
    const int all = v.tile_ptr[n_buckets];
    if (n_buckets <= 4 * kWave) {  // the first list in one round of loads
      int tiles[4], below = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        tiles[i] = v.tile_ptr[min((int)(threadIdx.x % kWave) + i * kWave, n_buckets)];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        below += __popcll(__ballot((int)(threadIdx.x % kWave) + i * kWave < n_buckets && tiles[i] <= t));
      if (t >= all) return RowTile{0, 0, -1};
      g = __builtin_amdgcn_readfirstlane(max(below - 1, 0));
    } else {
      if (t >= all) return RowTile{0, 0, -1};
      g = find_group(v.tile_ptr, n_buckets, t);
    }
    before = v.tile_ptr[g];
    from = v.row_ptr[g];
    to = v.row_ptr[g + 1];
  }
  // (unsigned: other numbers may wrap, and are then held to the rows)
  const int begin = max(0, (int)((uint32_t)from + ((uint32_t)t - (uint32_t)before) * (uint32_t)size));
  const int end = min(min(to, n_rows), (int)((uint32_t)begin + (uint32_t)size));
  return RowTile{begin, end, begin < end ? g : -1};
}

// The block's slot among those of the tiles that there are, in runs of one length for the XCDs (the launch has room for
// more: a tile more a group, whose blocks would be one XCD's), -1 where it has none (16,384 rows in 64 uneven groups,
// 1,024 x 1,024 in bfloat16: forward 69 us, so 58; 5,000 rows in 6 of 119, 250 -> 511 in float16: 20 us, so 11)
__device__ __forceinline__ int64_t tile_slot(const GroupView& v, int64_t tiles, int tiles_n, int parts, int64_t& there) {
  there = tiles;
  if (v.n_groups > 0)
    there = min(tiles, (int64_t)max(v.tile_ptr[v.n_groups + 1], 0) * tiles_n);
  const int64_t count = there * parts, each = (count + kXcds - 1) / kXcds, i = blockIdx.x / kXcds;
  const int64_t slot = blockIdx.x % kXcds * each + i;
  return i < each && slot < count ? slot : -1;
}

__device__ __forceinline__ int64_t group_row(const GroupView& v, int r) {
  return v.order == nullptr ? r : v.order[r];
}

// the tile's rows for its way out, -1 where it has none; the product's barriers are between this and their use
template <int BM>
__device__ __forceinline__ void note_rows(const GroupView& v, const RowTile& t, int n_rows, int32_t (&rows)[BM]) {
  for (int i = threadIdx.x; i < BM; i += blockDim.x) {
    const int64_t row = t.begin + i < t.end ? group_row(v, t.begin + i) : -1;
    rows[i] = row >= 0 && row < n_rows ? (int32_t)row : -1;
  }
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

// Phi(-|z|) / (t e) for t = 1 / (1 + 0.27 |z|), e = exp(-z^2 / 2): a smooth function of t in [0.2, 1]. FINE: the polynomial of
// degree 8 with the least relative error, 2.4e-8 (weighted least squares, the weights moved by Lawson's rule). Else
// erfc(x) = t (a1 + t (a2 + ...)) exp(-x^2), t = 1 / (1 + 0.3275911 x), x >= 0, to 1.5e-7 (Abramowitz and Stegun,
// Handbook of Mathematical Functions, 7.1.26): a twentieth of what 16 bits round, in four instructions less
template <bool FINE>
__device__ __forceinline__ float normal_tail(float a, float e) {
  if constexpr (FINE) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.27f, a, 1.0f));
    float q = fmaf(t, 0.028915273f, -0.12625526f);
    q = fmaf(t, q, 0.16929141f);
    q = fmaf(t, q, -0.068620972f);
    q = fmaf(t, q, 0.10739943f);
    q = fmaf(t, q, 0.072240293f);
    q = fmaf(t, q, 0.10175917f);
    q = fmaf(t, q, 0.10755051f);
    q = fmaf(t, q, 0.10772018f);
    return q * (t * e);
  } else {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678118654752f, a, 1.0f));
    float q = fmaf(t, 1.061405429f, -1.453152027f);
    q = fmaf(t, q, 1.421413741f);
    q = fmaf(t, q, -0.284496736f);
    q = fmaf(t, q, 0.254829592f);
    return q * (0.5f * t * e);
  }
}

// f(z) and f'(z), to a few float32 steps of the larger of 1 and |z|; FINE, for float32: gelu to a few of its own (72,000 x
// 128 -> 512 with its slope 137 us with the five terms, 149 so; 24,000 x 256 -> 1,024 106 and 112)
template <bool FINE>
__device__ __forceinline__ void activate(int kind, float z, float& y, float& slope) {
  if (kind == kSilu) {
    // the exponential's error is |z| 2^-24 of it, p (1 - p) |z| < 1/4 of that in p
    const float p = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * z));
    y = z * p;
    slope = p * fmaf(z, 1.0f - p, 1.0f);
  } else if (kind == kGelu) {
    // (its exponential is the slope's)
    const float e = __builtin_amdgcn_exp2f(-0.5f * kLog2e * z * z), q = normal_tail<FINE>(fabsf(z), e);
    float c = z < 0.0f ? q : 1.0f - q;
    if constexpr (FINE) {
      // 1 - q has lost 4e-7 where q is near a half: Phi(z) = 1/2 + z r(z^2) in |z| < 1, r fitted to 3e-10
      const float w = z * z;
      float r = fmaf(w, -7.6624747e-6f, 1.1350714e-4f);
      r = fmaf(w, r, -1.1863483e-3f);
      r = fmaf(w, r, 9.9733304e-3f);
      r = fmaf(w, r, -0.06649036f);
      r = fmaf(w, r, 0.39894229f);
      c = w < 1.0f ? fmaf(z, r, 0.5f) : c;
    }
    y = z * c;
    slope = fmaf(z * 0.39894228040143268f, e, c);
  } else if (kind == kTanh) {
    // by the exponential; y near zero, where that loses it, by the series (1 - y^2 would lose the slope where y is near 1)
    const float a = fabsf(z), e = __builtin_amdgcn_exp2f(-2.0f * kLog2e * a), w = z * z;
    const float r = __builtin_amdgcn_rcpf(1.0f + e), far = copysignf((1.0f - e) * r, z);
    float q = fmaf(w, 62.0f / 2835.0f, -17.0f / 315.0f);
    q = fmaf(w, q, 2.0f / 15.0f);
    q = fmaf(w, q, -1.0f / 3.0f);
    const float near = fmaf(z * w, q, z);
    y = a < 0.25f ? near : far;
    slope = 4.0f * e * r * r;
  } else {
    y = z;
    slope = 1.0f;
  }
}

// f'(z) as the backward pass gets it, so that d = g f'(z) is rounded once and not twice (the gradients' error is
// 1.4 times an output's rounding, 1.7 with f' in the type): float32 as it is; for bfloat16 2^15 times it in float16
// (f' is below 1.13), off by 2^-11 of it down to 2^-29; for float16 in 16 bits that are fine where f' is large and never
// coarser than the type where it is small (a loss scale makes such d large):
//   |f'| >= 2^-7   its root in steps of 1 / 30,000, off by 2^-14.8 root(f'): 2^-14.8 of it near 1, 2^-11.3 at 2^-7
//   below          2^5 times it in float16, off by 2^-11 of it down to 2^-19, by 2^-30 below
// Of 65,536 numbers, counted from one for zero, 13,312 are the float16 ones and then the roots up to 1.13's above it, and as
// many and the roots up to 0.13's below (no f' is less); the last one stands for NaN. (Both passes of 72,000 x 128 -> 512 with
// silu 153 us, 139 with the root alone, which was off by 0.4 % for silu at z = -12 and by 5 % for tanh at 8.)
template <typename T>
struct Slope {
  typedef T type;
};
template <>
struct Slope<bf16_t> {
  typedef f16_t type;
};
template <>
struct Slope<f16_t> {
  typedef uint16_t type;
};
constexpr float kSlopeScale = 32768.0f;
constexpr float kSlopeUnit = 30000.0f, kSlopeFine = 0x1p-7f, kSlopeFineScale = 32.0f;
constexpr int kSlopeFineLast = 0x3400;             // 2^5 2^-7 in float16
constexpr int kSlopeRoots = 10662;                 // the root of 2^-7, 2,652 steps, comes after it
constexpr int kSlopeZero = 21600, kSlopeNan = 65535;
static_assert(kSlopeRoots + 2652 == kSlopeFineLast + 2 && kSlopeZero + kSlopeRoots + 31950 < kSlopeNan &&
                  kSlopeZero > kSlopeRoots + 10850, "");
template <typename T>
__device__ __forceinline__ typename Slope<T>::type slope_stored(float s) {
  if constexpr (sizeof(T) == 4)
    return s;
  else if constexpr (__is_same(T, bf16_t))
    return (f16_t)(s * kSlopeScale);
  else {
    const float a = fabsf(s);
    const int fine = __builtin_bit_cast(uint16_t, (f16_t)(a * kSlopeFineScale));
    const int root = kSlopeRoots + __float2int_rn(kSlopeUnit * __builtin_amdgcn_sqrtf(a));
    const int n = a < kSlopeFine ? fine : root;
    return (uint16_t)(s == s ? kSlopeZero + (s < 0.0f ? -n : n) : kSlopeNan);
  }
}
template <typename T>
__device__ __forceinline__ float slope_value(typename Slope<T>::type s) {
  if constexpr (sizeof(T) == 4)
    return s;
  else if constexpr (__is_same(T, bf16_t))
    return (float)s * (1.0f / kSlopeScale);
  else {
    const float m = (float)s - (float)kSlopeZero, a = fabsf(m);
    const float root = fmaf(a, 1.0f / kSlopeUnit, -kSlopeRoots / kSlopeUnit);
    const float fine = (float)__builtin_bit_cast(f16_t, (uint16_t)a) * (1.0f / kSlopeFineScale);
    const float f = copysignf(a <= (float)kSlopeFineLast ? fine : root * root, m);
    return m > (float)(kSlopeNan - kSlopeZero - 1) ? __builtin_nanf("") : f;
  }
}

// ---------------------------------------------------------------- sizes
// BK: elements of the reduction a step
template <typename T, int BM_, int BN_, int WM_, int WN_, int BK_>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, kWavesM = WM_, kWavesN = WN_;
  static constexpr int MT = BM / WM_ / 32, NT = BN / WN_ / 32;   // 32 x 32 products of a wave
  static constexpr int BK = BK_;
  static_assert(WM_ * WN_ == kDenseWaves, "");
};

// an operand in LDS: ROWS outer indices
template <typename T, int ROWS, int BK, bool ALONG>
struct Place;
template <typename T, int ROWS, int BK>
struct Place<T, ROWS, BK, true> {  // rows along the reduction; 16 bytes more spread the banks
  static constexpr int kRow = BK * 2 + 16, kPlane = ROWS * kRow;
  static constexpr int kBytes = kPlane * Store<T>::kPlanes;
};
template <typename T, int ROWS, int BK>
struct Place<T, ROWS, BK, false> { // rows across it; 64 more: four rows of a transposing read on other banks
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

// the first `left` elements of a piece, zeros for the others
template <typename T>
__device__ __forceinline__ u32x4 piece_head(u32x4 x, int left) {
  constexpr int kWord = 4 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = left - i * kWord;
    x[i] = n >= kWord ? x[i] : n == 1 && kWord == 2 ? x[i] & 0xFFFFu : 0u;
  }
  return x;
}

// A piece from any address (the loads are unaligned ones, at full rate where the address happens to be aligned).
// One that reaches beyond its row's `left` elements is within the tensor where another row follows; in the last
// row it is taken element by element.
__device__ __forceinline__ u32x4 load_raw(const char* p) {
  u32x4 x;
  __builtin_memcpy(&x, p, sizeof(x));
  return x;
}
template <typename T>
__device__ __forceinline__ u32x4 load_raw(const char* p, int left, bool last) {
  constexpr int N = 16 / sizeof(T);
  if (left >= N || (left > 0 && !last)) return load_raw(p);
  Pack<T, N> x;
#pragma unroll
  for (int i = 0; i < N; ++i) x.v[i] = i < left ? reinterpret_cast<const T*>(p)[i] : (T)0.0f;
  return __builtin_bit_cast(u32x4, x);
}

// One piece to LDS: as it is, or in three planes of half the bytes
template <typename T>
__device__ __forceinline__ void put_piece(char* at, int plane, u32x4 x) {
  if constexpr (sizeof(T) == 4) {
    uint32_t a[3], b[3];
    rounded_planes(__uint_as_float(x[0]), __uint_as_float(x[1]), a);
    rounded_planes(__uint_as_float(x[2]), __uint_as_float(x[3]), b);
#pragma unroll
    for (int n = 0; n < 3; ++n) *reinterpret_cast<u32x2*>(at + n * plane) = u32x2{a[n], b[n]};
  } else {
    *reinterpret_cast<u32x4*>(at) = x;
  }
}

// d = g f'(z) of a piece
template <typename T>
__device__ __forceinline__ u32x4 times_slope(u32x4 g, u32x4 slope) {
  constexpr int N = 16 / sizeof(T);
  typedef typename Slope<T>::type S;
  const Pack<T, N> x = __builtin_bit_cast(Pack<T, N>, g);
  const Pack<S, N> y = __builtin_bit_cast(Pack<S, N>, slope);
  Pack<T, N> out;
#pragma unroll
  for (int i = 0; i < N; ++i) out.v[i] = (T)((float)x.v[i] * slope_value<T>(y.v[i]));
  return __builtin_bit_cast(u32x4, out);
}

// One operand on its way: a matrix of rows of `width` elements, row r at data + r stride (TIMES: times the slope's,
// of the same layout), of which LEN rows or columns are this tile's. ALONG: the tile's rows, along which the
// reduction runs; else its columns, and the reduction runs over the rows. Row r of the tile, or of the reduction,
// is order[first + r], or first + r without an order.
//
// Steps that begin before `fast` are of whole pieces, one address each that the step before has left: along the rows
// those that end within them; across them all but the last one where a piece may reach beyond its row (the
// tensor's last row is the last of its group).
template <typename T, int LEN, int BK, bool ALONG, bool TIMES = false, bool ORDERED = ALONG>
struct Operator {
  static constexpr int kPer = 16 / sizeof(T);
  static constexpr int kRows = ALONG ? LEN : BK, kCols = ALONG ? BK : LEN;   // of a staged step
  static constexpr int kChunks = kCols / kPer;
  static constexpr int kStep = kDenseThreads / kChunks;
  static constexpr int kCount = kRows / kStep;
  static_assert(kDenseThreads % kChunks == 0 && kRows % kStep == 0 && kCount <= 32, "");
  typedef Place<T, LEN, BK, ALONG> At;

  const char *data, *column;       // the tensor, and the thread's first piece of its row 0
  const int32_t* order;            // from `first` on
  int64_t stride, slope;           // bytes of a row, bytes from data to the slope
  int width, row, at, first, end, last, fast;   // last: the tensor's last row
  int most;                        // the last row that a whole piece may begin in
  uint32_t edges;                  // ALONG: pieces of the tensor's last row
  const char* p[kCount];           // pieces of the next step; across rows in an order
  int32_t index[!ALONG && ORDERED ? kCount : 1];   // those rows, whose loads have a step's time
  u32x4 x[kCount], y[TIMES ? kCount : 1];

  // rows [first_row, end_row), columns from first_col on
  __device__ __forceinline__ void init(const void* data_, const int32_t* order_, int64_t stride_,
                                       int tensor_rows, int width_, int first_row, int end_row,
                                       int first_col, const void* slope_ = nullptr) {
    data = (const char*)data_;
    slope = TIMES ? (const char*)slope_ - data : 0;
    order = order_ == nullptr ? nullptr : order_ + first_row;
    stride = stride_ * (int)sizeof(T);
    last = tensor_rows - 1;
    width = width_;
    row = threadIdx.x / kChunks;
    at = first_col + threadIdx.x % kChunks * kPer;
    if (!ALONG && at >= width) at = 0;                     // columns beyond the edge: any that exist
    column = data + at * (int)sizeof(T);
    first = first_row;
    end = end_row - first_row;
    const bool whole = width % kPer == 0;
    most = ALONG || whole ? last : max(last - 1, 0);
    fast = stride_ < kPer ? 0 : ALONG ? (width - first_col) / BK * BK : (whole ? end : end - 1) / BK * BK;
    edges = 0;
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const int i = row_of(row + n * kStep);
      if (ALONG && i == last) edges |= 1u << n;
      if constexpr (!ALONG && ORDERED) index[n] = i;
      p[n] = column + i * stride;
    }
  }
  __device__ __forceinline__ int row_of(int r) const {
    r = min(r, end - 1);
    if (!ORDERED || (ALONG && order == nullptr)) return first + r;
    return min(max(order[r], 0), last);
  }
  // the step from reduction index k0 < fast on
  __device__ __forceinline__ void fetch_fast(int k0) {
    if constexpr (!ALONG && ORDERED)
#pragma unroll
      for (int n = 0; n < kCount; ++n) p[n] = column + min(index[n], most) * stride;
    const int64_t step = ALONG ? BK * (int)sizeof(T) : BK * stride;
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      x[n] = load_raw(p[n]);
      if constexpr (TIMES) y[n] = load_raw(p[n] + slope);
      p[n] += step;
    }
    if constexpr (!ALONG && ORDERED)
#pragma unroll
      for (int n = 0; n < kCount; ++n) index[n] = row_of(k0 + BK + row + n * kStep);
  }
  // any step
  __device__ __forceinline__ void fetch(int k0) {
    if (k0 < fast) {
      fetch_fast(k0);
      return;
    }
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const int i = ALONG ? 0 : row_of(k0 + row + n * kStep);
      const char* q = ALONG ? p[n] : column + i * stride;
      const int left = width - at - (ALONG ? k0 : 0);
      const bool edge = (ALONG ? (edges >> n & 1) != 0 : i == last) || stride < 16;
      x[n] = load_raw<T>(q, left, edge);
      if constexpr (TIMES) y[n] = load_raw<T>(q + slope, left, edge);
      if (ALONG) p[n] += BK * (int)sizeof(T);
    }
  }
  // to LDS, TAIL: zeros beyond the reduction's `length`
  template <bool TAIL>
  __device__ __forceinline__ void commit(char* lds, int k0, int length) {
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const int r = row + n * kStep, c = threadIdx.x % kChunks * kPer;
      if constexpr (TIMES) x[n] = times_slope<T>(x[n], y[n]);
      u32x4 out = x[n];
      if constexpr (TAIL) out = piece_head<T>(out, ALONG ? length - k0 - c : k0 + r < length ? kPer : 0);
      put_piece<T>(lds + r * At::kRow + c * 2, At::kPlane, out);
    }
  }
  // the step's rows before `length`, added to each of the thread's columns (after commit, before the next fetch)
  __device__ __forceinline__ void add_rows(int k0, int length, float (&sums)[kPer]) const {
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const Pack<T, kPer> v = __builtin_bit_cast(Pack<T, kPer>, x[n]);
      const bool in = k0 + row + n * kStep < length;
#pragma unroll
      for (int i = 0; i < kPer; ++i) sums[i] += in ? (float)v.v[i] : 0.0f;
    }
  }
};

// operand `step` of 16 reduction indices for the 32 outer indices from `outer` on
template <typename T, int LEN, int BK, bool ALONG>
__device__ __forceinline__ Operand<T> dense_operand(const char* lds, int outer, int step) {
  typedef Place<T, LEN, BK, ALONG> At;
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

// N elements from any address, and from column `at` on of a row of `width` (as load_raw)
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

// ---------------------------------------------------------------- the product
// LDS of a block: one stage of both operands, and the waves' rows on their way out
template <typename L, typename T, bool ALONG_A, bool ALONG_B>
struct DenseLds {
  static constexpr int kA = Place<T, L::BM, L::BK, ALONG_A>::kBytes,
                       kB = Place<T, L::BN, L::BK, ALONG_B>::kBytes;
  static constexpr int kOutRow = L::NT * 32 + 4;                         // floats
  static constexpr int kOut = kDenseWaves * 32 * kOutRow * 4;
  static constexpr int kPlanes = Store<T>::kPlanes;
  static constexpr int kStages = 2 * (kA + kB) <= 150 * 1024 && sizeof(T) == 2 ? 2 : 1;
  static constexpr int kBytes = kStages * (kA + kB) > kOut ? kStages * (kA + kB) : kOut;
};

// The order of a region's instructions: among M products, READS reads of LDS in the first three quarters, WRITES writes
// to it and LOADS global loads evenly. Without it the compiler puts each kind in a row and the matrix cores wait.
template <int M, int READS, int WRITES, int LOADS, int I = 0>
__device__ __forceinline__ void interleave() {
  if constexpr (I < M) {
    constexpr auto reads = [](int i) { return i * READS * 4 / (3 * M) < READS ? i * READS * 4 / (3 * M) : READS; };
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if constexpr (reads(I + 1) > reads(I)) __builtin_amdgcn_sched_group_barrier(0x100, reads(I + 1) - reads(I), 0);
    if constexpr ((I + 1) * WRITES / M > I * WRITES / M)
      __builtin_amdgcn_sched_group_barrier(0x200, (I + 1) * WRITES / M - I * WRITES / M, 0);
    if constexpr ((I + 1) * LOADS / M > I * LOADS / M)
      __builtin_amdgcn_sched_group_barrier(0x020, (I + 1) * LOADS / M - I * LOADS / M, 0);
    interleave<M, READS, WRITES, LOADS, I + 1>();
  }
}

// The tile's sums over `length` reduction indices; seen(k) after each step that starts at k is in LDS. The rows of
// a 32 x 32 product are the output's columns, so that a lane holds four of them in a row.
template <typename T, typename L, bool ALONG_A, bool ALONG_B, typename A, typename B, typename F>
__device__ __forceinline__ void dense_product(A& a, B& b, int length, char* lds, f32x16 (&acc)[L::MT][L::NT],
                                              F&& seen) {
  typedef DenseLds<L, T, ALONG_A, ALONG_B> S;
  constexpr int BK = L::BK;
  const int wave = wave_in_block();
  const int m0 = wave / L::kWavesN * L::MT * 32, n0 = wave % L::kWavesN * L::NT * 32;
#pragma unroll
  for (int i = 0; i < L::MT; ++i)
#pragma unroll
    for (int j = 0; j < L::NT; ++j) acc[i][j] = f32x16{};
  // operands `step` of a stage, two steps' in registers: a step's are read while the products of the one before run
  constexpr int kSteps = BK / 16;
  static_assert(kSteps % 2 == 0, "");
  Operand<T> fa[2][L::MT], fb[2][L::NT];
  const auto read = [&](const char* s, int step) {
#pragma unroll
    for (int i = 0; i < L::MT; ++i) fa[step & 1][i] = dense_operand<T, L::BM, BK, ALONG_A>(s, m0 + 32 * i, step);
#pragma unroll
    for (int j = 0; j < L::NT; ++j)
      fb[step & 1][j] = dense_operand<T, L::BN, BK, ALONG_B>(s + S::kA, n0 + 32 * j, step);
  };
  const auto multiply = [&](int step) {
#pragma unroll
    for (int i = 0; i < L::MT; ++i)
#pragma unroll
      for (int j = 0; j < L::NT; ++j) mma<T>(fb[step & 1][j], fa[step & 1][i], acc[i][j]);
  };
  constexpr int kProducts = L::MT * L::NT * (S::kPlanes == 3 ? 6 : 1);          // of a step
  constexpr int kReads = (L::MT * (ALONG_A ? 1 : 2) + L::NT * (ALONG_B ? 1 : 2)) * S::kPlanes;
  constexpr int kMoves = A::kCount + B::kCount;
  const auto commit_fast = [&](char* s, int k) {
    a.template commit<false>(s, k, length);
    b.template commit<false>(s + S::kA, k, length);
    seen(k);
  };
  const auto commit = [&](char* s, int k) {
    if (k + BK <= length) {
      commit_fast(s, k);
    } else {
      a.template commit<true>(s, k, length);
      b.template commit<true>(s + S::kA, k, length);
      seen(k);
    }
  };
  const auto fetch = [&](int k) {
    a.fetch(k);
    b.fetch(k);
  };
  const auto fetch_fast = [&](int k) {
    a.fetch_fast(k);
    b.fetch_fast(k);
  };
  const int fast = min(min(a.fast, b.fast), length);
  int k = 0;
  fetch(k);
  if constexpr (S::kStages == 2) {
    constexpr int kStage = S::kA + S::kB;
    commit(lds, k);
    if (k + BK < length) fetch(k + BK);
    __syncthreads();
    int stage = 0;
    read(lds, 0);
    for (; k + 2 * BK < fast; k += BK, stage ^= 1) {
      commit_fast(lds + (stage ^ 1) * kStage, k + BK);
      fetch_fast(k + 2 * BK);
#pragma unroll
      for (int step = 0; step + 1 < kSteps; ++step) {
        read(lds + stage * kStage, step + 1);
        multiply(step);
      }
      interleave<kProducts * (kSteps - 1), kReads * (kSteps - 1), kMoves, kMoves>();
      __syncthreads();
      read(lds + (stage ^ 1) * kStage, 0);
      multiply(kSteps - 1);
      interleave<kProducts, kReads, 0, 0>();
    }
    for (; k < length; k += BK, stage ^= 1) {
      if (k + BK < length) commit(lds + (stage ^ 1) * kStage, k + BK);
      if (k + 2 * BK < length) fetch(k + 2 * BK);
#pragma unroll
      for (int step = 0; step + 1 < kSteps; ++step) {
        read(lds + stage * kStage, step + 1);
        multiply(step);
      }
      __syncthreads();
      if (k + BK < length) read(lds + (stage ^ 1) * kStage, 0);
      multiply(kSteps - 1);
    }
    __syncthreads();
  } else {
    const auto compute = [&]() {
      read(lds, 0);
#pragma unroll
      for (int step = 0; step < kSteps; ++step) {
        if (step + 1 < kSteps) read(lds, step + 1);
        __builtin_amdgcn_sched_barrier(0);
        multiply(step);
      }
    };
    for (; k + BK < fast; k += BK) {
      commit_fast(lds, k);
      __syncthreads();
      fetch_fast(k + BK);
      compute();
      __syncthreads();
    }
    for (; k < length; k += BK) {
      commit(lds, k);
      __syncthreads();
      if (k + BK < length) fetch(k + BK);
      compute();
      __syncthreads();
    }
  }
}

// The wave's sums by rows of the output, through its own part of the LDS: a lane has the N columns of a 16-byte store,
// the same in every row. put(row of the tile, its N sums) for each of them, begin(column of the tile) before
template <typename L, int N, typename G, typename F>
__device__ __forceinline__ void dense_rows(char* lds, const f32x16 (&acc)[L::MT][L::NT], G&& begin, F&& put) {
  constexpr int kRow = L::NT * 32 + 4, kLanes = L::NT * 32 / N, kRows = kWave / kLanes;
  const int wave = wave_in_block(), lane = threadIdx.x % kWave;
  const int m0 = wave / L::kWavesN * L::MT * 32, n0 = wave % L::kWavesN * L::NT * 32;
  float* s = reinterpret_cast<float*>(lds) + wave * 32 * kRow;
  begin(n0 + lane % kLanes * N);
#pragma unroll
  for (int i = 0; i < L::MT; ++i) {
#pragma unroll
    for (int j = 0; j < L::NT; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(s + lane % 32 * kRow + 32 * j + tile_row(4 * q, lane / 32)) =
            f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    wave_sync();
#pragma unroll 4
    for (int r = lane / kLanes; r < 32; r += kRows) {
      const float* p = s + r * kRow + lane % kLanes * N;
      float v[N];
#pragma unroll
      for (int q = 0; q < N; q += 4) load_pack<float, 4>(p + q, v + q);
      put(m0 + 32 * i + r, v);
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
// (STREAM: past the caches, for what is not read soon)
template <typename T, int N, bool STREAM = false, typename V>
__device__ __forceinline__ void store_row_part(T* row, int at, int width, const V* in) {
  if (at + N <= width) {
    Pack<T, N> x;
#pragma unroll
    for (int i = 0; i < N; ++i) x.v[i] = (T)in[i];
    if constexpr (STREAM) {
      typedef uint32_t Words __attribute__((ext_vector_type(sizeof(x) / 4), aligned(sizeof(T))));
      __builtin_nontemporal_store(__builtin_bit_cast(Words, x), reinterpret_cast<Words*>(row + at));
    } else {
      __builtin_memcpy(row + at, &x, sizeof(x));
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (at + i < width) row[at + i] = (T)in[i];
  }
}

// ---------------------------------------------------------------- outputs
// What becomes of the sums of a row: residual + f(v + bias), and the slope
struct Output {
  const void *bias, *residual;     // NULL: none
  void *out, *slope;
  float* part;                     // (parts, rows, width): sums of parts of the reduction
  GroupView groups;
  int n_rows, width, activation;
  float none;                      // in the rows of no group
  int stream;                      // out is larger than the caches of the dies
};

// An output that the L2 caches (4 MB a die) cannot hold for its reader goes past them, as the slope does, which the
// backward pass reads (24,000 x 4,096 in bfloat16: 274 us without an activation, past them 256; with gelu 396,
// the slope past them 376)
inline int past_caches(int64_t rows, int64_t width, size_t size) {
  return rows * width * (int64_t)size > ((int64_t)32 << 20);
}

template <typename T>
__device__ __forceinline__ void load_bias(const Output& o, int group, int c, float (&bias)[16 / sizeof(T)]) {
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < N; ++i) bias[i] = 0.0f;
  if (o.bias != nullptr && c < o.width)
    load_row_part<T, N>((const T*)o.bias + (int64_t)group * o.width, c, o.width, bias);
}

template <typename T>
__device__ __forceinline__ void put_row(const Output& o, int64_t row, int c, float (&v)[16 / sizeof(T)],
                                        const float (&bias)[16 / sizeof(T)]) {
  constexpr int N = 16 / sizeof(T);
  typedef typename Slope<T>::type S;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] += bias[i];
  if (o.activation != kNone) {
    S slope[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s;
      activate<sizeof(T) == 4>(o.activation, v[i], v[i], s);
      slope[i] = slope_stored<T>(s);
    }
    if (o.slope != nullptr) store_row_part<S, N, true>((S*)o.slope + row * o.width, c, o.width, slope);
  }
  if (o.residual != nullptr) {
    float z[N];
    load_row_part<T, N>((const T*)o.residual + row * o.width, c, o.width, z);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += z[i];
  }
  if (o.stream)
    store_row_part<T, N, true>((T*)o.out + row * o.width, c, o.width, v);
  else
    store_row_part<T, N>((T*)o.out + row * o.width, c, o.width, v);
}

// A tile's sums to where they go: the outputs, or the part's sums
template <typename T, typename L>
__device__ __forceinline__ void put_tile(char* lds, const f32x16 (&acc)[L::MT][L::NT], const Output& o, int parts,
                                         int part, int group, const int32_t (&rows)[L::BM], int n0) {
  int c;
  if (parts > 1) {
    float* to = o.part + (int64_t)part * o.n_rows * o.width;
    dense_rows<L, 4>(
        lds, acc, [&](int n) { c = n0 + n; },
        [&](int m, float(&v)[4]) {
          const int64_t row = rows[m];
          if (row >= 0 && c < o.width) store_row_part<float, 4>(to + row * o.width, c, o.width, v);
        });
    return;
  }
  constexpr int N = 16 / sizeof(T);
  float bias[N];
  dense_rows<L, N>(
      lds, acc,
      [&](int n) {
        c = n0 + n;
        load_bias<T>(o, group, c, bias);
      },
      [&](int m, float(&v)[N]) {
        const int64_t row = rows[m];
        if (row >= 0 && c < o.width) put_row<T>(o, row, c, v, bias);
      });
}

// The parts of a reduction added: a block has 4 sorted rows of 8 pieces of 16 bytes, eight threads an output, each with
// every eighth part in order, then those sums in order (one thread an output waited 12 us for 32 parts, whose
// lines other dies have written)
template <typename T>
__global__ __launch_bounds__(256) void dense_parts_kernel(Output o, int parts, int columns) {
  constexpr int N = 16 / sizeof(T);
  __shared__ __align__(16) float sums[8][32][N];
  const int lane = threadIdx.x % 8, line = threadIdx.x / 8 % 4, slice = threadIdx.x / 32;
  const int quarter = blockIdx.x / columns % 8;
  const RowTile t = row_tile(o.groups, o.groups.n_groups + 1, o.n_rows, blockIdx.x / (8 * columns), 32);
  if (t.group < 0) return;
  if (o.groups.n_groups > 0 && t.group == o.groups.n_groups) return;   // rows of no group: done
  const int c = (blockIdx.x % columns * 8 + lane) * N, r = t.begin + 4 * quarter + line;
  const int64_t row = r < t.end ? group_row(o.groups, r) : -1;
  const bool live = c < o.width && row >= 0 && row < o.n_rows;
  float v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.0f;
  if (live)
#pragma unroll 4
    for (int n = slice; n < parts; n += 8) {
      float x[N];
      load_row_part<float, N>(o.part + ((int64_t)n * o.n_rows + row) * o.width, c, o.width, x);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += x[i];
    }
  store_pack<float, N>(sums[slice][threadIdx.x % 32], v);
  __syncthreads();
  if (slice != 0 || !live) return;
  float bias[N];
  load_bias<T>(o, t.group, c, bias);
#pragma unroll
  for (int q = 1; q < 8; ++q)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += sums[q][threadIdx.x][i];
  put_row<T>(o, row, c, v, bias);
}

// ---------------------------------------------------------------- host side
// Tiles: 64 x 64; 128 x 128; in 16 bits 256 x 128. Steps of 32 leave LDS and registers for two blocks a CU, of 128
// x 128 in 16 bits three, one in its products while another loads or stores (24,000 x 1,024 x 4,096 in bfloat16
// with gelu: 256 x 256, one block a CU, 495 us; 256 x 128 398; 128 x 128 418, in steps of 64 470; 70,000 x 128 x
// 512 with silu: 128 x 128 47, in steps of 64 58).
enum TileKind : int { kTile64 = 0, kTile128 = 1, kTile256 = 2 };
template <typename T>
using Tile64 = Shape<T, 64, 64, 2, 2, 128 / sizeof(T)>;
template <typename T>
using Tile128 = Shape<T, 128, 128, 2, 2, 32>;
template <typename T>
using Tile256 = Shape<T, 256, 128, 2, 2, 32>;

// The kind for an output of m x n, in `groups` of rows where they are grouped (then a group's last tile is half empty;
// how many groups have rows is not known here, and that any has does not speak for smaller tiles).
// 256 x 128 tiles pay where they come in full rounds of two a CU, a last round of up to one a CU counting little more
// than half (9,000 x 512 x 2,048 with silu, 1.1 rounds: 78 us, 128 x 128 44; 24,000 x 1,024 x 4,096, 5.9: 398 and
// 418; 24,000 x 4,096 x 1,024, 1.5: 226 and 255); 64 x 64 where 128 x 128 are not one a CU (1,000^3: 10 us, 128 x 128
// 21).
inline int dense_tile(size_t size, int64_t m, int64_t n, int64_t groups) {
  const auto rounds = [&](int64_t bm, int64_t bn, int64_t more) {
    return (double)((m + bm - 1) / bm + more) * (double)((n + bn - 1) / bn) / 512;
  };
  const auto whole = [](double r) {
    const double f = r - std::floor(r);
    return std::floor(r) + (f == 0.0 ? 0.0 : f <= 0.5 ? 0.6 : 1.0);
  };
  if (n <= 64 || rounds(128, 128, 0) < 0.5) return kTile64;
  const int64_t more = groups / 2;
  return size == 2 && 1.8 * whole(rounds(256, 128, more)) <= whole(rounds(128, 128, more)) ? kTile256 : kTile128;
}

// One or two rows of up to 1,500 inputs are a stream of the weight.
// Against tiles, whose reduction is cut into parts that all CUs take (one row, 1,024 outputs): 1,024 inputs in bfloat16
// 5.7 us, tiles 10.5, in float32 5.4 and 7.3; 1,500 inputs 7.0 and 7.4, 6.6 and 8.3; 2,048 8.3 and 7.2, 7.8 and 8.9;
// 4,096 13.3 and 8.4, 19.1 and 12.3. Two rows cost 1 us more, tiles the same; of three (accumulators for four) 1,024
// inputs take 8.4 us in bfloat16 and 7.1 in float32, tiles 10.5 and 7.3, but 128 inputs 5.9 and tiles 4.2.
constexpr int kMaxFew = 2, kMaxFewInputs = 1500;
inline bool few_rows(int64_t n_rows, int32_t n_in) { return n_rows <= kMaxFew && n_in <= kMaxFewInputs; }

// call(Shape) for the kind
#define XNN_TILE_DISPATCH(kind, T, L, ...)           \
  do {                                               \
    if ((kind) == kTile64) {                         \
      typedef ::xnn::Tile64<T> L;                    \
      __VA_ARGS__;                                   \
    } else if (sizeof(T) == 4 || (kind) == kTile128) { \
      typedef ::xnn::Tile128<T> L;                   \
      __VA_ARGS__;                                   \
    } else if constexpr (sizeof(T) == 2) {           \
      typedef ::xnn::Tile256<T> L;                   \
      __VA_ARGS__;                                   \
    }                                                \
  } while (0)

// the first level of at least so many rows
inline int group_level(int64_t rows) {
  int s = 0;
  while (s < kGroupLevels - 1 && level_rows(s) < rows) ++s;
  return s;
}

// an upper bound of the tiles of `size` rows
inline int64_t row_tiles(int64_t n_rows, int64_t n_groups, bool grouped, int64_t size) {
  return grouped ? n_rows / size + std::min<int64_t>(n_groups + 1, n_rows) : (n_rows + size - 1) / size;
}

// The parts of a reduction of `length` for an output of m x n: more than one where its tiles leave the card idle,
// as many as the estimated time has its least with: steps of 0.3 us, in float32 0.5 (their loads' latency), a
// launch that adds the parts, their sums written and read at 4 TB/s. Each is of `steps` whole steps.
struct Split {
  int parts, steps;
  size_t bytes;
};
inline Split dense_split(size_t size, int kind, int64_t m, int64_t n, int64_t length) {
  const int64_t step = 128 / size, steps = (length + step - 1) / step;
  Split best{1, (int)steps, 0};
  if (kind != kTile64) return best;
  const int64_t tiles = ((m + 63) / 64) * ((n + 63) / 64);
  const double one = size == 2 ? 0.3 : 0.5;
  double least = one * (double)steps;
  for (int64_t p = 2; p <= steps && p * tiles <= 1024; ++p) {
    const int64_t each = (steps + p - 1) / p;
    if ((p - 1) * each >= steps) continue;                 // the last part would be empty
    const double time = one * (double)each * (p * tiles > 768 ? 2 : 1) + 5.0 + 0.03 * (double)p + (double)(p * m * n) * 8 / 4e6;
    if (time < least) {
      least = time;
      best = Split{(int)p, (int)each, (size_t)p * m * n * sizeof(float)};
    }
  }
  return best;
}

template <typename T>
static void parts_launch(const Output& o, const int32_t* plan, int n_groups, int parts, hipStream_t s) {
  Output q = o;
  q.groups = group_view(plan, o.n_rows, n_groups, 0);
  const int columns = (o.width + 8 * (int)(16 / sizeof(T)) - 1) / (8 * (int)(16 / sizeof(T)));
  const int64_t blocks = row_tiles(o.n_rows, n_groups, plan != nullptr, 32) * 8 * columns;
  hipLaunchKernelGGL(dense_parts_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, s, q, parts, columns);
}

// blocks of a launch: its threads are numbered in 32 bits
constexpr int64_t kMaxBlocks = ((int64_t)1 << 32) / kDenseThreads - kXcds;

inline int dense_sizes(int dtype, int64_t n_rows, int32_t n_in, int32_t n_out, const int32_t* plan,
                       int32_t n_groups) {
  XNN_REQUIRE(is_storage(dtype), "dtype must be XNN_F32, XNN_BF16 or XNN_F16");
  XNN_REQUIRE(n_rows >= 0 && n_rows < ((int64_t)1 << 30), "n_rows must be in [0, 2^30)");
  XNN_REQUIRE(n_in >= 1 && n_in < (1 << 20) && n_out >= 1 && n_out < (1 << 20), "widths must be in [1, 2^20)");
  XNN_REQUIRE(n_groups >= 1 && n_groups <= kMaxGroups, "n_groups must be in [1, %d]", kMaxGroups);
  XNN_REQUIRE(plan != nullptr || n_groups == 1 || n_rows == 0, "groups need a plan");
  XNN_REQUIRE(((n_rows >> 6) + n_groups + 2) * ((std::max(n_in, n_out) >> 6) + 1) < kMaxBlocks, "too many tiles");
  return XNN_OK;
}

}  // namespace xnn
