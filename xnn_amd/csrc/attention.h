// Tiles of attention within structures, shared by the forward and the backward kernels
// (gfx950, wave64).
//
// A wave owns 32 rows (query rows, or keys in the kernel of their gradients) and walks the other
// side in tiles that the block's waves stage in LDS. All products are 32 x 32 matrix-core tiles
// oriented so that the wave's own rows are the tile's COLUMNS: a lane then holds one own row
// (lane % 32) and 16 of the 32 walked rows, row(r) = 8 (r / 4) + 4 (lane / 32) + r % 4 in
// register r. Softmax statistics are one value a lane, and the registers of a product are at once
// the operand of the next one, because the order of a contraction index is free as long as both
// operands use the same: the walked row of operand element e is the one the product left there.
//
//   walk(tile) x own       = tile (rows from LDS, 16 bytes a lane)  x  own (registers)
//   own^T     += tile^T x weights: tile read across its rows by the transposing LDS read
//
// 16-bit types use v_mfma_f32_32x32x16_{bf16,f16} (sums in float32). float32 is taken apart into
// three bfloat16 planes of 8 bits each by truncation, x = h + m + l exactly, and a product is the
// six plane products of order 2^-16 and larger (h h, h m, m h, h l, l h, m m; the dropped ones
// are 2^-24 of it, as a float32 rounding): six instructions of the 16-bit rate in place of eight of
// a sixteenth of it, 2.7 times the rate of v_mfma_f32_32x32x2_f32. An operand that is not finite
// makes the products it enters NaN.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "common.h"
#include "device.h"
#include "storage.h"

namespace xnn {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

constexpr int kOwn = 32;           // own rows of a wave
constexpr float kLog2e = 1.4426950408889634f;

// row of register r in a 32 x 32 tile, for the half wave `half` = lane / 32
__host__ __device__ constexpr int tile_row(int r, int half) {
  return 8 * (r / 4) + 4 * half + r % 4;
}

template <typename T>
struct Store {                     // bfloat16, float16: one plane, the value itself
  typedef T Element;
  static constexpr int kPlanes = 1;
};
template <>
struct Store<float> {
  typedef bf16_t Element;
  static constexpr int kPlanes = 3;
};
template <typename E>
struct FragOf {
  typedef bf16x8 type;
};
template <>
struct FragOf<f16_t> {
  typedef f16x8 type;
};
// the eight elements of a lane in an operand of one instruction, and its planes
template <typename T>
using Frag = typename FragOf<typename Store<T>::Element>::type;
template <typename T, int PLANES = Store<T>::kPlanes>
struct Operand {
  Frag<T> p[PLANES];
};

__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// c += a b over the plane products of order max(NA, NB) - 1 and lower, the smallest first
template <typename T, int NA, int NB>
__device__ __forceinline__ void mma(const Operand<T, NA>& a, const Operand<T, NB>& b, f32x16& c) {
  constexpr int kMost = NA > NB ? NA : NB;
#pragma unroll
  for (int order = kMost - 1; order >= 0; --order)
#pragma unroll
    for (int i = 0; i <= order; ++i)
      if (i < NA && order - i < NB) c = mfma(a.p[i], b.p[order - i], c);
}

// the upper halves of two float32, the first in the low half: truncated bfloat16s
__device__ __forceinline__ uint32_t upper_halves(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ float truncated(float x) {
  return __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
}

// the planes of two float32
__device__ __forceinline__ void planes_of(float a, float b, uint32_t (&out)[3]) {
  out[0] = upper_halves(a, b);
  a -= truncated(a);
  b -= truncated(b);
  out[1] = upper_halves(a, b);
  a -= truncated(a);
  b -= truncated(b);
  out[2] = upper_halves(a, b);
}

// Sizes of a head padded to DP elements (16, 32, 64, 96 or 128; zeros beyond the head). Heads of 65 to 96
// have rows of 128 in LDS, which the threads of a block divide evenly, and products of 96: what stands in a
// row beyond them is in no product (8,000 rows, 2 heads of 96, both passes: 1,543 us in float32 and 509 in
// bfloat16, padded to 128 2,252 and 684, the keys' gradients in float32 with spilled registers)
template <typename T, int DP, int TILE = 64>
struct Head {
  static constexpr int kPlanes = Store<T>::kPlanes;
  static constexpr int kSteps = DP / 16;                 // operands along the head
  static constexpr int kBlocks = (DP + 31) / 32;         // 32-element blocks of an output
  static constexpr int kHead = DP;
  static constexpr int kWide = DP == 96 ? 128 : DP;      // elements of a staged row
  static constexpr int kRow = kWide * 2 + 16;            // its bytes in a plane: 16 more spread the banks
  // walked rows of a staged tile: 32 also where three planes of 64 would leave a CU one block
  static constexpr int kTile = kPlanes == 3 && DP > 64 ? 32 : TILE;
  static constexpr int kPlane = kTile * kRow;
  // waves of a SIMD: two share its matrix core and vector unit where their registers fit
  static constexpr int kOccupancy = DP <= 32 || (kPlanes == 1 && DP == 64) ? 2 : 1;
  static constexpr int kForward = DP <= 64 || kPlanes == 1 ? 2 : 1;
  static constexpr int kBytes = kPlanes * kPlane;
};

// Operand f (of two) along the 32 walked rows of a product's registers, the weights of the next
// product. WP planes: float32 in three; 16 bits in one, rounded to nearest, or in two, the second
// one the rounding error of the first.
template <typename T, int WP>
__device__ __forceinline__ Operand<T, WP> weight_operand(const f32x16& p, int f) {
  Operand<T, WP> out;
  if constexpr (sizeof(T) == 4) {
    u32x4 w[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t x[3];
      planes_of(p[8 * f + 2 * i], p[8 * f + 2 * i + 1], x);
#pragma unroll
      for (int n = 0; n < 3; ++n) w[n][i] = x[n];
    }
#pragma unroll
    for (int n = 0; n < 3; ++n) out.p[n] = __builtin_bit_cast(Frag<T>, w[n]);
  } else {
    typedef T Two __attribute__((ext_vector_type(2)));
    u32x4 w[WP];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 x = {p[8 * f + 2 * i], p[8 * f + 2 * i + 1]};
      const Two y = __builtin_convertvector(x, Two);
      w[0][i] = __builtin_bit_cast(uint32_t, y);
      if constexpr (WP == 2)
        w[1][i] = __builtin_bit_cast(
            uint32_t, __builtin_convertvector(x - __builtin_convertvector(y, f32x2), Two));
    }
#pragma unroll
    for (int n = 0; n < WP; ++n) out.p[n] = __builtin_bit_cast(Frag<T>, w[n]);
  }
  return out;
}

// operand `step` along the head of walked row `row`
template <typename T, typename S>
__device__ __forceinline__ Operand<T> natural_operand(const char* tile, int row, int step, int half) {
  Operand<T> out;
#pragma unroll
  for (int n = 0; n < S::kPlanes; ++n)
    out.p[n] = *reinterpret_cast<const Frag<T>*>(tile + n * S::kPlane + row * S::kRow + 32 * step +
                                                 16 * half);
  return out;
}

// operand f along the 32 walked rows from `row0`, for the head's elements 32 block + lane % 32:
// sixteen lanes read four rows of sixteen elements and get a column of four each (a head of 16 gives
// the upper lanes the same columns again: outputs beyond the head, which are not stored)
template <typename T, typename S>
__device__ __forceinline__ Operand<T> transposed_operand(const char* tile, int row0, int block, int f,
                                                         int lane) {
  constexpr int kRow = S::kRow;
  typedef __attribute__((address_space(3))) s16x4* lds_ptr;
  const int l = lane % 16;
  const char* p = tile + (row0 + 16 * f + 4 * (lane / 32) + l / 4) * kRow +
                  (32 * block + (S::kWide == 16 ? 0 : 16 * ((lane / 16) & 1)) + 4 * (l % 4)) * 2;
  Operand<T> out;
#pragma unroll
  for (int n = 0; n < S::kPlanes; ++n) {
    const char* q = p + n * S::kPlane;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)q);
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(q + 8 * kRow));
    out.p[n] = __builtin_bit_cast(Frag<T>, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  return out;
}

// N elements of a row from element d on, zeros beyond the head's D elements
template <typename T, int N, bool VEC>
__device__ __forceinline__ Pack<T, N> load_row(const T* row, int d, int D) {
  Pack<T, N> out;
  if constexpr (VEC) {
    if (d < D) {
      out = *reinterpret_cast<const Pack<T, N>*>(row + d);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) out.v[i] = (T)0.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out.v[i] = row[d + i < D ? d + i : 0];
#pragma unroll
    for (int i = 0; i < N; ++i) out.v[i] = d + i < D ? out.v[i] : (T)0.0f;
  }
  return out;
}

// The own row's operands, zeros where the row does not exist. Scores are in base 2: float32 takes
// `scale` into the operands here (one more rounding of each, no product a score); 16 bits would
// lose the operands' last bits and scales the scores.
template <typename T, int DP, bool VEC>
__device__ __forceinline__ void load_own(const T* base, int64_t stride, int64_t row, bool live, int D,
                                         int half, float scale,
                                         Operand<T> (&out)[Head<T, DP>::kSteps]) {
  const T* p = base + (live ? row : 0) * stride;
  D = live ? D : 0;
#pragma unroll
  for (int c = 0; c < Head<T, DP>::kSteps; ++c) {
    const int d = 16 * c + 8 * half;
    if constexpr (sizeof(T) == 4) {
      u32x4 w[3];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const Pack<T, 4> x = load_row<T, 4, VEC>(p, d + 4 * i, D);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t y[3];
          planes_of(x.v[2 * j] * scale, x.v[2 * j + 1] * scale, y);
#pragma unroll
          for (int n = 0; n < 3; ++n) w[n][2 * i + j] = y[n];
        }
      }
#pragma unroll
      for (int n = 0; n < 3; ++n) out[c].p[n] = __builtin_bit_cast(Frag<T>, w[n]);
    } else {
      out[c].p[0] = __builtin_bit_cast(Frag<T>, load_row<T, 8, VEC>(p, d, D));
    }
  }
}
template <typename T>
__device__ __forceinline__ float score(float s, float scale) {
  return sizeof(T) == 4 ? s : s * scale;
}
// exp2(score - base)
template <typename T>
__device__ __forceinline__ float weight(float s, float scale, float base) {
  return __builtin_amdgcn_exp2f(sizeof(T) == 4 ? s - base : fmaf(s, scale, -base));
}

// the larger of a lane's value and that of the lane 32 away
__device__ __forceinline__ float max_xor32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// A tile of walked rows on its way to LDS: fetched to registers before the products of the tile
// before, written after them, so that the products cover the memory latency. A thread moves the same
// 16 bytes of every kStep-th row. Rows beyond the structure, elements beyond the head and rows that
// the mask leaves out become zeros as they are written, so that what they hold reaches no sum: no
// address waits for the mask (24,000 rows of 4 heads with a tenth masked,
// both passes 4.01 ms where they did, 3.24 so). A thread whose piece is beyond the head reads its row's
// first one (8,000 rows, 2 heads of 80 in float32, both passes: 1,553 us, with an address a row 1,742). Loads beyond the structure go to the tile's first row,
// which exists.
template <typename T, typename S, int THREADS, bool VEC>
struct Stage {
  static constexpr int kPer = 16 / sizeof(T);
  static constexpr int kChunks = S::kWide / kPer;          // 16-byte pieces of a row
  static constexpr int kStep = THREADS / kChunks;
  static constexpr int kCount = (S::kTile + kStep - 1) / kStep;
  static_assert(THREADS % kChunks == 0, "a thread keeps its place in the rows");
  typedef Pack<T, kPer> Piece;
  static constexpr uint64_t kAll = ~0ull >> (64 - S::kTile);
  Piece x[kCount];
  bool full;                                               // no elements beyond the head in its products
  bool near;                                               // 16-byte pieces, and a tile spans less than 2 GB
  int row, at;                                             // its first row, its element of a row
  int64_t offset;

  __device__ __forceinline__ void init(int64_t stride, int D) {
    row = threadIdx.x / kChunks;
    at = threadIdx.x % kChunks * kPer;
    offset = (row < S::kTile ? row : 0) * stride + (at < D ? at : 0);   // heads of 16: more threads than pieces
    full = VEC && D == S::kHead;
    near = stride >= (VEC ? 0 : kPer) && stride < (int64_t)1 << 22;
  }
  // `tile`: the first of `rows` rows
  __device__ __forceinline__ void fetch(const T* tile, int64_t stride, int64_t rows, int D) {
    // One address a thread, the rest scalar. Pieces without alignment may reach beyond their head, which
    // is within the tensor where another row follows the tile's (8,000 rows, 2 heads of 33 in bfloat16,
    // both passes: 281 us, element by element 460; the elements beyond are zeros from commit on).
    if (near && rows >= S::kTile + (VEC ? 0 : 1)) {
      const uint32_t bytes = (uint32_t)offset * (uint32_t)sizeof(T);
#pragma unroll
      for (int n = 0; n < kCount; ++n) {
        const char* p = reinterpret_cast<const char*>(tile + n * kStep * stride) + bytes;
        if constexpr (VEC)
          x[n] = *reinterpret_cast<const Pack<T, kPer>*>(p);
        else
          __builtin_memcpy(&x[n], p, sizeof(x[n]));
      }
      return;
    }
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const int r = row + n * kStep;
      const T* p = at < D && r < rows && r < S::kTile ? tile + n * kStep * stride + offset : tile;
      if constexpr (VEC) {
        x[n] = *reinterpret_cast<const Pack<T, kPer>*>(p);
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) x[n].v[j] = p[at + j < D ? j : 0];
      }
    }
  }
  // `keep`: a bit a row of the tile
  __device__ __forceinline__ void commit(char* tile, int D, uint64_t keep) {
    if (!full || keep != kAll) {
      const uint64_t mine = row < S::kTile && at < D ? keep >> row : 0;
#pragma unroll
      for (int n = 0; n < kCount; ++n) {
        const bool kept = (mine >> (n * kStep)) & 1;
        if (!VEC) {
#pragma unroll
          for (int j = 0; j < kPer; ++j) x[n].v[j] = kept && at + j < D ? x[n].v[j] : (T)0.0f;
          continue;
        }
        u32x4 w = __builtin_bit_cast(u32x4, x[n]);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = kept ? w[j] : 0u;
        x[n] = __builtin_bit_cast(Piece, w);
      }
    }
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const int r = row + n * kStep;
      if (S::kTile % kStep != 0 && r >= S::kTile) break;
      char* p = tile + r * S::kRow + at * 2;
      const u32x4 w = __builtin_bit_cast(u32x4, x[n]);
      if constexpr (sizeof(T) == 4) {
        uint32_t a[3], b[3];
        planes_of(__uint_as_float(w[0]), __uint_as_float(w[1]), a);
        planes_of(__uint_as_float(w[2]), __uint_as_float(w[3]), b);
#pragma unroll
        for (int m = 0; m < 3; ++m) *reinterpret_cast<u32x2*>(p + m * S::kPlane) = u32x2{a[m], b[m]};
      } else {
        *reinterpret_cast<u32x4*>(p) = w;
      }
    }
  }
};

// This lane's byte of the mask (NULL: none) for a tile on its way, zero for rows from `end` on. A bit a
// row is the ballot of it, formed where the tile is used.
template <int ROWS>
__device__ __forceinline__ uint8_t row_byte(int64_t first, int64_t end, const uint8_t* mask, int lane) {
  const int64_t row = first + lane;
  if (lane >= ROWS || row >= end) return 0;
  return mask == nullptr ? 1 : mask[row];
}

// Whether the walked row of this lane in register r is among `rows` (a bit a row of a 32-row product): a
// mask of lanes from two scalar bits, so that the choice costs one vector instruction
__device__ __forceinline__ bool has_row(uint32_t rows, int r) {
  const uint32_t low = (uint32_t)((int32_t)(rows << (31 - tile_row(r, 0))) >> 31);
  const uint32_t high = (uint32_t)((int32_t)(rows << (31 - tile_row(r, 1))) >> 31);
  return __builtin_amdgcn_inverse_ballot_w64(low | (uint64_t)high << 32);
}

// a bit a row of a tile with `rows` (at least one) before its end
template <int ROWS>
__device__ __forceinline__ uint64_t rows_before(int64_t rows) {
  return ~0ull >> (64 - (rows < ROWS ? (int)rows : ROWS));
}

// the wave's result, own rows as columns: element 32 b + row(r) of own row `out` = acc[b][r] * factor
template <typename T, int BLOCKS>
__device__ __forceinline__ void store_own(T* out, const f32x16 (&acc)[BLOCKS], float factor, int D,
                                          bool vec, int half) {
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * b + 8 * g + 4 * half;
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = acc[b][4 * g + j] * factor;
      if (vec) {
        if (d < D) store_pack<T, 4>(out + d, v);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (d + j < D) out[d + j] = (T)v[j];
      }
    }
  }
}

// what a launch is given, by value
struct AttentionArgs {
  const void *q, *k, *v, *out, *grad;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;
  int64_t n_tokens;
  const int32_t* tiles;            // (first row, end of its structure, begin of its structure) each
  int64_t n_tiles;
  const uint8_t* mask;
  int heads, kv_heads, D;
  int splits;                      // parts of the walked side, each with results of its own
  bool vec, vec_out;
  bool head_major;                 // blocks walk a head's tiles in turn, not a tile's heads
  float scale;
  float *lse, *delta;              // (heads, tokens): base-2 logarithm of the sums; rows' dot products
  float *part, *part_lse;          // of the parts: results, logarithms
  void *dq, *dk, *dv, *result;
};

struct Tile {
  int64_t first, end, begin;
  int head, split;
};

// The block's tile, head and part. The plan lists the tiles of longer structures first, and blocks
// start in their order: the long ones do not come last.
__device__ __forceinline__ void block_tile(const AttentionArgs& a, int heads, Tile& t) {
  int64_t slot = blockIdx.x, tile;
  if (a.head_major) {
    tile = slot % a.n_tiles;
    slot /= a.n_tiles;
    t.split = (int)(slot % a.splits);
    t.head = (int)(slot / a.splits);
  } else {
    t.head = (int)(slot % heads);
    slot /= heads;
    t.split = (int)(slot % a.splits);
    tile = slot / a.splits;
  }
  // a tile that is not of these tokens reads and writes none outside them
  t.first = max(a.tiles[3 * tile], 0);
  t.end = min((int64_t)a.tiles[3 * tile + 1], a.n_tokens);
  t.begin = max(a.tiles[3 * tile + 2], 0);
}

// part `split` of `n` walked tiles: [from, to)
__device__ __forceinline__ void walk_part(int64_t n, const AttentionArgs& a, int split, int64_t& from,
                                          int64_t& to) {
  from = n * split / a.splits;
  to = n * (split + 1) / a.splits;
}

constexpr int kCus = 256;
constexpr int kMostSplits = 16;

// Walked rows of a part, at least: some ten microseconds of walking, beside which a join is small (512 rows
// of 64 elements in 16 bits; fewer of wider heads, and a sixth in float32, which has six products for one).
inline int64_t split_rows(int dtype, int D) {
  return std::max<int64_t>(64, 512 * 64 / (std::max(D, 32) * (dtype == XNN_F32 ? 6 : 1)));
}

// Parts of the walked side, for `blocks` blocks of equal length without: as few as give every one of the
// chip's 256 CUs `each` blocks and leave none idle for more than a tenth of the time.
inline int attention_splits(int64_t blocks, int64_t walked, int64_t rows, int each) {
  const int64_t most = std::min<int64_t>(kMostSplits, walked / rows);
  int best = 1;
  double best_use = 0.0;
  for (int s = 1; s <= std::max<int64_t>(most, 1); ++s) {
    const int64_t n = blocks * s;
    const double use = (double)n / ((n + kCus - 1) / kCus * kCus) *
                       (n < each * kCus ? 0.6 + 0.2 * n / (each * kCus) : 1.0);
    if (use > best_use * 1.03) {
      best = s;
      best_use = use;
    }
    if (best_use >= 0.9) break;
  }
  return best;
}
// Two blocks a CU for the forward pass (24,000 rows of 4 heads, 752 blocks: 752 us undivided, 799 in two
// parts, with the join); four for the gradients, two of which a CU holds at a time (2,430 us undivided,
// 2,278 in two parts). 9,000 rows of 4 heads, 284 blocks: five parts for all.
inline int forward_splits(int64_t blocks, int64_t walked, int64_t rows) {
  return attention_splits(blocks, walked, rows, 2);
}
inline int backward_splits(int64_t blocks, int64_t walked, int64_t rows) {
  return attention_splits(blocks, walked, rows, 4);
}

// Rows of a block: 32, one wave, where no structure is longer than 64 (the other waves of a larger
// block would idle) and one wave's registers hold a tile on its way, otherwise 128. Both passes in
// float32, blocks of 32 and of 128: 1,024 structures of 10 to 60 atoms, 4 heads of 16, 75 and 99 us; 256 of
// 64 to 128 atoms 76 and 69; 128 of 128 to 256, heads of 32, 135 and 124.
inline bool short_head(int bytes, int D) { return bytes * D <= 128; }
inline int attention_rows(const xnn_attention_tiles* plan, int bytes, int D) {
  return plan->max_atoms <= 64 && short_head(bytes, D) ? 32 : 128;
}

// blocks of a launch without parts
inline int64_t attention_blocks(const xnn_attention_tiles* plan, int heads) {
  return plan->n_tiles128 * heads;
}

// Planes of the weights (probabilities, score gradients). float32 has three. In 16 bits one: its rounding
// is of the size of the output's own, 1.4 times the error of an output that is rounded once, whatever the
// length. Where few elements average it a second plane, the rounding error of the first, is taken as
// well: in blocks of one wave, whose products are not what bounds them (1,024 molecules of 10 to 60 atoms: the
// same time), and where all scores are some microseconds of work (4 heads of 64, both passes: 1,400 atoms 81
// us with and without; 4,000 atoms 176 with, 152 without). So it is for the queries' gradient in
// heads of at most 32 elements: the row's weights sum to zero, so that what is left of a sum over few
// elements is smaller than its parts (1.45 to 1.67 times the output's rounding with one plane).
constexpr int64_t kFineScores = (int64_t)1 << 23;
inline bool fine_weights(const AttentionArgs& a, const xnn_attention_tiles* plan) {
  return a.n_tokens * plan->max_atoms * a.heads <= kFineScores;
}
inline bool fine_query_gradient(const AttentionArgs& a, const xnn_attention_tiles* plan) {
  return a.D <= 32 || fine_weights(a, plan);
}

// Probabilities of a long structure are small beside float16's least normal number, 2^-14: the gradients
// carry them, and what is formed from them, 2^this times larger (half the average 1 / n at most, and no
// more than 2^5) and take the factor back at the end. Exact; the other types have the exponents.
template <typename T>
__device__ __forceinline__ int carried(int64_t n) {
  if constexpr (Store<T>::kPlanes == 3 || __is_same(T, bf16_t)) return 0;
  return max(0, min(5, 63 - __clzll((long long)n) - 9));
}

// Score gradients on their way to float16, whose largest number they can pass where the gradients do not (a
// peaked row, large cotangents). A row that passes 2^15 goes on in units that are a power of two larger: its
// score gradients and what they have summed so far shrink with `unit`, which the result takes back. Exact; what
// it costs is the largest of a product's score gradients (both passes, without and with it: 8,000 rows, 2
// heads of 64, 239 and 252 us, 24,000 rows, 4 heads of 64, 3.04 and 3.16 ms, 1,000 structures of 35, 4 heads of
// 16, 85 and 84 us).
template <typename T>
struct GradientRange {
  template <int BLOCKS>
  __device__ __forceinline__ void hold(f32x16&, f32x16 (&)[BLOCKS]) {}
  __device__ __forceinline__ float back() const { return 1.0f; }
};
template <>
struct GradientRange<f16_t> {
  float unit = 1.0f;
  bool smaller = false;            // some row of the wave is in other units

  // `x`: a product's score gradients; `sum`: the rows' sums of them
  template <int BLOCKS>
  __device__ __forceinline__ void hold(f32x16& x, f32x16 (&sum)[BLOCKS]) {
    if (smaller) {
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] *= unit;
    }
    float most = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(x[r]));
    if (!__any(most > 0x1p15f)) return;
    most = max_xor32(most);                                // a row is in two lanes
    const int e = most > 0x1p15f && most < INFINITY ? (int)(__float_as_uint(most) >> 23) - 127 - 14 : 0;
    const float shrink = ldexpf(1.0f, -e);
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] *= shrink;
#pragma unroll
    for (int d = 0; d < BLOCKS; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum[d][r] *= shrink;
    unit *= shrink;
    smaller = true;
  }
  __device__ __forceinline__ float back() const { return 1.0f / unit; }
};

// the tiles of a launch; rows that are not moved 16 bytes at a time are always walked by 128
inline int attention_pick(AttentionArgs& a, const xnn_attention_tiles* plan, int dtype) {
  const int rows = a.vec ? attention_rows(plan, storage_bytes(dtype), a.D) : 128;
  a.tiles = rows == 32 ? plan->tiles32 : plan->tiles128;
  a.n_tiles = rows == 32 ? plan->n_tiles32 : plan->n_tiles128;
  return rows;
}

// the checks and the choices that forward and backward share
inline int attention_args(AttentionArgs& a, int dtype, const xnn_heads* q, const xnn_heads* k,
                          const xnn_heads* v, int64_t n_tokens, int32_t head_dim,
                          const xnn_attention_tiles* plan, const uint8_t* mask, float scale) {
  XNN_REQUIRE(is_storage(dtype), "dtype must be XNN_F32, XNN_BF16 or XNN_F16");
  XNN_REQUIRE(q && k && v && plan, "NULL heads or plan");
  XNN_REQUIRE(n_tokens >= 0 && n_tokens < ((int64_t)1 << 31) - 128, "token count out of range");
  XNN_REQUIRE(head_dim >= 1 && head_dim <= 128, "head_dim must be in [1, 128]");
  XNN_REQUIRE(q->n_heads >= 1 && k->n_heads >= 1 && k->n_heads == v->n_heads &&
                  q->n_heads % k->n_heads == 0,
              "the heads must be a multiple of those of keys and values");
  XNN_REQUIRE(scale > 0.0f && scale < INFINITY, "scale must be positive and finite");
  XNN_REQUIRE(plan->n_tokens == n_tokens, "the plan is of another number of tokens");
  a = AttentionArgs{};
  if (n_tokens == 0) return XNN_OK;
  XNN_REQUIRE(q->data && k->data && v->data, "NULL input");
  XNN_REQUIRE(plan->tiles32 && plan->tiles128 && plan->n_tiles32 > 0 && plan->n_tiles128 > 0,
              "empty plan");
  XNN_REQUIRE(plan->n_tiles32 * q->n_heads <= (int64_t)1 << 26, "too many tiles");
  a.q = q->data;
  a.k = k->data;
  a.v = v->data;
  a.q_token = q->token_stride;
  a.q_head = q->head_stride;
  a.k_token = k->token_stride;
  a.k_head = k->head_stride;
  a.v_token = v->token_stride;
  a.v_head = v->head_stride;
  a.n_tokens = n_tokens;
  a.heads = q->n_heads;
  a.kv_heads = k->n_heads;
  a.D = head_dim;
  a.mask = mask;
  a.scale = scale;
  a.splits = 1;
  const int per = 16 / storage_bytes(dtype);
  a.vec = ((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v) % 16 == 0 &&
          (a.q_token | a.q_head | a.k_token | a.k_head | a.v_token | a.v_head) % per == 0 &&
          head_dim % per == 0;
  // Keys and values of all heads of a structure within half an XCD's 4 MB of L2: its heads side by side,
  // which spreads the longest structures over the chip (64 of 10 to 1,000 atoms, 8 heads of 64 in 16 bits: 33 us
  // forward, one head after the other 42; neighbouring blocks are on different XCDs, so that each fetches the
  // lines of packed projections for itself, 40.6 MB for 20.2). Otherwise one head after the other (24,000 atoms, 16
  // heads of 64 on 4, both passes: 11.25 ms, side by side 11.2 to 11.7; 3 heads 2.28 and 2.30).
  a.head_major = plan->max_atoms * a.kv_heads * head_dim * storage_bytes(dtype) * 2 > (2 << 20);
  return XNN_OK;
}

}  // namespace xnn

// One launch of kernel<T, DP, waves, tile, vec, weight planes> for arguments `a` of `rows` rows a block on
// stream `s`
#define XNN_ATTENTION_LAUNCH(kernel, grid, fine)                                                    \
  do {                                                                                              \
    constexpr int kOne = Store<T>::kPlanes, kFine = kOne == 3 ? 3 : 2;                              \
    if (!a.vec && fine)                                                                             \
      hipLaunchKernelGGL((kernel<T, DP, 4, 64, false, kFine>), grid, dim3(256), 0, s, a);           \
    else if (!a.vec)                                                                                \
      hipLaunchKernelGGL((kernel<T, DP, 4, 64, false, kOne>), grid, dim3(256), 0, s, a);            \
    else if (rows == 128 && fine)                                                                   \
      hipLaunchKernelGGL((kernel<T, DP, 4, 64, true, kFine>), grid, dim3(256), 0, s, a);            \
    else if (rows == 128)                                                                           \
      hipLaunchKernelGGL((kernel<T, DP, 4, 64, true, kOne>), grid, dim3(256), 0, s, a);             \
    else if constexpr (sizeof(T) * DP <= 128)                                                       \
      hipLaunchKernelGGL((kernel<T, DP, 1, 32, true, kFine>), grid, dim3(64), 0, s, a);             \
  } while (0)
