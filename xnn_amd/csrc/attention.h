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
//   walk(tile) x own   = tile (natural rows from LDS, 16 bytes a lane)  x  own (registers)
//   own^T += tile^T x weights: tile read across its rows (float32: one element a lane and row;
//            16 bits: the transposing LDS read, four rows a lane)
//
// float32 uses v_mfma_f32_32x32x2_f32 (products and sums in float32), 16 bits
// v_mfma_f32_32x32x16_{bf16,f16} (sums in float32).
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "common.h"
#include "device.h"
#include "storage.h"

namespace xnn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
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

// 16 bytes of one row a lane: the unit of loads and of operands
template <typename T>
struct Mma;
template <>
struct Mma<float> {
  typedef f32x4 Frag;
  static __device__ __forceinline__ void mma(Frag a, Frag b, f32x16& c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
  }
};
template <>
struct Mma<bf16_t> {
  typedef bf16x8 Frag;
  static __device__ __forceinline__ void mma(Frag a, Frag b, f32x16& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<f16_t> {
  typedef f16x8 Frag;
  static __device__ __forceinline__ void mma(Frag a, Frag b, f32x16& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

// Sizes of a head padded to DP elements (16, 32, 64 or 128; zeros beyond the head)
template <typename T, int DP>
struct Head {
  static constexpr int kPer = 16 / sizeof(T);            // elements of 16 bytes
  static constexpr int kSteps = DP * sizeof(T) / 32;     // operands along the head (natural)
  static constexpr int kBlocks = (DP + 31) / 32;         // 32-element blocks of an output
  static constexpr int kWide = kBlocks * 32;             // elements of a staged row
  static constexpr int kRow = kWide * sizeof(T) + 16;    // its bytes: 16 more spread the banks
  static constexpr int kFrags = sizeof(T);               // operands along 32 walked rows
};

// operand f of the weights: registers of a 32 x 32 product, rounded to T
template <typename T>
__device__ __forceinline__ typename Mma<T>::Frag weight_frag(const f32x16& p, int f) {
  typename Mma<T>::Frag out;
  constexpr int kPer = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < kPer; ++i) out[i] = (T)p[f * kPer + i];
  return out;
}

// operand `step` along the head of walked row `row` (natural order)
template <typename T, int DP>
__device__ __forceinline__ typename Mma<T>::Frag natural_frag(const char* tile, int row, int step,
                                                              int half) {
  return *reinterpret_cast<const typename Mma<T>::Frag*>(tile + row * Head<T, DP>::kRow +
                                                         32 * step + 16 * half);
}

// operand f along the 32 walked rows from `row0`, transposed: own side's elements 32 block + lane % 32
template <typename T, int DP>
__device__ __forceinline__ typename Mma<T>::Frag transposed_frag(const char* tile, int row0,
                                                                 int block, int f, int lane) {
  constexpr int kRow = Head<T, DP>::kRow;
  const int half = lane / 32;
  if constexpr (sizeof(T) == 4) {
    const char* p = tile + (row0 + 8 * f + 4 * half) * kRow + (32 * block + lane % 32) * 4;
    f32x4 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = *reinterpret_cast<const float*>(p + i * kRow);
    return out;
  } else {
    // sixteen lanes read four rows of sixteen elements and get a column of four each
    const int l = lane % 16;
    const char* p = tile + (row0 + 16 * f + 4 * half + l / 4) * kRow +
                    (32 * block + 16 * ((lane / 16) & 1) + 4 * (l % 4)) * 2;
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p);
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 8 * kRow));
    const s16x8 both = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(typename Mma<T>::Frag, both);
  }
}

// 16 bytes of a row from element d on, zeros beyond the head's D elements
template <typename T>
__device__ __forceinline__ typename Mma<T>::Frag load_frag(const T* row, int d, int D, bool vec) {
  typedef typename Mma<T>::Frag Frag;
  constexpr int kPer = 16 / sizeof(T);
  Frag out;
  if (vec) {
    if (d < D) {
      out = *reinterpret_cast<const Frag*>(row + d);
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) out[i] = (T)0.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) out[i] = d + i < D ? row[d + i] : (T)0.0f;
  }
  return out;
}

// the own row's operands in registers, zeros where the row does not exist
template <typename T, int DP>
__device__ __forceinline__ void load_own(const T* base, int64_t stride, int64_t row, bool live,
                                         int D, bool vec, int half,
                                         typename Mma<T>::Frag (&out)[Head<T, DP>::kSteps]) {
  constexpr int kPer = Head<T, DP>::kPer;
#pragma unroll
  for (int c = 0; c < Head<T, DP>::kSteps; ++c)
    out[c] = load_frag<T>(base + (live ? row : 0) * stride, (2 * c + half) * kPer, live ? D : 0, vec);
}

// Scores in base 2. float32 takes the scale into the own row's operands once (one more rounding of
// each, no product a score); 16 bits would lose the operands' last bits and scale the scores.
template <typename T, int DP>
__device__ __forceinline__ void scale_own(float scale,
                                          typename Mma<T>::Frag (&own)[Head<T, DP>::kSteps]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int c = 0; c < Head<T, DP>::kSteps; ++c) own[c] *= scale;
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

// Rows [first, first + ROWS) of one head into LDS; zeros beyond `end`, beyond the head and in rows
// that `skip` (a mask's zeros, NULL: none) leaves out, so that what they hold reaches no sum.
template <typename T, int DP, int ROWS, int THREADS>
__device__ __forceinline__ void stage(const T* base, int64_t stride, int64_t first, int64_t end,
                                      int D, bool vec, const uint8_t* mask, char* tile) {
  typedef Head<T, DP> S;
  constexpr int kChunks = S::kWide / S::kPer;
#pragma unroll
  for (int i0 = 0; i0 < ROWS * kChunks; i0 += THREADS) {
    const int i = i0 + threadIdx.x;
    if (ROWS * kChunks % THREADS != 0 && i >= ROWS * kChunks) break;
    const int r = i / kChunks, c = i % kChunks;
    const int64_t row = first + r;
    const bool live = row < end && (mask == nullptr || mask[row] != 0);
    *reinterpret_cast<typename Mma<T>::Frag*>(tile + r * S::kRow + 16 * c) =
        load_frag<T>(base + (live ? row : 0) * stride, c * S::kPer, live ? D : 0, vec);
  }
}

// one bit a walked row of a tile of 64: rows before `end` that the mask keeps (the whole wave calls)
__device__ __forceinline__ uint64_t live_rows(int64_t first, int64_t end, const uint8_t* mask,
                                              int lane) {
  const int64_t row = first + lane;
  return __ballot(row < end && (mask == nullptr || mask[row] != 0));
}

// the wave's result, own rows as columns: element 32 b + row(r) of own row `out` = acc[b][r] * factor
template <typename T, int DP>
__device__ __forceinline__ void store_own(T* out, const f32x16 (&acc)[Head<T, DP>::kBlocks],
                                          float factor, int D, bool vec, int half) {
#pragma unroll
  for (int b = 0; b < Head<T, DP>::kBlocks; ++b) {
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
  bool vec, vec_out;
  bool head_major;                 // blocks walk a head's tiles in turn, not a tile's heads
  float scale;
  float *lse, *delta;              // (heads, tokens): base-2 logarithm of the sums; rows' dot products
  void *dq, *dk, *dv, *result;
};

struct Tile {
  int64_t first, end, begin;
  int head;
};

// the block's tile and head; consecutive slots lie in one XCD and share its L2
__device__ __forceinline__ bool block_tile(const AttentionArgs& a, int heads, Tile& t) {
  const int64_t slot = xcd_slot();
  if (slot >= a.n_tiles * heads) return false;
  const int64_t tile = a.head_major ? slot % a.n_tiles : slot / heads;
  t.head = (int)(a.head_major ? slot / a.n_tiles : slot % heads);
  t.first = a.tiles[3 * tile];
  t.end = a.tiles[3 * tile + 1];
  t.begin = a.tiles[3 * tile + 2];
  return true;
}

// The checks and the choices that forward and backward share. `rows`: of a tile, 128 where that
// still gives every SIMD of the chip (1,024) a wave, 64 below and where no structure is longer.
inline int attention_args(AttentionArgs& a, int dtype, const xnn_heads* q, const xnn_heads* k,
                          const xnn_heads* v, int64_t n_tokens, int32_t head_dim,
                          const xnn_attention_tiles* plan, const uint8_t* mask, float scale,
                          int& rows) {
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
  XNN_REQUIRE(plan->tiles64 && plan->tiles128 && plan->n_tiles64 > 0 && plan->n_tiles128 > 0,
              "empty plan");
  XNN_REQUIRE(plan->n_tiles64 * q->n_heads <= (int64_t)1 << 30, "too many tiles");
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
  const int per = 16 / storage_bytes(dtype);
  a.vec = ((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v) % 16 == 0 &&
          (a.q_token | a.q_head | a.k_token | a.k_head | a.v_token | a.v_head) % per == 0 &&
          head_dim % per == 0;
  rows = plan->max_atoms <= 64 || plan->n_tiles128 * q->n_heads * 4 < 1024 ? 64 : 128;
  a.tiles = rows == 64 ? plan->tiles64 : plan->tiles128;
  a.n_tiles = rows == 64 ? plan->n_tiles64 : plan->n_tiles128;
  // keys and values of all heads of a structure within half an XCD's 4 MB of L2: its heads side by
  // side (they share the lines of packed projections), otherwise one head after the other
  a.head_major = plan->max_atoms * a.kv_heads * head_dim * storage_bytes(dtype) * 2 > (2 << 20);
  return XNN_OK;
}

}  // namespace xnn
