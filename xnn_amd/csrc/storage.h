// Element types of the attention operators: float32, bfloat16 and float16 in memory, float32
// in the registers; rounding to 16 bits is to nearest even, once per stored value.
#pragma once
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "xnn_amd.h"

namespace xnn {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

inline bool is_storage(int dtype) {
  return dtype == XNN_F32 || dtype == XNN_BF16 || dtype == XNN_F16;
}
inline int storage_bytes(int dtype) { return dtype == XNN_F32 ? 4 : 2; }

// N consecutive elements, loaded and stored as one access where N fills one
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_pack(const T* __restrict__ p, float* out) {
  const Pack<T, N> x = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = (float)x.v[i];
}

template <typename T, int N>
__device__ __forceinline__ void store_pack(T* __restrict__ p, const float* in) {
  Pack<T, N> x;
#pragma unroll
  for (int i = 0; i < N; ++i) x.v[i] = (T)in[i];
  *reinterpret_cast<Pack<T, N>*>(p) = x;
}

}  // namespace xnn

// One call of `fn<T>(...)` by dtype code
#define XNN_STORAGE_DISPATCH(dtype, T, ...)  \
  do {                                       \
    if ((dtype) == XNN_F32) {                \
      typedef float T;                       \
      __VA_ARGS__;                           \
    } else if ((dtype) == XNN_BF16) {        \
      typedef ::xnn::bf16_t T;               \
      __VA_ARGS__;                           \
    } else {                                 \
      typedef ::xnn::f16_t T;                \
      __VA_ARGS__;                           \
    }                                        \
  } while (0)
