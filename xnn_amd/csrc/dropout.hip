// Dropout from a counter-based generator with an optional residual (gfx950, wave64).
//
//   out[e] = residual[e] + keep(e) x[e] 65536 / (65536 - drop)
//
// keep(e) compares a 16-bit draw with `drop`. The draws of elements 8 i .. 8 i + 7 are the half
// words of one Philox4x32-10 block (Salmon, Moraes, Dror and Shaw, SC 2011) with counter
// (i, offset) and key `seed`: a function of the element's index alone, so the backward pass
// forms the mask again and none is stored. The probability is a multiple of 1/65536 and the factor
// is that of the rounded probability, so the mean is kept exactly.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.h"
#include "device.h"
#include "storage.h"

namespace xnn {

struct Philox {
  uint32_t c[4];
};

__device__ __forceinline__ Philox philox(uint64_t index, uint64_t offset, uint64_t seed) {
  uint32_t c0 = (uint32_t)index, c1 = (uint32_t)(index >> 32);
  uint32_t c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Philox{{c0, c1, c2, c3}};
}

// VEC: the arrays are 16-byte aligned; a thread takes the eight elements of one block of draws. A stream:
// twenty 32-bit products for eight elements hide behind their bytes. 72,000 x 512 in bfloat16 with a
// residual 37 us for 221 MB, 6.0 TB/s, without one 27 us for 147 MB; 9,000 x 128 in float32 4 us, the
// launch. Sixteen bits a draw in place of thirty-two halve the products.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dropout_kernel(const T* __restrict__ x,
                                                      const T* __restrict__ residual, int64_t n,
                                                      uint32_t drop, float factor, uint64_t seed,
                                                      uint64_t offset,
                                                      const int64_t* __restrict__ offset_add,
                                                      T* __restrict__ out) {
  if (offset_add != nullptr) offset += (uint64_t)*offset_add;
  const int64_t blocks = (n + 7) / 8;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < blocks;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t e = 8 * i;
    const bool whole = VEC && e + 8 <= n;
    float a[8], b[8];
    if (whole) {
      constexpr int kPer = 16 / sizeof(T);
#pragma unroll
      for (int j = 0; j < 8; j += kPer) load_pack<T, kPer>(x + e + j, a + j);
      if (residual != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; j += kPer) load_pack<T, kPer>(residual + e + j, b + j);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        a[j] = e + j < n ? (float)x[e + j] : 0.0f;
        if (residual != nullptr) b[j] = e + j < n ? (float)residual[e + j] : 0.0f;
      }
    }
    const Philox r = philox((uint64_t)i, offset, seed);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t draw = (j & 1) ? r.c[j / 2] >> 16 : r.c[j / 2] & 0xFFFFu;
      a[j] = draw >= drop ? a[j] * factor : 0.0f;
      if (residual != nullptr) a[j] += b[j];
    }
    if (whole) {
      constexpr int kPer = 16 / sizeof(T);
#pragma unroll
      for (int j = 0; j < 8; j += kPer) store_pack<T, kPer>(out + e + j, a + j);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (e + j < n) out[e + j] = (T)a[j];
    }
  }
}

template <typename T>
static int dropout(const void* x, const void* residual, int64_t n, uint32_t drop, uint64_t seed,
                   uint64_t offset, const int64_t* offset_add, void* out, hipStream_t s) {
  const float factor = drop < 65536u ? 65536.0f / (float)(65536u - drop) : 0.0f;
  const bool vec = ((uintptr_t)x | (uintptr_t)residual | (uintptr_t)out) % 16 == 0;
  const int64_t blocks = (n + 2047) / 2048;
  const dim3 grid((unsigned)std::min<int64_t>(blocks, 1 << 20)), block(256);
  const T* xt = static_cast<const T*>(x);
  const T* rt = static_cast<const T*>(residual);
  T* o = static_cast<T*>(out);
  if (vec)
    hipLaunchKernelGGL((dropout_kernel<T, true>), grid, block, 0, s, xt, rt, n, drop, factor, seed,
                       offset, offset_add, o);
  else
    hipLaunchKernelGGL((dropout_kernel<T, false>), grid, block, 0, s, xt, rt, n, drop, factor,
                       seed, offset, offset_add, o);
  XNN_LAUNCH_CHECK();
  return XNN_OK;
}

}  // namespace xnn

using namespace xnn;

extern "C" {

int xnn_dropout_add(int dtype, const void* x, const void* residual, int64_t n, int32_t drop,
                    uint64_t seed, uint64_t offset, const int64_t* offset_add, void* out,
                    xnn_stream_t stream) {
  XNN_REQUIRE(is_storage(dtype), "dtype must be XNN_F32, XNN_BF16 or XNN_F16");
  XNN_REQUIRE(n >= 0, "negative size");
  XNN_REQUIRE(drop >= 0 && drop <= 65536, "drop must be in [0, 65536]");
  if (n == 0) return XNN_OK;
  XNN_REQUIRE(x && out, "NULL input or output");
  XNN_STORAGE_DISPATCH(dtype, T,
                       return dropout<T>(x, residual, n, (uint32_t)drop, seed, offset, offset_add,
                                         out, as_hip(stream)));
}

}  // extern "C"
