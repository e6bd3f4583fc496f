// The 8-bit forms a paged cache holds its rows in, for the kernels that write and read one (hstu_append.cu; hstu_decode8.cu,
// hstu_rows8.cu and hstu_paged.cu through hstu_mma8.cuh): value = number * scale, one fp32 scale per block of tokens and head.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "hstu_common.cuh"

namespace hstu {

struct E4m3 {
  // the scale of a block: amax / scale <= 448 = 1.75 * 2^8
  static constexpr int kExp = 8;
  static constexpr uint32_t kFraction = 0x600000u;
  static __device__ __forceinline__ uint8_t from_float(float x) {   // round to nearest even, +-448 beyond, NaN stays NaN
    return static_cast<uint8_t>(__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3));
  }
  static __device__ __forceinline__ uint32_t from_floats(float a, float b) {   // two of them, the first in the low byte
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  }
  static __device__ __forceinline__ float to_float(uint8_t v) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3)));
  }
};
struct Int8 {
  // amax / scale <= 127 = 1.984375 * 2^6
  static constexpr int kExp = 6;
  static constexpr uint32_t kFraction = 0x7e0000u;
  static __device__ __forceinline__ uint8_t from_float(float x) {   // round to nearest even, +-127 beyond, NaN becomes 0
    int v = __float2int_rn(x);
    v = v > 127 ? 127 : v < -127 ? -127 : v;
    return static_cast<uint8_t>(static_cast<int8_t>(v));
  }
  static __device__ __forceinline__ uint32_t from_floats(float a, float b) {
    return static_cast<uint32_t>(from_float(a)) | (static_cast<uint32_t>(from_float(b)) << 8);
  }
  static __device__ __forceinline__ float to_float(uint8_t v) { return static_cast<float>(static_cast<int8_t>(v)); }
};

// The smallest power of two that amax fits, from 2^-100 on.  Powers of two: the quotient is exact, so a row is rounded once
// and the result does not depend on how the division is done; a scale that grows later only shifts what the block holds.
template <typename H> __device__ __forceinline__ float block_scale(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  int e = static_cast<int>(bits >> 23) - 127 - H::kExp + ((bits & 0x7fffffu) > H::kFraction ? 1 : 0);
  if (e < -100 || bits < 0x800000u) e = -100;
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

}  // namespace hstu
