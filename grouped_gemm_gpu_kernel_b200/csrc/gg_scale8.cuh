// gg_scale8.cuh -- a block of 128 values in 8 bits with one FP32 scale, as the norm and the gated 8-bit product write it.
#pragma once

#include <cuda_fp8.h>

#include <cstdint>

namespace gg {

// A value's bits without the sign: as numbers they are ordered like the magnitudes, infinity above the finite ones
// and NaN above that, so a maximum over them finds a value that is not finite.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// scale = the block's largest magnitude over the type's largest number; values are multiplied by its inverse, taken once.
// Below 2^-100 the scale would leave FP32's normal numbers: such a block is held as zeros. A block with an
// infinity or a NaN gets a scale that is not finite.
struct Scale8 {
  float scale, inverse;
  __device__ __forceinline__ Scale8(uint32_t top, float largest) {
    const float most = __uint_as_float(top);
    const bool none = most < 7.888609e-31f;  // 2^-100; false for NaN
    scale = none ? 0.0f : most / largest;
    inverse = none ? 0.0f : largest / most;
  }
  // Four values rounded to nearest even, x in the low byte. The product may pass the largest number by a rounding of
  // FP32; the conversion saturates.
  __device__ __forceinline__ uint32_t four(float x, float y, float z, float w, bool e5m2) const {
    const __nv_fp8_interpretation_t kind = e5m2 ? __NV_E5M2 : __NV_E4M3;
    const float2 lo = make_float2(x * inverse, y * inverse), hi = make_float2(z * inverse, w * inverse);
    return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, kind)) |
           static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, kind)) << 16;
  }
};

}  // namespace gg
