// gg_scale8.cuh -- a block of 128 values in 8 bits with one FP32 scale, as the norm and the gated 8-bit product write it.
#pragma once

#include <cuda_fp8.h>

#include <cstdint>

namespace gg {

// A value's bits without the sign: as numbers they are ordered like the magnitudes, infinity above the finite ones
// and NaN above that, so a maximum over them finds a value that is not finite.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Four values rounded to nearest even, x in the low byte. A quotient may pass the largest number by a rounding of FP32; the
// conversion saturates.
__device__ __forceinline__ uint32_t round_8bit(float x, float y, float z, float w, bool e5m2) {
  const __nv_fp8_interpretation_t kind = e5m2 ? __NV_E5M2 : __NV_E4M3;
  return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, kind)) |
         static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(z, w), __NV_SATFINITE, kind)) << 16;
}

// scale = the block's largest magnitude over the type's largest number. Below 2^-100 the scale would leave FP32's normal numbers:
// such a block is held as zeros. A block with an infinity or a NaN gets a scale that is not finite.
//
// A value is held as v * largest / top, rounded once from that quotient: both types' largest numbers are 0.875 times a power of two
// (which goes to the divisor, so that no product leaves the range), 0.875 v is held in two parts, and a first quotient by a rounded
// inverse is corrected by its remainder. That leaves the FP32 number nearest to the quotient but for some 2^-44 of it, and the
// quotient itself where it is one: a tie between two 8-bit values stays a tie. The inverse alone took values at and next to a
// tie to either side. The epilogue does this once for a tile's outputs, beside all its blocks of k.
struct Scale8 {
  float scale, most, near;  // most: top over that power of two; near: about the inverse of that
  __device__ __forceinline__ Scale8(uint32_t bits, bool e5m2) {
    const float top = __uint_as_float(bits);
    const bool none = top < 7.888609e-31f;  // 2^-100; false for NaN
    scale = none ? 0.0f : top / (e5m2 ? 57344.0f : 448.0f);
    most = top * (e5m2 ? 1.0f / 65536 : 1.0f / 512);
    near = __fdividef(1.0f, most);
    if (none) most = near = 0.0f;
    if (bits == 0x7f800000u) most = 0.0f;  // near is 0: finite values next to an infinity
  }
  __device__ __forceinline__ float quotient(float v) const {
    const float u = 0.875f * v, rest = fmaf(0.875f, v, -u), q = u * near;
    return fmaf(fmaf(-q, most, u) + rest, near, q);
  }
  __device__ __forceinline__ uint32_t four(float x, float y, float z, float w, bool e5m2) const {
    return round_8bit(quotient(x), quotient(y), quotient(z), quotient(w), e5m2);
  }
};

// The same for values v * factor, of which v is exact: a product of two 16-bit numbers. Quotients of such v are often ties
// between two 8-bit values (1 in 10000 or so), which multiplying by a rounded inverse takes to either side. So the quotient is
// corrected by its remainder, after which it is exact where it can be. Both types' largest numbers are 1.75 times a power of two, and
// 1.75 * v is still exact with products of BF16 (of FP16 it has up to 25 bits).
struct ExactScale8 {
  float top, most, near;  // the largest v; over that power of two; about the inverse of that
  __device__ __forceinline__ ExactScale8(uint32_t bits, float factor, bool e5m2) {
    top = __uint_as_float(bits);
    most = top * (e5m2 ? 1.0f / 32768 : 1.0f / 256);
    near = __fdividef(1.0f, most);
    if (top * factor < 7.888609e-31f) top = most = near = 0.0f;
    if (bits == 0x7f800000u) most = 0.0f;
  }
  __device__ __forceinline__ float scale(float factor, bool e5m2) const { return top * factor / (e5m2 ? 57344.0f : 448.0f); }
  __device__ __forceinline__ float quotient(float v) const {
    const float u = 1.75f * v, q = u * near;
    return fmaf(fmaf(-q, most, u), near, q);
  }
  __device__ __forceinline__ uint32_t four(float x, float y, float z, float w, bool e5m2) const {
    return round_8bit(quotient(x), quotient(y), quotient(z), quotient(w), e5m2);
  }
};

}  // namespace gg
