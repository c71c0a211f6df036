// gg_rows.cu -- the rows of a mixture-of-experts layer into expert order and back:
//   dispatch          packed[pos(t, j), :] = x[t, :]
//   combine           out[t, :] = sum_j w(t, j) packed[pos(t, j), :]
//   combine backward  grad_packed[pos(t, j), :] = w(t, j) grad_out[t, :],
//                     grad_weights(t, j) = <grad_out[t, :], packed[pos(t, j), :]>
// All three move bytes and compute next to nothing: memory bandwidth bounds them.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gg_epilogue_ops.cuh"
#include "grouped_gemm_b200.h"

namespace gg {
namespace {

constexpr int kRowsThreads = 256;

template <typename U>
__global__ void __launch_bounds__(kRowsThreads) dispatch_kernel(const U* __restrict__ x, int64_t ldx,
                                                                const int* __restrict__ positions, int top_k, int units,
                                                                U* __restrict__ packed, int packed_rows, int64_t ldp) {
  const int t = static_cast<int>(blockIdx.x);
  for (int u = threadIdx.x; u < units; u += kRowsThreads) {
    const U v = x[t * ldx + u];
    for (int j = 0; j < top_k; ++j) {
      const int p = positions[static_cast<int64_t>(t) * top_k + j];
      if (p >= 0 && p < packed_rows) packed[p * ldp + u] = v;
    }
  }
}

template <int PF, int OF>
__global__ void __launch_bounds__(kRowsThreads) combine_kernel(const void* __restrict__ packed, int packed_rows, int64_t ldp,
                                                               const int* __restrict__ positions,
                                                               const float* __restrict__ weights, int top_k, int width,
                                                               void* __restrict__ out, int64_t ldo) {
  const int t = static_cast<int>(blockIdx.x);
  for (int c = threadIdx.x; c < width; c += kRowsThreads) {
    float sum = 0.0f;
    for (int j = 0; j < top_k; ++j) {
      const int64_t s = static_cast<int64_t>(t) * top_k + j;
      const int p = positions[s];
      if (p < 0 || p >= packed_rows) continue;
      const float v = load_out<PF>(packed, p * ldp + c);
      sum = weights ? fmaf(weights[s], v, sum) : sum + v;
    }
    store_out<OF>(out, t * ldo + c, sum);
  }
}

template <int PF, int OF>
__global__ void __launch_bounds__(kRowsThreads) combine_backward_kernel(
    const void* __restrict__ grad_out, int64_t ldo, const void* packed, int packed_rows, int64_t ldp,
    const int* __restrict__ positions, const float* __restrict__ weights, int top_k, int width, void* grad_packed,
    int64_t ldgp, float* __restrict__ grad_weights) {
  __shared__ float part[kRowsThreads / 32];
  const int t = static_cast<int>(blockIdx.x);
  for (int j = 0; j < top_k; ++j) {
    const int64_t s = static_cast<int64_t>(t) * top_k + j;
    const int p = positions[s];
    float dot = 0.0f;
    if (p >= 0 && p < packed_rows) {
      const float w = weights[s];
      for (int c = threadIdx.x; c < width; c += kRowsThreads) {
        const float g = load_out<OF>(grad_out, t * ldo + c);
        float y;
        if constexpr (PF == kOutF32) y = static_cast<const float*>(packed)[p * ldp + c];
        else y = widen16<PF>(static_cast<const unsigned short*>(packed)[p * ldp + c]);
        dot = fmaf(g, y, dot);
        store_out<PF>(grad_packed, p * ldgp + c, w * g);
      }
    }
    for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
    __syncthreads();
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = dot;
    __syncthreads();
    if (threadIdx.x == 0) {
      float sum = 0.0f;
      for (int i = 0; i < kRowsThreads / 32; ++i) sum += part[i];
      grad_weights[s] = sum;
    }
  }
}

bool out_type_ok(int t) { return t == GG_OUTPUT_F32 || t == GG_OUTPUT_F16 || t == GG_OUTPUT_BF16; }

// Calls f with the packed and the out format as compile-time constants.
template <typename F>
void with_formats(int packed_type, int out_type, F f) {
  auto inner = [&](auto pf) {
    if (out_type == GG_OUTPUT_F32) f(pf, std::integral_constant<int, kOutF32>());
    else if (out_type == GG_OUTPUT_F16) f(pf, std::integral_constant<int, kOutF16>());
    else f(pf, std::integral_constant<int, kOutBF16>());
  };
  if (packed_type == GG_OUTPUT_F32) inner(std::integral_constant<int, kOutF32>());
  else if (packed_type == GG_OUTPUT_F16) inner(std::integral_constant<int, kOutF16>());
  else inner(std::integral_constant<int, kOutBF16>());
}

}  // namespace
}  // namespace gg

extern "C" {

int gg_moe_dispatch(const void* x, int ldx, const int* positions, int tokens, int top_k, int width, int elem_bytes,
                    void* packed, int packed_rows, int ldp, void* stream) {
  if (tokens < 0 || top_k < 1 || width < 0 || packed_rows < 0 || (elem_bytes != 1 && elem_bytes != 2 && elem_bytes != 4) ||
      ldx < std::max(1, width) || ldp < std::max(1, width))
    return cudaErrorInvalidValue;
  if (tokens == 0 || width == 0 || packed_rows == 0) return cudaSuccess;
  if (!x || !positions || !packed) return cudaErrorInvalidValue;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto launch = [&](auto unit) {
    using U = decltype(unit);
    gg::dispatch_kernel<U><<<tokens, gg::kRowsThreads, 0, s>>>(static_cast<const U*>(x), ldx, positions, top_k, width,
                                                               static_cast<U*>(packed), packed_rows, ldp);
  };
  if (elem_bytes == 4) launch(uint32_t());
  else if (elem_bytes == 2) launch(uint16_t());
  else launch(uint8_t());
  return cudaGetLastError();
}

int gg_moe_combine(const void* packed, int packed_type, int packed_rows, int ldp, const int* positions,
                   const float* weights, int tokens, int top_k, int width, void* out, int out_type, int ldo,
                   void* stream) {
  if (tokens < 0 || top_k < 1 || width < 0 || packed_rows < 0 || !gg::out_type_ok(packed_type) ||
      !gg::out_type_ok(out_type) || ldp < std::max(1, width) || ldo < std::max(1, width))
    return cudaErrorInvalidValue;
  if (tokens == 0 || width == 0) return cudaSuccess;
  if (!out || !positions || (!packed && packed_rows > 0)) return cudaErrorInvalidValue;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  gg::with_formats(packed_type, out_type, [&](auto pf, auto of) {
    gg::combine_kernel<pf(), of()><<<tokens, gg::kRowsThreads, 0, s>>>(packed, packed_rows, ldp, positions, weights,
                                                                       top_k, width, out, ldo);
  });
  return cudaGetLastError();
}

int gg_moe_combine_backward(const void* grad_out, int out_type, int ldo, const void* packed, int packed_type,
                            int packed_rows, int ldp, const int* positions, const float* weights, int tokens,
                            int top_k, int width, void* grad_packed, int ldgp, float* grad_weights, void* stream) {
  if (tokens < 0 || top_k < 1 || width < 0 || packed_rows < 0 || !gg::out_type_ok(packed_type) ||
      !gg::out_type_ok(out_type) || ldp < std::max(1, width) || ldo < std::max(1, width) ||
      ldgp < std::max(1, width))
    return cudaErrorInvalidValue;
  if (tokens == 0) return cudaSuccess;
  if (!positions || !weights || !grad_weights || (width > 0 && !grad_out) ||
      (packed_rows > 0 && width > 0 && (!packed || !grad_packed)))
    return cudaErrorInvalidValue;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  gg::with_formats(packed_type, out_type, [&](auto pf, auto of) {
    gg::combine_backward_kernel<pf(), of()><<<tokens, gg::kRowsThreads, 0, s>>>(
        grad_out, ldo, packed, packed_rows, ldp, positions, weights, top_k, width, grad_packed, ldgp, grad_weights);
  });
  return cudaGetLastError();
}

}  // extern "C"
