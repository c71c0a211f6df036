// gg_norm.cu -- root-mean-square norm of rows with the residual's addition before it, its result in the rows' type, in
// 8 bits with a scale for each row and 128 columns, or both; and its gradient.
//
//   h = x + residual,  rstd = 1 / sqrt(mean h^2 + eps),  y = h * rstd * weight
//   grad_x = rstd * (g - xhat * mean(g * xhat)) + grad_h  with  g = grad_y * weight, xhat = h * rstd
//   grad_weight = sum over rows of grad_y * xhat
//
// Memory bounds it: a row is read once, stays in registers through the sum over it, and is written once. A row
// belongs to a team of 32 to 1024 threads of a block. A team goes through it in spans of 256 values for a
// warp, 8 for a thread: 8 in a piece where rows are aligned (16 bytes of 16-bit values), so that 16 lanes hold a block of 128
// columns, and else every 32nd of 256, so that a warp's loads of single values are whole lines, and 4 of a lane's 8 are of
// one block. h is rounded to its type first and the norm is of what is stored, as the gradient finds it.
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <new>

#include "gg_epilogue_ops.cuh"
#include "gg_internal.h"
#include "gg_launch.cuh"
#include "gg_scale8.cuh"
#include "grouped_gemm_b200.h"

namespace gg {
namespace {

constexpr int kSpan = 256;  // values that a warp takes in one piece
constexpr int kManyRows = 2048;

// Warps of a row at most, where each holds so many spans: by registers (8 values a span, three times that in the gradient).
__host__ __device__ constexpr int most_warps(int spans, bool gradient) { return gradient && spans > 1 ? 16 : 32; }

struct NormParams {
  const void* x;
  const void* residual;
  void* residual_out;
  const void* weight;
  void* y;
  unsigned char* q;
  float* scales;
  float* rstd;
  int64_t ldx, ldr, ldro, ldy, ldq, lds;
  int rows, width;
  float eps, largest;  // largest: of the 8-bit type
  bool e5m2;
};

struct NormGradientParams {
  const void* h;
  const void* weight;
  const float* rstd;
  const void* grad_y;
  const void* grad_h;
  void* grad_x;
  float* partial;  // NULL: no gradient of the weight; [grid * teams][width]
  int64_t ldh, ldgy, ldgh, ldgx;
  int rows, width;
};

// Column of value j of this lane in a span.
template <bool kVec>
__device__ __forceinline__ int column(int span, int lane, int j) {
  return span * kSpan + (kVec ? lane * 8 + j : j * 32 + lane);
}

// This lane's 8 values of a span of a row of `width` (zeros past it).
template <int F, bool kVec>
__device__ __forceinline__ void load8(const void* base, int64_t at, int span, int lane, int width, float (&v)[8]) {
  const int c0 = column<kVec>(span, lane, 0);
  if (kVec && c0 + 8 <= width) {
    const char* p = static_cast<const char*>(base) + (at + c0) * OutFormat<F>::kBytes;
    if constexpr (F == kOutF32) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 16);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<F>(w[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int c = column<kVec>(span, lane, j);
    v[j] = 0.0f;
    if (c < width) {
      if constexpr (F == kOutF32) v[j] = static_cast<const float*>(base)[at + c];
      else v[j] = widen16<F>(static_cast<const unsigned short*>(base)[at + c]);
    }
  }
}

template <int F, bool kVec>
__device__ __forceinline__ void store8(void* base, int64_t at, int span, int lane, int width, const float (&v)[8]) {
  const int c0 = column<kVec>(span, lane, 0);
  if (kVec && c0 + 8 <= width) {
    char* p = static_cast<char*>(base) + (at + c0) * OutFormat<F>::kBytes;
    if constexpr (F == kOutF32) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(p + 16) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(p) = make_uint4(pack2<F>(v[0], v[1]), pack2<F>(v[2], v[3]), pack2<F>(v[4], v[5]), pack2<F>(v[6], v[7]));
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int c = column<kVec>(span, lane, j);
    if (c < width) store_out<F>(base, at + c, v[j]);
  }
}

template <int F>
__device__ __forceinline__ float rounded(float v) {
  if constexpr (F == kOutF32) return v;
  else if constexpr (F == kOutF16) return __half2float(__float2half_rn(v));
  else return __bfloat162float(__float2bfloat16_rn(v));
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The sum over a team of `warps` warps (a whole block where it is more than one), the same in every thread. `sums`: 32
// floats of shared memory, used by one sum at a time.
__device__ __forceinline__ float team_sum(float v, int warps, float* sums) {
  v = warp_sum(v);
  if (warps == 1) return v;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  __syncthreads();
  if (lane == 0) sums[warp] = v;
  __syncthreads();
  return warp_sum(lane < warps ? sums[lane] : 0.0f);
}

// F: type of the rows; W: of the weight; kSpans: spans that a warp holds; kVec: rows aligned.
template <int F, int W, int kSpans, bool kVec>
__global__ void __launch_bounds__(32 * most_warps(kSpans, false)) norm_kernel(const NormParams p, int warps) {
  __shared__ float sums[32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, member = warps == 1 ? 0 : warp;
  const int64_t row = warps == 1 ? static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + warp : blockIdx.x;
  chained_begin();
  if (row >= p.rows) return;  // whole teams
  float h[kSpans][8];
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kSpans; ++i) load8<F, kVec>(p.x, row * p.ldx, member + i * warps, lane, p.width, h[i]);
  if (p.residual) {
#pragma unroll
    for (int i = 0; i < kSpans; ++i) {
      float r[8];
      load8<F, kVec>(p.residual, row * p.ldr, member + i * warps, lane, p.width, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] = rounded<F>(h[i][j] + r[j]);
    }
  }
#pragma unroll
  for (int i = 0; i < kSpans; ++i) {
    if (p.residual_out) store8<F, kVec>(p.residual_out, row * p.ldro, member + i * warps, lane, p.width, h[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(h[i][j], h[i][j], sum);
  }
  sum = team_sum(sum, warps, sums);
  // no reciprocal square root of its own: both steps are correctly rounded
  const float rstd = __frcp_rn(__fsqrt_rn(sum / static_cast<float>(p.width) + p.eps));
  if (p.rstd && member == 0 && lane == 0) p.rstd[row] = rstd;
#pragma unroll
  for (int i = 0; i < kSpans; ++i) {
    const int span = member + i * warps;
    if (span * kSpan >= p.width) break;
    float w[8];
    if (p.weight) {
      load8<W, kVec>(p.weight, 0, span, lane, p.width, w);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = 1.0f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] *= h[i][j] * rstd;
    if (p.y) store8<F, kVec>(p.y, row * p.ldy, span, lane, p.width, w);
    if (!p.q) continue;
    const int c0 = column<kVec>(span, lane, 0);
    if constexpr (kVec) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, magnitude(w[j]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const Scale8 s(top, p.largest);
      if (lane % 16 == 0 && c0 < p.width) p.scales[row * p.lds + c0 / GG_SCALE_BLOCK] = s.scale;
      const uint2 b = make_uint2(s.four(w[0], w[1], w[2], w[3], p.e5m2), s.four(w[4], w[5], w[6], w[7], p.e5m2));
      unsigned char* q = p.q + row * p.ldq + c0;
      if (c0 + 8 <= p.width) {
        *reinterpret_cast<uint2*>(q) = b;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c0 + j < p.width) q[j] = static_cast<unsigned char>((j < 4 ? b.x : b.y) >> (8 * (j % 4)));
      }
    } else {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) top = max(top, magnitude(w[4 * half + j]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const Scale8 s(top, p.largest);
        const int b0 = span * kSpan + half * GG_SCALE_BLOCK;
        if (lane == 0 && b0 < p.width) p.scales[row * p.lds + b0 / GG_SCALE_BLOCK] = s.scale;
        const uint32_t b = s.four(w[4 * half], w[4 * half + 1], w[4 * half + 2], w[4 * half + 3], p.e5m2);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = b0 + j * 32 + lane;
          if (c < p.width) p.q[row * p.ldq + c] = static_cast<unsigned char>(b >> (8 * j));
        }
      }
    }
  }
}

// The grid's teams go through the rows; each thread adds up its columns' part of grad_weight on the way.
template <int F, int W, int kSpans, bool kVec>
__global__ void __launch_bounds__(32 * most_warps(kSpans, true)) norm_gradient_kernel(const NormGradientParams p, int warps) {
  __shared__ float sums[32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, member = warps == 1 ? 0 : warp;
  const int teams = warps == 1 ? blockDim.x / 32 : 1;
  const int64_t team = static_cast<int64_t>(blockIdx.x) * teams + (warps == 1 ? warp : 0);
  chained_begin();
  float gw[kSpans][8];
#pragma unroll
  for (int i = 0; i < kSpans; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) gw[i][j] = 0.0f;
  for (int64_t row = team; row < p.rows; row += static_cast<int64_t>(gridDim.x) * teams) {
    float h[kSpans][8], g[kSpans][8];
#pragma unroll
    for (int i = 0; i < kSpans; ++i) {
      load8<F, kVec>(p.h, row * p.ldh, member + i * warps, lane, p.width, h[i]);
      load8<F, kVec>(p.grad_y, row * p.ldgy, member + i * warps, lane, p.width, g[i]);
    }
    const float rstd = p.rstd[row];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kSpans; ++i) {
      float w[8];
      if (p.weight) {
        load8<W, kVec>(p.weight, 0, member + i * warps, lane, p.width, w);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = 1.0f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[i][j] *= rstd;
        gw[i][j] = fmaf(g[i][j], h[i][j], gw[i][j]);
        g[i][j] *= w[j];
        sum = fmaf(g[i][j], h[i][j], sum);
      }
    }
    const float mean = team_sum(sum, warps, sums) / static_cast<float>(p.width);
#pragma unroll
    for (int i = 0; i < kSpans; ++i) {
      const int span = member + i * warps;
      float past[8];
      if (p.grad_h) {
        load8<F, kVec>(p.grad_h, row * p.ldgh, span, lane, p.width, past);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) past[j] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) past[j] = fmaf(rstd, fmaf(-h[i][j], mean, g[i][j]), past[j]);
      store8<F, kVec>(p.grad_x, row * p.ldgx, span, lane, p.width, past);
    }
  }
  if (!p.partial) return;
#pragma unroll
  for (int i = 0; i < kSpans; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column<kVec>(member + i * warps, lane, j);
      if (c < p.width) p.partial[team * p.width + c] = gw[i][j];
    }
}

// grad_weight[c] = the sum of the teams' parts, a warp's every 32nd part first, then the warps'.
constexpr int kSumWarps = 32;
__global__ void __launch_bounds__(32 * kSumWarps) norm_weight_sum_kernel(const float* partial, int parts, int width, float* out) {
  __shared__ float sums[kSumWarps][33];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, c = blockIdx.x * 32 + lane;
  chained_begin();
  float v = 0.0f;
  if (c < width) {
#pragma unroll 8
    for (int i = warp; i < parts; i += kSumWarps) v += partial[static_cast<int64_t>(i) * width + c];
  }
  sums[warp][lane] = v;
  __syncthreads();
  const float s = warp_sum(sums[lane][warp]);  // column `warp` of the block's 32
  if (lane == 0 && blockIdx.x * 32 + warp < width) out[blockIdx.x * 32 + warp] = s;
}

// The warps that hold a row, and the spans that each of them does.
struct Team {
  int warps, spans;
};
Team team_of(int width, int64_t rows, bool gradient) {
  const int spans = (width - 1) / kSpan + 1, most = gradient ? 8 : 4;
  // with rows enough to fill the GPU a few warps that hold more each (fewer sums across warps), else all the warps there are
  for (int each = 1;; each *= 2) {
    const int warps = (spans + each - 1) / each;
    if (warps <= (rows >= kManyRows ? 4 : most_warps(each, gradient))) return {warps, each};
    if (each == most || (warps <= most_warps(each, gradient) && each >= 4)) return {warps, each};
  }
}

template <typename Do>
void with_types(int type, int weight_type, Do go) {
  using std::integral_constant;
  if (type == GG_OUTPUT_F32) go(integral_constant<int, kOutF32>(), integral_constant<int, kOutF32>());
  else if (type == GG_OUTPUT_F16 && weight_type == type) go(integral_constant<int, kOutF16>(), integral_constant<int, kOutF16>());
  else if (type == GG_OUTPUT_F16) go(integral_constant<int, kOutF16>(), integral_constant<int, kOutF32>());
  else if (weight_type == type) go(integral_constant<int, kOutBF16>(), integral_constant<int, kOutBF16>());
  else go(integral_constant<int, kOutBF16>(), integral_constant<int, kOutF32>());
}

template <bool kGradient, typename Do>
void with_spans(int spans, bool vec, Do go) {
  using std::integral_constant;
  const auto one = [&](auto v) {
    if (spans == 1) go(integral_constant<int, 1>(), v);
    else if (spans == 2) go(integral_constant<int, 2>(), v);
    else if (spans == 4 || !kGradient) go(integral_constant<int, 4>(), v);
    else go(integral_constant<int, kGradient ? 8 : 4>(), v);
  };
  if (vec) one(std::true_type());
  else one(std::false_type());
}

int bytes_of(int type) { return type == GG_OUTPUT_F32 ? 4 : 2; }

// Whether a matrix that is there has rows that start on `to`-byte boundaries.
bool rows_on(const void* p, int64_t ld, int bytes, int to) {
  return !p || (reinterpret_cast<uintptr_t>(p) % to == 0 && ld * bytes % to == 0);
}

}  // namespace
}  // namespace gg

struct gg_norm_plan {
  gg_norm_config config{};
  float* partial = nullptr;
  int device = 0, sms = 0;
};

namespace {
// Teams that go through the rows of a gradient: enough threads to keep memory busy, and no more parts of
// grad_weight than that.
constexpr int kGradientThreads = 1024;
int gradient_teams(const gg_norm_plan* plan, const gg::Team& t) { return plan->sms * std::max(1, kGradientThreads / (32 * t.warps)); }
}  // namespace

extern "C" {

int gg_norm_create(const gg_norm_config* config, gg_norm_plan** out) {
  if (!out) return cudaErrorInvalidValue;
  *out = nullptr;
  if (!config || config->width < 1 || config->width > GG_NORM_MAX_WIDTH || config->type < GG_OUTPUT_F32 ||
      config->type > GG_OUTPUT_BF16 || (config->weight_type != config->type && config->weight_type != GG_OUTPUT_F32) ||
      !(config->eps >= 0.0f) || !std::isfinite(config->eps))
    return cudaErrorInvalidValue;
  gg_norm_plan* plan = new (std::nothrow) gg_norm_plan();
  if (!plan) return cudaErrorMemoryAllocation;
  plan->config = *config;
  cudaError_t st = cudaGetDevice(&plan->device);
  if (st == cudaSuccess) st = cudaDeviceGetAttribute(&plan->sms, cudaDevAttrMultiProcessorCount, plan->device);
  if (st == cudaSuccess) {
    const size_t teams = static_cast<size_t>(std::max(gradient_teams(plan, gg::team_of(config->width, INT32_MAX, true)),
                                                      gradient_teams(plan, gg::team_of(config->width, 1, true))));
    st = cudaMalloc(reinterpret_cast<void**>(&plan->partial), teams * config->width * sizeof(float));
  }
  if (st != cudaSuccess) {
    delete plan;
    return st;
  }
  *out = plan;
  return cudaSuccess;
}

int gg_norm_run(const gg_norm_plan* plan, const gg_norm* call, void* stream) {
  if (!plan || !plan->partial) return cudaErrorInvalidDevicePointer;
  if (!call || call->rows < 0) return cudaErrorInvalidValue;
  const gg_norm& q = *call;
  const int w = plan->config.width, b = gg::bytes_of(plan->config.type);
  if (q.rows == 0) return cudaSuccess;
  if (!q.x || (q.q && (!q.scales || (q.q_type != GG_OUTPUT_E4M3 && q.q_type != GG_OUTPUT_E5M2))) || q.ldx < w || (q.residual && q.ldr < w) ||
      (q.residual_out && q.ldro < w) || (q.y && q.ldy < w) || (q.q && (q.ldq < w || q.lds < (w - 1) / GG_SCALE_BLOCK + 1)))
    return cudaErrorInvalidValue;
  cudaError_t st = gg::expect_device(plan->device);
  if (st != cudaSuccess) return st;
  gg::NormParams p{};
  p.x = q.x, p.residual = q.residual, p.residual_out = q.residual_out, p.weight = q.weight, p.y = q.y;
  p.q = static_cast<unsigned char*>(q.q), p.scales = q.scales, p.rstd = q.rstd;
  p.ldx = q.ldx, p.ldr = q.ldr, p.ldro = q.ldro, p.ldy = q.ldy, p.ldq = q.ldq, p.lds = q.lds;
  p.rows = q.rows, p.width = w, p.eps = plan->config.eps;
  p.e5m2 = q.q_type == GG_OUTPUT_E5M2;
  p.largest = p.e5m2 ? 57344.0f : 448.0f;
  const bool vec = gg::rows_on(q.x, q.ldx, b, 16) && gg::rows_on(q.residual, q.ldr, b, 16) && gg::rows_on(q.residual_out, q.ldro, b, 16) &&
                   gg::rows_on(q.y, q.ldy, b, 16) && gg::rows_on(q.q, q.ldq, 1, 8) && gg::rows_on(q.weight, 0, 1, 16);
  const gg::Team t = gg::team_of(w, q.rows, false);
  const int teams = t.warps == 1 ? 4 : 1;
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(q.rows) + teams - 1) / teams);
  gg::with_types(plan->config.type, plan->config.weight_type, [&](auto f, auto wt) {
    gg::with_spans<false>(t.spans, vec, [&](auto n, auto v) {
      st = gg::launch_chained(gg::norm_kernel<f(), wt(), n(), v()>, dim3(grid), static_cast<unsigned>(32 * t.warps * teams), 0,
                              static_cast<cudaStream_t>(stream), 1, p, t.warps);
    });
  });
  return st;
}

int gg_norm_backward(gg_norm_plan* plan, const gg_norm_gradient* gradient, void* stream) {
  if (!plan || !plan->partial) return cudaErrorInvalidDevicePointer;
  if (!gradient || gradient->rows < 0) return cudaErrorInvalidValue;
  const gg_norm_gradient& q = *gradient;
  const int w = plan->config.width, b = gg::bytes_of(plan->config.type);
  if (q.rows > 0 && (!q.h || !q.rstd || !q.grad_y || !q.grad_x || q.ldh < w || q.ldgy < w || (q.grad_h && q.ldgh < w) || q.ldgx < w))
    return cudaErrorInvalidValue;
  cudaError_t st = gg::expect_device(plan->device);
  if (st != cudaSuccess) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  gg::NormGradientParams p{};
  p.h = q.h, p.weight = q.weight, p.rstd = q.rstd, p.grad_y = q.grad_y, p.grad_h = q.grad_h, p.grad_x = q.grad_x;
  p.partial = q.grad_weight ? plan->partial : nullptr;
  p.ldh = q.ldh, p.ldgy = q.ldgy, p.ldgh = q.ldgh, p.ldgx = q.ldgx;
  p.rows = q.rows, p.width = w;
  const bool vec = gg::rows_on(q.h, q.ldh, b, 16) && gg::rows_on(q.grad_y, q.ldgy, b, 16) && gg::rows_on(q.grad_h, q.ldgh, b, 16) &&
                   gg::rows_on(q.grad_x, q.ldgx, b, 16) && gg::rows_on(q.weight, 0, 1, 16);
  const gg::Team t = gg::team_of(w, q.rows, true);
  const int per = t.warps == 1 ? 4 : 1;
  const int most = gradient_teams(plan, t);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(std::max(1, most / per), (static_cast<int64_t>(q.rows) + per - 1) / per));
  if (q.rows > 0)
    gg::with_types(plan->config.type, plan->config.weight_type, [&](auto f, auto wt) {
      gg::with_spans<true>(t.spans, vec, [&](auto n, auto v) {
        st = gg::launch_chained(gg::norm_gradient_kernel<f(), wt(), n(), v()>, dim3(grid), static_cast<unsigned>(32 * t.warps * per), 0, s,
                                1, p, t.warps);
      });
    });
  if (st == cudaSuccess && q.grad_weight)
    st = gg::launch_chained(gg::norm_weight_sum_kernel, dim3(static_cast<unsigned>((w + 31) / 32)), 32 * gg::kSumWarps, 0, s, 1,
                            static_cast<const float*>(plan->partial), static_cast<int>(grid) * per, w, q.grad_weight);
  return st;
}

void gg_norm_destroy(gg_norm_plan* plan) {
  if (!plan) return;
  if (plan->partial) cudaFree(plan->partial);
  delete plan;
}

}  // extern "C"
