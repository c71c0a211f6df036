// gg_norm.cu -- root-mean-square norm of rows with the residual's addition before it, its result in the rows' type, in
// 8 bits with a scale for each row and 128 columns, or both; and its gradient.
//
//   h = x + residual,  rstd = 1 / sqrt(mean h^2 + eps),  y = h * rstd * weight
//   grad_x = rstd * (g - xhat * mean(g * xhat)) + grad_h  with  g = grad_y * weight, xhat = h * rstd
//   grad_weight = sum over rows of grad_y * xhat
//
// Memory bounds it: a row is read once, stays in registers through the sum over it, and is written once. A row
// belongs to a team of 1 to 16 warps (more than one: a whole block), each of which holds 1 to 8 spans of 256 of its values, 8 of
// each a thread (team_of). In a span a thread has 8 values in a piece where rows are
// aligned (16 bytes of 16-bit values), so that 16 lanes hold a block of 128 columns, and else every 32nd of 256, so that a
// warp's loads of single values are whole lines, and 4 of a lane's 8 are of one block. The teams that fit the GPU go through the rows,
// and a team asks for its next row before it adds this one up (asks_ahead). h is rounded to its type first and the norm is of
// what is stored, as the gradient finds it.
//
// 16384 rows of 4096 in BF16, with the residual: forward 93 us, 5.8 TB/s; gradient with the residual's and the weight's 101 us,
// 5.3 TB/s, 6 us of it the last sum over the blocks' parts. FP32: 166 us and 174, 6.5 and 6.2 TB/s. 32768 rows into 16 and 8 bits: 230 to
// 240 us, 5.1 to 5.3; 16384 into 8 bits alone, without a residual, 97 us, by the instructions of the 8-bit form. A copy has 6.55. Rows that are
// not aligned to 16 bytes go value by value: 67041 rows of 1001 in BF16 182 us and 208. Wide rows hold fewer blocks an SM: 2048
// rows of 32768 in BF16 154 us and 379 (the gradient keeps two rows and the weight's sums, 8 spans of each, and spills).
// 4 rows of 4096 with 8-bit results: 5 us, a launch and the latency of one row.
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

constexpr int kMostWarps = 16;  // of a row, which leaves a thread 128 registers
// Whether the next row's values fit beside this one's: 16384 wide rows of 16 bits take 192 us where they are not asked for ahead
// and 96 where they are; of FP32, with 4 spans a warp, a quarter more than where they are not.
__host__ __device__ constexpr bool asks_ahead(int type, int spans) { return spans <= (type == GG_OUTPUT_F32 ? 2 : 8); }
__host__ __device__ constexpr bool gradient_asks_ahead(int spans) { return spans <= 2; }

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
  float eps;
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

// This lane's 8 values of a span of a row of `width` (zeros past it), as they are stored.
template <int F, bool kVec>
struct Eight {
  static constexpr int kWords = F == kOutF32 ? 8 : 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const void* base, int64_t at, int span, int lane, int width) {
    const int c0 = column<kVec>(span, lane, 0);
    if (kVec && c0 + 8 <= width) {
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(base) + (at + c0) * OutFormat<F>::kBytes);
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 u = p[i];
        w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column<kVec>(span, lane, j);
      if (c < width) {
        if constexpr (F == kOutF32) w[j] = static_cast<const uint32_t*>(base)[at + c];
        else w[j / 2] |= static_cast<uint32_t>(static_cast<const unsigned short*>(base)[at + c]) << (16 * (j % 2));
      }
    }
  }
  __device__ __forceinline__ void store(void* base, int64_t at, int span, int lane, int width) const {
    const int c0 = column<kVec>(span, lane, 0);
    if (kVec && c0 + 8 <= width) {
      uint4* p = reinterpret_cast<uint4*>(static_cast<char*>(base) + (at + c0) * OutFormat<F>::kBytes);
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) p[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column<kVec>(span, lane, j);
      if (c < width) {
        if constexpr (F == kOutF32) static_cast<uint32_t*>(base)[at + c] = w[j];
        else static_cast<unsigned short*>(base)[at + c] = static_cast<unsigned short>(w[j / 2] >> (16 * (j % 2)));
      }
    }
  }
  // Rounded to the type.
  __device__ __forceinline__ void set(int pair, float x, float y) {
    if constexpr (F == kOutF32) w[2 * pair] = __float_as_uint(x), w[2 * pair + 1] = __float_as_uint(y);
    else w[pair] = pack2<F>(x, y);
  }
  __device__ __forceinline__ float value(int j) const {
    if constexpr (F == kOutF32) return __uint_as_float(w[j]);
    else return widen16<F>(static_cast<unsigned short>(w[j / 2] >> (16 * (j % 2))));
  }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The sum over a team of `warps` warps (a whole block where it is more than one), the same in every thread. `sums`: two times 32
// floats of shared memory, taken in turn (`turn`).
__device__ __forceinline__ float team_sum(float v, int warps, float* sums, int turn) {
  v = warp_sum(v);
  if (warps == 1) return v;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  float* at = sums + 32 * (turn & 1);
  if (lane == 0) at[warp] = v;
  __syncthreads();
  return warp_sum(lane < warps ? at[lane] : 0.0f);
}

// Which row a thread's team starts with, how far it is to its next one, and which of the team's warps this is.
struct Place {
  int64_t row, step;
  int member;
  __device__ __forceinline__ Place(int warps) {
    const int warp = threadIdx.x / 32, teams = warps == 1 ? blockDim.x / 32 : 1;
    row = static_cast<int64_t>(blockIdx.x) * teams + (warps == 1 ? warp : 0);
    step = static_cast<int64_t>(gridDim.x) * teams;
    member = warps == 1 ? 0 : warp;
  }
};

// y = t * factor in 8 bits: a span's part of this lane.
template <bool kVec>
__device__ __forceinline__ void store_8bit(const NormParams& p, int64_t row, int span, int lane, const float (&t)[8], float factor) {
  if constexpr (kVec) {
    const int c0 = column<kVec>(span, lane, 0);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, magnitude(t[j]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const ExactScale8 s(top, factor, p.e5m2);
    if (lane % 16 == 0 && c0 < p.width) p.scales[row * p.lds + c0 / GG_SCALE_BLOCK] = s.scale(factor, p.e5m2);
    const uint2 b = make_uint2(s.four(t[0], t[1], t[2], t[3], p.e5m2), s.four(t[4], t[5], t[6], t[7], p.e5m2));
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
      for (int j = 0; j < 4; ++j) top = max(top, magnitude(t[4 * half + j]));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const ExactScale8 s(top, factor, p.e5m2);
      const int b0 = span * kSpan + half * GG_SCALE_BLOCK;
      if (lane == 0 && b0 < p.width) p.scales[row * p.lds + b0 / GG_SCALE_BLOCK] = s.scale(factor, p.e5m2);
      const uint32_t b = s.four(t[4 * half], t[4 * half + 1], t[4 * half + 2], t[4 * half + 3], p.e5m2);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = b0 + j * 32 + lane;
        if (c < p.width) p.q[row * p.ldq + c] = static_cast<unsigned char>(b >> (8 * j));
      }
    }
  }
}

// F: type of the rows; W: of the weight; kSpans: spans that a warp holds; kVec: rows aligned.
template <int F, int W, int kSpans, bool kVec>
__global__ void __launch_bounds__(32 * kMostWarps, kSpans == 1 ? 2 : 1) norm_kernel(const NormParams p, int warps) {
  __shared__ float sums[64];
  const int lane = threadIdx.x % 32;
  const Place at(warps);
  chained_begin();
  Eight<F, kVec> x[kSpans], r[kSpans];
  const auto ask = [&](int64_t row) {
    if (row >= p.rows) return;
#pragma unroll
    for (int i = 0; i < kSpans; ++i) x[i].load(p.x, row * p.ldx, at.member + i * warps, lane, p.width);
    if (p.residual) {
#pragma unroll
      for (int i = 0; i < kSpans; ++i) r[i].load(p.residual, row * p.ldr, at.member + i * warps, lane, p.width);
    }
  };
  constexpr bool kAhead = asks_ahead(F, kSpans);
  if constexpr (kAhead) ask(at.row);
  int turn = 0;
  for (int64_t row = at.row; row < p.rows; row += at.step, ++turn) {  // whole teams
    if constexpr (!kAhead) ask(row);
    Eight<F, kVec> h[kSpans];
    float sum = 0.0f;
    const auto account = [&](int i) {
      if (p.residual_out) h[i].store(p.residual_out, row * p.ldro, at.member + i * warps, lane, p.width);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(h[i].value(j), h[i].value(j), sum);
    };
    // Span by span where the values were asked for a row ago, which leaves the most room for the next row's (16384 wide rows of
    // 16 bits: 95 us, and 132 as below). Values just asked for are all taken before the first branch, which would have each span
    // wait for its own (FP32: 188 us then, and 270 as above).
    if constexpr (kAhead) {
#pragma unroll
      for (int i = 0; i < kSpans; ++i) {
        h[i] = x[i];
        if (p.residual) {
#pragma unroll
          for (int j = 0; j < 8; j += 2) h[i].set(j / 2, x[i].value(j) + r[i].value(j), x[i].value(j + 1) + r[i].value(j + 1));
        }
        account(i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kSpans; ++i)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          h[i].set(j / 2, p.residual ? x[i].value(j) + r[i].value(j) : x[i].value(j),
                   p.residual ? x[i].value(j + 1) + r[i].value(j + 1) : x[i].value(j + 1));
        }
#pragma unroll
      for (int i = 0; i < kSpans; ++i) account(i);
    }
    if constexpr (kAhead) ask(row + at.step);
    sum = team_sum(sum, warps, sums, turn);
    // both steps are correctly rounded
    const float rstd = __frcp_rn(__fsqrt_rn(sum / static_cast<float>(p.width) + p.eps));
    if (p.rstd && at.member == 0 && lane == 0) p.rstd[row] = rstd;
    if (!p.y && !p.q) continue;
    // For 8 bits rstd = power * factor, a power of two and a number from 2 to 4: h * power * weight is exact with 16-bit rows and
    // weights, and stays below y.
    float factor = 1.0f, power = rstd;
    if (p.q) {
      factor = __uint_as_float((__float_as_uint(rstd) & 0x007fffffu) | 0x40000000u);
      if (rstd == rstd) power = 0.5f * __uint_as_float(__float_as_uint(rstd) & 0x7f800000u);
    }
#pragma unroll
    for (int i = 0; i < kSpans; ++i) {
      const int span = at.member + i * warps;
      if (span * kSpan >= p.width) break;
      float t[8];  // y over `factor`
      if (p.weight) {
        Eight<W, kVec> w;
        w.load(p.weight, 0, span, lane, p.width);
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = h[i].value(j) * power * w.value(j);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = h[i].value(j) * power;
      }
      if (p.y) {
        Eight<F, kVec> out;
#pragma unroll
        for (int j = 0; j < 8; j += 2) out.set(j / 2, t[j] * factor, t[j + 1] * factor);
        out.store(p.y, row * p.ldy, span, lane, p.width);
      }
      if (p.q) store_8bit<kVec>(p, row, span, lane, t, factor);
    }
  }
}

// Each thread adds up its columns' part of grad_weight on its team's way through the rows.
template <int F, int W, int kSpans, bool kVec>
__global__ void __launch_bounds__(32 * kMostWarps, kSpans == 1 && F != kOutF32 ? 2 : 1) norm_gradient_kernel(const NormGradientParams p, int warps) {
  __shared__ float sums[64];
  const int lane = threadIdx.x % 32;
  const Place at(warps);
  chained_begin();
  float gw[kSpans][8];
#pragma unroll
  for (int i = 0; i < kSpans; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) gw[i][j] = 0.0f;
  constexpr bool kAhead = gradient_asks_ahead(kSpans);
  Eight<F, kVec> rh[kSpans], rg[kSpans], rp[kSpans];
  float rstd_next = 0.0f;
  const auto ask = [&](int64_t row) {
    if (row >= p.rows) return;
#pragma unroll
    for (int i = 0; i < kSpans; ++i) {
      rh[i].load(p.h, row * p.ldh, at.member + i * warps, lane, p.width);
      rg[i].load(p.grad_y, row * p.ldgy, at.member + i * warps, lane, p.width);
      if (kAhead && p.grad_h) rp[i].load(p.grad_h, row * p.ldgh, at.member + i * warps, lane, p.width);
    }
    rstd_next = p.rstd[row];
  };
  if constexpr (kAhead) ask(at.row);
  int turn = 0;
  for (int64_t row = at.row; row < p.rows; row += at.step, ++turn) {
    if constexpr (!kAhead) ask(row);
    const float rstd = rstd_next;
    float h[kSpans][8], g[kSpans][8];
    Eight<F, kVec> past[kSpans];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kSpans; ++i) {
      Eight<W, kVec> w;
      if (p.weight) w.load(p.weight, 0, at.member + i * warps, lane, p.width);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[i][j] = rh[i].value(j) * rstd;
        gw[i][j] = fmaf(rg[i].value(j), h[i][j], gw[i][j]);
        g[i][j] = p.weight ? rg[i].value(j) * w.value(j) : rg[i].value(j);
        sum = fmaf(g[i][j], h[i][j], sum);
      }
      if constexpr (kAhead) past[i] = rp[i];
    }
    if constexpr (kAhead) ask(row + at.step);
    const float mean = team_sum(sum, warps, sums, turn) / static_cast<float>(p.width);
#pragma unroll
    for (int i = 0; i < kSpans; ++i) {
      const int span = at.member + i * warps;
      if constexpr (!kAhead) {
        if (p.grad_h) past[i].load(p.grad_h, row * p.ldgh, span, lane, p.width);
      }
      float gx[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) gx[j] = fmaf(rstd, fmaf(-h[i][j], mean, g[i][j]), p.grad_h ? past[i].value(j) : 0.0f);
      Eight<F, kVec> out;
#pragma unroll
      for (int j = 0; j < 8; j += 2) out.set(j / 2, gx[j], gx[j + 1]);
      out.store(p.grad_x, row * p.ldgx, span, lane, p.width);
    }
  }
  if (!p.partial) return;
  if (warps == 1) {  // a block of several teams, each of which is one warp with one span (team_of): their sum, in order
    __shared__ float part[kMostWarps][kSpan];
#pragma unroll
    for (int j = 0; j < 8; ++j) part[threadIdx.x / 32][column<kVec>(0, lane, j)] = gw[0][j];
    __syncthreads();
    for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
      float v = 0.0f;
      for (unsigned t = 0; t < blockDim.x / 32; ++t) v += part[t][c];
      p.partial[static_cast<int64_t>(blockIdx.x) * p.width + c] = v;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kSpans; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column<kVec>(at.member + i * warps, lane, j);
      if (c < p.width) p.partial[static_cast<int64_t>(blockIdx.x) * p.width + c] = gw[i][j];
    }
}

// grad_weight[c] = the sum of the blocks' parts, a warp's every 32nd part first, then the warps'.
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

// The warps that hold a row, the spans that each of them does, and the threads of a block. Rows of FP32: as few spans as the warps
// allow (16384 rows of 4096: 170 us with 1 and 188 with 2, the gradient 174 and 191). Of 16 bits: 1 as long as the warps allow
// (91 us with 1, 100 with 2), then 4 (8192 rows of 8192: 102 us with 2, 95 with 4; 13421 of 5000: 150 and 109, since a block of 10
// warps leaves no room for a second); the gradient 2 from 4 spans on (16384 rows of 4096: 123 us with 1, 101 with 2).
struct Team {
  int warps, spans, threads;
};
Team team_of(int width, int type, bool gradient) {
  const int spans = (width - 1) / kSpan + 1;
  int each = 1;
  if (type != GG_OUTPUT_F32) each = gradient ? (spans >= 4 ? 2 : 1) : (spans > kMostWarps ? 4 : 1);
  while ((spans + each - 1) / each > kMostWarps) each *= 2;
  const int warps = (spans + each - 1) / each;
  return {warps, each, 32 * (warps > 1 ? warps : gradient ? 16 : 4)};
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

// kTwo: a warp may hold 2 spans (a forward pass of 16 bits goes from 1 to 4).
template <bool kTwo, typename Do>
void with_spans(int spans, bool vec, Do go) {
  using std::integral_constant;
  const auto one = [&](auto v) {
    if constexpr (kTwo) {
      if (spans == 2) return go(integral_constant<int, 2>(), v);
    }
    if (spans == 1) go(integral_constant<int, 1>(), v);
    else if (spans == 4) go(integral_constant<int, 4>(), v);
    else go(integral_constant<int, 8>(), v);
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
  gg::Team team{}, gradient_team{};
  int blocks[2] = {}, gradient_blocks[2] = {};  // that the GPU holds at a time; [aligned rows]
  int device = 0;
};

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
  int sms = 0;
  if (st == cudaSuccess) st = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, plan->device);
  plan->team = gg::team_of(config->width, config->type, false);
  plan->gradient_team = gg::team_of(config->width, config->type, true);
  gg::with_types(config->type, config->weight_type, [&](auto f, auto wt) {
    for (int vec = 0; vec < 2; ++vec) {
      const auto count = [&](auto kernel, int threads, int* blocks) {
        int per_sm = 0;
        if (st == cudaSuccess) st = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, 0);
        *blocks = sms * std::max(1, per_sm);
      };
      gg::with_spans<f() == gg::kOutF32>(plan->team.spans, vec != 0, [&](auto n, auto v) {
        count(gg::norm_kernel<f(), wt(), n(), v()>, plan->team.threads, &plan->blocks[vec]);
      });
      gg::with_spans<true>(plan->gradient_team.spans, vec != 0, [&](auto n, auto v) {
        count(gg::norm_gradient_kernel<f(), wt(), n(), v()>, plan->gradient_team.threads, &plan->gradient_blocks[vec]);
      });
    }
  });
  if (st == cudaSuccess)
    st = cudaMalloc(reinterpret_cast<void**>(&plan->partial),
                    static_cast<size_t>(std::max(plan->gradient_blocks[0], plan->gradient_blocks[1])) * config->width * sizeof(float));
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
  const bool vec = gg::rows_on(q.x, q.ldx, b, 16) && gg::rows_on(q.residual, q.ldr, b, 16) && gg::rows_on(q.residual_out, q.ldro, b, 16) &&
                   gg::rows_on(q.y, q.ldy, b, 16) && gg::rows_on(q.q, q.ldq, 1, 8) && gg::rows_on(q.weight, 0, 1, 16);
  const gg::Team& t = plan->team;
  const int teams = t.threads / (32 * t.warps);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(plan->blocks[vec], (static_cast<int64_t>(q.rows) + teams - 1) / teams));
  gg::with_types(plan->config.type, plan->config.weight_type, [&](auto f, auto wt) {
    gg::with_spans<f() == gg::kOutF32>(t.spans, vec, [&](auto n, auto v) {
      st = gg::launch_chained(gg::norm_kernel<f(), wt(), n(), v()>, dim3(grid), static_cast<unsigned>(t.threads), 0,
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
  const gg::Team& t = plan->gradient_team;
  const int teams = t.threads / (32 * t.warps);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(plan->gradient_blocks[vec], (static_cast<int64_t>(q.rows) + teams - 1) / teams));
  if (q.rows > 0)
    gg::with_types(plan->config.type, plan->config.weight_type, [&](auto f, auto wt) {
      gg::with_spans<true>(t.spans, vec, [&](auto n, auto v) {
        st = gg::launch_chained(gg::norm_gradient_kernel<f(), wt(), n(), v()>, dim3(grid), static_cast<unsigned>(t.threads), 0, s,
                                1, p, t.warps);
      });
    });
  if (st == cudaSuccess && q.grad_weight)
    st = gg::launch_chained(gg::norm_weight_sum_kernel, dim3(static_cast<unsigned>((w + 31) / 32)), 32 * gg::kSumWarps, 0, s, 1,
                            static_cast<const float*>(plan->partial), static_cast<int>(grid), w, q.grad_weight);
  return st;
}

void gg_norm_destroy(gg_norm_plan* plan) {
  if (!plan) return;
  if (plan->partial) cudaFree(plan->partial);
  delete plan;
}

}  // extern "C"
