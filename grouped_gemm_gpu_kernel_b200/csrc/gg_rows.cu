// gg_rows.cu -- the rows of a mixture-of-experts layer into expert order and back:
//   dispatch          packed[pos(t, j), :] = x[t, :]
//   combine           out[t, :] = sum_j w(t, j) packed[pos(t, j), :]
//   combine backward  grad_packed[pos(t, j), :] = w(t, j) grad_out[t, :],
//                     grad_weights(t, j) = <grad_out[t, :], packed[pos(t, j), :]>
// All three move bytes and compute next to nothing: memory bandwidth bounds them. A token's row is
// read once whatever top_k is (dispatch) or written once (combine), in 16-byte units where the rows allow.
// Measured (B200, 8192 tokens of 4096 BF16, top 2, inputs past L2; share of the measured copy rate of 6.54 TB/s):
// dispatch 32.3 us (0.95), combine 31.5 us (0.97), its gradient 57.8 us (0.89). Small calls are one launch:
// 4 tokens of 4096, top 2, 1.7 and 1.9 us on the GPU, 3.4 us each on the host.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "gg_epilogue_ops.cuh"
#include "gg_launch.cuh"
#include "grouped_gemm_b200.h"

namespace gg {
namespace {

constexpr int kRowsThreads = 256;

// A block's threads split into groups of 2^shift, one group per token; thread `in` of a group takes the
// units in, in + 2^shift, ... of the row (UN of them, loaded together, per turn).
struct RowsShape {
  int tokens, top_k, packed_rows;
  int units;  // units (vectors) a row
  int shift;  // log2 of a group's threads
};

struct RowsPlace {
  int64_t t;
  int in, group;
};

__device__ __forceinline__ RowsPlace rows_place(int shift) {
  const int tid = static_cast<int>(threadIdx.x);
  RowsPlace p;
  p.t = (static_cast<int64_t>(blockIdx.x) << (8 - shift)) + (tid >> shift);
  p.in = tid & ((1 << shift) - 1);
  p.group = 1 << shift;
  return p;
}
static_assert(kRowsThreads == 1 << 8, "rows_place");

// A position as the row that it names, -1 where it names none.
__device__ __forceinline__ int row_of(const int* __restrict__ positions, int64_t slot, int packed_rows) {
  const int p = __ldg(positions + slot);
  return p < packed_rows ? p : -1;
}

// Every thread reads its units of x once and writes them to all rows of the token, so the row is read
// once whatever top_k is. A warp writes whole 128-byte lines of one row at a time.
template <typename U, int UN>
__global__ void __launch_bounds__(kRowsThreads) dispatch_kernel(RowsShape sh, const U* __restrict__ x, int64_t ldx,
                                                                const int* __restrict__ positions,
                                                                U* __restrict__ packed, int64_t ldp) {
  chained_begin();
  const RowsPlace at = rows_place(sh.shift);
  if (at.t >= sh.tokens) return;
  const U* row = x + at.t * ldx;
  for (int u = blockIdx.y * at.group * UN + at.in; u < sh.units; u += gridDim.y * at.group * UN) {
    U v[UN];
#pragma unroll
    for (int i = 0; i < UN; ++i)
      if (u + i * at.group < sh.units) v[i] = row[u + i * at.group];
    for (int j = 0; j < sh.top_k; ++j) {
      const int p = row_of(positions, at.t * sh.top_k + j, sh.packed_rows);
      if (p < 0) continue;
      U* to = packed + p * ldp + u;
#pragma unroll
      for (int i = 0; i < UN; ++i)
        if (u + i * at.group < sh.units) to[i * at.group] = v[i];
    }
  }
}

// N elements of format F as they lie in memory, in 4-byte words (they are widened where they are used,
// so that loads in flight hold no more registers than bytes).
template <int F, int N>
struct Raw {
  static constexpr int kWords = F == kOutF32 ? N : (N + 1) / 2;
  uint32_t w[kWords];
  __device__ __forceinline__ float at(int i) const {  // i is known at compile time after unrolling
    if constexpr (F == kOutF32) return __uint_as_float(w[i]);
    else return widen16<F>(static_cast<unsigned short>(i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu));
  }
};

// The elements at `at` of base; the first `have` of them exist, the others give 0. base + at is aligned
// to N elements (to 16 bytes at most) where all exist.
template <int F, int N>
__device__ __forceinline__ void load_vec(const void* base, int64_t at, int have, Raw<F, N>& v) {
  constexpr int kWords = Raw<F, N>::kWords;
  const char* p = static_cast<const char*>(base) + at * OutFormat<F>::kBytes;
  if (N > 1 && have >= N) {
    if constexpr (kWords % 4 == 0) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 q = reinterpret_cast<const uint4*>(p)[i];
        v.w[4 * i] = q.x, v.w[4 * i + 1] = q.y, v.w[4 * i + 2] = q.z, v.w[4 * i + 3] = q.w;
      }
    } else if constexpr (kWords == 2) {
      const uint2 q = *reinterpret_cast<const uint2*>(p);
      v.w[0] = q.x, v.w[1] = q.y;
    } else {
      v.w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kWords; ++i) v.w[i] = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < have) {
        if constexpr (F == kOutF32) v.w[i] = reinterpret_cast<const uint32_t*>(p)[i];
        else v.w[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const unsigned short*>(p)[i]) << (16 * (i % 2));
      }
  }
}

// The first `have` of N elements to `at` of base, each rounded once to the format.
template <int F, int N>
__device__ __forceinline__ void store_vec(void* base, int64_t at, int have, const float (&v)[N]) {
  if (N > 1 && have >= N) {
    if constexpr (F == kOutF32) {
      float* p = static_cast<float*>(base) + at;
      if constexpr (N == 2) {
        *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
      } else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i)
          *reinterpret_cast<float4*>(p + 4 * i) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      }
    } else {
      unsigned short* p = static_cast<unsigned short*>(base) + at;
      if constexpr (N == 2) *reinterpret_cast<uint32_t*>(p) = pack2<F>(v[0], v[1]);
      else if constexpr (N == 4) *reinterpret_cast<uint2*>(p) = make_uint2(pack2<F>(v[0], v[1]), pack2<F>(v[2], v[3]));
      else if constexpr (N == 8)
        *reinterpret_cast<uint4*>(p) =
            make_uint4(pack2<F>(v[0], v[1]), pack2<F>(v[2], v[3]), pack2<F>(v[4], v[5]), pack2<F>(v[6], v[7]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < have) store_out<F>(base, at + i, v[i]);
  }
}

// Slots of a token worked on together (KS): the smallest of 2, 4 and, where the vectors are wide, 8 that
// holds top_k. Units a thread loads per turn: as many as make 8 wide loads, or 16 narrow ones, in flight
// whatever top_k is. (The combine of 16384 rows of 4096 BF16, top 2: 31.6 us; 61 with 4
// slots of 2 units, half of the loads dead.)
constexpr int units_per_turn(int N, int KS) { return (N >= 4 ? 8 : 16) / KS; }

template <int PF, int OF, int N, int KS>
__global__ void __launch_bounds__(kRowsThreads) combine_kernel(RowsShape sh, const void* __restrict__ packed, int64_t ldp,
                                                               const int* __restrict__ positions,
                                                               const float* __restrict__ weights, int width,
                                                               void* __restrict__ out, int64_t ldo) {
  constexpr int UN = units_per_turn(N, KS);
  chained_begin();
  const RowsPlace at = rows_place(sh.shift);
  if (at.t >= sh.tokens) return;
  const int64_t slot0 = at.t * sh.top_k;
  for (int u = blockIdx.y * at.group * UN + at.in; u < sh.units; u += gridDim.y * at.group * UN) {
    float sum[UN][N];
#pragma unroll
    for (int i = 0; i < UN; ++i)
#pragma unroll
      for (int x = 0; x < N; ++x) sum[i][x] = 0.0f;
    // with 2 slots at a time top_k is at most 2: one turn, whose sums live one unit long
    for (int j0 = 0; j0 < (KS == 2 ? 1 : sh.top_k); j0 += KS) {
      Raw<PF, N> v[KS][UN];
      float w[KS];
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const int p = j0 + j < sh.top_k ? row_of(positions, slot0 + j0 + j, sh.packed_rows) : -1;
        w[j] = p >= 0 ? (weights ? __ldg(weights + slot0 + j0 + j) : 1.0f) : 0.0f;
#pragma unroll
        for (int i = 0; i < UN; ++i) {
          const int c = (u + i * at.group) * N;
          load_vec<PF, N>(packed, p * ldp + c, p >= 0 ? width - c : 0, v[j][i]);
        }
      }
#pragma unroll
      for (int i = 0; i < UN; ++i) {
#pragma unroll
        for (int j = 0; j < KS; ++j)
#pragma unroll
          for (int x = 0; x < N; ++x) sum[i][x] = fmaf(w[j], v[j][i].at(x), sum[i][x]);
        if constexpr (KS == 2) {
          const int c = (u + i * at.group) * N;
          store_vec<OF, N>(out, at.t * ldo + c, width - c, sum[i]);
        }
      }
    }
    if constexpr (KS != 2) {
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        const int c = (u + i * at.group) * N;
        store_vec<OF, N>(out, at.t * ldo + c, width - c, sum[i]);
      }
    }
  }
}

// One pass over grad_out and packed gives both gradients: a thread reads its units of both, writes those
// of grad_packed and keeps its share of the dot products, which the group then adds up.
template <int PF, int OF, int N, int KS>
__global__ void __launch_bounds__(kRowsThreads) combine_backward_kernel(
    RowsShape sh, const void* __restrict__ grad_out, int64_t ldo, const void* packed, int64_t ldp,
    const int* __restrict__ positions, const float* __restrict__ weights, int width, void* grad_packed, int64_t ldgp,
    float* __restrict__ grad_weights) {
  constexpr int UN = units_per_turn(N, KS);
  __shared__ float s_part[kRowsThreads / 32][KS];
  chained_begin();
  const RowsPlace at = rows_place(sh.shift);
  const int warp = static_cast<int>(threadIdx.x) / 32, lane = static_cast<int>(threadIdx.x) % 32;
  const bool live = at.t < sh.tokens;
  const int64_t slot0 = at.t * sh.top_k;
  for (int j0 = 0; j0 < sh.top_k; j0 += KS) {
    int p[KS];
    float w[KS], dot[KS];
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      p[j] = live && j0 + j < sh.top_k ? row_of(positions, slot0 + j0 + j, sh.packed_rows) : -1;
      w[j] = p[j] >= 0 ? __ldg(weights + slot0 + j0 + j) : 0.0f;
      dot[j] = 0.0f;
    }
    for (int u = at.in; live && u < sh.units; u += at.group * UN) {
      Raw<OF, N> g[UN];
      Raw<PF, N> y[KS][UN];
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        const int c = (u + i * at.group) * N;
        load_vec<OF, N>(grad_out, at.t * ldo + c, width - c, g[i]);
      }
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int i = 0; i < UN; ++i) {
          const int c = (u + i * at.group) * N;
          load_vec<PF, N>(packed, p[j] * ldp + c, p[j] >= 0 ? width - c : 0, y[j][i]);
        }
#pragma unroll
      for (int j = 0; j < KS; ++j)
        if (p[j] >= 0)
#pragma unroll
          for (int i = 0; i < UN; ++i) {
            const int c = (u + i * at.group) * N;
            float o[N];
#pragma unroll
            for (int x = 0; x < N; ++x) {
              dot[j] = fmaf(g[i].at(x), y[j][i].at(x), dot[j]);
              o[x] = w[j] * g[i].at(x);
            }
            store_vec<PF, N>(grad_packed, p[j] * ldgp + c, width - c, o);
          }
    }
#pragma unroll
    for (int j = 0; j < KS; ++j)
      for (int d = min(16, at.group / 2); d > 0; d >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], d);
    if (sh.shift > 5) {  // a group of several warps
      if (j0 > 0) __syncthreads();
      if (lane == 0)
#pragma unroll
        for (int j = 0; j < KS; ++j) s_part[warp][j] = dot[j];
      __syncthreads();
      if (at.in == 0)
#pragma unroll
        for (int j = 0; j < KS; ++j)
          for (int i = 1; i < at.group / 32; ++i) dot[j] += s_part[warp + i][j];
    }
    if (live && at.in == 0)
#pragma unroll
      for (int j = 0; j < KS; ++j)
        if (j0 + j < sh.top_k) grad_weights[slot0 + j0 + j] = dot[j];
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

// Calls f with a vector length (`n`: 8, 4 for FP32, 2 or 1) and the slots worked on together.
template <typename F>
void with_vector_and_slots(int top_k, int n, F f) {
  using std::integral_constant;
  if (n == 2 && top_k <= 2) f(integral_constant<int, 2>(), integral_constant<int, 2>());
  else if (n == 2) f(integral_constant<int, 2>(), integral_constant<int, 4>());
  else if (n == 1 && top_k <= 2) f(integral_constant<int, 1>(), integral_constant<int, 2>());
  else if (n == 1) f(integral_constant<int, 1>(), integral_constant<int, 4>());
  else if (top_k <= 2) f(integral_constant<int, 8>(), integral_constant<int, 2>());
  else if (top_k <= 4) f(integral_constant<int, 8>(), integral_constant<int, 4>());
  else f(integral_constant<int, 8>(), integral_constant<int, 8>());
}

// The largest vector, in elements, of which both matrices' rows are made up: `most` where every row start
// is aligned to `most` elements (16 bytes at most), else 2, else 1.
int vector_of(int most, const void* a, int64_t lda, int a_bytes, const void* b, int64_t ldb, int b_bytes,
              const void* c = nullptr, int64_t ldc = 0) {
  const auto fits = [&](const void* p, int64_t ld, int bytes, int n) {
    const uintptr_t unit = static_cast<uintptr_t>(std::min(16, n * bytes));
    return reinterpret_cast<uintptr_t>(p) % unit == 0 && static_cast<uintptr_t>(ld * bytes) % unit == 0;
  };
  for (int n : {most, 2})
    if (fits(a, lda, a_bytes, n) && fits(b, ldb, b_bytes, n) && fits(c, ldc, a_bytes, n)) return n;
  return 1;
}

// Threads of a group: about `per_thread` units each, between a fraction of a warp and the block.
int group_shift(int units, int per_thread) {
  int shift = 3;
  while (shift < 8 && (1 << shift) * per_thread < units) ++shift;
  return shift;
}

unsigned token_blocks(int tokens, int shift) {
  return static_cast<unsigned>((static_cast<int64_t>(tokens) + (gg::kRowsThreads >> shift) - 1) / (gg::kRowsThreads >> shift));
}

int bytes_of(int type) { return type == GG_OUTPUT_F32 ? 4 : 2; }

}  // namespace
}  // namespace gg

extern "C" {

int gg_moe_dispatch(const void* x, int ldx, const int* positions, int tokens, int top_k, int width, int elem_bytes,
                    void* packed, int packed_rows, int ldp, void* stream) {
  if (tokens < 0 || top_k < 1 || width < 0 || width > GG_MOE_MAX_WIDTH || packed_rows < 0 || (elem_bytes != 1 && elem_bytes != 2 && elem_bytes != 4) ||
      ldx < std::max(1, width) || ldp < std::max(1, width))
    return cudaErrorInvalidValue;
  if (tokens == 0 || width == 0 || packed_rows == 0) return cudaSuccess;
  if (!x || !positions || !packed) return cudaErrorInvalidValue;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // the widest unit that the bases, the pitches and the row's length are made up of
  const uint64_t row = static_cast<uint64_t>(width) * elem_bytes;
  const uint64_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(packed) | row |
                       static_cast<uint64_t>(ldx) * elem_bytes | static_cast<uint64_t>(ldp) * elem_bytes;
  cudaError_t st = cudaSuccess;
  auto launch = [&](auto unit, auto per_turn) {
    using U = decltype(unit);
    constexpr int bytes = sizeof(U), UN = per_turn();
    gg::RowsShape sh{tokens, top_k, packed_rows, static_cast<int>(row / bytes), 0};
    sh.shift = gg::group_shift(sh.units, UN);
    const int turn = UN << sh.shift;
    const dim3 grid(gg::token_blocks(tokens, sh.shift), static_cast<unsigned>(std::min(65535, (sh.units - 1) / turn + 1)));
    st = gg::launch_chained(gg::dispatch_kernel<U, UN>, grid, gg::kRowsThreads, 0, s, 1, sh, static_cast<const U*>(x),
                            static_cast<int64_t>(ldx) * elem_bytes / bytes, positions, static_cast<U*>(packed),
                            static_cast<int64_t>(ldp) * elem_bytes / bytes);
  };
  using std::integral_constant;
  if (all % 16 == 0) launch(uint4(), integral_constant<int, 4>());
  else if (all % 8 == 0) launch(uint2(), integral_constant<int, 4>());
  else if (all % 4 == 0) launch(uint32_t(), integral_constant<int, 8>());
  else if (all % 2 == 0) launch(uint16_t(), integral_constant<int, 8>());
  else launch(uint8_t(), integral_constant<int, 8>());
  return st;
}

int gg_moe_combine(const void* packed, int packed_type, int packed_rows, int ldp, const int* positions,
                   const float* weights, int tokens, int top_k, int width, void* out, int out_type, int ldo,
                   void* stream) {
  if (tokens < 0 || top_k < 1 || width < 0 || width > GG_MOE_MAX_WIDTH || packed_rows < 0 || !gg::out_type_ok(packed_type) ||
      !gg::out_type_ok(out_type) || ldp < std::max(1, width) || ldo < std::max(1, width))
    return cudaErrorInvalidValue;
  if (tokens == 0 || width == 0) return cudaSuccess;
  if (!out || !positions || (!packed && packed_rows > 0)) return cudaErrorInvalidValue;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t st = cudaSuccess;
  gg::with_formats(packed_type, out_type, [&](auto pf, auto of) {
    gg::with_vector_and_slots(top_k, gg::vector_of(pf() == gg::kOutF32 ? 4 : 8, packed, ldp, gg::bytes_of(packed_type), out, ldo,
                                  gg::bytes_of(out_type)), [&](auto vec, auto slots) {
      constexpr int N = pf() == gg::kOutF32 && vec() == 8 ? 4 : vec(), KS = slots(), UN = gg::units_per_turn(N, KS);
      gg::RowsShape sh{tokens, top_k, packed_rows, (width - 1) / N + 1, 0};
      sh.shift = gg::group_shift(sh.units, UN);
      const int turn = UN << sh.shift;
      const dim3 grid(gg::token_blocks(tokens, sh.shift), static_cast<unsigned>(std::min(65535, (sh.units - 1) / turn + 1)));
      st = gg::launch_chained(gg::combine_kernel<pf(), of(), N, KS>, grid, gg::kRowsThreads, 0, s, 1, sh, packed,
                              static_cast<int64_t>(ldp), positions, weights, width, out, static_cast<int64_t>(ldo));
    });
  });
  return st;
}

int gg_moe_combine_backward(const void* grad_out, int out_type, int ldo, const void* packed, int packed_type,
                            int packed_rows, int ldp, const int* positions, const float* weights, int tokens,
                            int top_k, int width, void* grad_packed, int ldgp, float* grad_weights, void* stream) {
  if (tokens < 0 || top_k < 1 || width < 0 || width > GG_MOE_MAX_WIDTH || packed_rows < 0 || !gg::out_type_ok(packed_type) ||
      !gg::out_type_ok(out_type) || ldp < std::max(1, width) || ldo < std::max(1, width) ||
      ldgp < std::max(1, width))
    return cudaErrorInvalidValue;
  if (tokens == 0) return cudaSuccess;
  if (!positions || !weights || !grad_weights || (width > 0 && !grad_out) ||
      (packed_rows > 0 && width > 0 && (!packed || !grad_packed)))
    return cudaErrorInvalidValue;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t st = cudaSuccess;
  gg::with_formats(packed_type, out_type, [&](auto pf, auto of) {
    gg::with_vector_and_slots(top_k, gg::vector_of(pf() == gg::kOutF32 ? 4 : 8, packed, ldp, gg::bytes_of(packed_type), grad_out, ldo,
                                  gg::bytes_of(out_type), grad_packed, ldgp), [&](auto vec, auto slots) {
      constexpr int N = pf() == gg::kOutF32 && vec() == 8 ? 4 : vec(), KS = slots();
      gg::RowsShape sh{tokens, top_k, packed_rows, width > 0 ? (width - 1) / N + 1 : 0, 0};
      sh.shift = gg::group_shift(sh.units, 2 * gg::units_per_turn(N, KS));
      st = gg::launch_chained(gg::combine_backward_kernel<pf(), of(), N, KS>, dim3(gg::token_blocks(tokens, sh.shift)),
                              gg::kRowsThreads, 0, s, 1, sh, grad_out, static_cast<int64_t>(ldo), packed, static_cast<int64_t>(ldp),
                              positions, weights, width, grad_packed, static_cast<int64_t>(ldgp), grad_weights);
    });
  });
  return st;
}

}  // extern "C"
