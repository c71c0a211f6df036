// gg_q4.cu -- rows of a mixture-of-experts layer against expert weights held in 4 bits with a scale
// per output and group of k (the decoding form of the mixture-of-experts plan):
//   D[r, o] = act(sum_g scale(o, g) * sum_{k in g} A[r, k] (q(o, k) - zero(o, g)) + bias(o)).
//
// With few rows an expert the weights' bytes bound it, so the kernel is built around reading them
// once, whole lines at a time. The weights stand as the A operand of mma.sync m16n8k16 (16 outputs
// a tile, 8 rows of the activations as its columns): the differences q - zero are small integers,
// exact in FP16 and BF16, so the tensor pipe's products are exact and its sums FP32, and the group's
// scale multiplies the FP32 sum. tcgen05 would want 128 outputs and the unpacked operand in shared
// or tensor memory, a detour that costs more than the matrix work of 8 columns; a fragment in
// registers is fed from the unpacking directly.
//
// Weights are laid out once (gg_q4_plan_create), per expert as blocks of 16 outputs x 128 k, 1 KB:
//   [half h][lane][4 words]: lane l, word i, half h hold output 16 tile + 8 h + l / 4 and
//   k = 128 block + 32 i + 8 (l % 4) + 0..7, the eight values in the nibbles (0, 4, 1, 5, 2, 6, 3, 7)
//   from the low end, so that one mask gives the pair (x, x + 1) in the two halves of a register
// and per block the scales as [l / 4][group of the block][half], the zeros alike.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <new>
#include <vector>

#include "gg_epilogue_ops.cuh"
#include "grouped_gemm_b200.h"

namespace gg {
namespace {

constexpr int kQ4Threads = 256;
constexpr int kQ4Warps = kQ4Threads / 32;
constexpr int kTileN = 16;   // outputs a block of weights covers
constexpr int kBlockK = 128; // k values a block covers
constexpr int kBlockBytes = kTileN * kBlockK / 2;

struct Q4Params {
  const unsigned char* q;       // [experts][n_tiles][k_blocks][1024]
  const unsigned short* scales; // [experts][n_tiles][k_blocks][8][groups of a block][2]
  const unsigned char* zeros;   // the same, bytes; NULL: all 8
  const float* const* bias;     // [experts]; NULL: none
  int* status;
  int experts, n, k, n_tiles, k_blocks, output_type, activation;
  // of a run
  const void* a;
  const int* row_tokens;
  const int* rows;
  void* d;
  int64_t lda, ldd;
  int a_rows, capacity_rows;
  int vec_a;
};

struct Q4PackParams {
  const unsigned char* const* q;
  const void* const* scales;
  const unsigned char* const* zeros;
  unsigned char* out_q;
  unsigned short* out_scales;
  unsigned char* out_zeros;
  int experts, n, k, group, n_tiles, k_blocks, per_block;
  int64_t ldq;
};

// One thread per 16-byte piece (expert, tile, block, half, lane), and one per scale.
__global__ void __launch_bounds__(kQ4Threads) q4_pack_kernel(Q4PackParams p) {
  const int64_t blocks = static_cast<int64_t>(p.experts) * p.n_tiles * p.k_blocks;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kQ4Threads;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kQ4Threads + threadIdx.x;
  for (int64_t i = first; i < blocks * 64; i += stride) {
    const int64_t b = i / 64;
    const int h = static_cast<int>(i / 32 % 2), lane = static_cast<int>(i % 32);
    const int kb = static_cast<int>(b % p.k_blocks), tile = static_cast<int>(b / p.k_blocks % p.n_tiles);
    const int e = static_cast<int>(b / p.k_blocks / p.n_tiles);
    const int o = kTileN * tile + 8 * h + lane / 4;
    unsigned w[4];
    for (int x = 0; x < 4; ++x) {
      unsigned word = 0;
      for (int v = 0; v < 8; ++v) {
        const int k = kBlockK * kb + 32 * x + 8 * (lane % 4) + v;
        unsigned q = 8;
        if (o < p.n && k < p.k) q = (p.q[e][o * p.ldq + k / 2] >> (4 * (k % 2))) & 15u;
        const int place = (v / 2) + 4 * (v % 2);
        word |= q << (4 * place);
      }
      w[x] = word;
    }
    reinterpret_cast<uint4*>(p.out_q)[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  const int per = 16 * p.per_block;
  const int groups = (p.k + p.group - 1) / p.group;
  for (int64_t i = first; i < blocks * per; i += stride) {
    const int64_t b = i / per;
    const int in = static_cast<int>(i % per);
    const int h = in % 2, sub = in / 2 % p.per_block, row = in / 2 / p.per_block;
    const int kb = static_cast<int>(b % p.k_blocks), tile = static_cast<int>(b / p.k_blocks % p.n_tiles);
    const int e = static_cast<int>(b / p.k_blocks / p.n_tiles);
    const int o = kTileN * tile + 8 * h + row;
    const int k = kBlockK * kb + kBlockK / p.per_block * sub;
    const bool in_range = o < p.n && k < p.k;
    const int64_t at = static_cast<int64_t>(o) * groups + k / p.group;
    p.out_scales[i] = in_range ? static_cast<const unsigned short*>(p.scales[e])[at] : static_cast<unsigned short>(0);
    if (p.out_zeros) p.out_zeros[i] = in_range ? p.zeros[e][at] & 15 : 8;
  }
}

template <bool kBf16>
struct Q4Type;
template <>
struct Q4Type<false> {
  static constexpr int kOut = kOutF16;
  static constexpr unsigned kMagic = 0x64006400u;  // 1024: the low mantissa bits count in ones
};
template <>
struct Q4Type<true> {
  static constexpr int kOut = kOutBF16;
  static constexpr unsigned kMagic = 0x43004300u;  // 128
};

// (a - b) of two pairs of 16-bit numbers; exact here (whole numbers below 2048, below 256 in BF16).
template <bool kBf16>
__device__ __forceinline__ unsigned sub2(unsigned a, unsigned b) {
  unsigned d;
  if constexpr (kBf16) asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  if constexpr (kBf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float q4_activate(float x, int act) {
  if (act == GG_ACT_RELU) return x < 0.0f ? 0.0f : x;
  if (act == GG_ACT_GELU) return x / (1.0f + expf(-1.5957691216057308f * fmaf(0.044715f * x, x * x, x)));
  return x;
}

// Eight activations from k on of row `row` (elements past k are zero), as four packed pairs.
__device__ __forceinline__ uint4 load_a(const Q4Params& p, int64_t row, int k) {
  const unsigned short* at = static_cast<const unsigned short*>(p.a) + row * p.lda + k;
  if (p.vec_a && k + 8 <= p.k) return __ldg(reinterpret_cast<const uint4*>(at));
  unsigned v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = k + i < p.k ? __ldg(at + i) : 0u;
  return make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
}

// kPer: groups per 128-k block (1, 2 or 4).
template <bool kBf16, int kPer, bool kZeros>
__global__ void __launch_bounds__(kQ4Threads) q4_kernel(Q4Params p) {
  __shared__ int s_row0[GG_Q4_MAX_EXPERTS];   // first packed row of each busy expert
  __shared__ int s_rows[GG_Q4_MAX_EXPERTS];
  __shared__ int s_item[GG_Q4_MAX_EXPERTS + 1];  // first item of each busy expert
  __shared__ int s_expert[GG_Q4_MAX_EXPERTS];
  __shared__ int s_busy, s_bad;
  __shared__ float s_sum[kQ4Warps][kTileN * 8];
  using Type = Q4Type<kBf16>;
  const int tid = static_cast<int>(threadIdx.x), warp = tid / 32, lane = tid % 32;
  const int g = lane / 4, t = lane % 4;

  if (warp == 0) {  // the busy experts, in order
    int busy = 0, item = 0;
    int64_t row = 0;
    bool bad = false;
    for (int e0 = 0; e0 < p.experts; e0 += 32) {
      const int e = e0 + lane;
      const int rows = e >= p.experts ? 0 : p.rows ? p.rows[e] : p.capacity_rows;
      bad |= rows < 0;
      // sums clamped per expert, so that no count overflows before it is refused
      const int64_t mine = max(0, rows);
      int64_t upto = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += up;
      }
      const unsigned has = __ballot_sync(0xffffffffu, mine > 0);
      const int at = busy + __popc(has & ((1u << lane) - 1u));
      if (mine > 0) {
        s_expert[at] = e;
        s_rows[at] = static_cast<int>(mine);
        s_row0[at] = static_cast<int>(min(static_cast<int64_t>(p.capacity_rows), row + upto - mine));
      }
      busy += __popc(has);
      row += __shfl_sync(0xffffffffu, upto, 31);
    }
    bad = __any_sync(0xffffffffu, bad) || row > p.capacity_rows || (p.row_tokens == nullptr && row > p.a_rows);
    __syncwarp();
    if (lane == 0) {
      if (!bad)
        for (int i = 0; i < busy; ++i) {
          s_item[i] = item;
          item += (s_rows[i] + 7) / 8 * p.n_tiles;
        }
      s_item[busy] = item;
      s_busy = busy;
      s_bad = bad;
      if (bad && blockIdx.x == 0) atomicOr(p.status, GG_STATUS_BAD_ROWS);
    }
  }
  __syncthreads();
  if (s_bad) return;
  const int items = s_item[s_busy];
  int cur = 0;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    while (s_item[cur + 1] <= item) ++cur;
    const int in = item - s_item[cur];
    const int tile = in % p.n_tiles, chunk = in / p.n_tiles;
    const int e = s_expert[cur];
    const int row0 = s_row0[cur] + 8 * chunk, count = min(8, s_rows[cur] - 8 * chunk);
    // this lane's row of the activations: column g of the product
    int64_t arow = -1;
    if (g < count) {
      arow = p.row_tokens ? p.row_tokens[row0 + g] : row0 + g;
      if (arow >= p.a_rows) arow = -1;
    }
    const int64_t blk0 = (static_cast<int64_t>(e) * p.n_tiles + tile) * p.k_blocks;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int kb = warp; kb < p.k_blocks; kb += kQ4Warps) {
      const uint4* wq = reinterpret_cast<const uint4*>(p.q + (blk0 + kb) * kBlockBytes) + lane;
      const uint4 w0 = __ldg(wq), w1 = __ldg(wq + 32);
      const unsigned lo[4] = {w0.x, w0.y, w0.z, w0.w}, hi[4] = {w1.x, w1.y, w1.z, w1.w};
      const int64_t meta = ((blk0 + kb) * 8 + g) * kPer * 2;
#pragma unroll
      for (int sub = 0; sub < kPer; ++sub) {
        const unsigned sc = __ldg(reinterpret_cast<const unsigned*>(p.scales + meta) + sub);
        const float2 s = unpack2<Type::kOut>(sc);
        unsigned z0 = 8, z1 = 8;
        if constexpr (kZeros) z0 = __ldg(p.zeros + meta + 2 * sub), z1 = __ldg(p.zeros + meta + 2 * sub + 1);
        const unsigned b0 = Type::kMagic + z0 * 0x10001u, b1 = Type::kMagic + z1 * 0x10001u;
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = sub * (4 / kPer); i < (sub + 1) * (4 / kPer); ++i) {
          uint4 x = make_uint4(0u, 0u, 0u, 0u);
          if (arow >= 0) x = load_a(p, arow, kBlockK * kb + 32 * i + 8 * t);
          unsigned f0[4], f1[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            f0[v] = sub2<kBf16>(((lo[i] >> (4 * v)) & 0x000f000fu) | Type::kMagic, b0);
            f1[v] = sub2<kBf16>(((hi[i] >> (4 * v)) & 0x000f000fu) | Type::kMagic, b1);
          }
          const unsigned a0[4] = {f0[0], f1[0], f0[1], f1[1]}, a1[4] = {f0[2], f1[2], f0[3], f1[3]};
          mma16816<kBf16>(part, a0, x.x, x.y);
          mma16816<kBf16>(part, a1, x.z, x.w);
        }
        acc[0] = fmaf(s.x, part[0], acc[0]);
        acc[1] = fmaf(s.x, part[1], acc[1]);
        acc[2] = fmaf(s.y, part[2], acc[2]);
        acc[3] = fmaf(s.y, part[3], acc[3]);
      }
    }
    // sums of the warps, in warp order: [row of the activations][output]
    __syncthreads();
    s_sum[warp][(2 * t) * kTileN + g] = acc[0];
    s_sum[warp][(2 * t + 1) * kTileN + g] = acc[1];
    s_sum[warp][(2 * t) * kTileN + g + 8] = acc[2];
    s_sum[warp][(2 * t + 1) * kTileN + g + 8] = acc[3];
    __syncthreads();
    if (tid < kTileN * 8) {
      const int r = tid / kTileN, o = kTileN * tile + tid % kTileN;
      if (r < count && o < p.n) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kQ4Warps; ++w) sum += s_sum[w][tid];
        if (p.bias && p.bias[e]) sum += p.bias[e][o];
        store_out_rt(p.output_type, p.d, (row0 + r) * p.ldd + o, q4_activate(sum, p.activation));
      }
    }
  }
}

template <typename F>
void with_q4(bool bf16, int per_block, bool zeros, F f) {
  using std::bool_constant;
  using std::integral_constant;
  auto types = [&](auto b) {
    auto per = [&](auto n) {
      if (zeros) f(b, n, bool_constant<true>());
      else f(b, n, bool_constant<false>());
    };
    if (per_block == 1) per(integral_constant<int, 1>());
    else if (per_block == 2) per(integral_constant<int, 2>());
    else per(integral_constant<int, 4>());
  };
  if (bf16) types(bool_constant<true>());
  else types(bool_constant<false>());
}

}  // namespace
}  // namespace gg

struct gg_q4_plan {
  void* block = nullptr;  // weights | scales | zeros | bias table | status
  gg::Q4Params params{};
  bool bf16 = false;
  int per_block = 1;
  int grid = 0;
};

extern "C" {

int gg_q4_plan_create(const gg_q4_problem* problem, void* stream, gg_q4_plan** out) {
  if (!out) return cudaErrorInvalidValue;
  *out = nullptr;
  if (!problem) return cudaErrorInvalidValue;
  const gg_q4_problem& q = *problem;
  if (q.experts < 1 || q.experts > GG_Q4_MAX_EXPERTS || q.n < 1 || q.k < 1 || q.ldq < (q.k + 1) / 2 || !q.q || !q.scales ||
      (q.group != 32 && q.group != 64 && (q.group < 128 || q.group % 128 != 0)) ||
      (q.input_type != GG_INPUT_F16 && q.input_type != GG_INPUT_BF16) || q.output_type < GG_OUTPUT_F32 ||
      q.output_type > GG_OUTPUT_BF16 || q.activation < GG_ACT_NONE || q.activation > GG_ACT_GELU)
    return cudaErrorInvalidValue;
  for (int e = 0; e < q.experts; ++e)
    if (!q.q[e] || !q.scales[e] || (q.zeros && !q.zeros[e])) return cudaErrorInvalidValue;
  const size_t E = static_cast<size_t>(q.experts);
  const int n_tiles = (q.n - 1) / gg::kTileN + 1, k_blocks = (q.k - 1) / gg::kBlockK + 1;
  const int per_block = q.group >= gg::kBlockK ? 1 : gg::kBlockK / q.group;
  const size_t blocks = E * n_tiles * k_blocks;
  const auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  const size_t scales_at = up(blocks * gg::kBlockBytes);
  const size_t zeros_at = up(scales_at + blocks * 16 * per_block * 2);
  const size_t bias_at = up(zeros_at + (q.zeros ? blocks * 16 * per_block : 0));
  const size_t status_at = up(bias_at + E * sizeof(void*));
  const size_t tables_at = up(status_at + sizeof(int));  // the caller's pointers, read once
  const size_t bytes = tables_at + 3 * E * sizeof(void*);

  gg_q4_plan* plan = new (std::nothrow) gg_q4_plan();
  if (!plan) return cudaErrorMemoryAllocation;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  std::vector<const void*> tables(3 * E);
  for (size_t e = 0; e < E; ++e) {
    tables[e] = q.q[e];
    tables[E + e] = q.scales[e];
    tables[2 * E + e] = q.zeros ? q.zeros[e] : nullptr;
  }
  int device = 0, sms = 0, per_sm = 0;
  cudaError_t st = cudaGetDevice(&device);
  if (st == cudaSuccess) st = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (st == cudaSuccess)
    gg::with_q4(q.input_type == GG_INPUT_BF16, per_block, q.zeros != nullptr, [&](auto b, auto n, auto z) {
      st = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, gg::q4_kernel<b(), n(), z()>, gg::kQ4Threads, 0);
    });
  if (st == cudaSuccess) st = cudaMalloc(&plan->block, bytes);
  if (st != cudaSuccess) {
    delete plan;
    return st;
  }
  unsigned char* base = static_cast<unsigned char*>(plan->block);
  st = cudaMemcpyAsync(base + tables_at, tables.data(), tables.size() * sizeof(void*), cudaMemcpyHostToDevice, s);
  if (st == cudaSuccess && q.bias)
    st = cudaMemcpyAsync(base + bias_at, q.bias, E * sizeof(void*), cudaMemcpyHostToDevice, s);
  if (st == cudaSuccess) st = cudaMemsetAsync(base + status_at, 0, sizeof(int), s);
  if (st == cudaSuccess) {
    const unsigned char* const* table = reinterpret_cast<const unsigned char* const*>(base + tables_at);
    gg::Q4PackParams pk{table,
                        reinterpret_cast<const void* const*>(table + E),
                        table + 2 * E,
                        base,
                        reinterpret_cast<unsigned short*>(base + scales_at),
                        q.zeros ? base + zeros_at : nullptr,
                        q.experts,
                        q.n,
                        q.k,
                        q.group,
                        n_tiles,
                        k_blocks,
                        per_block,
                        q.ldq};
    const size_t want = (blocks * 64 + gg::kQ4Threads - 1) / gg::kQ4Threads;
    gg::q4_pack_kernel<<<static_cast<unsigned>(std::min<size_t>(want, 1u << 16)), gg::kQ4Threads, 0, s>>>(pk);
    st = cudaGetLastError();
  }
  if (st == cudaSuccess) st = cudaStreamSynchronize(s);
  if (st != cudaSuccess) {
    cudaFree(plan->block);
    delete plan;
    return st;
  }
  gg::Q4Params& p = plan->params;
  p.q = base;
  p.scales = reinterpret_cast<const unsigned short*>(base + scales_at);
  p.zeros = q.zeros ? base + zeros_at : nullptr;
  p.bias = q.bias ? reinterpret_cast<const float* const*>(base + bias_at) : nullptr;
  p.status = reinterpret_cast<int*>(base + status_at);
  p.experts = q.experts;
  p.n = q.n;
  p.k = q.k;
  p.n_tiles = n_tiles;
  p.k_blocks = k_blocks;
  p.output_type = q.output_type;
  p.activation = q.activation;
  plan->bf16 = q.input_type == GG_INPUT_BF16;
  plan->per_block = per_block;
  plan->grid = std::max(1, sms * per_sm);
  *out = plan;
  return cudaSuccess;
}

int gg_q4_plan_run(gg_q4_plan* plan, const void* a, int lda, int a_rows, const int* row_tokens, const int* rows,
                   void* d, int ldd, int capacity_rows, void* stream) {
  if (!plan || !plan->block) return cudaErrorInvalidDevicePointer;
  gg::Q4Params p = plan->params;
  if (capacity_rows < 0 || a_rows < 0 || lda < p.k || ldd < p.n || (!rows && p.experts != 1)) return cudaErrorInvalidValue;
  if (capacity_rows == 0 && !rows) return cudaSuccess;
  if ((capacity_rows > 0 && !d) || (a_rows > 0 && !a)) return cudaErrorInvalidValue;
  // items are counted in an int: (rows / 8 + experts) tiles of 16 outputs
  if ((static_cast<int64_t>(capacity_rows) / 8 + p.experts) * p.n_tiles > INT32_MAX) return cudaErrorInvalidValue;
  p.a = a;
  p.lda = lda;
  p.a_rows = a_rows;
  p.row_tokens = row_tokens;
  p.rows = rows;
  p.d = d;
  p.ldd = ldd;
  p.capacity_rows = capacity_rows;
  p.vec_a = (reinterpret_cast<uintptr_t>(a) & 15u) == 0 && lda % 8 == 0;
  const int64_t most = (static_cast<int64_t>(capacity_rows) / 8 + std::min(capacity_rows, p.experts)) * p.n_tiles;
  const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(plan->grid, most)));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  gg::with_q4(plan->bf16, plan->per_block, p.zeros != nullptr, [&](auto b, auto n, auto z) {
    gg::q4_kernel<b(), n(), z()><<<grid, gg::kQ4Threads, 0, s>>>(p);
  });
  return cudaGetLastError();
}

int gg_q4_plan_status(gg_q4_plan* plan, int* status) {
  if (!plan || !plan->block) return cudaErrorInvalidDevicePointer;
  if (!status) return cudaErrorInvalidValue;
  cudaError_t st = cudaDeviceSynchronize();
  if (st != cudaSuccess) return st;
  st = cudaMemcpy(status, plan->params.status, sizeof(int), cudaMemcpyDeviceToHost);
  if (st != cudaSuccess) return st;
  return cudaMemset(plan->params.status, 0, sizeof(int));
}

void gg_q4_plan_destroy(gg_q4_plan* plan) {
  if (!plan) return;
  if (plan->block) cudaFree(plan->block);
  delete plan;
}

}  // extern "C"
