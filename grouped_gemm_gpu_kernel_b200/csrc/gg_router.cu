// gg_router.cu -- the mixture-of-experts router: top-k experts of every token, their weights, the
// row counts, the places of the rows in packed order, the balance and z losses, and the gradient of
// all of them with respect to the logits.
//
// Forward. A group of G lanes holds one token's logits, V consecutive experts a lane (G * V >=
// experts), so a warp works on 32 / G tokens at once. Choosing is on the logits themselves, through
// an integer key that orders like the value, so equal logits tie exactly and rounding of exp() never
// decides. Every warp owns a contiguous range of tokens and counts its choices per expert as it
// goes; a slot's rank among its warp's earlier slots of the same expert is its place up to an offset
// that only depends on (expert, warp). Those offsets need the counts of all warps, so a second
// kernel adds them (for few tokens the blocks of one cluster do both in one launch). No atomics: ranks and
// sums have a fixed order, and the same inputs give the same bits.
//
// What bounds it (B200): up to some ten thousand tokens the launches (4 tokens of 64 experts 5.5 us, 999 of 37 8.5 us,
// 16384 of 64 11.8 us, where the logits' bytes would take 0.6); then the instructions of choosing (131072 tokens of 256
// FP32 logits, top 8: 85 us, 80 % of the forward kernel's issue slots, some 484 a token; the bytes would take
// 24 us), all the more where the choice goes by rounds of maxima: 233 us there with top 16, 432 with top 32. 32768 tokens
// of 512 experts, top 8, take 54 us, of 1024, 32 experts a lane in 8 warps an SM, 169. The gradient reads the logits and
// writes their gradient once: 51 us for 131072 of 256, 0.81 of the copy rate.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstring>
#include <new>

#include "gg_epilogue_ops.cuh"
#include "gg_launch.cuh"
#include "grouped_gemm_b200.h"

namespace gg {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kMaxBlocks = 148;  // one forward block per SM at most

struct RouterShape {
  int experts, top_k, normalize;
};

// What a forward pass leaves per block and warp for the second kernel.
struct RouterWork {
  int* warp_before;   // [blocks][warps][experts] rows of the block's earlier warps
  int* block_count;   // [blocks][experts]
  float* block_prob;  // [blocks][experts] sums of p
  float* block_z;     // [blocks][2]: sum of lse^2, valid tokens
};

constexpr int kTaken = INT32_MIN;             // below every key
constexpr int kClosed = static_cast<int>(0x807fffffu);  // the key of -infinity: an expert that cannot be taken

// A signed integer that orders like the float: adding 0 turns -0 into +0 and every NaN into the
// positive one, which is above +infinity; negative numbers order backwards in their low 31 bits.
__device__ __forceinline__ int order_key(float v) {
  const int b = __float_as_int(v + 0.0f);
  return b ^ ((b >> 31) & 0x7fffffff);
}

__device__ __forceinline__ float key_value(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }

template <int G>
__device__ __forceinline__ int group_max(int v) {
  if constexpr (G == 32) {
    return __reduce_max_sync(kFull, v);
  } else {
#pragma unroll
    for (int d = G / 2; d > 0; d >>= 1) v = max(v, __shfl_xor_sync(kFull, v, d));
    return v;
  }
}

// exp(x) for x <= 0: 2^-22 + |x| 2^-23 relative (the exponential unit, and the roundings of log2(e) and of the scaled
// argument), and 0 below 2^-126. expf() costs four times the instructions for 2^-23. What that would gain is lost on a
// probability before: the terms that make up a sum have |x| of a few units, so its error is a few 2^-22, and a term of
// larger |x| is off by more of itself, but is that much smaller (1e-5 of e^-64 at x = -64).
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float exp_fast(float x) { return exp2_fast(x * kLog2e); }

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int d = G / 2; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  return v;
}

// V consecutive elements from p (element count `have` of them exist; the rest read as `fill`).
template <int F, int V>
__device__ __forceinline__ void load_row(const void* base, int64_t at, int have, bool vec, float fill, float (&v)[V]) {
  if (vec && have >= V) {
    if constexpr (F == kOutF32) {
      const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        const float4 q = __ldg(p + i);
        v[4 * i] = q.x, v[4 * i + 1] = q.y, v[4 * i + 2] = q.z, v[4 * i + 3] = q.w;
      }
    } else {
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(base) + at);
#pragma unroll
      for (int i = 0; i < V / 8; ++i) {
        const uint4 q = __ldg(p + i);
        const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const float2 f = unpack2<F>(w[h]);
          v[8 * i + 2 * h] = f.x, v[8 * i + 2 * h + 1] = f.y;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = i < have ? load_out<F>(base, at + i) : fill;
  }
}

// Warps of a forward block (one block an SM): as many as the registers of V experts a lane allow.
__host__ __device__ constexpr int router_warps(int V) { return V <= 8 ? 32 : V <= 16 ? 16 : 8; }
constexpr int kClusterMost = 8;   // blocks of a cluster that any launch may ask for
constexpr int kFewWarps = 4;  // of a forward block that takes few tokens
constexpr int kBackwardWarps = 8;
constexpr int kBackwardBlocks = 4;  // of them an SM: the grid is one wave, and a warp walks its tokens

constexpr int kForwardSmemMost = 160 * 1024;
constexpr int kCandidates = 64;  // see choose_of_candidates
// Slots a warp gathers before it places them: 32 (one a lane) or, where its tokens of one turn have more,
// theirs. At least one turn, at most 32 tokens.
__host__ __device__ __forceinline__ int slots_held(int at_once, int top_k) {
  return at_once * top_k > 32 ? at_once * top_k : 32;
}

// Shared memory of a forward block, in 4-byte words: counts [warps][experts], sums of p
// [warps][experts], per warp the held slots (index and key) and the factor of the weights and the
// largest logit of their tokens (32 at most), z and valid tokens per warp; where a warp takes one
// token at once, its candidates (keys, then experts).
size_t forward_smem(int G, int warps, int experts, int top_k) {
  return 4ull * (2ull * warps * experts + warps * (2ull * slots_held(32 / G, top_k) + 64) + 2ull * warps +
                 (G == 32 ? 2ull * kCandidates * warps : 0));
}

// Parts the blocks' counts are summed in: what the threads allow, so that each sums few rows.
__host__ __device__ __forceinline__ int place_parts(int threads, int experts) {
  const int p = threads / (experts % 4 == 0 ? experts / 4 : experts);
  return p < 1 ? 1 : p > 16 ? 16 : p;
}
size_t place_smem(int threads, int experts) {
  return 4ull * ((3ull * place_parts(threads, experts) + 2 + threads / 32) * experts + 64);
}

struct PlaceArgs {
  RouterShape shape;
  RouterWork work;
  int tokens, tokens_per_warp, blocks;
  int cluster;  // blocks of the forward kernel's one cluster; 0: it has none, and a second kernel places the slots
  const int* indices;
  int* positions;
  int* rows;
  int* row_tokens;
  float* prob_mean;
  float* losses;
};

__device__ __forceinline__ float block_sum(float v, float* s_warp) {
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  __syncthreads();
  if (threadIdx.x % 32 == 0) s_warp[threadIdx.x / 32] = v;
  __syncthreads();
  float s = 0.0f;
  for (int i = 0; i < static_cast<int>(blockDim.x) / 32; ++i) s += s_warp[i];
  return s;
}

// Sums over the rows of a [rows][E] table, N columns (1 or 4) and one of `parts` of the rows a thread, eight rows
// loaded before the first is added (one after the other, they would cost a trip to L2 each). total and, where
// given, below (the rows before `split`) become [parts][E] partial sums.
template <int N, typename T>
__device__ __forceinline__ void sum_rows(const T* table, int E, int rows, int parts, int split, T* total, T* below) {
  const int columns = E / N;
  for (int i = threadIdx.x; i < parts * columns; i += blockDim.x) {
    const int part = i / columns, e = (i - part * columns) * N;
    T all[N], low[N];
#pragma unroll
    for (int x = 0; x < N; ++x) all[x] = low[x] = T(0);
    for (int b = part; b < rows; b += 8 * parts) {
      T c[8][N];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int at = b + r * parts;
        const T* from = table + static_cast<int64_t>(at) * E + e;
        if constexpr (N == 4) {
          int4 q = make_int4(0, 0, 0, 0);
          if (at < rows) q = *reinterpret_cast<const int4*>(from);
          memcpy(c[r], &q, sizeof(q));
        } else {
          c[r][0] = at < rows ? *from : T(0);
        }
      }
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int x = 0; x < N; ++x) {
          all[x] += c[r][x];
          low[x] += b + r * parts < split ? c[r][x] : T(0);
        }
    }
#pragma unroll
    for (int x = 0; x < N; ++x) {
      total[part * E + e + x] = all[x];
      if (below) below[part * E + e + x] = low[x];
    }
  }
}

// Turns the ranks of a block's slots into packed rows (slots), and what the blocks left behind into the
// counts, means and losses (losses). smem: place_smem bytes.
__device__ void place_block(const PlaceArgs& a, int block, bool slots, bool losses, unsigned char* smem) {
  const int E = a.shape.experts, K = a.shape.top_k;
  const int tid = static_cast<int>(threadIdx.x), threads = static_cast<int>(blockDim.x);
  const int warps = threads / 32, warp = tid / 32, lane = tid % 32;
  const int parts = place_parts(threads, E);
  int* s_before = reinterpret_cast<int*>(smem);                   // [parts][E]
  int* s_total = s_before + parts * E;                            // [parts][E]
  float* s_prob = reinterpret_cast<float*>(s_total + parts * E);  // [parts][E]
  int* s_base = reinterpret_cast<int*>(s_prob + parts * E);       // [E]
  int* s_sum = s_base + E;                                        // [E]
  float* s_warp = reinterpret_cast<float*>(s_sum + E);            // [64]
  int* first = reinterpret_cast<int*>(s_warp + 64) + warp * E;    // of every expert, the first row of this warp

  // this warp's first slots and its experts' earlier rows, on their way during the sums
  const int unit = block * warps + warp;
  const int t0 = static_cast<int>(min(static_cast<int64_t>(a.tokens), static_cast<int64_t>(unit) * a.tokens_per_warp));
  const int s_end = (a.tokens - t0 > a.tokens_per_warp ? t0 + a.tokens_per_warp : a.tokens) * K;
  constexpr int kBatch = 4;  // slots a lane loads before it stores the first
  int e_of[kBatch], rank[kBatch];
  const auto load_slots = [&](int s0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const bool in = s_end - s0 > 32 * i;
      e_of[i] = in ? a.indices[s0 + 32 * i] : -1;
      rank[i] = in ? a.positions[s0 + 32 * i] : 0;
    }
  };
  if (slots) {
    load_slots(t0 * K + lane);
    for (int e = lane; e < E; e += 32) first[e] = a.work.warp_before[static_cast<int64_t>(unit) * E + e];
  }
  float z = 0.0f, n = 0.0f;
  if (losses)
    for (int b = tid; b < a.blocks; b += threads) z += a.work.block_z[2 * b], n += a.work.block_z[2 * b + 1];
  if (E % 4 == 0) {
    sum_rows<4>(a.work.block_count, E, a.blocks, parts, block, s_total, s_before);
    if (losses) sum_rows<4>(a.work.block_prob, E, a.blocks, parts, 0, s_prob, static_cast<float*>(nullptr));
  } else {
    sum_rows<1>(a.work.block_count, E, a.blocks, parts, block, s_total, s_before);
    if (losses) sum_rows<1>(a.work.block_prob, E, a.blocks, parts, 0, s_prob, static_cast<float*>(nullptr));
  }
  __syncthreads();
  for (int e = tid; e < E; e += threads) {
    int before = 0, total = 0;
    for (int p = 0; p < parts; ++p) before += s_before[p * E + e], total += s_total[p * E + e];
    s_base[e] = before;
    s_sum[e] = total;
  }
  __syncthreads();
  if (tid < 32) {  // the experts' offsets: an exclusive scan of the totals
    int run = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + tid;
      const int c = e < E ? s_sum[e] : 0;
      int inc = c;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(kFull, inc, d);
        if (tid >= d) inc += up;
      }
      if (e < E) s_base[e] += run + inc - c;
      run += __shfl_sync(kFull, inc, 31);
    }
    if (tid == 0) s_warp[32] = __int_as_float(run);
  }
  __syncthreads();
  const int routed = __float_as_int(s_warp[32]);

  if (slots) {
    for (int s0 = t0 * K + lane; s0 < s_end; s0 += 32 * kBatch) {
      if (s0 != t0 * K + lane) load_slots(s0);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int s = s0 + 32 * i, e = e_of[i];
        if (s_end - s0 <= 32 * i) break;
        int p = -1;
        if (e >= 0) {
          p = s_base[e] + first[e] + rank[i];
          if (a.row_tokens) a.row_tokens[p] = static_cast<int>(static_cast<unsigned>(s) / static_cast<unsigned>(K));
        }
        a.positions[s] = p;
      }
      if (s_end - s0 <= 32 * kBatch) break;
    }
    if (a.row_tokens)
      for (int64_t s = routed + static_cast<int64_t>(block) * threads + tid; s < static_cast<int64_t>(a.tokens) * K;
           s += static_cast<int64_t>(a.blocks) * threads)
        a.row_tokens[s] = -1;
  }
  if (!losses) return;

  z = block_sum(z, s_warp);
  n = block_sum(n, s_warp);
  const float inv_n = 1.0f / fmaxf(n, 1.0f);
  const float inv_routed = 1.0f / static_cast<float>(max(routed, 1));
  float balance = 0.0f;
  for (int e = tid; e < E; e += threads) {
    float sum = 0.0f;
    for (int p = 0; p < parts; ++p) sum += s_prob[p * E + e];
    const float mean = sum * inv_n;
    if (a.prob_mean) a.prob_mean[e] = mean;
    a.rows[e] = s_sum[e];
    balance = fmaf(static_cast<float>(s_sum[e]) * inv_routed, mean, balance);
  }
  balance = block_sum(balance, s_warp);
  if (tid == 0) {
    a.losses[0] = static_cast<float>(E) * balance;
    a.losses[1] = z * inv_n;
    a.losses[2] = n;
  }
}

struct ForwardArgs {
  const void* logits;
  const unsigned char* mask;
  int* indices;
  float* weights;
  float* lse;
  int64_t ld;
  int vec;  // rows can be read 16 bytes at a time
  PlaceArgs place;
};

// The keys in list[0, n) (a multiple of 8 is read; those past n are kTaken) above `own`, which is at `at`; with
// `ties` the equal ones before it as well.
__device__ __forceinline__ int keys_above(const int* list, int n, int own, int at, bool ties) {
  int rank = 0;
  if (!ties) {
    for (int c = 0; c < n; c += 8) {
      const int4 x = *reinterpret_cast<const int4*>(list + c), y = *reinterpret_cast<const int4*>(list + c + 4);
      const int k[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        asm("{ .reg .pred p; setp.gt.s32 p, %1, %2; @p add.s32 %0, %0, 1; }" : "+r"(rank) : "r"(k[i]), "r"(own));
    }
  } else {
    for (int c = 0; c < n; ++c) rank += c < at ? list[c] >= own : list[c] > own;
  }
  return rank;
}

// The top_k largest keys of a token that a whole warp holds, V consecutive experts a lane, when
// top_k <= 8: the smallest of the maxima of eight groups of four lanes bounds the 8th largest key from below,
// so only keys from it on are candidates. On random logits that leaves about 22 (the draws until
// every group was hit), where every group has an open expert: with 225 to 256 experts, 449 to 512 or 897 to 1024.
// With fewer a group holds none, all open experts are candidates, too many, and the bound and the scan are spent for
// nothing (131072 tokens of 160 experts, top 8: 147 us forward, 84 of 256; 32768 of 384: 77, of 512: 54). Candidates
// are gathered in shared memory in the order of experts, one a lane (two where they are
// more than 32), and each lane counts the keys above its own: that is its slot. The counts depend on no
// other lane's, unlike rounds that take one maximum after the other (131072 tokens of 256 experts, top 8: this kernel
// 77 us, 91 with such rounds on the candidates, 114 with rounds on all keys). Equal keys give a slot twice, and leave
// one empty unless it is the last; then, and only then, the keys before a lane's own are counted from its own on (BF16
// logits near 100, most of whose tokens tie: 132 us forward, 98 near 0). Writes the slots and returns the
// lane's part of the sum of exp(key - top); fits: false where there are more than kCandidates, and nothing is written.
template <int V>
__device__ __forceinline__ float choose_of_candidates(const int (&key)[V], int mine, int e0, int K, int* s_list, unsigned list, int lane,
                                                      int* s_slot, int* s_key, float top, bool* fits) {
  int bound = max(mine, __shfl_xor_sync(kFull, mine, 1));
  bound = max(bound, __shfl_xor_sync(kFull, bound, 2));
  bound = max(__reduce_min_sync(kFull, bound), kClosed + 1);
  int upto = 0;
#pragma unroll
  for (int i = 0; i < V; ++i)
    asm("{ .reg .pred p; setp.ge.s32 p, %1, %2; @p add.s32 %0, %0, 1; }" : "+r"(upto) : "r"(key[i]), "r"(bound));
  const int count = upto;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1)
    asm volatile("{ .reg .s32 r; .reg .pred p; shfl.sync.up.b32 r|p, %0, %1, 0, -1; @p add.s32 %0, %0, r; }" : "+r"(upto) : "r"(d));
  const int n = __shfl_sync(kFull, upto, 31);
  *fits = n <= kCandidates;
  if (n > kCandidates) return 0.0f;
  // `list`: s_list as a shared address; keys, then kCandidates words further their experts
  unsigned to = list + 4 * (upto - count);
#pragma unroll
  for (int i = 0; i < V; ++i)
    asm volatile("{ .reg .pred p; setp.ge.s32 p, %1, %2; @p st.shared.s32 [%0], %1; @p st.shared.s32 [%0 + %4], %3; @p add.u32 %0, %0, 4; }"
                 : "+r"(to)
                 : "r"(key[i]), "r"(bound), "r"(e0 + i), "n"(4 * kCandidates)
                 : "memory");
  if (lane < 8 && n + lane < kCandidates) s_list[n + lane] = kTaken;
  __syncwarp();
  const int slots = min(K, n);
  float part = 0.0f;
  bool ties = false;
  while (true) {
    int taken = 0, takers = 0;
    part = 0.0f;
    for (int first = 0; first < n; first += 32) {
      const int at = first + lane, own = at < n ? s_list[at] : kTaken;
      const int rank = keys_above(s_list, n, own, at, ties);
      const bool in = at < n && rank < K;
      takers += __popc(__ballot_sync(kFull, in));
      if (in) {
        taken |= 1 << rank;
        s_slot[rank] = s_list[kCandidates + at];
        s_key[rank] = own;
        part += exp_fast(key_value(own) - top);
      }
    }
    if (ties || (takers == slots && __reduce_or_sync(kFull, taken) == (1 << slots) - 1)) break;
    ties = true;
    __syncwarp();
  }
  if (lane >= n && lane < K) s_slot[lane] = -1, s_key[lane] = kTaken;  // fewer experts than slots
  return part;
}

template <int F, int G, int V, int W>
__global__ void __launch_bounds__(32 * W) router_forward_kernel(ForwardArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int kWarps = W, kAtOnce = 32 / G;
  const int E = a.place.shape.experts, K = a.place.shape.top_k, T = a.place.tokens;
  const int tid = static_cast<int>(threadIdx.x), warp = tid / 32, lane = tid % 32;
  const int group = lane / G, gl = lane % G;
  int* s_list = reinterpret_cast<int*>(smem) + warp * 2 * kCandidates;
  int* s_count = reinterpret_cast<int*>(smem + (G == 32 ? 8 * kCandidates * kWarps : 0));
  float* s_prob = reinterpret_cast<float*>(s_count + kWarps * E);
  const int held = slots_held(kAtOnce, K);  // slots a warp keeps until it places them together
  int* s_slot = reinterpret_cast<int*>(s_prob + kWarps * E) + warp * (2 * held + 64);
  int* s_key = s_slot + held;
  float* s_factor = reinterpret_cast<float*>(s_key + held);  // [32] factors of the weights, then [32] largest logits
  float* s_z = s_prob + kWarps * E + kWarps * (2 * held + 64);
  int* count = s_count + warp * E;
  for (int e = lane; e < E; e += 32) count[e] = 0;
  __syncwarp();

  // this warp's tokens (the host keeps tokens * top_k in an int)
  chained_begin();
  const int per_warp = a.place.tokens_per_warp;
  const int unit = static_cast<int>(blockIdx.x) * kWarps + warp;
  const int t0 = static_cast<int>(min(static_cast<int64_t>(T), static_cast<int64_t>(unit) * per_warp));
  const int t1 = T - t0 > per_warp ? t0 + per_warp : T;
  const int e0 = gl * V, have = max(0, min(V, E - e0));
  const char* row = static_cast<const char*>(a.logits) + ((t0 + group) * a.ld + e0) * OutFormat<F>::kBytes;
  const int64_t next_row = kAtOnce * a.ld * OutFormat<F>::kBytes;
  float prob[V];
#pragma unroll
  for (int i = 0; i < V; ++i) prob[i] = 0.0f;
  float z = 0.0f, n = 0.0f;

  // Tokens held at a time: as many whole turns as fill the lanes with slots. The first of them is th.
  const int turns = max(1, 32 / (kAtOnce * K));
  const int lane_token = lane / K;  // the held token of this lane's slot among the first 32
  int turn = 0;
  int th = t0;
  for (int tb = t0; tb < t1; tb += kAtOnce, row += next_row) {
    const int t = tb + group;
    const int slot0 = (turn * kAtOnce + group) * K;
    float v[V];
    int key[V];
    load_row<F, V>(row, 0, t < t1 ? have : 0, a.vec != 0, -INFINITY, v);
    if (a.mask != nullptr && t < t1 && a.mask[t] == 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = order_key(v[i]);
    int mine = key[0];
#pragma unroll
    for (int i = 1; i < V; ++i) mine = max(mine, key[i]);
    const int largest = group_max<G>(mine);
    const bool valid = largest > kClosed;
    const float top = key_value(largest);
    float chosen = 0.0f;  // the sum of exp(logit - top) over the chosen experts
    bool done = false;
    if constexpr (G == 32) {
      if (K >= 4 && K <= 8) {
        chosen = choose_of_candidates<V>(key, mine, e0, K, s_list, static_cast<unsigned>(__cvta_generic_to_shared(s_list)), lane, s_slot + slot0, s_key + slot0, top, &done);
        chosen = group_sum<32>(chosen);
      }
    }
    if (!done) {
      int best = largest;
      for (int j = 0; j < K; ++j) {
        const unsigned holders = __ballot_sync(kFull, mine == best);
        const unsigned of_group = G == 32 ? holders : (holders >> (group * G)) & ((1u << (G & 31)) - 1u);
        const int owner = __ffs(of_group) - 1;  // experts are in lane order: the lowest lane has the lowest expert
        if (best > kClosed) chosen += exp_fast(key_value(best) - top);
        if (gl == owner) {
          int at = 0;
#pragma unroll
          for (int i = V - 1; i >= 0; --i) at = key[i] == best ? i : at;
#pragma unroll
          for (int i = 0; i < V; ++i) key[i] = i == at ? kTaken : key[i];
          s_slot[slot0 + j] = best > kClosed ? e0 + at : -1;
          s_key[slot0 + j] = best;
        }
        if (j + 1 == K) break;
        mine = key[0];
#pragma unroll
        for (int i = 1; i < V; ++i) mine = max(mine, key[i]);
        best = group_max<G>(mine);
      }
    }
    // The difference first, whose rounding is relative to it and not to top, and which no finite logits overflow
    // (to -infinity at most). Without a valid logit all of them are -infinity, and give 0.
    float sum = 0.0f;
    float ex[V];
    const float from = valid ? top : 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      ex[i] = exp_fast(v[i] - from);
      sum += ex[i];
    }
    sum = group_sum<G>(sum);
    const float inv = valid ? __fdividef(1.0f, sum) : 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) prob[i] = fmaf(ex[i], inv, prob[i]);
    const float lse = valid ? top + __logf(sum) : 0.0f;
    if (gl == 0) {
      z = fmaf(lse, lse, z);
      n += valid ? 1.0f : 0.0f;
      if (a.lse && t < t1) a.lse[t] = lse;
      s_factor[turn * kAtOnce + group] = a.place.shape.normalize ? __fdividef(1.0f, chosen) : inv;
      s_factor[32 + turn * kAtOnce + group] = top;
    }
    __syncwarp();
    if (++turn < turns && tb + kAtOnce < t1) continue;
    // the slots of the held tokens, in order, 32 at a time
    const int slots = (min(t1, tb + kAtOnce) - th) * K;
    for (int s0 = 0; s0 < slots; s0 += 32) {
      const int s = s0 + lane;
      const int e = s < slots ? s_slot[s] : -1;
      const unsigned same = __match_any_sync(kFull, e);
      const int seen = e >= 0 ? count[e] : 0;
      __syncwarp();
      if (e >= 0 && lane == 31 - __clz(same)) count[e] = seen + __popc(same);
      __syncwarp();
      if (s < slots) {
        const int h = s0 == 0 ? lane_token : s / K;
        const int at = th * K + s;
        a.indices[at] = e;
        a.weights[at] = e >= 0 ? exp_fast(key_value(s_key[s]) - s_factor[32 + h]) * s_factor[h] : 0.0f;
        a.place.positions[at] = seen + __popc(same & ((1u << lane) - 1u));
      }
    }
    __syncwarp();
    turn = 0;
    th = tb + kAtOnce;
  }

  // the block's sums: over the groups of a warp, then over the warps
#pragma unroll
  for (int d = G; d < 32; d <<= 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) prob[i] += __shfl_xor_sync(kFull, prob[i], d);
    z += __shfl_xor_sync(kFull, z, d);
    n += __shfl_xor_sync(kFull, n, d);
  }
  if (group == 0)
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < have) s_prob[warp * E + e0 + i] = prob[i];
  if (lane == 0) s_z[2 * warp] = z, s_z[2 * warp + 1] = n;
  __syncthreads();
  const RouterWork& w = a.place.work;
  for (int e = tid; e < E; e += 32 * kWarps) {
    int run = 0;
    float p = 0.0f;
    static_assert(kWarps % 4 == 0, "four warps' numbers are read before the first is used");
    for (int i0 = 0; i0 < kWarps; i0 += 4) {
      int c[4];
      float f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = s_count[(i0 + i) * E + e], f[i] = s_prob[(i0 + i) * E + e];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w.warp_before[(static_cast<int64_t>(blockIdx.x) * kWarps + i0 + i) * E + e] = run;
        run += c[i];
        p += f[i];
      }
    }
    w.block_count[static_cast<int64_t>(blockIdx.x) * E + e] = run;
    w.block_prob[static_cast<int64_t>(blockIdx.x) * E + e] = p;
  }
  if (tid < 2) {
    float sum = 0.0f;
    for (int i = 0; i < kWarps; ++i) sum += s_z[2 * i + tid];
    w.block_z[2 * blockIdx.x + tid] = sum;
  }
  if (a.place.cluster > 0) {  // the grid is one cluster: its blocks meet here, and place their own slots
    if (a.place.cluster == 1) __syncthreads();
    else asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    place_block(a.place, static_cast<int>(blockIdx.x), true, blockIdx.x == 0, smem);
  }
}

__global__ void __launch_bounds__(1024) router_place_kernel(PlaceArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  chained_begin();
  const int block = static_cast<int>(blockIdx.x);
  place_block(a, block, block < a.blocks, block == a.blocks, smem);  // the last block, without slots, sums the losses
}

struct BackwardArgs {
  RouterShape shape;
  const void* logits;
  const int* indices;
  const float* weights;
  const int* rows;
  const float* losses;
  const float* lse;
  const float* grad_weights;
  const float* grad_losses;
  void* grad;
  int tokens;
  int64_t ld, ldg;
  int vec, vec_grad;
};

// p = exp(l - lse) is off by lse's rounding to FP32, 2^-24 |lse| relative: up to here no more than by the exponential
// itself (1e-6). A token past it has its p divided by their sum, which takes the common factor out (131072 tokens of
// 256 FP32 logits: 51.6 us with no token past it, 54.4 with all of them, 50.0 without the check).
constexpr float kRoughLse = 16.0f;

// dl = p (c_e - <c, p> + 2 g1 lse / n) + the weights' part, with c_e = g0 E f(e) / n. One pass: a
// group of lanes reads its token's logits once and writes the gradient once; all loads of a turn are
// issued before the first is used.
template <int F, int G, int V>
__global__ void __launch_bounds__(32 * kBackwardWarps, V == 8 ? kBackwardBlocks : 1) router_backward_kernel(BackwardArgs a) {
  constexpr int kWarps = kBackwardWarps, kAtOnce = 32 / G;
  constexpr int kSlotTurns = (GG_ROUTER_MAX_TOP_K + G - 1) / G;
  // the weights' part of each token's gradient: expert v of a lane at [v / 4][lane][v % 4], so that a lane
  // reads its experts four at a time and no two lanes of a quarter warp meet in a bank
  __shared__ float4 s_part[kWarps][V / 4][32];
  __shared__ float s_sum[kWarps];
  const int E = a.shape.experts, K = a.shape.top_k;
  const int tid = static_cast<int>(threadIdx.x), warp = tid / 32, lane = tid % 32;
  const int group = lane / G, gl = lane % G;
  const int e0 = gl * V, have = max(0, min(V, E - e0));
  chained_begin();
  const float n = a.losses[2];
  const float inv_n = n > 0.0f ? 1.0f / n : 0.0f;
  const float g0 = a.grad_losses ? a.grad_losses[0] : 0.0f, g1 = a.grad_losses ? a.grad_losses[1] : 0.0f;
  float routed = 0.0f;
  for (int e = tid; e < E; e += 32 * kWarps) routed += static_cast<float>(a.rows[e]);
  routed = block_sum(routed, s_sum);
  const float scale = routed > 0.0f ? g0 * static_cast<float>(E) * inv_n / routed : 0.0f;
  float c[V];
#pragma unroll
  for (int i = 0; i < V; ++i) c[i] = i < have ? scale * static_cast<float>(a.rows[e0 + i]) : 0.0f;
  float* part = reinterpret_cast<float*>(s_part[warp]);
  const auto place = [&](int e) { return (e % V / 4 * 32 + group * G + e / V) * 4 + e % 4; };
#pragma unroll
  for (int i = 0; i < V / 4; ++i) s_part[warp][i][lane] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  __syncwarp();

  const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps * kAtOnce;
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * kWarps + warp) * kAtOnce;
  float next[V];
  load_row<F, V>(a.logits, (first + group) * a.ld + e0, first + group < a.tokens ? have : 0, a.vec != 0, -INFINITY, next);
  for (int64_t tb = first; tb < a.tokens; tb += step) {
    const int64_t t = tb + group;
    const bool in = t < a.tokens;
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = next[i];
    // slot j of a token by lane j of its group (and j + G, ... where top_k is larger)
    int e[kSlotTurns];
    float w[kSlotTurns], gw[kSlotTurns];
#pragma unroll
    for (int i = 0; i < kSlotTurns; ++i) {
      const int j = gl + i * G;
      const bool slot = in && j < K;
      e[i] = slot ? a.indices[t * K + j] : -1;
      w[i] = slot ? a.weights[t * K + j] : 0.0f;
      gw[i] = slot && a.grad_weights ? a.grad_weights[t * K + j] : 0.0f;
      if (i * G + G >= K) break;
    }
    const float lse = in ? a.lse[t] : 0.0f;
    load_row<F, V>(a.logits, (t + step) * a.ld + e0, t + step < a.tokens ? have : 0, a.vec != 0, -INFINITY, next);
    const bool live = __shfl_sync(kFull, e[0], group * G) >= 0;  // a token that was routed has a first slot
    float dot_w = 0.0f;
#pragma unroll
    for (int i = 0; i < kSlotTurns; ++i) {
      if (e[i] >= 0) dot_w = fmaf(w[i], gw[i], dot_w);
      if (i * G + G >= K) break;
    }
    dot_w = group_sum<G>(dot_w);
#pragma unroll
    for (int i = 0; i < kSlotTurns; ++i) {
      if (e[i] >= 0 && e[i] < E) part[place(e[i])] = w[i] * (gw[i] - (a.shape.normalize ? dot_w : 0.0f));
      if (i * G + G >= K) break;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = i < have && live ? exp_fast(v[i] - lse) : 0.0f;
    const bool rough = live && fabsf(lse) > kRoughLse;
    if (__any_sync(kFull, rough)) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) sum += v[i];
      sum = group_sum<G>(sum);
      const float inv = rough ? __fdividef(1.0f, sum) : 1.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] *= inv;
    }
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) dot = fmaf(c[i], v[i], dot);
    dot = group_sum<G>(dot);
    const float common = 2.0f * g1 * inv_n * lse - dot - (a.shape.normalize ? 0.0f : dot_w);
    __syncwarp();
    if (in) {
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        const float4 p = s_part[warp][i][lane];
        const float q[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
        for (int x = 0; x < 4; ++x) v[4 * i + x] = live ? fmaf(v[4 * i + x], c[4 * i + x] + common, q[x]) : 0.0f;
      }
      const int64_t at = t * a.ldg + e0;
      if (a.vec_grad && have == V) {
        if constexpr (F == kOutF32) {
#pragma unroll
          for (int i = 0; i < V / 4; ++i)
            store_out4<F>(static_cast<float*>(a.grad) + at + 4 * i,
                          make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
        } else {
#pragma unroll
          for (int i = 0; i < V / 8; ++i)
            *reinterpret_cast<uint4*>(static_cast<unsigned short*>(a.grad) + at + 8 * i) =
                make_uint4(pack2<F>(v[8 * i], v[8 * i + 1]), pack2<F>(v[8 * i + 2], v[8 * i + 3]),
                           pack2<F>(v[8 * i + 4], v[8 * i + 5]), pack2<F>(v[8 * i + 6], v[8 * i + 7]));
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i < have) store_out<F>(a.grad, at + i, v[i]);
      }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kSlotTurns; ++i) {
      if (e[i] >= 0 && e[i] < E) part[place(e[i])] = 0.0f;
      if (i * G + G >= K) break;
    }
    __syncwarp();
  }
}

// The lane layout for a number of experts: G lanes a token, V experts a lane.
template <typename Fn>
void with_layout(int experts, Fn f) {
  using std::integral_constant;
  if (experts <= 32) f(integral_constant<int, 4>(), integral_constant<int, 8>());
  else if (experts <= 64) f(integral_constant<int, 8>(), integral_constant<int, 8>());
  else if (experts <= 128) f(integral_constant<int, 16>(), integral_constant<int, 8>());
  else if (experts <= 256) f(integral_constant<int, 32>(), integral_constant<int, 8>());
  else if (experts <= 512) f(integral_constant<int, 32>(), integral_constant<int, 16>());
  else f(integral_constant<int, 32>(), integral_constant<int, 32>());
}

template <typename Fn>
void with_logits(int type, Fn f) {
  if (type == GG_OUTPUT_F32) f(std::integral_constant<int, kOutF32>());
  else if (type == GG_OUTPUT_F16) f(std::integral_constant<int, kOutF16>());
  else f(std::integral_constant<int, kOutBF16>());
}

int type_bytes(int type) { return type == GG_OUTPUT_F32 ? 4 : 2; }

// Rows of `ld` elements from `p` whose every element at a multiple of 8 is 16-byte aligned.
bool rows_aligned(const void* p, int64_t ld, int type) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * type_bytes(type)) % 16 == 0;
}

}  // namespace
}  // namespace gg

struct gg_router {
  gg_router_config config{};
  void* block = nullptr;
  gg::RouterWork work{};
  int device = 0;
};

extern "C" {

int gg_router_create(const gg_router_config* config, gg_router** out) {
  if (!out) return cudaErrorInvalidValue;
  *out = nullptr;
  if (!config) return cudaErrorInvalidValue;
  const gg_router_config& c = *config;
  if (c.experts < 1 || c.experts > GG_ROUTER_MAX_EXPERTS || c.top_k < 1 || c.top_k > GG_ROUTER_MAX_TOP_K ||
      c.capacity_tokens < 0 || static_cast<int64_t>(c.capacity_tokens) * c.top_k > GG_ROUTER_MAX_SLOTS ||
      (c.logit_type != GG_OUTPUT_F32 && c.logit_type != GG_OUTPUT_F16 && c.logit_type != GG_OUTPUT_BF16))
    return cudaErrorInvalidValue;
  gg_router* r = new (std::nothrow) gg_router();
  if (!r) return cudaErrorMemoryAllocation;
  r->config = c;
  size_t warps = 0;
  cudaError_t st = cudaGetDevice(&r->device);
  if (st != cudaSuccess) {
    delete r;
    return st;
  }
  gg::with_logits(c.logit_type, [&](auto f) {
    gg::with_layout(c.experts, [&](auto g, auto v) {
      constexpr int W = gg::router_warps(v());
      warps = W;
      // the most any router of this kernel takes: the attribute is the kernel's, not the router's
      st = cudaFuncSetAttribute(gg::router_forward_kernel<f(), g(), v(), W>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                gg::kForwardSmemMost);
    });
  });
  if (st == cudaSuccess)
    st = cudaFuncSetAttribute(gg::router_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, gg::kForwardSmemMost);
  if (st != cudaSuccess) {
    delete r;
    return st;
  }
  const size_t E = static_cast<size_t>(c.experts), B = gg::kMaxBlocks;
  const size_t words = B * warps * E + 2 * B * E + 2 * B;
  st = cudaMalloc(&r->block, words * 4);
  if (st != cudaSuccess) {
    delete r;
    return st;
  }
  r->work.warp_before = static_cast<int*>(r->block);
  r->work.block_count = r->work.warp_before + B * warps * E;
  r->work.block_prob = reinterpret_cast<float*>(r->work.block_count + B * E);
  r->work.block_z = r->work.block_prob + B * E;
  *out = r;
  return cudaSuccess;
}

int gg_router_run(gg_router* router, const gg_route* route, void* stream) {
  if (!router || !router->block) return cudaErrorInvalidDevicePointer;
  if (!route) return cudaErrorInvalidValue;
  const gg_router_config& c = router->config;
  const gg_route& q = *route;
  if (q.tokens < 0 || q.tokens > c.capacity_tokens || q.ld < c.experts || !q.rows || !q.losses) return cudaErrorInvalidValue;
  if (q.tokens > 0 && (!q.logits || !q.indices || !q.weights || !q.positions)) return cudaErrorInvalidValue;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t st = gg::expect_device(router->device);
  if (st != cudaSuccess) return st;
  gg::with_logits(c.logit_type, [&](auto f) {
    gg::with_layout(c.experts, [&](auto g, auto v) {
      constexpr int G = g(), V = v(), at_once = 32 / G;
      const auto launch = [&](auto warps_c) {
        constexpr int warps = warps_c();
        // One cluster of blocks, where it has room for the tokens: they exchange their counts behind a barrier of the
        // cluster, and the second launch falls away. Else as many blocks as there are SMs, tokens a warp in
        // whole turns.
        const int64_t turn = static_cast<int64_t>(warps) * at_once;
        int cluster = 0;
        if (warps == gg::kFewWarps && q.tokens <= gg::kClusterMost * turn)
          for (cluster = 1; cluster * turn < q.tokens;) cluster *= 2;
        const int64_t most = (cluster > 0 ? cluster : gg::kMaxBlocks) * turn;
        const int64_t per_warp = std::max<int64_t>(1, (q.tokens + most - 1) / most) * at_once;
        const int blocks = cluster > 0 ? cluster : static_cast<int>(std::max<int64_t>(1, (q.tokens + per_warp * warps - 1) / (per_warp * warps)));
        gg::ForwardArgs a{};
        a.logits = q.logits;
        a.mask = q.token_mask;
        a.indices = q.indices;
        a.weights = q.weights;
        a.lse = q.lse;
        a.ld = q.ld;
        a.vec = gg::rows_aligned(q.logits, q.ld, c.logit_type);
        a.place = {{c.experts, c.top_k, c.normalize != 0}, router->work, q.tokens, static_cast<int>(per_warp), blocks, cluster,
                   q.indices, q.positions, q.rows, q.row_tokens, q.prob_mean, q.losses};
        const size_t place = gg::place_smem(32 * warps, c.experts);
        const size_t forward = gg::forward_smem(G, warps, c.experts, c.top_k);
        st = gg::launch_chained(gg::router_forward_kernel<f(), G, V, warps>, dim3(blocks), 32 * warps,
                                cluster > 0 ? std::max(place, forward) : forward, s, cluster, a);
        if (st == cudaSuccess && cluster == 0)
          st = gg::launch_chained(gg::router_place_kernel, dim3(blocks + 1), 32 * warps, place, s, 1, a.place);
      };
      // Few tokens: small blocks, so that all SMs work on them (a full block's warps share one SM's issue slots), as
      // long as every warp has one turn (999 tokens of 37 experts, top 5: 8.5 us against 13.1 in full blocks; 4 tokens
      // of 64, top 2: 5.5 against 8.7).
      constexpr int kFew = V == 8 ? gg::kFewWarps : gg::router_warps(V);
      if (q.tokens <= static_cast<int64_t>(gg::kMaxBlocks) * kFew * at_once) launch(std::integral_constant<int, kFew>());
      else launch(std::integral_constant<int, gg::router_warps(V)>());
    });
  });
  return st;
}

int gg_router_backward(const gg_router* router, const gg_route_gradient* gradient, void* stream) {
  if (!router) return cudaErrorInvalidDevicePointer;
  if (!gradient) return cudaErrorInvalidValue;
  const gg_router_config& c = router->config;
  const gg_route_gradient& q = *gradient;
  if (q.tokens < 0 || q.tokens > c.capacity_tokens || q.ld < c.experts || q.ld_grad < c.experts) return cudaErrorInvalidValue;
  if (q.tokens == 0) return cudaSuccess;
  if (!q.logits || !q.indices || !q.weights || !q.rows || !q.losses || !q.lse || !q.grad_logits) return cudaErrorInvalidValue;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t st = gg::expect_device(router->device);
  if (st != cudaSuccess) return st;
  gg::with_logits(c.logit_type, [&](auto f) {
    gg::with_layout(c.experts, [&](auto g, auto v) {
      constexpr int G = g(), V = v();
      constexpr int warps = gg::kBackwardWarps, at_once = 32 / G;
      gg::BackwardArgs a{{c.experts, c.top_k, c.normalize != 0}, q.logits, q.indices, q.weights, q.rows, q.losses, q.lse,
                         q.grad_weights, q.grad_losses, q.grad_logits, q.tokens, q.ld, q.ld_grad,
                         gg::rows_aligned(q.logits, q.ld, c.logit_type),
                         gg::rows_aligned(q.grad_logits, q.ld_grad, c.logit_type)};
      const int64_t blocks = (static_cast<int64_t>(q.tokens) + warps * at_once - 1) / (warps * at_once);
      st = gg::launch_chained(gg::router_backward_kernel<f(), G, V>,
                              dim3(static_cast<unsigned>(std::min<int64_t>(blocks, gg::kBackwardBlocks * gg::kMaxBlocks))), 32 * warps, 0,
                              s, 1, a);
    });
  });
  return st;
}

void gg_router_destroy(gg_router* router) {
  if (!router) return;
  if (router->block) cudaFree(router->block);
  delete router;
}

}  // extern "C"
