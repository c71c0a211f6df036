// gg_gated.cu -- the gated feed-forward of experts, h = act(x Wg) * (x Wu), and its gradient, on packed rows whose counts are in
// device memory.
//
// Three products of one shape, a 128 x 256 tile from stages of 64 deep (kind::f16, FP32 sums in tensor memory, two
// accumulators so that one tile is taken out while the next is computed):
//   forward   columns 0-127 of a tile are x Wg and 128-255 x Wu for the same 128 inner columns, so h is made from
//             two columns of one lane and gate and up need not leave the SM;
//   rows      grad_x = grad_gate Wg^T + grad_up Wu^T is one sum along both matrices' inner size;
//   weights   grad_Wg and grad_Wu = x^T [grad_gate | grad_up], the forward's tile with the expert's rows as the inner
//             size. The last stage of an expert can hold rows of the next one: a warp of its own clears them in
//             shared memory (at most 15 rows: up to the next multiple of 16, the depth of a product) before that
//             stage is handed over.
// Each comes in two forms. On one CTA a tile takes 48 KB of operands for a stage of 64, which its shared memory both takes in and
// feeds to the tensor cores: 96 KB in 512 cycles of products at their full rate, and 128 bytes a cycle is what it has. On a
// pair (cta_group::2, 256 x 256) each CTA has 128 rows of the one operand and half of the other: 32 KB, six stages in
// place of four, and a third less from L2. Tiles of 256 rows leave more of an expert's last tile empty.
// Before the two gradients one pass over gate, up and grad_h makes grad_gate and grad_up.
//
// What bounds it: few rows, the weights from memory (16 rows on 8 experts of 2 x 14336 x 4096: 299 us, 6.3 TB/s of the 6.55 of a
// copy). Many rows, the tensor cores and then the card's power limit. 8192 rows on one expert of 4096 x 4096: 1.56 PFLOP/s in all three
// products. 8192 rows on 8 experts of 14336 x 4096 (1.92 TFLOP a product): forward 1400 us, 1.37 PFLOP/s, the pass before the
// gradients 210 us, 5.6 TB/s, rows 1530 us, 1.26 PFLOP/s, weights 1900 us, 1.0. The card is at its power limit, which does not explain the
// last: with 2048 rows on 2 experts of 4096 x 4096 its tensor pipe is 66 % busy, the others' 88 and 90, at about one clock (1.54 to 1.59 GHz);
// neither without its stores nor without its loads does it take less. Pairs against single CTAs, at 1024 rows an expert: forward 1430 us and
// 1520, rows 1590 and 1660; at 512 the same. Tile rows gone through 2, 4 or 8 at a time in place of 16: no less.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <memory>
#include <new>

#include "gg_expert_tiles.cuh"
#include "gg_internal.h"
#include "gg_launch.cuh"
#include "grouped_gemm_b200.h"

namespace gg {
namespace {

using namespace tiles;

constexpr int kForward = 0, kRowGradient = 1, kWeightGradient = 2;
constexpr int kClearWarp = 9;
constexpr int kBN = 256;       // columns of an accumulator
constexpr int kDepth = 64;     // values of k of a stage
constexpr int kAcc = 2;
template <bool kPair>
struct GatedShape {
  static constexpr int kStages = kPair ? 6 : 4;
  static constexpr int kStageBytes = kABytes + kBN / (kPair ? 2 : 1) * kRowBytes;
  static constexpr int kBars = 3 * kStages + 2 * kAcc + 1;
  static constexpr int kStretch = kPair ? 2 * kTileRows : kTileRows;  // rows of a tile
  static constexpr int smem(int experts) { return layout(kStages * kStageBytes, experts, kBars).bytes; }
  static_assert(layout(kStages * kStageBytes, kMaxExperts, kBars).bytes <= 232448, "shared memory of a block");
};
constexpr int kChunkBytes = kDepth * kRowBytes;  // 64 columns x 64 values of k, a row of shared memory for each k

struct GatedParams {
  CUtensorMap in[4];        // forward: x; rows: grad_gate, grad_up (each 128 rows, then boxes); weights: x, grad_gate, grad_up
  const CUtensorMap* maps;  // [experts][2]: Wg's and Wu's
  const int* rows;
  char* out[3];             // forward: h, gate, up (the last two may be NULL); rows: grad_x; weights: grad_Wg, grad_Wu
  int64_t pitch[3];         // bytes
  int64_t expert_bytes;     // weights: from one expert's gradient to the next
  int experts, inner, tiles_m, tiles_n, columns, out_rows, capacity, type, out_type, activation;
  // inner: forward k, rows n; tiles_m, out_rows: weights (k); columns: of the outputs
  bool aligned[3], wide[3];  // rows start on 16- and on 32-byte boundaries
  int* status;
  unsigned long long timeout_ns;
};

// Zeros in the rows `left` and on, up to the next multiple of 16, of kChunks pieces of shared memory that hold a 128-byte row of 64
// columns for each k. By one warp, between the loads' barrier and a proxy fence.
template <int kChunks>
__device__ __forceinline__ void clear_after(uint8_t* stage, int left, int lane) {
  const int first = left % kDepth, rows = 16 - first % 16;
  for (int i = lane; i < rows * kChunks * 8; i += 32)
    *reinterpret_cast<uint4*>(stage + i / (rows * 8) * kChunkBytes + (first + i / 8 % rows) * kRowBytes + i % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
}

template <int kMode, bool kPair>
__global__ void __launch_bounds__(kTileThreads, 1) gated_kernel(const __grid_constant__ GatedParams p) {
  using S = GatedShape<kPair>;
  constexpr int kStages = S::kStages, kStageBytes = S::kStageBytes;
  constexpr int kWidth = kMode == kRowGradient ? kBN : kBN / 2;  // output columns of a tile
  extern __shared__ uint8_t smem_dyn[];
  uint8_t* smem = smem_dyn + ((1024u - (ptx::smem_addr(smem_dyn) & 1023u)) & 1023u);
  const uint32_t sbase = ptx::smem_addr(smem);
  const Layout l = layout(kStages * kStageBytes, p.experts, S::kBars);
  int* first_row = reinterpret_cast<int*>(smem + l.table);
  int* first_tile = first_row + p.experts + 1;
  const uint32_t bar0 = sbase + l.bars;
  const auto full = [&](int s) { return bar0 + 8u * s; };
  const auto empty = [&](int s) { return bar0 + 8u * (kStages + s); };
  const auto ready = [&](int b) { return bar0 + 8u * (2 * kStages + b); };
  const auto taken = [&](int b) { return bar0 + 8u * (2 * kStages + kAcc + b); };
  const uint32_t drained = bar0 + 8u * (2 * kStages + 2 * kAcc);
  const auto cut = [&](int s) { return bar0 + 8u * (2 * kStages + 2 * kAcc + 1 + s); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + l.words);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + l.words + 4);
  // Stages that each loading warp has asked for. Who waits for a whole tile, or for several, waits as long as these go on.
  volatile uint32_t* progress = reinterpret_cast<volatile uint32_t*>(smem + l.words + 8);

  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
  const int rank = kPair ? static_cast<int>(ptx::cluster_ctarank()) : 0;
  if (threadIdx.x == 0) {
    // a pair's stages and accumulators are counted on the barriers of its first CTA
    for (int s = 0; s < kStages; ++s) ptx::mbar_init(full(s), kPair ? 2 : 1), ptx::mbar_init(empty(s), 1), ptx::mbar_init(cut(s), 1);
    for (int b = 0; b < kAcc; ++b) ptx::mbar_init(ready(b), 1), ptx::mbar_init(taken(b), (kPair ? 2 : 1) * kEpilogueWarps);
    ptx::mbar_init(drained, 1);
    *abort_flag = 0;
    progress[0] = progress[1] = 0;
    ptx::fence_mbar_init();
  }
  if constexpr (kPair) ptx::cluster_sync();  // the barriers are there before the other CTA uses them
  if (warp == kProductWarp) {
    if constexpr (kPair) {
      ptx::tmem_alloc_pair(ptx::smem_addr(tmem_slot), kAcc * kBN);
      ptx::tmem_relinquish_pair();
    } else {
      ptx::tmem_alloc(ptx::smem_addr(tmem_slot), kAcc * kBN);
      ptx::tmem_relinquish();
    }
  }
  if constexpr (kMode != kWeightGradient && !kPair) clear_rows<kStages, kStageBytes>(smem);
  chained_begin();
  if (warp == 0) expert_table<S::kStretch>(p.rows, p.experts, p.capacity, p.tiles_n, first_row, first_tile, p.status, lane);
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  const int grid = static_cast<int>(gridDim.x) / (kPair ? 2 : 1), block = static_cast<int>(blockIdx.x) / (kPair ? 2 : 1);
  const int per_expert = p.tiles_m * p.tiles_n;  // weights
  const bool bad = first_tile[p.experts] < 0;
  const int total = bad ? 0 : kMode == kWeightGradient ? p.experts * per_expert : first_tile[p.experts];

  struct Tile {
    int e, row, rows, m, n, depth;  // this CTA's first packed row and rows of the tile (weights: of the expert); stages of 64
  };
  const auto tile_at = [&](int t) {
    Tile x;
    if constexpr (kMode == kWeightGradient) {
      x.e = t / per_expert;
      place(t - x.e * per_expert, p.tiles_m, p.tiles_n, x.m, x.n);
      x.row = first_row[x.e];
      x.rows = first_row[x.e + 1] - x.row;
      x.depth = (x.rows + kDepth - 1) / kDepth;
    } else {
      x.e = expert_of(first_tile, p.experts, t);
      const int count = first_row[x.e + 1] - first_row[x.e];
      place(t - first_tile[x.e], stretches_of<S::kStretch>(count), p.tiles_n, x.m, x.n);
      x.row = first_row[x.e] + x.m * S::kStretch + rank * kTileRows;
      x.rows = min(kTileRows, count - x.m * S::kStretch - rank * kTileRows);  // none for the second CTA of a pair: not positive
      x.depth = (kMode == kRowGradient ? 2 : 1) * ((p.inner + kDepth - 1) / kDepth);
    }
    return x;
  };
  // Whether stage kb of a tile ends within 16 rows of k: what follows there is another expert's, or no row.
  const auto is_cut = [&](const Tile& x, int kb) { return kMode == kWeightGradient && kb + 1 == x.depth && x.rows % 16 != 0; };
  // the first of this CTA's 128 columns of A of the weights' gradient
  const auto first_k = [&](const Tile& x) { return x.m * S::kStretch + rank * kTileRows; };

  if (warp >= kLoadWarp) {
    const bool leader = ptx::elect_one();
    RowLoads<kStages> rows;
    Ring<kStages, 2> stage;
    stage.at = warp - kLoadWarp;
    int skip = stage.at;  // stages of 64 until this warp's next
    uint32_t asked = 0;
    bool ok = true;
    for (int t = block; ok && t < total; t += grid) {
      const Tile x = tile_at(t);
      const CUtensorMap* maps = p.maps + 2 * x.e;
      int kb = skip;
      for (; kb < x.depth; kb += 2) {
        ok = __all_sync(0xffffffffu, wait_phase_inline(empty(stage.at), stage.phase ^ 1u, abort_flag, p.status, p.timeout_ns, GG_STATUS_TIMEOUT_PRODUCER));
        if (!ok) break;
        const uint32_t a = sbase + static_cast<uint32_t>(stage.at * kStageBytes), b = a + kABytes;
        const uint32_t counted = kPair ? ptx::mapa_shared(full(stage.at), 0) : full(stage.at);
        const bool clear = is_cut(x, kb);  // handed over by the warp that clears it
        const uint32_t bar = clear ? cut(stage.at) : counted;
        const auto load = [&](uint32_t to, const CUtensorMap* map, int at, int row) {
          if (kPair && !clear) ptx::tma_load_2d_pair(to, map, bar, at, row);
          else ptx::tma_load_2d(to, map, bar, at, row);
        };
        const uint32_t bytes = kPair || kMode == kWeightGradient ? kStageBytes : rows.bytes(stage.at / 2, x.rows) + kBN * kRowBytes;
        if (leader) {
          if (clear || !kPair) ptx::mbar_arrive_expect_tx(bar, bytes);
          else if (rank == 0) ptx::mbar_arrive_expect_tx(full(stage.at), 2 * kStageBytes);
          if constexpr (kMode == kForward) {
            if constexpr (kPair) {
              load(a, &p.in[0], kb * kDepth, x.row);
#pragma unroll
              for (int i = 0; i < 2; ++i) load(b + i * kChunkBytes, maps + rank, x.n * kWidth + i * kDepth, kb * kDepth);
            } else {
              rows.load(&p.in[0], &p.in[1], a, bar, kb * kDepth, x.row, p.capacity);
#pragma unroll
              for (int i = 0; i < 4; ++i) load(b + i * kChunkBytes, maps + i / 2, x.n * kWidth + i % 2 * kDepth, kb * kDepth);
            }
          } else if constexpr (kMode == kRowGradient) {
            const int second = kb >= x.depth / 2, at = (second ? kb - x.depth / 2 : kb) * kDepth;
            if constexpr (kPair) {
              load(a, &p.in[2 * second], at, x.row);
              load(b, maps + second, at, x.n * kWidth + rank * kTileRows);
            } else {
              rows.load(&p.in[2 * second], &p.in[2 * second + 1], a, bar, at, x.row, p.capacity);
#pragma unroll
              for (int i = 0; i < 2; ++i) load(b + i * kTileRows * kRowBytes, maps + second, at, x.n * kWidth + i * kTileRows);
            }
          } else {
            const int at = x.row + kb * kDepth;
#pragma unroll
            for (int i = 0; i < 2; ++i) load(a + i * kChunkBytes, &p.in[0], first_k(x) + i * kDepth, at);
#pragma unroll
            for (int i = 0; i < (kPair ? 2 : 4); ++i)
              load(b + i * kChunkBytes, &p.in[1 + (kPair ? rank : i / 2)], x.n * kWidth + i % 2 * kDepth, at);
          }
          if (kPair && !clear && rank != 0) ptx::mbar_arrive_cluster_relaxed(counted);  // counts; the bytes are tracked by themselves
          progress[warp - kLoadWarp] = ++asked;
        }
        __syncwarp();
        stage.next();
      }
      skip = kb - x.depth;
    }
    if (rank == 0) drain_loads<kStages>(stage, full);
  } else if (kMode == kWeightGradient && warp == kClearWarp) {
    uint32_t it = 0, turns = 0;  // a bit for each stage: the parity of its next cut
    bool ok = true;
    for (int t = block; ok && t < total; t += grid) {
      const Tile x = tile_at(t);
      it += static_cast<uint32_t>(x.depth);
      if (x.depth == 0 || !is_cut(x, x.depth - 1)) continue;
      const int at = static_cast<int>((it - 1) % kStages);
      // through all the tiles without a cut before this one
      ok = __all_sync(0xffffffffu, wait_progress_inline(cut(at), turns >> at & 1u, abort_flag, p.status, p.timeout_ns, GG_STATUS_TIMEOUT_PRODUCER, progress));
      if (!ok) break;
      turns ^= 1u << at;
      clear_after<kStageBytes / kChunkBytes>(smem + at * kStageBytes, x.rows % kDepth, lane);
      ptx::fence_proxy_async_all();  // the tensor cores read it, on a pair the other CTA's too
      __syncwarp();
      if (lane == 0) {
        if (rank == 0) ptx::mbar_arrive(full(at));
        else ptx::mbar_arrive_cluster(ptx::mapa_shared(full(at), 0));
      }
    }
  } else if (warp == kProductWarp) {
    if (rank == 0) {
      // the forward's weights and all of the weights' gradient have k as their rows in shared memory
      constexpr bool kAWide = kMode == kWeightGradient, kBWide = kMode != kRowGradient;
      const bool leader = ptx::elect_one();
      const uint32_t idesc = ptx::idesc_f32acc(S::kStretch, kBN, static_cast<uint32_t>(p.type), kAWide, kBWide);
      // descriptors of a stage's operands: an address in units of 16 bytes in their low bits, so a stage and a step of K are additions
      constexpr uint32_t kStepA = (kAWide ? 2048 : 32) / 16, kStepB = (kBWide ? 2048 : 32) / 16;
      const uint64_t a0 = ptx::smem_desc_sw128(sbase, kAWide ? kChunkBytes : 16u, 1024u);
      const uint64_t b0 = ptx::smem_desc_sw128(sbase + kABytes, kBWide ? kChunkBytes : 16u, 1024u);
      Ring<kStages> stage;
      Ring<kAcc> acc;
      bool ok = true;
      for (int t = block; ok && t < total; t += grid) {
        const Tile x = tile_at(t);
        ok = __all_sync(0xffffffffu, wait_phase_inline<kPair>(taken(acc.at), acc.phase ^ 1u, abort_flag, p.status, p.timeout_ns, GG_STATUS_TIMEOUT_MMA));
        if (!ok) break;
        ptx::tc_fence_after_sync();
        const uint32_t d = tmem + static_cast<uint32_t>(acc.at * kBN);
        for (int kb = 0; kb < x.depth; ++kb) {
          ok = __all_sync(0xffffffffu, wait_phase_inline<kPair>(full(stage.at), stage.phase, abort_flag, p.status, p.timeout_ns, GG_STATUS_TIMEOUT_MMA));
          if (!ok) break;
          int steps = kDepth / 16;
          if constexpr (kMode == kWeightGradient) {
            const int left = x.rows - kb * kDepth;
            if (left < kDepth) steps = (left + 15) / 16;
          }
          ptx::tc_fence_after_sync();
          const uint64_t a = a0 + static_cast<uint32_t>(stage.at * (kStageBytes / 16)), b = b0 + static_cast<uint32_t>(stage.at * (kStageBytes / 16));
          if (leader) {
#pragma unroll
            for (uint32_t kk = 0; kk < kDepth / 16; ++kk)
              if (kMode != kWeightGradient || static_cast<int>(kk) < steps) {
                if constexpr (kPair) ptx::tc_mma_f16_pair(d, a + kStepA * kk, b + kStepB * kk, idesc, kb != 0 || kk != 0);
                else ptx::tc_mma_f16(d, a + kStepA * kk, b + kStepB * kk, idesc, kb != 0 || kk != 0);
              }
            if constexpr (kPair) ptx::tc_commit_pair_mc(empty(stage.at), 0x3);
            else ptx::tc_commit(empty(stage.at));
          }
          __syncwarp();
          stage.next();
        }
        if (!ok) break;
        if (leader) {
          if (x.depth > 0) {
            if constexpr (kPair) ptx::tc_commit_pair_mc(ready(acc.at), 0x3);
            else ptx::tc_commit(ready(acc.at));
          } else {  // an expert without rows: zeros
            ptx::mbar_arrive(ready(acc.at));
            if constexpr (kPair) ptx::mbar_arrive_cluster(ptx::mapa_shared(ready(acc.at), 1));
          }
        }
        __syncwarp();
        acc.next();
      }
      if (leader) {
        // before tensor memory is freed
        if constexpr (kPair) ptx::tc_commit_pair(drained);
        else ptx::tc_commit(drained);
        wait_drain_inline(drained, 0u, 100000000ull);
      }
      __syncwarp();
    }
  } else if (warp < kEpilogueWarps) {
    const int quarter = warp & 3, half = warp >> 2;
    unsigned char* stage = smem + l.staging + warp * kStagingBytes;
    uint32_t done = 0;
    for (int t = block; t < total; t += grid, ++done) {
      const Tile x = tile_at(t);
      const int buf = static_cast<int>(done % kAcc);
      if (!__all_sync(0xffffffffu, wait_progress_inline(ready(buf), (done / kAcc) & 1u, abort_flag, p.status, p.timeout_ns, GG_STATUS_TIMEOUT_EPILOGUE,
                                                        progress)))
        break;
      ptx::tc_fence_after_sync();
      const uint32_t from = tmem + static_cast<uint32_t>(buf * kBN) + (static_cast<uint32_t>(quarter * 32) << 16);
      const int rows = (kMode == kWeightGradient ? p.out_rows - first_k(x) : x.rows) - quarter * 32;  // from this warp's first on
      const int64_t row0 = (kMode == kWeightGradient ? first_k(x) : x.row) + quarter * 32;
      const auto out = [&](int i) {
        return Out{p.out[i] + row0 * p.pitch[i] + (kMode == kWeightGradient ? x.e * p.expert_bytes : 0), p.pitch[i], min(32, rows), p.columns,
                   p.aligned[i], p.wide[i]};
      };
      if (rows > 0) {
        if constexpr (kMode == kForward) {
#pragma unroll 1
          for (int c = half * 64; c < half * 64 + 64; c += 32) {
            uint32_t g[32], u[32];
            tmem_read(from + c, g);
            tmem_read(from + 128 + c, u);
            const int column = x.n * kWidth + c;
            float v[32];
            if (p.out[1]) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(g[j]);
              store_columns(stage, lane, v, p.out_type, out(1), column);
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(u[j]);
              store_columns(stage, lane, v, p.out_type, out(2), column);
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(g[j]);
            activate_all(v, p.activation);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] *= __uint_as_float(u[j]);
            store_columns(stage, lane, v, p.out_type, out(0), column);
          }
        } else {
          // half a tile: 128 columns of grad_x, or grad_Wg's (half 0) or grad_Wu's (half 1)
          const Out o = out(kMode == kWeightGradient ? half : 0);
#pragma unroll 1
          for (int c = 0; c < 128; c += 32) {
            uint32_t r[32];
            float v[32];
            if (kMode == kWeightGradient && x.depth == 0) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = 0.0f;
            } else {
              tmem_read(from + half * 128 + c, r);
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
            }
            store_columns(stage, lane, v, p.out_type, o, x.n * kWidth + (kMode == kWeightGradient ? 0 : half * 128) + c);
          }
        }
      }
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if (rank == 0) ptx::mbar_arrive(taken(buf));
        else ptx::mbar_arrive_cluster(ptx::mapa_shared(taken(buf), 0));
      }
    }
  }

  if constexpr (kPair) {
    __syncwarp();
    ptx::cluster_sync();  // neither CTA ends while the other may still use its shared memory
  } else {
    __syncthreads();
  }
  if (*abort_flag) {  // after an abort, loads may still be landing
    const uint64_t t0 = ptx::global_timer_ns();
    while (ptx::global_timer_ns() - t0 < 200000ull) {
    }
  }
  if (warp == kProductWarp) {
    ptx::tc_fence_after_sync();
    if constexpr (kPair) ptx::tmem_dealloc_pair(tmem, kAcc * kBN);
    else ptx::tmem_dealloc(tmem, kAcc * kBN);
  }
}

// act'(x) and act(x), with the forward pass's exponential and division.
__device__ __forceinline__ void slope_of(float x, int act, float& slope, float& value) {
  if (act == GG_ACT_SILU) {
    const float s = over_logistic(1.0f, x);
    value = x * s;
    slope = s * fmaf(x, 1.0f - s, 1.0f);
  } else if (act == GG_ACT_GELU) {
    // x s(z) with s the logistic function: its derivative is s + x s (1 - s) z'. Far out s is 0 or 1 and the second term 0, while z'
    // leaves FP32 (past |x| = 5e19).
    const float s = over_logistic(1.0f, gelu_exponent(x)), bend = x * s * (1.0f - s);
    value = x * s;
    slope = bend == 0.0f ? s : fmaf(bend, 1.5957691216057308f * fmaf(3.0f * 0.044715f * x, x, 1.0f), s);
  } else if (act == GG_ACT_RELU) {
    value = fmaxf(x, 0.0f);
    slope = x > 0.0f ? 1.0f : 0.0f;
  } else {
    value = x;
    slope = 1.0f;
  }
}

struct GateGradientParams {
  const void* gate;
  const void* up;
  const void* grad_h;
  void* grad_gate;
  void* grad_up;
  const int* rows;
  int64_t ldg, ldgh, ldgg;
  int experts, n, capacity, activation;
  int* status;
};

constexpr int kGateThreads = 256;

// grad_gate and grad_up of the rows that are there: eight columns a thread and step.
template <int F, bool kVec>
__global__ void __launch_bounds__(kGateThreads) gate_gradient_kernel(const GateGradientParams p) {
  __shared__ long long s_rows;
  __shared__ int s_bad;
  if (threadIdx.x == 0) s_rows = p.rows ? 0 : p.capacity, s_bad = 0;
  chained_begin();
  __syncthreads();
  if (p.rows) {  // their sum
    long long sum = 0;
    bool bad = false;
    for (int e = threadIdx.x; e < p.experts; e += kGateThreads) {
      const int r = p.rows[e];
      bad = bad || r < 0;
      sum += r;
    }
    atomicAdd(reinterpret_cast<unsigned long long*>(&s_rows), static_cast<unsigned long long>(sum));
    if (bad) s_bad = 1;
  }
  __syncthreads();
  if (s_bad || s_rows > p.capacity) {
    if (blockIdx.x == 0 && threadIdx.x == 0) atomicOr(p.status, GG_STATUS_BAD_ROWS);
    return;
  }
  const int per_row = (p.n + 7) / 8;
  const int64_t pieces = s_rows * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kGateThreads + threadIdx.x; i < pieces; i += static_cast<int64_t>(gridDim.x) * kGateThreads) {
    const int64_t r = i / per_row;
    const int c = static_cast<int>(i % per_row) * 8;
    const unsigned short* gate = static_cast<const unsigned short*>(p.gate) + r * p.ldg + c;
    const unsigned short* up = static_cast<const unsigned short*>(p.up) + r * p.ldg + c;
    const unsigned short* gh = static_cast<const unsigned short*>(p.grad_h) + r * p.ldgh + c;
    unsigned short* gg = static_cast<unsigned short*>(p.grad_gate) + r * p.ldgg + c;
    unsigned short* gu = static_cast<unsigned short*>(p.grad_up) + r * p.ldgg + c;
    if (kVec && c + 8 <= p.n) {
      const uint4 a = *reinterpret_cast<const uint4*>(gate), b = *reinterpret_cast<const uint4*>(up), d = *reinterpret_cast<const uint4*>(gh);
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w}, dw[4] = {d.x, d.y, d.z, d.w};
      uint32_t gw[4], uw[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = unpack2<F>(aw[j]), u = unpack2<F>(bw[j]), g = unpack2<F>(dw[j]);
        float s0, v0, s1, v1;
        slope_of(x.x, p.activation, s0, v0);
        slope_of(x.y, p.activation, s1, v1);
        gw[j] = pack2<F>(g.x * u.x * s0, g.y * u.y * s1);
        uw[j] = pack2<F>(g.x * v0, g.y * v1);
      }
      *reinterpret_cast<uint4*>(gg) = make_uint4(gw[0], gw[1], gw[2], gw[3]);
      *reinterpret_cast<uint4*>(gu) = make_uint4(uw[0], uw[1], uw[2], uw[3]);
    } else {
      for (int j = 0; j < 8 && c + j < p.n; ++j) {
        const float x = widen16<F>(gate[j]), u = widen16<F>(up[j]), g = widen16<F>(gh[j]);
        float s, v;
        slope_of(x, p.activation, s, v);
        store_out<F>(gg, j, g * u * s);
        store_out<F>(gu, j, g * v);
      }
    }
  }
}

bool on(int bytes, const void* p, int64_t pitch) { return reinterpret_cast<uintptr_t>(p) % bytes == 0 && pitch % bytes == 0; }
bool on16(const void* p, int64_t pitch) { return on(16, p, pitch); }

}  // namespace
}  // namespace gg

struct gg_gated_plan {
  gg_gated_problem problem{};
  unsigned char* block = nullptr;        // maps forward | maps rows | status
  const CUtensorMap* maps[2] = {};
  int* status = nullptr;
  int device = 0, sms = 0;
  int pairs = 0;  // that the GPU holds at a time
};

namespace {

constexpr int kPairRows = 512;     // rows of an expert that the capacity has, in the mean, from which on its tiles are of 256
constexpr int kPairColumns = 256;  // k from which on the weights' gradients' are

gg::GatedParams common(const gg_gated_plan* plan, const int* rows, int capacity) {
  gg::GatedParams p{};
  p.rows = rows;
  p.experts = plan->problem.experts;
  p.capacity = capacity;
  p.type = plan->problem.type;
  p.out_type = plan->problem.type == GG_INPUT_F16 ? GG_OUTPUT_F16 : GG_OUTPUT_BF16;
  p.activation = plan->problem.activation;
  p.status = plan->status;
  p.timeout_ns = gg::wait_limit_ns();
  return p;
}

void set_out(gg::GatedParams& p, int i, void* out, int ld, int bytes) {
  p.out[i] = static_cast<char*>(out);
  p.pitch[i] = static_cast<int64_t>(ld) * bytes;
  p.aligned[i] = gg::on(16, out, p.pitch[i]);
  p.wide[i] = gg::on(32, out, p.pitch[i]);
}

// The kernel of one form: `most` tiles at most.
template <int kMode, bool kPair>
cudaError_t launch(const gg_gated_plan* plan, const gg::GatedParams& p, int64_t most, cudaStream_t stream) {
  const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(kPair ? plan->pairs : plan->sms, most)) * (kPair ? 2 : 1);
  return gg::launch_chained(gg::gated_kernel<kMode, kPair>, dim3(static_cast<unsigned>(grid)), gg::tiles::kTileThreads,
                            static_cast<size_t>(gg::GatedShape<kPair>::smem(p.experts)), stream, kPair ? 2 : 1, p);
}

template <int kMode, bool kPair>
cudaError_t prepare(gg_gated_plan* plan) {
  const int smem = gg::GatedShape<kPair>::smem(gg::tiles::kMaxExperts);
  cudaError_t st = cudaFuncSetAttribute(gg::gated_kernel<kMode, kPair>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (!kPair || st != cudaSuccess) return st;
  return gg::resident_pairs(gg::gated_kernel<kMode, kPair>, gg::tiles::kTileThreads, static_cast<size_t>(smem), &plan->pairs);
}

// The maps of packed rows for RowLoads: whole tiles and boxes.
bool encode_both(CUtensorMap* maps, int type, const void* rows, int columns, int count, int ld) {
  const int kind = type == GG_INPUT_F16 ? 2 : 3;
  return gg::encode_rows(&maps[0], kind, rows, columns, count, static_cast<int64_t>(ld) * 2, gg::kDepth, gg::tiles::kTileRows) &&
         gg::encode_rows(&maps[1], kind, rows, columns, count, static_cast<int64_t>(ld) * 2, gg::kDepth, gg::tiles::kBoxRows);
}

// Tile rows (128 or 256 of an expert) of all experts at most.
int64_t stretches(const gg_gated_plan* plan, int capacity, bool pair) {
  return std::min<int64_t>(capacity, static_cast<int64_t>(capacity) / (pair ? 256 : 128) + plan->problem.experts);
}

// Whether tiles of 256 rows on pairs of CTAs take the rows, or of 128.
bool rows_in_pairs(const gg_gated_plan* plan, int capacity) { return capacity / plan->problem.experts >= kPairRows; }

}  // namespace

extern "C" {

int gg_gated_plan_create(const gg_gated_problem* problem, gg_gated_plan** out) {
  if (!out) return cudaErrorInvalidValue;
  *out = nullptr;
  if (!problem) return cudaErrorInvalidValue;
  const gg_gated_problem& q = *problem;
  const auto off16 = [](const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 != 0; };
  if (q.experts < 1 || q.experts > GG_GATED_MAX_EXPERTS || q.n < 1 || q.n > gg::tiles::kMostSize || q.k < 1 || q.k > gg::tiles::kMostSize || q.ldw < q.n || q.ldw % 8 != 0 || !q.gate || !q.up ||
      (q.type != GG_INPUT_F16 && q.type != GG_INPUT_BF16) || q.activation < GG_ACT_NONE || q.activation > GG_ACT_SILU)
    return cudaErrorInvalidValue;
  for (int e = 0; e < q.experts; ++e)
    if (!q.gate[e] || !q.up[e] || off16(q.gate[e]) || off16(q.up[e])) return cudaErrorInvalidValue;

  gg_gated_plan* plan = new (std::nothrow) gg_gated_plan();
  if (!plan) return cudaErrorMemoryAllocation;
  const size_t E = static_cast<size_t>(q.experts), map_bytes = 2 * E * sizeof(CUtensorMap), status_at = 2 * map_bytes;
  const size_t host_bytes = status_at + sizeof(int);
  // aligned as tensor maps want it
  const std::unique_ptr<CUtensorMap[]> host(new (std::nothrow) CUtensorMap[(host_bytes - 1) / sizeof(CUtensorMap) + 1]());
  if (!host) {
    delete plan;
    return cudaErrorMemoryAllocation;
  }
  CUtensorMap* forward = host.get();
  CUtensorMap* rows = forward + 2 * E;
  const int kind = q.type == GG_INPUT_F16 ? 2 : 3;
  const int64_t pitch = static_cast<int64_t>(q.ldw) * 2;
  cudaError_t st = cudaGetDevice(&plan->device);
  if (st == cudaSuccess) st = cudaDeviceGetAttribute(&plan->sms, cudaDevAttrMultiProcessorCount, plan->device);
  for (int e = 0; e < q.experts && st == cudaSuccess; ++e)
    for (int i = 0; i < 2 && st == cudaSuccess; ++i) {
      const void* w = i == 0 ? q.gate[e] : q.up[e];
      if (!gg::encode_rows(&forward[2 * e + i], kind, w, q.n, q.k, pitch, 64, gg::kDepth) ||
          !gg::encode_rows(&rows[2 * e + i], kind, w, q.n, q.k, pitch, gg::kDepth, gg::tiles::kTileRows))
        st = cudaErrorInvalidValue;
    }
  if (st == cudaSuccess) st = prepare<gg::kForward, false>(plan);
  if (st == cudaSuccess) st = prepare<gg::kRowGradient, false>(plan);
  if (st == cudaSuccess) st = prepare<gg::kWeightGradient, false>(plan);
  if (st == cudaSuccess) st = prepare<gg::kForward, true>(plan);
  if (st == cudaSuccess) st = prepare<gg::kRowGradient, true>(plan);
  if (st == cudaSuccess) st = prepare<gg::kWeightGradient, true>(plan);
  if (st == cudaSuccess) st = cudaMalloc(reinterpret_cast<void**>(&plan->block), host_bytes);
  if (st == cudaSuccess) st = cudaMemcpy(plan->block, host.get(), host_bytes, cudaMemcpyHostToDevice);
  if (st == cudaSuccess) st = cudaDeviceSynchronize();
  if (st != cudaSuccess) {
    if (plan->block) cudaFree(plan->block);
    delete plan;
    return st;
  }
  plan->problem = q;
  plan->maps[0] = reinterpret_cast<const CUtensorMap*>(plan->block);
  plan->maps[1] = plan->maps[0] + 2 * E;
  plan->status = reinterpret_cast<int*>(plan->block + status_at);
  *out = plan;
  return cudaSuccess;
}

int gg_gated_plan_run(gg_gated_plan* plan, const gg_gated* call, void* stream) {
  if (!plan || !plan->block) return cudaErrorInvalidDevicePointer;
  const gg_gated_problem& q = plan->problem;
  if (!call || call->capacity_rows < 0 || call->capacity_rows > gg::tiles::kMostRows || (!call->rows && q.experts != 1)) return cudaErrorInvalidValue;
  const gg_gated& c = *call;
  if (c.capacity_rows == 0 && !c.rows) return cudaSuccess;
  if (c.capacity_rows > 0 && (!c.x || !c.h || c.ldx < q.k || !gg::on16(c.x, static_cast<int64_t>(c.ldx) * 2) || c.ldh < q.n ||
                              (!c.gate != !c.up) || (c.gate && c.ldg < q.n)))
    return cudaErrorInvalidValue;
  cudaError_t st = gg::expect_device(plan->device);
  if (st != cudaSuccess) return st;
  gg::GatedParams p = common(plan, c.rows, c.capacity_rows);
  p.maps = plan->maps[0];
  p.inner = q.k;
  p.columns = q.n;
  p.tiles_n = (q.n - 1) / 128 + 1;
  set_out(p, 0, c.h, c.ldh, 2);
  set_out(p, 1, c.gate, c.ldg, 2);
  set_out(p, 2, c.up, c.ldg, 2);
  if (c.capacity_rows > 0 && !encode_both(&p.in[0], q.type, c.x, q.k, c.capacity_rows, c.ldx)) return cudaErrorInvalidValue;
  const bool pair = rows_in_pairs(plan, c.capacity_rows);
  const int64_t most = stretches(plan, c.capacity_rows, pair) * p.tiles_n;
  if (most > gg::tiles::kMostTiles) return cudaErrorInvalidValue;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return pair ? launch<gg::kForward, true>(plan, p, most, s) : launch<gg::kForward, false>(plan, p, most, s);
}

int gg_gated_plan_backward(gg_gated_plan* plan, const gg_gated_gradient* gradient, void* stream) {
  if (!plan || !plan->block) return cudaErrorInvalidDevicePointer;
  const gg_gated_problem& q = plan->problem;
  if (!gradient || gradient->capacity_rows < 0 || gradient->capacity_rows > gg::tiles::kMostRows || (!gradient->rows && q.experts != 1)) return cudaErrorInvalidValue;
  const gg_gated_gradient& c = *gradient;
  const int type16 = q.type == GG_INPUT_F16 ? GG_OUTPUT_F16 : GG_OUTPUT_BF16;
  if ((!c.grad_wg != !c.grad_wu) || (c.grad_wg && ((c.weight_grad_type != GG_OUTPUT_F32 && c.weight_grad_type != type16) || c.ldgw < q.n ||
                                                   (q.experts > 1 && c.expert_stride < static_cast<int64_t>(q.k - 1) * c.ldgw + q.n))))
    return cudaErrorInvalidValue;
  if (c.capacity_rows > 0 &&
      (!c.gate || !c.up || !c.grad_h || !c.grad_gate || !c.grad_up || c.ldg < q.n || c.ldgh < q.n || c.ldgg < q.n ||
       !gg::on16(c.grad_gate, static_cast<int64_t>(c.ldgg) * 2) || !gg::on16(c.grad_up, static_cast<int64_t>(c.ldgg) * 2) ||
       (c.grad_x && c.ldgx < q.k) || (c.grad_wg && (!c.x || c.ldx < q.k || !gg::on16(c.x, static_cast<int64_t>(c.ldx) * 2)))))
    return cudaErrorInvalidValue;
  cudaError_t st = gg::expect_device(plan->device);
  if (st != cudaSuccess) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int kind = q.type == GG_INPUT_F16 ? 2 : 3;
  const int64_t pitch_g = static_cast<int64_t>(c.ldgg) * 2;
  const bool pair_x = rows_in_pairs(plan, c.capacity_rows), pair_w = q.k >= kPairColumns;
  // nothing is launched before every check has passed
  gg::GatedParams px = common(plan, c.rows, c.capacity_rows), pw = px;
  if (c.capacity_rows > 0 && c.grad_x) {
    px.maps = plan->maps[1];
    px.inner = q.n;
    px.columns = q.k;
    px.tiles_n = (q.k - 1) / gg::kBN + 1;
    set_out(px, 0, c.grad_x, c.ldgx, 2);
    if (!encode_both(&px.in[0], q.type, c.grad_gate, q.n, c.capacity_rows, c.ldgg) ||
        !encode_both(&px.in[2], q.type, c.grad_up, q.n, c.capacity_rows, c.ldgg))
      return cudaErrorInvalidValue;
  }
  if (c.grad_wg) {
    const int bytes = c.weight_grad_type == GG_OUTPUT_F32 ? 4 : 2;
    pw.maps = plan->maps[0];
    pw.columns = q.n;
    pw.out_rows = q.k;
    pw.tiles_m = (q.k - 1) / (pair_w ? 256 : 128) + 1;
    pw.tiles_n = (q.n - 1) / 128 + 1;
    pw.out_type = c.weight_grad_type;
    set_out(pw, 0, c.grad_wg, c.ldgw, bytes);
    set_out(pw, 1, c.grad_wu, c.ldgw, bytes);
    pw.expert_bytes = c.expert_stride * bytes;
    for (int i = 0; i < 2; ++i) {
      pw.aligned[i] = pw.aligned[i] && (q.experts == 1 || pw.expert_bytes % 16 == 0);
      pw.wide[i] = pw.wide[i] && (q.experts == 1 || pw.expert_bytes % 32 == 0);
    }
    if (c.capacity_rows > 0 &&
        (!gg::encode_rows(&pw.in[0], kind, c.x, q.k, c.capacity_rows, static_cast<int64_t>(c.ldx) * 2, 64, gg::kDepth) ||
         !gg::encode_rows(&pw.in[1], kind, c.grad_gate, q.n, c.capacity_rows, pitch_g, 64, gg::kDepth) ||
         !gg::encode_rows(&pw.in[2], kind, c.grad_up, q.n, c.capacity_rows, pitch_g, 64, gg::kDepth)))
      return cudaErrorInvalidValue;
  }
  const int64_t most_x = px.maps ? stretches(plan, c.capacity_rows, pair_x) * px.tiles_n : 0;
  const int64_t most_w = pw.maps ? static_cast<int64_t>(q.experts) * pw.tiles_m * pw.tiles_n : 0;
  if (most_x > gg::tiles::kMostTiles || most_w > gg::tiles::kMostTiles) return cudaErrorInvalidValue;

  if (c.capacity_rows > 0 || c.rows) {  // without room for rows: for the counts' check
    gg::GateGradientParams g{c.gate, c.up, c.grad_h, c.grad_gate, c.grad_up, c.rows, c.ldg, c.ldgh, c.ldgg, q.experts, q.n, c.capacity_rows, q.activation, plan->status};
    const bool vec = gg::on16(c.gate, static_cast<int64_t>(c.ldg) * 2) && gg::on16(c.up, static_cast<int64_t>(c.ldg) * 2) &&
                     gg::on16(c.grad_h, static_cast<int64_t>(c.ldgh) * 2);
    const int64_t want = (static_cast<int64_t>(c.capacity_rows) * ((q.n + 7) / 8) + gg::kGateThreads - 1) / gg::kGateThreads;
    const dim3 grid(static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(want, static_cast<int64_t>(plan->sms) * 8))));
    const auto go = [&](auto kernel) { st = gg::launch_chained(kernel, grid, gg::kGateThreads, 0, s, 1, g); };
    if (kind == 2) vec ? go(gg::gate_gradient_kernel<gg::kOutF16, true>) : go(gg::gate_gradient_kernel<gg::kOutF16, false>);
    else vec ? go(gg::gate_gradient_kernel<gg::kOutBF16, true>) : go(gg::gate_gradient_kernel<gg::kOutBF16, false>);
  }
  if (st == cudaSuccess && px.maps)
    st = pair_x ? launch<gg::kRowGradient, true>(plan, px, most_x, s) : launch<gg::kRowGradient, false>(plan, px, most_x, s);
  if (st == cudaSuccess && pw.maps)
    st = pair_w ? launch<gg::kWeightGradient, true>(plan, pw, most_w, s) : launch<gg::kWeightGradient, false>(plan, pw, most_w, s);
  return st;
}

int gg_gated_plan_status(gg_gated_plan* plan, int* status) {
  if (!plan || !plan->block) return cudaErrorInvalidDevicePointer;
  if (!status) return cudaErrorInvalidValue;
  cudaError_t st = gg::expect_device(plan->device);
  if (st == cudaSuccess) st = cudaDeviceSynchronize();
  if (st == cudaSuccess) st = cudaMemcpy(status, plan->status, sizeof(int), cudaMemcpyDeviceToHost);
  if (st != cudaSuccess) return st;
  return cudaMemset(plan->status, 0, sizeof(int));
}

void gg_gated_plan_destroy(gg_gated_plan* plan) {
  if (!plan) return;
  if (plan->block) cudaFree(plan->block);
  delete plan;
}

}  // extern "C"
