// gg_f8.cu -- rows in 8 bits against expert weights in 8 bits, with a scale for each row and 128 values of k on the one
// side and for each block of 128 outputs x 128 values of k on the other:
//   G(r, o) = sum over b of sa(r, b) * sb(o / 128, b) * P_b(r, o),   P_b(r, o) = sum over k in block b of A(r, k) * B(o, k)
//   D = act(G + bias), or act(G) * U with a second matrix of weights.
//
// tcgen05 (kind::f8f6f4) computes P_b of a 128 x BN tile into tensor memory, a new accumulator for each b: one stage of
// shared memory is one b (128 bytes a row), four products of K = 32. The scales are FP32 numbers, so they cannot be left to
// the scaled form of the instruction, whose scales are powers of two: eight warps read each P_b back and add it, times its scale, to
// sums in their registers, BN / 2 a thread, two at a time (fma.rn.f32x2). Meanwhile the tensor cores work on the next b.
//
// What bounds it: few rows an expert, the weights from memory (64 rows on 8 experts of 4096 x 14336: 86 us, 5.5 TB/s of the 6.55 of a
// copy; gated, of two 14336 x 4096: 182 us, 5.2; one row on one
// expert: 33 us, 128 tiles of 32 outputs, each with 112 blocks of k one after another). Many rows,
// the way of each accumulator: 128 x 256 sums leave tensor memory for every 512 cycles' products, and its 512 columns
// hold two of them, so that the products of the next but one wait for the sums' way out (the tensor pipe is 46 % busy with 4096 rows on 8
// experts of 4096 x 4096, 92 us). 16384 rows on 64 experts, 14336 x 4096: 1345 us, 1.43 PFLOP/s; 16 experts of 1024 rows each 1044 us, 1.84; 4096 rows
// on 8 experts, gated, into 8 bits: 520 us, 1.85, where the product alone would be 2.8 (3.3 at full clock). Calls back to back are slowed by the card's power limit: 1610 us.
// Tried and slower: pairs of CTAs (2470 us: the sums' release crosses to the other CTA for every block), sums kept in tensor memory
// (2280). No difference: other boxes, element types and L2 promotions of the loads, a k of its own to start with for each CTA.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <memory>
#include <new>
#include <type_traits>

#include "gg_expert_tiles.cuh"
#include "gg_internal.h"
#include "gg_launch.cuh"
#include "gg_scale8.cuh"
#include "grouped_gemm_b200.h"

namespace gg {
namespace {

using namespace tiles;

// Scales in shared memory, brought there by a warp of its own (a row's lie in a line of their own, which can be as far as L2 or
// DRAM: read by the warps that use them, a kblock waits for them): kScaleSlots slots of kScaleBlocks blocks of k, each the tile's
// 128 rows' and two of the weights', kScaleSlots + 2 slots ahead.
constexpr int kScaleWarp = 9;
constexpr int kScaleBlocks = 4;
constexpr int kScaleSlots = 3;
constexpr int kScaleBytes = kScaleBlocks * (kTileRows + 2) * 4 + 16;  // and which tile they are of

struct F8Params {
  CUtensorMap a_map, a_box;     // 128 rows, and kBoxRows, x 128 bytes
  const CUtensorMap* maps;      // [experts][2]: the weights', boxes of a tile's outputs x 128 bytes
  const float* const* b_scales; // [experts]
  const float* const* up_scales;
  const float* const* bias;     // NULL: none
  const float* a_scales;
  const int* rows;
  char* d;
  float* d_scales;
  int64_t d_pitch, ldas, ldds;  // d_pitch in bytes
  int experts, n, k_blocks, tiles_n, capacity, input_format, output_type, activation;
  bool aligned, wide;   // D's rows start on 16- and on 32-byte boundaries
  bool scales_aligned;  // A's scales' rows start on 16-byte boundaries
  int* status;
  unsigned long long timeout_ns;
};

template <int BN>
struct F8Shape {
  static constexpr int kStageBytes = kABytes + BN * kRowBytes;
  static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 6 : 8;  // even: each loading warp has its own
  static constexpr int kAccumulators = BN == 256 ? 2 : 4;
  static constexpr int kTmemColumns = kAccumulators * BN;
  static constexpr int kBars = 2 * kStages + 2 * kAccumulators + 4 + 2 * kScaleSlots + 1;
  static_assert(kStages % 2 == 0 && kTmemColumns >= 32 && kTmemColumns <= 512);
  static_assert(layout(kStages * kStageBytes, kMaxExperts, kBars, kScaleSlots * kScaleBytes).bytes + 2048 <= 232448, "shared memory of a block");
};

// acc += p * s for two values.
__device__ __forceinline__ void fma2(uint64_t& acc, uint32_t p0, uint32_t p1, uint64_t s) {
  asm("{\n\t.reg .b64 p;\n\tmov.b64 p, {%1, %2};\n\tfma.rn.f32x2 %0, p, %3, %0;\n\t}" : "+l"(acc) : "r"(p0), "r"(p1), "l"(s));
}
__device__ __forceinline__ float half_of(uint64_t v, int i) { return __uint_as_float(static_cast<uint32_t>(v >> (32 * i))); }
__device__ __forceinline__ uint64_t twice(float s) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %1};" : "=l"(v) : "r"(__float_as_uint(s)));
  return v;
}

template <int BN, bool kGated>
__global__ void __launch_bounds__(kTileThreads, 1) f8_kernel(const __grid_constant__ F8Params p) {
  using S = F8Shape<BN>;
  constexpr int kStages = S::kStages, kAcc = S::kAccumulators;
  constexpr int kWidth = kGated ? BN / 2 : BN;  // outputs of a tile
  constexpr int kMine = kWidth / 2;             // outputs of an epilogue warp

  extern __shared__ uint8_t smem_dyn[];
  uint8_t* smem = smem_dyn + ((1024u - (ptx::smem_addr(smem_dyn) & 1023u)) & 1023u);
  const uint32_t sbase = ptx::smem_addr(smem);
  const Layout l = layout(kStages * S::kStageBytes, p.experts, S::kBars, kScaleSlots * kScaleBytes);
  int* first_row = reinterpret_cast<int*>(smem + l.table);
  int* first_tile = first_row + p.experts + 1;
  const uint32_t bar0 = sbase + l.bars;
  const auto full = [&](int s) { return bar0 + 8u * s; };
  const auto empty = [&](int s) { return bar0 + 8u * (kStages + s); };
  const auto ready = [&](int b) { return bar0 + 8u * (2 * kStages + b); };
  const auto taken = [&](int b) { return bar0 + 8u * (2 * kStages + kAcc + b); };
  const auto pair = [&](int q) { return bar0 + 8u * (2 * kStages + 2 * kAcc + q); };
  const auto scales_in = [&](uint32_t i) { return bar0 + 8u * (2 * kStages + 2 * kAcc + 4 + i); };
  const auto scales_used = [&](uint32_t i) { return bar0 + 8u * (2 * kStages + 2 * kAcc + 4 + kScaleSlots + i); };
  const uint32_t drained = bar0 + 8u * (2 * kStages + 2 * kAcc + 4 + 2 * kScaleSlots);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + l.words);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + l.words + 4);
  __shared__ float top[2][2][kTileRows];  // largest magnitudes of the 8-bit output: [tile parity][half][row]

  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) ptx::mbar_init(full(s), 1), ptx::mbar_init(empty(s), 1);
    for (int b = 0; b < kAcc; ++b) ptx::mbar_init(ready(b), 1), ptx::mbar_init(taken(b), kEpilogueWarps);
    for (int q = 0; q < 4; ++q) ptx::mbar_init(pair(q), 2);
    for (uint32_t i = 0; i < kScaleSlots; ++i) ptx::mbar_init(scales_in(i), 1), ptx::mbar_init(scales_used(i), kEpilogueWarps);
    ptx::mbar_init(drained, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == kProductWarp) {
    ptx::tmem_alloc(ptx::smem_addr(tmem_slot), S::kTmemColumns);
    ptx::tmem_relinquish();
  }
  clear_rows<kStages, S::kStageBytes>(smem);
  chained_begin();
  if (warp == 0) expert_table(p.rows, p.experts, p.capacity, p.tiles_n, first_row, first_tile, p.status, lane);
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  const int total = first_tile[p.experts], grid = static_cast<int>(gridDim.x);

  // What every role knows of tile t: its expert, first packed row, rows there, and place along the outputs.
  struct alignas(16) Tile {
    int e, row, rows, n;
  };
  const auto tile_at = [&](int t) {
    Tile x;
    x.e = expert_of(first_tile, p.experts, t);
    const int count = first_row[x.e + 1] - first_row[x.e];
    int m;
    place(t - first_tile[x.e], stretches_of<kTileRows>(count), p.tiles_n, m, x.n);
    x.row = first_row[x.e] + m * kTileRows;
    x.rows = min(kTileRows, count - m * kTileRows);
    return x;
  };

  if (warp < kEpilogueWarps) {
    epilogue_registers();
    const int quarter = warp & 3, half = warp >> 2;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    unsigned char* stage = smem + l.staging + warp * kStagingBytes;
    uint32_t it = 0, done = 0, slot = 0;
    bool ok = true;
    for (int t = static_cast<int>(blockIdx.x); t < total; t += grid, ++done) {
      // the tile comes with its first scales: finding it takes the warp that brings them 1000 cycles
      const auto slot_at = [&](uint32_t i) { return smem + l.own + i % kScaleSlots * kScaleBytes; };
      ok = __all_sync(0xffffffffu, wait_phase_inline(scales_in(slot % kScaleSlots), (slot / kScaleSlots) & 1u, abort_flag, p.status, p.timeout_ns,
                                                     GG_STATUS_TIMEOUT_EPILOGUE));
      if (!ok) break;
      const Tile x = *reinterpret_cast<const Tile*>(slot_at(slot) + kScaleBytes - 16);
      const bool mine = quarter * 32 < x.rows;  // some of the warp's rows are there
      const int row = quarter * 32 + lane, column = x.n * kWidth + half * kMine;
      uint64_t acc[BN / 4];  // this row's sums: kMine outputs, and as many of U
#pragma unroll
      for (int j = 0; j < BN / 4; ++j) acc[j] = 0;
      for (int kb0 = 0; ok && kb0 < p.k_blocks; kb0 += kScaleBlocks, ++slot) {
        const float* scales = reinterpret_cast<const float*>(slot_at(slot));
        ok = kb0 == 0 || __all_sync(0xffffffffu, wait_phase_inline(scales_in(slot % kScaleSlots), (slot / kScaleSlots) & 1u, abort_flag, p.status, p.timeout_ns,
                                                       GG_STATUS_TIMEOUT_EPILOGUE));
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < kScaleBlocks; ++i) {
          if (kb0 + i >= p.k_blocks) break;
          const float a = scales[i * kTileRows + row];
          const float2 b = *reinterpret_cast<const float2*>(scales + kScaleBlocks * kTileRows + 2 * i);
          const uint64_t s0 = twice(a * (kGated || half == 0 ? b.x : b.y)), s1 = kGated ? twice(a * b.y) : 0;
          const uint32_t buf = it % kAcc;
          ok = __all_sync(0xffffffffu, wait_phase_inline(ready(static_cast<int>(buf)), (it / kAcc) & 1u, abort_flag, p.status, p.timeout_ns,
                                                         GG_STATUS_TIMEOUT_EPILOGUE));
          if (!ok) break;
          ++it;
          ptx::tc_fence_after_sync();
          constexpr int kPiece = kMine < 32 ? 16 : 32, kPieces = (kGated ? 2 : 1) * kMine / kPiece;
          const uint32_t from = lanes + buf * BN + static_cast<uint32_t>(half * kMine);
          const auto at_piece = [&](int c) { return from + static_cast<uint32_t>(kGated && c * kPiece >= kMine ? kWidth + c * kPiece - kMine : c * kPiece); };
          // One piece at a time: two, each read while the one before it is added up, leave too few registers (16384 rows on 64
          // experts of 14336 x 4096: pieces of 32, 1345 us, of 16, 1395; two of 16 in turn 1430, two of 32 1860).
          uint32_t r[kPiece];
          if (mine) tmem_start(at_piece(0), r);
#pragma unroll
          for (int c = 0; c < kPieces; ++c) {
            if (mine) {
              if (c) tmem_start(at_piece(c), r);
              tmem_wait(r);
            }
            if (c + 1 == kPieces) {  // all of it is read
              ptx::tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) ptx::mbar_arrive(taken(static_cast<int>(buf)));
            }
            if (mine) {
#pragma unroll
              for (int j = 0; j < kPiece / 2; ++j)
                fma2(acc[c * kPiece / 2 + j], r[2 * j], r[2 * j + 1], kGated && c * kPiece >= kMine ? s1 : s0);
            }
          }
        }
        if (!ok) break;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(scales_used(slot % kScaleSlots));
      }
      if (!ok) break;
      const Out o{p.d + static_cast<int64_t>(x.row + quarter * 32) * p.d_pitch, p.d_pitch, min(32, x.rows - quarter * 32), p.n, p.aligned, p.wide};
      const float* bias = !kGated && p.bias ? p.bias[x.e] : nullptr;
      // N of the warp's outputs from c on, before their rounding
      const auto values = [&](auto& v, int c) {
        constexpr int N = sizeof(v) / sizeof(float);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = half_of(acc[(c + j) / 2], j % 2);
        if (!kGated && bias) {
#pragma unroll
          for (int j = 0; j < N; ++j)
            if (column + c + j < p.n) v[j] += __ldg(bias + column + c + j);
        }
        activate_all(v, p.activation);
        if constexpr (kGated) {
#pragma unroll
          for (int j = 0; j < N; ++j) v[j] *= half_of(acc[(kMine + c + j) / 2], j % 2);
        }
      };
      bool eight = false;
      if constexpr (BN == 256 && kGated) eight = p.output_type > GG_OUTPUT_BF16;
      if (!eight) {
        if (mine) {
          constexpr int kPiece = kMine < 32 ? kMine : 32;
#pragma unroll
          for (int c = 0; c < kMine; c += kPiece) {
            float v[kPiece];
            values(v, c);
            store_columns(stage, lane, v, p.output_type, o, column + c);
          }
        }
      } else if constexpr (BN == 256 && kGated) {
        // a tile's 128 outputs are one block of the result: its largest magnitude is of this warp's 64 and its partner's
        float v[kMine];
        values(v, 0);
        uint32_t most = 0;
#pragma unroll
        for (int c = 0; c < kMine; ++c) most = max(most, magnitude(v[c]));
        top[done & 1u][half][row] = __uint_as_float(most);
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(pair(quarter));
        ok = __all_sync(0xffffffffu, wait_phase_inline(pair(quarter), done & 1u, abort_flag, p.status, p.timeout_ns, GG_STATUS_TIMEOUT_EPILOGUE));
        if (!ok) break;
        most = max(most, __float_as_uint(top[done & 1u][half ^ 1][row]));
        if (mine) {
          const bool e5m2 = p.output_type == GG_OUTPUT_E5M2;
          const Scale8 s(most, e5m2);
          if (half == 0 && row < x.rows) p.d_scales[static_cast<int64_t>(x.row + row) * p.ldds + x.n] = s.scale;
          const auto put = [&](auto kind) {
            uint32_t w[kMine / 4];
#pragma unroll
            for (int i = 0; i < kMine / 4; ++i) w[i] = s.four(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], kind());
            store_bytes(stage, lane, w, o, column);
          };
          if (e5m2) put(std::true_type());
          else put(std::false_type());
        }
      }
    }
    __syncthreads();
    return;
  }
  other_registers();
  if (warp >= kLoadWarp) {
    const bool leader = ptx::elect_one();
    RowLoads<kStages> rows;
    Ring<kStages, 2> stage;
    stage.at = warp - kLoadWarp;
    int skip = stage.at;  // blocks of k until this warp's next
    bool ok = true;
    for (int t = static_cast<int>(blockIdx.x); ok && t < total; t += grid) {
      const Tile x = tile_at(t);
      const CUtensorMap* maps = p.maps + 2 * x.e;
      int kb = skip;
      for (; kb < p.k_blocks; kb += 2) {
        ok = __all_sync(0xffffffffu, wait_phase_inline(empty(stage.at), stage.phase ^ 1u, abort_flag, p.status, p.timeout_ns, GG_STATUS_TIMEOUT_PRODUCER));
        if (!ok) break;
        const uint32_t a = sbase + static_cast<uint32_t>(stage.at * S::kStageBytes), b = a + kABytes, bar = full(stage.at);
        const uint32_t bytes = rows.bytes(stage.at / 2, x.rows) + BN * kRowBytes;
        if (leader) {
          ptx::mbar_arrive_expect_tx(bar, bytes);
          rows.load(&p.a_map, &p.a_box, a, bar, kb * kRowBytes, x.row, p.capacity);
          ptx::tma_load_2d(b, maps, bar, kb * kRowBytes, x.n * kWidth);
          if constexpr (kGated) ptx::tma_load_2d(b + kWidth * kRowBytes, maps + 1, bar, kb * kRowBytes, x.n * kWidth);
        }
        __syncwarp();
        stage.next();
      }
      skip = kb - p.k_blocks;
    }
    drain_loads<kStages>(stage, full);
  } else if (warp == kScaleWarp) {
    const int last = (p.n - 1) / GG_SCALE_BLOCK;
    uint32_t slot = 0;
    bool ok = true;
    for (int t = static_cast<int>(blockIdx.x); ok && t < total; t += grid) {
      const Tile x = tile_at(t);
      // of the weights: lane 2 i + w takes block i of k, w: the tile's first or second half of outputs, or gated B or U
      const int64_t column = x.n * kWidth + (kGated ? 0 : lane % 2 * (kWidth / 2));
      const float* const* table = kGated && lane % 2 ? p.up_scales : p.b_scales;
      const float* sb = table[x.e] + min(column / GG_SCALE_BLOCK, static_cast<int64_t>(last)) * p.k_blocks;
      const float* sa[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) sa[j] = p.a_scales + static_cast<int64_t>(x.row + min(j * 32 + lane, x.rows - 1)) * p.ldas;
      // A slot's scales are asked for two slots before they are written: their way from L2 takes longer than a slot lasts.
      // The rows' by ordinary loads: the kernel before, which wrote them, may have run beside this one's beginning, and __ldg
      // is for what nothing writes as long as the kernel lasts.
      struct Group {
        float a[4][kScaleBlocks], b;
      };
      const auto fetch = [&](Group& g, int kb0) {
        g.b = lane < 2 * kScaleBlocks && kb0 + lane / 2 < p.k_blocks ? __ldg(sb + kb0 + lane / 2) : 0.0f;
        const bool four = p.scales_aligned && kb0 + kScaleBlocks <= p.k_blocks;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j * 32 < x.rows && four) {
            const float4 v = *reinterpret_cast<const float4*>(sa[j] + kb0);
            g.a[j][0] = v.x, g.a[j][1] = v.y, g.a[j][2] = v.z, g.a[j][3] = v.w;
          } else {
#pragma unroll
            for (int i = 0; i < kScaleBlocks; ++i) g.a[j][i] = j * 32 < x.rows && kb0 + i < p.k_blocks ? sa[j][kb0 + i] : 0.0f;
          }
        }
      };
      const auto hand_over = [&](const Group& g) {
        ok = __all_sync(0xffffffffu, wait_phase_inline(scales_used(slot % kScaleSlots), ((slot / kScaleSlots) & 1u) ^ 1u, abort_flag, p.status,
                                                       p.timeout_ns, GG_STATUS_TIMEOUT_PRODUCER));
        if (!ok) return;
        float* to = reinterpret_cast<float*>(smem + l.own + slot % kScaleSlots * kScaleBytes);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < kScaleBlocks; ++i) to[i * kTileRows + j * 32 + lane] = g.a[j][i];
        if (lane < 2 * kScaleBlocks) to[kScaleBlocks * kTileRows + lane] = g.b;
        if (lane == 0) *reinterpret_cast<Tile*>(reinterpret_cast<unsigned char*>(to) + kScaleBytes - 16) = x;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(scales_in(slot % kScaleSlots));
        ++slot;
      };
      Group even, odd;
      fetch(even, 0);
      fetch(odd, kScaleBlocks);
      for (int kb0 = 0; ok && kb0 < p.k_blocks; kb0 += 2 * kScaleBlocks) {
        hand_over(even);
        fetch(even, kb0 + 2 * kScaleBlocks);
        if (!ok || kb0 + kScaleBlocks >= p.k_blocks) break;
        hand_over(odd);
        fetch(odd, kb0 + 3 * kScaleBlocks);
      }
    }
  } else if (warp == kProductWarp) {
    const bool leader = ptx::elect_one();
    const uint32_t idesc = ptx::idesc_f32acc(kTileRows, BN, static_cast<uint32_t>(p.input_format - GG_INPUT_E4M3), false, false);
    // descriptors of a stage's operands: an address in units of 16 bytes in their low bits, so a stage and a step of K are additions
    const uint64_t a0 = ptx::smem_desc_sw128(sbase, 16u, 1024u), b0 = ptx::smem_desc_sw128(sbase + kABytes, 16u, 1024u);
    Ring<kStages> stage;
    Ring<kAcc> acc;
    bool ok = true, have = false;  // have: the next block of k has been seen to be there, with room for its products
    for (int t = static_cast<int>(blockIdx.x); ok && t < total; t += grid) {
      for (int kb = 0; kb < p.k_blocks; ++kb) {
        if (!have)
          ok = __all_sync(0xffffffffu, wait_phase_inline(full(stage.at), stage.phase, abort_flag, p.status, p.timeout_ns, GG_STATUS_TIMEOUT_MMA) &&
                                           wait_phase_inline(taken(acc.at), acc.phase ^ 1u, abort_flag, p.status, p.timeout_ns, GG_STATUS_TIMEOUT_MMA));
        if (!ok) break;
        ptx::tc_fence_after_sync();
        const uint64_t a = a0 + static_cast<uint32_t>(stage.at * (S::kStageBytes / 16)), b = b0 + static_cast<uint32_t>(stage.at * (S::kStageBytes / 16));
        const uint32_t d = tmem + static_cast<uint32_t>(acc.at * BN), done_stage = empty(stage.at), done_acc = ready(acc.at);
        stage.next();
        acc.next();
        // asked before this block's products are issued, so that the answer is on its way meanwhile
        const bool next_full = ptx::mbar_test_wait(full(stage.at), stage.phase), next_taken = ptx::mbar_test_wait(taken(acc.at), acc.phase ^ 1u);
        if (leader) {
#pragma unroll
          for (uint32_t kk = 0; kk < 4; ++kk) ptx::tc_mma_f8(d, a + 2 * kk, b + 2 * kk, idesc, kk != 0);
          ptx::tc_commit(done_stage);
          ptx::tc_commit(done_acc);
        }
        have = __all_sync(0xffffffffu, next_full && next_taken);
      }
    }
    if (leader) {
      ptx::tc_commit(drained);  // before tensor memory is freed
      wait_drain_inline(drained, 0u, 100000000ull);
    }
    __syncwarp();
  }

  __syncthreads();
  if (warp == kProductWarp) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem, S::kTmemColumns);
  }
}

template <typename Do>
void with_shape(int bn, bool gated, Do go) {
  using std::integral_constant;
  if (gated) {
    if (bn == 256) go(integral_constant<int, 256>(), std::true_type());
    else if (bn == 128) go(integral_constant<int, 128>(), std::true_type());
    else go(integral_constant<int, 64>(), std::true_type());
  } else {
    if (bn == 256) go(integral_constant<int, 256>(), std::false_type());
    else if (bn == 128) go(integral_constant<int, 128>(), std::false_type());
    else if (bn == 64) go(integral_constant<int, 64>(), std::false_type());
    else go(integral_constant<int, 32>(), std::false_type());
  }
}

constexpr int kShapes = 4;  // 256, 128, 64, 32
int width_of(int shape) { return 256 >> shape; }

// What a run with tiles of one width takes: its tiles go over the SMs in rounds, in each of which a block of k takes an SM so
// long (0.50, 0.345, 0.30 and 0.28 us, measured with one round of 148 tiles), or memory so long as the round's weights
// take it, and a tile some 4 us more (2.3 with the narrowest). 64 rows on 8 experts of 4096 x 14336 are 128 tiles of 256, one round, or
// 256 of 128, two: 82 us against 87; of 4736 x 14336, 152 and 296 tiles, two rounds each: 146 us against 79.
double expected_us(int shape, int64_t stretches, int64_t tiles_n, int k_blocks, int experts, int sms) {
  constexpr double kBlock[kShapes] = {0.50, 0.345, 0.30, 0.28}, kTile[kShapes] = {4.2, 2.9, 2.4, 2.3};
  constexpr double kBytesPerUs = 6.5e6;
  const int64_t tiles = stretches * tiles_n;
  // an expert's weights come from memory once, from L2 for its further rows
  const double bytes = width_of(shape) * 128.0 * std::min(1.0, static_cast<double>(experts) / std::max<int64_t>(1, stretches));
  const auto round = [&](int64_t n) { return k_blocks * std::max(kBlock[shape], n * bytes / kBytesPerUs) + kTile[shape]; };
  return static_cast<double>(tiles / sms) * round(sms) + (tiles % sms ? round(tiles % sms) : 0.0);
}

}  // namespace
}  // namespace gg

struct gg_f8_plan {
  gg_f8_problem problem{};
  unsigned char* block = nullptr;  // maps of every shape | tables of scales and biases | status
  const CUtensorMap* maps[gg::kShapes] = {};
  gg::F8Params params{};
  int device = 0, sms = 0;
};

extern "C" {

int gg_f8_plan_create(const gg_f8_problem* problem, gg_f8_plan** out) {
  if (!out) return cudaErrorInvalidValue;
  *out = nullptr;
  if (!problem) return cudaErrorInvalidValue;
  const gg_f8_problem& q = *problem;
  const bool gated = q.up != nullptr, eight = q.output_type > GG_OUTPUT_BF16;
  const auto off16 = [](const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 != 0; };
  if (q.experts < 1 || q.experts > GG_F8_MAX_EXPERTS || q.n < 1 || q.n > gg::tiles::kMostSize || q.k < 1 || q.k > gg::tiles::kMostSize || q.ldb < q.k || q.ldb % 16 != 0 || !q.b || !q.b_scales ||
      (gated != (q.up_scales != nullptr)) || (gated && q.bias) || (q.input_type != GG_INPUT_E4M3 && q.input_type != GG_INPUT_E5M2) ||
      q.output_type < GG_OUTPUT_F32 || q.output_type > GG_OUTPUT_E5M2 || (eight && !gated) || q.activation < GG_ACT_NONE ||
      q.activation > GG_ACT_SILU)
    return cudaErrorInvalidValue;
  for (int e = 0; e < q.experts; ++e)
    if (!q.b[e] || !q.b_scales[e] || off16(q.b[e]) || (gated && (!q.up[e] || !q.up_scales[e] || off16(q.up[e])))) return cudaErrorInvalidValue;

  gg_f8_plan* plan = new (std::nothrow) gg_f8_plan();
  if (!plan) return cudaErrorMemoryAllocation;
  const size_t E = static_cast<size_t>(q.experts);
  const size_t map_bytes = 2 * E * sizeof(CUtensorMap), tables_at = gg::kShapes * map_bytes, status_at = tables_at + 3 * E * sizeof(void*);
  const size_t host_bytes = status_at + sizeof(int);
  // aligned as tensor maps want it
  const std::unique_ptr<CUtensorMap[]> host(new (std::nothrow) CUtensorMap[(host_bytes - 1) / sizeof(CUtensorMap) + 1]());
  if (!host) {
    delete plan;
    return cudaErrorMemoryAllocation;
  }
  unsigned char* base = reinterpret_cast<unsigned char*>(host.get());
  const auto maps = [&](int shape) { return reinterpret_cast<CUtensorMap*>(base + shape * map_bytes); };
  const float** tables = reinterpret_cast<const float**>(base + tables_at);
  cudaError_t st = cudaGetDevice(&plan->device);
  if (st == cudaSuccess) st = cudaDeviceGetAttribute(&plan->sms, cudaDevAttrMultiProcessorCount, plan->device);
  for (int e = 0; e < q.experts && st == cudaSuccess; ++e) {
    tables[e] = q.b_scales[e];
    tables[E + e] = gated ? q.up_scales[e] : nullptr;
    tables[2 * E + e] = q.bias ? q.bias[e] : nullptr;
    for (int s = 0; s < gg::kShapes && st == cudaSuccess; ++s) {
      const int box = gg::width_of(s) / (gated ? 2 : 1);
      if (!gg::encode_rows(&maps(s)[2 * e], 1, q.b[e], q.k, q.n, q.ldb, 128, box) ||
          (gated && !gg::encode_rows(&maps(s)[2 * e + 1], 1, q.up[e], q.k, q.n, q.ldb, 128, box)))
        st = cudaErrorInvalidValue;
    }
  }
  for (int s = 0; s < gg::kShapes && st == cudaSuccess; ++s)
    gg::with_shape(gg::width_of(s), gated, [&](auto bn, auto g) {
      using S = gg::F8Shape<bn()>;
      cudaFuncAttributes attributes{};
      st = cudaFuncGetAttributes(&attributes, gg::f8_kernel<bn(), g()>);
      // what the warpgroups take and give up has to be what the block is launched with
      if (st == cudaSuccess && attributes.numRegs != gg::tiles::kLaunchRegisters) st = cudaErrorInvalidConfiguration;
      if (st == cudaSuccess) st = cudaFuncSetAttribute(gg::f8_kernel<bn(), g()>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                gg::tiles::layout(S::kStages * S::kStageBytes, gg::tiles::kMaxExperts, S::kBars, gg::kScaleSlots * gg::kScaleBytes).bytes);
    });
  if (st == cudaSuccess) st = cudaMalloc(reinterpret_cast<void**>(&plan->block), host_bytes);
  if (st == cudaSuccess) st = cudaMemcpy(plan->block, host.get(), host_bytes, cudaMemcpyHostToDevice);
  if (st == cudaSuccess) st = cudaDeviceSynchronize();
  if (st != cudaSuccess) {
    if (plan->block) cudaFree(plan->block);
    delete plan;
    return st;
  }
  plan->problem = q;
  for (int s = 0; s < gg::kShapes; ++s) plan->maps[s] = reinterpret_cast<const CUtensorMap*>(plan->block + s * map_bytes);
  const float* const* on = reinterpret_cast<const float* const*>(plan->block + tables_at);
  gg::F8Params& p = plan->params;
  p.b_scales = on;
  p.up_scales = on + E;
  p.bias = q.bias ? on + 2 * E : nullptr;
  p.experts = q.experts;
  p.n = q.n;
  p.k_blocks = (q.k - 1) / 128 + 1;
  p.input_format = q.input_type;
  p.output_type = q.output_type;
  p.activation = q.activation;
  p.status = reinterpret_cast<int*>(plan->block + status_at);
  p.timeout_ns = gg::wait_limit_ns();
  *out = plan;
  return cudaSuccess;
}

int gg_f8_plan_run(gg_f8_plan* plan, const void* a, int lda, const float* a_scales, int ldas, const int* rows, void* d, int ldd,
                   float* d_scales, int ldds, int capacity_rows, void* stream) {
  if (!plan || !plan->block) return cudaErrorInvalidDevicePointer;
  const gg_f8_problem& q = plan->problem;
  gg::F8Params p = plan->params;
  const bool gated = q.up != nullptr, eight = q.output_type > GG_OUTPUT_BF16;
  if (capacity_rows < 0 || capacity_rows > gg::tiles::kMostRows || (!rows && q.experts != 1)) return cudaErrorInvalidValue;
  if (capacity_rows == 0 && !rows) return cudaSuccess;
  if (capacity_rows > 0 && (!a || !a_scales || !d || lda < q.k || lda % 16 != 0 || reinterpret_cast<uintptr_t>(a) % 16 != 0 || ldas < p.k_blocks ||
                            ldd < q.n || (eight && (!d_scales || ldds < (q.n - 1) / GG_SCALE_BLOCK + 1))))
    return cudaErrorInvalidValue;
  cudaError_t st = gg::expect_device(plan->device);
  if (st != cudaSuccess) return st;
  const int bytes = q.output_type == GG_OUTPUT_F32 ? 4 : eight ? 1 : 2;
  p.a_scales = a_scales;
  p.ldas = ldas;
  p.scales_aligned = reinterpret_cast<uintptr_t>(a_scales) % 16 == 0 && ldas % 4 == 0;
  p.rows = rows;
  p.d = static_cast<char*>(d);
  p.d_pitch = static_cast<int64_t>(ldd) * bytes;
  p.d_scales = d_scales;
  p.ldds = ldds;
  p.capacity = capacity_rows;
  p.aligned = reinterpret_cast<uintptr_t>(d) % 16 == 0 && p.d_pitch % 16 == 0;
  p.wide = reinterpret_cast<uintptr_t>(d) % 32 == 0 && p.d_pitch % 32 == 0;
  if (capacity_rows > 0 && (!gg::encode_rows(&p.a_map, 1, a, q.k, capacity_rows, lda, 128, gg::tiles::kTileRows) ||
                            !gg::encode_rows(&p.a_box, 1, a, q.k, capacity_rows, lda, 128, gg::tiles::kBoxRows)))
    return cudaErrorInvalidValue;
  // 128-row tiles at most, if every expert's rows end in a part of one
  const int64_t stretches = std::min<int64_t>(capacity_rows, static_cast<int64_t>(capacity_rows) / gg::tiles::kTileRows + q.experts);
  const auto tiles_n = [&](int s) { return (static_cast<int64_t>(q.n) * (gated ? 2 : 1) - 1) / gg::width_of(s) + 1; };
  // and as many as there are likely to be: one for each expert, or half of an expert's last one empty; each has a row at least
  // (2 rows on 64 experts of 4096 x 14336: 39.7 us with a width for 32 of them, 36.7 for the 2 that can be; 4 on 32: 58.8 and 44.4)
  const int64_t likely = std::min<int64_t>(capacity_rows, std::max<int64_t>(q.experts, (capacity_rows / gg::tiles::kTileRows) + q.experts / 2));
  int shape = 0;
  for (int s = 1; !eight && s < (gated ? 3 : gg::kShapes); ++s)
    if (gg::expected_us(s, likely, tiles_n(s), p.k_blocks, q.experts, plan->sms) < gg::expected_us(shape, likely, tiles_n(shape), p.k_blocks, q.experts, plan->sms))
      shape = s;
  const int64_t most = stretches * tiles_n(shape);
  if (most > gg::tiles::kMostTiles) return cudaErrorInvalidValue;
  p.tiles_n = static_cast<int>(tiles_n(shape));
  p.maps = plan->maps[shape];
  const unsigned grid = static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(plan->sms, most)));
  gg::with_shape(gg::width_of(shape), gated, [&](auto bn, auto g) {
    using S = gg::F8Shape<bn()>;
    st = gg::launch_chained(gg::f8_kernel<bn(), g()>, dim3(grid), gg::tiles::kTileThreads,
                            static_cast<size_t>(gg::tiles::layout(S::kStages * S::kStageBytes, q.experts, S::kBars, gg::kScaleSlots * gg::kScaleBytes).bytes),
                            static_cast<cudaStream_t>(stream), 1, p);
  });
  return st;
}

int gg_f8_plan_status(gg_f8_plan* plan, int* status) {
  if (!plan || !plan->block) return cudaErrorInvalidDevicePointer;
  if (!status) return cudaErrorInvalidValue;
  cudaError_t st = gg::expect_device(plan->device);
  if (st == cudaSuccess) st = cudaDeviceSynchronize();
  if (st == cudaSuccess) st = cudaMemcpy(status, plan->params.status, sizeof(int), cudaMemcpyDeviceToHost);
  if (st != cudaSuccess) return st;
  return cudaMemset(plan->params.status, 0, sizeof(int));
}

void gg_f8_plan_destroy(gg_f8_plan* plan) {
  if (!plan) return;
  if (plan->block) cudaFree(plan->block);
  delete plan;
}

}  // extern "C"
