// gg_expert_tiles.cuh -- what the 8-bit product (gg_f8.cu) and the gated block (gg_gated.cu) share: persistent kernels
// over the output tiles of experts whose row counts are in device memory.
//
// A block of 384 threads has an SM to itself: warps 0-7 take results out of tensor memory (two to each quarter of its
// lanes), warp 8 issues the products, warp 10 the TMA loads. Every block works out the experts' first rows and first
// tiles by itself at its start (one warp, one pass over the counts), so a run is one launch and no role needs the
// others to know its tiles: block b takes tiles b, b + grid, ...
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "gg_epilogue_ops.cuh"
#include "gg_ptx.cuh"
#include "gg_wait.cuh"
#include "grouped_gemm_b200.h"

namespace gg {
namespace tiles {

constexpr int kTileThreads = 384;
constexpr int kEpilogueWarps = 8;
constexpr int kProductWarp = 8;
constexpr int kLoadWarp = 10;
constexpr int kTileRows = 128;                 // rows of a tile: M of the products
constexpr int kRowBytes = 128;                 // of a stage's row: 64 values of 16 bits or 128 of 8
constexpr int kABytes = kTileRows * kRowBytes; // of a stage
constexpr int kBoxRows = 32;                   // rows that one load of packed rows takes: a tile loads the boxes that hold its rows
constexpr int kStagingBytes = 2048;            // of an epilogue warp: 32 rows of 64 bytes
constexpr int kMaxExperts = 1024;
constexpr int kRaster = 16;                    // tile rows that are gone through before the next tile column

// Shared memory after the stages: staging, the experts' tables, barriers.
struct Layout {
  int staging, table, bars, words, bytes;
};
constexpr Layout layout(int stage_bytes, int experts, int bars) {
  Layout l{};
  l.staging = stage_bytes;
  l.table = l.staging + kEpilogueWarps * kStagingBytes;
  l.bars = (l.table + 2 * (experts + 1) * 4 + 7) / 8 * 8;
  l.words = l.bars + 8 * bars;
  l.bytes = l.words + 16 + 1024;  // slack: stages start on 1024 bytes
  return l;
}

__device__ __forceinline__ float activate_more(float x, int act) {
  // x / (1 + exp(-x)); past exp(80) the result is below 1e-33 either way, and __fdividef wants less than 2^126
  if (act == GG_ACT_SILU) return __fdividef(x, 1.0f + __expf(fminf(-x, 80.0f)));
  return activate(x, act);
}

// first_row[e], first_tile[e] for e = 0..experts (totals at the end), by one warp. `per_row_tile`: tiles of one 128-row
// stretch of an expert. Counts that are negative or sum to more than `capacity` leave no rows, and -1 as the total of tiles.
__device__ __forceinline__ void expert_table(const int* rows, int experts, int capacity, int per_row_tile, int* first_row, int* first_tile,
                                             int* status, int lane) {
  int row = 0, tile = 0;
  bool bad = false;
  if (!rows) {
    if (lane == 0) {
      first_row[0] = first_tile[0] = 0;
      first_row[1] = capacity;
      first_tile[1] = (capacity + kTileRows - 1) / kTileRows * per_row_tile;
    }
    return;
  }
  int next = lane < experts ? rows[lane] : 0;
  for (int e0 = 0; e0 < experts; e0 += 32) {
    const int r = next;
    if (e0 + 32 + lane < experts) next = rows[e0 + 32 + lane];
    else next = 0;
    // a count above capacity - row, or a negative one, ends it, so no sum passes 32 bits: 32 counts of at most capacity
    bad = bad || __any_sync(0xffffffffu, r < 0 || r > capacity);
    if (bad) break;
    long long sum = r;
    int t = (r + kTileRows - 1) / kTileRows * per_row_tile;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long s = __shfl_up_sync(0xffffffffu, sum, o);
      const int u = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) sum += s, t += u;
    }
    bad = __any_sync(0xffffffffu, sum + row > capacity);
    if (bad) break;
    if (e0 + lane < experts) {
      first_row[e0 + lane + 1] = row + static_cast<int>(sum);
      first_tile[e0 + lane + 1] = tile + t;
    }
    row += static_cast<int>(__shfl_sync(0xffffffffu, sum, 31));
    tile += __shfl_sync(0xffffffffu, t, 31);
  }
  if (bad) {
    for (int e = lane; e <= experts; e += 32) first_row[e] = 0, first_tile[e] = e < experts ? 0 : -1;
    if (lane == 0) atomicOr(status, GG_STATUS_BAD_ROWS);
  } else if (lane == 0) {
    first_row[0] = first_tile[0] = 0;
  }
}

// The expert whose tiles hold `tile`: the last e with first_tile[e] <= tile (experts without tiles are passed over).
__device__ __forceinline__ int expert_of(const int* first_tile, int experts, int tile) {
  int lo = 0, hi = experts;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first_tile[mid] <= tile) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Tile `local` of tiles_m x tiles_n: stretches of kRaster tile rows, in each of which the row runs fastest, so that the
// blocks at work share both operands in L2.
__device__ __forceinline__ void place(int local, int tiles_m, int tiles_n, int& m, int& n) {
  const int span = kRaster * tiles_n, g = local / span, first = g * kRaster;
  const int rows = min(kRaster, tiles_m - first), in = local - g * span;
  m = first + in % rows;
  n = in / rows;
}

// N (8, 16 or 32) columns of the warp's 32 lanes of tensor memory; the wait is apart (tmem_wait).
template <int N>
__device__ __forceinline__ void tmem_read(uint32_t addr, uint32_t (&r)[N]) {
  if constexpr (N == 32) {
    ptx::tmem_load_32cols(addr, r);
  } else {
    static_assert(N == 16);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
  }
}

// Where a warp's 32 rows of an output go.
struct Out {
  char* base;      // of the first row
  int64_t pitch;   // bytes
  int rows;        // rows that are there, at most 32
  int columns;     // of the whole matrix
  bool aligned;    // rows start on 16-byte boundaries
};

// The warp's staging rows (64 bytes, 16-byte unit u of row r at u ^ (r / 2 % 4)) to the output from byte `at` of its rows on;
// kUnits units of each row are filled. kBytes: of an element.
template <int kBytes, int kUnits>
__device__ __forceinline__ void write_out(const unsigned char* stage, int lane, const Out& o, int column) {
  constexpr int kPer = 16 / kBytes;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int idx = i * 32 + lane, r = idx / kUnits, u = idx % kUnits, c = column + u * kPer;
    if (r < o.rows && c < o.columns) {
      const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 64 + ((u ^ (r >> 1 & 3)) << 4));
      char* to = o.base + r * o.pitch + static_cast<int64_t>(c) * kBytes;
      if (o.aligned && c + kPer <= o.columns) {
        *reinterpret_cast<uint4*>(to) = v;
      } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          if (c + j >= o.columns) break;
          if constexpr (kBytes == 4) reinterpret_cast<uint32_t*>(to)[j] = w[j];
          else if constexpr (kBytes == 2) reinterpret_cast<unsigned short*>(to)[j] = static_cast<unsigned short>(w[j / 2] >> (16 * (j % 2)));
          else reinterpret_cast<unsigned char*>(to)[j] = static_cast<unsigned char>(w[j / 4] >> (8 * (j % 4)));
        }
      }
    }
  }
  __syncwarp();
}

__device__ __forceinline__ uint4* staging_unit(unsigned char* stage, int lane, int u) {
  return reinterpret_cast<uint4*>(stage + lane * 64 + ((u ^ (lane >> 1 & 3)) << 4));
}

// N (16 or 32) columns of the lane's row, rounded to `type` (FP32 or 16 bits), to columns column..column + N - 1.
template <int N>
__device__ __forceinline__ void store_columns(unsigned char* stage, int lane, const float (&v)[N], int type, const Out& o, int column) {
  if (type == GG_OUTPUT_F32) {
#pragma unroll
    for (int c = 0; c < N; c += 16) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        *staging_unit(stage, lane, u) = make_uint4(__float_as_uint(v[c + 4 * u]), __float_as_uint(v[c + 4 * u + 1]),
                                                   __float_as_uint(v[c + 4 * u + 2]), __float_as_uint(v[c + 4 * u + 3]));
      write_out<4, 4>(stage, lane, o, column + c);
    }
  } else {
#pragma unroll
    for (int u = 0; u < N / 8; ++u)
      *staging_unit(stage, lane, u) = make_uint4(pack2_rt(type, v[8 * u], v[8 * u + 1]), pack2_rt(type, v[8 * u + 2], v[8 * u + 3]),
                                                 pack2_rt(type, v[8 * u + 4], v[8 * u + 5]), pack2_rt(type, v[8 * u + 6], v[8 * u + 7]));
    write_out<2, N / 8>(stage, lane, o, column);
  }
}

// After an abort: waits, bounded, for the loads into the last stages before the block ends.
template <int kStages, typename FullBar>
__device__ __forceinline__ void drain_loads(uint32_t issued, FullBar full) {
  const uint32_t back = issued < kStages ? issued : kStages;
  for (uint32_t j = 1; j <= back; ++j) {
    const uint32_t i = issued - j;
    wait_drain(full(static_cast<int>(i % kStages)), (i / kStages) & 1u, 100000000ull);
  }
}

}  // namespace tiles
}  // namespace gg
