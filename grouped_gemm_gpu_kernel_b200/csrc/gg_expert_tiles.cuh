// gg_expert_tiles.cuh -- what the 8-bit product (gg_f8.cu) and the gated block (gg_gated.cu) share: persistent kernels
// over the output tiles of experts whose row counts are in device memory.
//
// A block of 384 threads has an SM to itself: warps 0-7 take results out of tensor memory (two to each quarter of its
// lanes), warp 8 issues the products, warps 10 and 11 the TMA loads. Every block works out the experts' first rows and first
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
constexpr int kLoadWarp = 10;                  // and the next one, which take the stages in turn: one warp takes 500 cycles for a stage's loads
constexpr int kTileRows = 128;                 // rows of a tile: M of the products
constexpr int kRowBytes = 128;                 // of a stage's row: 64 values of 16 bits or 128 of 8
constexpr int kABytes = kTileRows * kRowBytes; // of a stage
constexpr int kBoxRows = 16;                   // rows that one load of a part of a tile takes
constexpr int kStagingBytes = 2048;            // of an epilogue warp: 32 rows of 64 bytes
constexpr int kMaxExperts = 1024;
// Limits that keep rows, columns and tiles, and what a role adds to them, within 32 bits.
constexpr int kMostRows = 2147483647 - 65536;
constexpr int kMostSize = 1 << 30;
constexpr long long kMostTiles = 2147483647 - 65536;
constexpr int kRaster = 16;                    // tile rows that are gone through before the next tile column

// Shared memory after the stages: staging, what a kernel wants for itself, the experts' tables, barriers.
struct Layout {
  int staging, own, table, bars, words, bytes;
};
constexpr Layout layout(int stage_bytes, int experts, int bars, int own = 0) {
  Layout l{};
  l.staging = stage_bytes;
  l.own = l.staging + kEpilogueWarps * kStagingBytes;
  l.table = l.own + own;
  l.bars = (l.table + 2 * (experts + 1) * 4 + 7) / 8 * 8;
  l.words = l.bars + 8 * bars;
  l.bytes = l.words + 16 + 1024;  // words: tensor memory's address, the abort flag, two of progress; slack: stages start on 1024 bytes
  return l;
}

// x / (1 + exp(-z)), within 4e-5 of it: a fast exponential and a fast division, since a tile's end has thousands of them (in FP32
// results too, whose sums have some 1e-5 of their own). Where exp(-z) passes 2^126, __fdividef gives 0, which the result is
// within 1e-32 of for both uses below: z = x, and z about 0.07 x^3.
__device__ __forceinline__ float over_logistic(float x, float z) { return __fdividef(x, 1.0f + __expf(-z)); }
// GELU in its tanh form: x / (1 + exp(-2u)), u = sqrt(2 / pi) (x + 0.044715 x^3).
__device__ __forceinline__ float gelu_exponent(float x) { return 1.5957691216057308f * fmaf(0.044715f * x, x * x, x); }

// act of N values. The choice is made once for all of them: code for every value's own choice, unrolled, is more than the
// instruction caches hold, and a tile's end then takes 15 us.
template <int N>
__device__ __forceinline__ void activate_all(float (&v)[N], int act) {
  if (act == GG_ACT_SILU) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = over_logistic(v[j], v[j]);
  } else if (act == GG_ACT_GELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = over_logistic(v[j], gelu_exponent(v[j]));
  } else if (act == GG_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = fmaxf(v[j], 0.0f);
  }
}

// first_row[e], first_tile[e] for e = 0..experts (totals at the end), by one warp. `per_row_tile`: tiles of one stretch of kStretch
// rows of an expert. Counts that are negative or sum to more than `capacity` leave no rows, and -1 as the total of tiles.
template <int kStretch>
__device__ __forceinline__ int stretches_of(int rows) {
  return rows / kStretch + (rows % kStretch != 0);
}
template <int kStretch = kTileRows>
__device__ __forceinline__ void expert_table(const int* rows, int experts, int capacity, int per_row_tile, int* first_row, int* first_tile,
                                             int* status, int lane) {
  int row = 0, tile = 0;
  bool bad = false;
  if (!rows) {
    if (lane == 0) {
      first_row[0] = first_tile[0] = 0;
      first_row[1] = capacity;
      first_tile[1] = stretches_of<kStretch>(capacity) * per_row_tile;
    }
    return;
  }
  int next = lane < experts ? rows[lane] : 0;
  for (int e0 = 0; e0 < experts; e0 += 32) {
    const int r = next;
    if (e0 + 32 + lane < experts) next = rows[e0 + 32 + lane];
    else next = 0;
    // sums of 32 counts of at most capacity take 64 bits; tiles are counted only where the rows fit
    bad = bad || __any_sync(0xffffffffu, r < 0 || r > capacity);
    if (bad) break;
    long long sum = r;
    unsigned t = static_cast<unsigned>(stretches_of<kStretch>(r)) * static_cast<unsigned>(per_row_tile);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long s = __shfl_up_sync(0xffffffffu, sum, o);
      const unsigned u = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) sum += s, t += u;
    }
    bad = __any_sync(0xffffffffu, sum + row > capacity);
    if (bad) break;
    if (e0 + lane < experts) {
      first_row[e0 + lane + 1] = row + static_cast<int>(sum);
      first_tile[e0 + lane + 1] = tile + static_cast<int>(t);
    }
    row += static_cast<int>(__shfl_sync(0xffffffffu, sum, 31));
    tile += static_cast<int>(__shfl_sync(0xffffffffu, t, 31));
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

// N (16 or 32) columns of the warp's 32 lanes of tensor memory, started; tmem_wait makes the registers valid.
template <int N>
__device__ __forceinline__ void tmem_start(uint32_t addr, uint32_t (&r)[N]) {
  static_assert(N == 16 || N == 32);
  if constexpr (N == 32) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
          "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
          "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
          "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
  } else {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
  }
}
// Waits for every read that was started, and names the registers so that no use of them moves ahead of it.
template <int N>
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[N]) {
  if constexpr (N == 32) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                   "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
                   "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                   "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                   "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
  } else {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                   "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
                   "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
  }
}
template <int N>
__device__ __forceinline__ void tmem_read(uint32_t addr, uint32_t (&r)[N]) {
  tmem_start(addr, r);
  tmem_wait(r);
}

// Gives registers up, or takes them, for this warpgroup: a block of 384 threads is launched with kLaunchRegisters a thread, of
// which the two warpgroups of the epilogue take 208 and the third keeps 88: 2 * 208 + 88 = 3 * 168.
constexpr int kLaunchRegisters = 168;
__device__ __forceinline__ void epilogue_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 208;"); }
__device__ __forceinline__ void other_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 88;"); }

// A place in a ring of N and the parity of its round.
template <int N, int kStep = 1>
struct Ring {
  int at = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    at += kStep;
    if (at >= N) at -= N, phase ^= 1u;
  }
};

// Where a warp's 32 rows of an output go.
struct Out {
  char* base;      // of the first row
  int64_t pitch;   // bytes
  int rows;        // rows that are there, at most 32
  int columns;     // of the whole matrix
  bool aligned;    // rows start on 16-byte boundaries
  bool wide;       // and on 32-byte boundaries
};
__device__ __forceinline__ void store_32_bytes(char* to, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
               "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// The warp's staging rows (64 bytes, 16-byte unit u of row r at u ^ (r / 2 % 4)) to the output from `column` on;
// kUnits units of each row are filled. kBytes: of an element.
template <int kBytes, int kUnits>
__device__ __forceinline__ void write_out(const unsigned char* stage, int lane, const Out& o, int column) {
  constexpr int kPer = 16 / kBytes;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int idx = i * 32 + lane, r = idx / kUnits, u = idx % kUnits, c = column + u * kPer;
    if (r < o.rows && c < o.columns) {
      const unsigned char* from = stage + r * 64 + ((u ^ (r >> 1 & 3)) << 4);
      char* to = o.base + r * o.pitch + static_cast<int64_t>(c) * kBytes;
      if (o.aligned && c + kPer <= o.columns) {
        *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
      } else {
        const int bytes = min(16, (o.columns - c) * kBytes);
#pragma unroll 1
        for (int j = 0; j < bytes; j += kBytes) {
          if constexpr (kBytes == 4) *reinterpret_cast<uint32_t*>(to + j) = *reinterpret_cast<const uint32_t*>(from + j);
          else if constexpr (kBytes == 2) *reinterpret_cast<unsigned short*>(to + j) = *reinterpret_cast<const unsigned short*>(from + j);
          else to[j] = static_cast<char>(from[j]);
        }
      }
    }
  }
  __syncwarp();
}

__device__ __forceinline__ uint4* staging_unit(unsigned char* stage, int lane, int u) {
  return reinterpret_cast<uint4*>(stage + lane * 64 + ((u ^ (lane >> 1 & 3)) << 4));
}

// N (16 or 32) columns of the lane's row, rounded to the output type F, to columns column..column + N - 1. Where rows start on
// 32-byte boundaries and all columns are there, each lane writes its own row's, 32 bytes (a whole sector) at a time, straight
// from its registers: through staging, 32 columns take 800 cycles of one round trip after another. Else the staging rows
// bring the pieces of a row together.
template <int F, int N>
__device__ __forceinline__ void store_columns_as(unsigned char* stage, int lane, const float (&v)[N], const Out& o, int column) {
  if (o.wide && column + N <= o.columns) {
    if (lane >= o.rows) return;
    char* to = o.base + lane * o.pitch + static_cast<int64_t>(column) * OutFormat<F>::kBytes;
    constexpr int kPer = 32 / OutFormat<F>::kBytes;
#pragma unroll
    for (int c = 0; c < N; c += kPer) {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (F == GG_OUTPUT_F32) w[i] = __float_as_uint(v[c + i]);
        else w[i] = pack2<F>(v[c + 2 * i], v[c + 2 * i + 1]);
      }
      store_32_bytes(to + c * OutFormat<F>::kBytes, w);
    }
    return;
  }
  if constexpr (F == GG_OUTPUT_F32) {
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
      *staging_unit(stage, lane, u) = make_uint4(pack2<F>(v[8 * u], v[8 * u + 1]), pack2<F>(v[8 * u + 2], v[8 * u + 3]),
                                                 pack2<F>(v[8 * u + 4], v[8 * u + 5]), pack2<F>(v[8 * u + 6], v[8 * u + 7]));
    write_out<2, N / 8>(stage, lane, o, column);
  }
}
template <int N>
__device__ __forceinline__ void store_columns(unsigned char* stage, int lane, const float (&v)[N], int type, const Out& o, int column) {
  if (type == GG_OUTPUT_BF16) store_columns_as<GG_OUTPUT_BF16>(stage, lane, v, o, column);
  else if (type == GG_OUTPUT_F16) store_columns_as<GG_OUTPUT_F16>(stage, lane, v, o, column);
  else store_columns_as<GG_OUTPUT_F32>(stage, lane, v, o, column);
}

// 64 columns of the lane's row in 8 bits.
__device__ __forceinline__ void store_bytes(unsigned char* stage, int lane, const uint32_t (&w)[16], const Out& o, int column) {
  if (o.wide && column + 64 <= o.columns) {
    if (lane >= o.rows) return;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint32_t q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = w[8 * c + i];
      store_32_bytes(o.base + lane * o.pitch + column + 32 * c, q);
    }
    return;
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) *staging_unit(stage, lane, u) = make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
  write_out<1, 4>(stage, lane, o, column);
}

// The packed rows of a tile into a stage. A whole tile is one load; a part of one is the boxes of kBoxRows that hold it, and
// the rows of the stage past them are zeros: what is multiplied there is never stored, but the products of what an
// earlier tile left take power, which the clock goes by. `dirty`: the boxes of each stage that are not zeros; at the kernel's
// start all of shared memory's are.
template <int kStages>
struct RowLoads {
  static constexpr int kBoxes = kTileRows / kBoxRows;
  int dirty[kStages / 2] = {};  // of the stages of this loading warp
  int boxes = 0, most = 0;
  // For a tile of `rows` rows; then the bytes that load() brings.
  __device__ __forceinline__ uint32_t bytes(int mine, int rows) {
    boxes = (rows + kBoxRows - 1) / kBoxRows;
    most = boxes;
#pragma unroll
    for (int i = 0; i < kStages / 2; ++i)
      if (i == mine) most = max(most, dirty[i]), dirty[i] = boxes;
    return static_cast<uint32_t>(most * kBoxRows * kRowBytes);
  }
  // zeros_at: a row past the matrix, where a box is filled with zeros.
  __device__ __forceinline__ void load(const CUtensorMap* whole, const CUtensorMap* box, uint32_t a, uint32_t bar, int k, int row, int zeros_at) const {
    if (boxes == kBoxes) {
      ptx::tma_load_2d(a, whole, bar, k, row);
    } else {
      for (int i = 0; i < most; ++i) ptx::tma_load_2d(a + i * kBoxRows * kRowBytes, box, bar, k, i < boxes ? row + i * kBoxRows : zeros_at);
    }
  }
};
// At the start, by all threads: zeros in the rows' part of every stage (before the barrier that the roles start behind).
template <int kStages, int kStageBytes>
__device__ __forceinline__ void clear_rows(uint8_t* smem) {
  for (int i = static_cast<int>(threadIdx.x); i < kStages * (kABytes / 16); i += kTileThreads)
    *reinterpret_cast<uint4*>(smem + i / (kABytes / 16) * kStageBytes + i % (kABytes / 16) * 16) = make_uint4(0u, 0u, 0u, 0u);
  ptx::fence_proxy_async_smem();
}

// At the end of a loading warp: waits, bounded, for the loads of its stages, since a block must not end while they may still land in
// its shared memory. The products wait for them too, unless another warp has given up, before this one's end or after it, so this
// does not ask whether one has. `stage` is the next that the warp would have filled; one that it had not filled yet is passed at once,
// and one that never completes runs out its limit.
template <int kStages, typename FullBar>
__device__ __forceinline__ void drain_loads(Ring<kStages, 2> stage, FullBar full) {
  for (int j = 0; j < kStages / 2; ++j) {
    wait_drain_inline(full(stage.at), stage.phase ^ 1u, 100000000ull);  // the round before
    stage.next();
  }
}

}  // namespace tiles
}  // namespace gg
