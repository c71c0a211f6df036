// gg_q4.cu -- rows of a mixture-of-experts layer against expert weights held in 4 bits with a scale
// per output and group of k (the decoding form of the mixture-of-experts plan):
//   D[r, o] = act(sum_g scale(o, g) * sum_{k in g} A[r, k] (q(o, k) - zero(o, g)) + bias(o)).
//
// With few rows an expert the weights' bytes bound it, so the kernel is built around reading them
// once, whole lines at a time. The weights stand as the A operand of mma.sync m16n8k16 (16 outputs
// a tile, 8 rows of the activations as its columns): the differences q - zero are small integers,
// exact in FP16 and BF16, so the tensor pipe's products are exact and its sums FP32, and the group's
// scale multiplies the FP32 sum. tcgen05 takes 128 outputs a tile, and the unpacked operand from shared or tensor
// memory: through one matrix of 4096 or 14336 outputs that is 32 or 112 tiles for 148 SMs without a split of k over
// blocks; a fragment in registers is fed from the unpacking directly. With experts enough for the tiles and rows enough
// to pay for the way through shared memory, tcgen05 would unpack a tile once, where this kernel does for every 16 rows:
// that form is not here.
//
// Measured (B200, FP16, group 128, inputs past L2): one row through 14336 x 4096, 12.1 us (2.4 TB/s of weights; 4.5 us
// at the copy rate), of which some 5 are the start and the end of the kernel (4096 x 4096 takes 6.6); eight experts of
// 4096 x 14336 with one row each, 52 us (4.5 TB/s), 8 each 62, 64 rows as 3 to 14 each 70. The copies alone, without the
// arithmetic, run at 39 us there; the arithmetic alone, without the copies, at 47: about 165 instructions a block of
// 1 KB, of which 98 are the unpacking and the products, at half of the issue slots (dependent steps of 16 warps an SM;
// 24 warps at 80 registers take 20 % more instructions and no less time). Past 8 rows an expert the activations,
// read once a tile from L1 or L2, are more bytes than the weights, and past 16 the unpacking is done again: 256
// rows 151 us, 1024 673, 8192 6.2 ms. Two tiles a task, which halves those reads,
// gained 4 to 12 % above 16 rows and lost 8 to 10 % below and with group 64 and zeros: not kept.
//
// Weights are laid out once (gg_q4_plan_create), per expert as blocks of 16 outputs x 128 k, tile by tile
// and along k in a tile. A block is what one step of a warp reads, in one piece:
//   1024 bytes of weights [half h][lane][4 words]: lane l, word i, half h hold output 16 tile + 8 h + l / 4
//   and k = 128 block + 32 i + 8 (l % 4) + 0..7, the eight values in the nibbles (0, 4, 1, 5, 2, 6, 3, 7)
//   from the low end, so that one mask gives the pair (x, x + 1) in the two halves of a register;
//   its scales [l / 4][group of the block][half], 16 bits each; the zeros alike, 8 bits each (if any).
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <new>
#include <type_traits>

#include "gg_epilogue_ops.cuh"
#include "gg_internal.h"
#include "gg_launch.cuh"
#include "gg_ptx.cuh"
#include "grouped_gemm_b200.h"

namespace gg {
namespace {

constexpr int kQ4Threads = 256;
constexpr int kQ4Warps = kQ4Threads / 32;
constexpr int kTileN = 16;   // outputs a block of weights covers
constexpr int kBlockK = 128; // k values a block covers
constexpr int kBlockBytes = kTileN * kBlockK / 2;

// Bytes of a block with `per` groups along its k.
__host__ __device__ constexpr int record_bytes(int per, bool zeros) {
  return kBlockBytes + kTileN * per * 2 + (zeros ? kTileN * per : 0);
}

struct Q4Params {
  const unsigned char* blocks;  // [experts][n_tiles][k_blocks][record_bytes]
  const float* const* bias;     // [experts]; NULL: none
  int* status;
  int experts, n, k, n_tiles, k_blocks, output_type, activation, sms;
  unsigned long long timeout_ns;
  // of a run
  const void* a;
  const int* row_tokens;
  const int* rows;
  void* d;
  int64_t lda, ldd;
  int a_rows, capacity_rows;
  const unsigned short* no_row; // k zeros, for a gathered row that does not exist
};

struct Q4PackParams {
  const unsigned char* const* q;
  const void* const* scales;
  const unsigned char* const* zeros;  // its entries are NULL without zeros
  unsigned char* out;
  int experts, n, k, group, n_tiles, k_blocks, per_block, record, with_zeros;
  int64_t ldq;
};

// One thread per 16-byte piece of the weights (block, half, lane), and one per scale and zero.
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
    const unsigned char* row = o < p.n ? p.q[e] + o * p.ldq : nullptr;
    const bool words = (reinterpret_cast<uintptr_t>(row) & 3u) == 0;
    unsigned w[4];
    for (int x = 0; x < 4; ++x) {
      const int k = kBlockK * kb + 32 * x + 8 * (lane % 4);
      unsigned in = 0x88888888u;  // eight values from k on; past k: 8
      if (row && k + 8 <= p.k && words) {
        in = *reinterpret_cast<const unsigned*>(row + k / 2);
      } else if (row) {
        for (int v = 0; v < 8 && k + v < p.k; ++v)
          in = (in & ~(15u << (4 * v))) | ((row[(k + v) / 2] >> (4 * (v % 2))) & 15u) << (4 * v);
      }
      // the even values to the low half, the odd ones to the high half
      unsigned even = in & 0x0f0f0f0fu, odd = (in >> 4) & 0x0f0f0f0fu;
      even = (even | even >> 4) & 0x00ff00ffu, odd = (odd | odd >> 4) & 0x00ff00ffu;
      w[x] = ((even | even >> 8) & 0xffffu) | (odd | odd >> 8) << 16;
    }
    reinterpret_cast<uint4*>(p.out + b * p.record)[i % 64] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  const int per = kTileN * p.per_block;
  const int groups = (p.k - 1) / p.group + 1;
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
    unsigned char* record = p.out + b * p.record + kBlockBytes;
    reinterpret_cast<unsigned short*>(record)[in] =
        in_range ? static_cast<const unsigned short*>(p.scales[e])[at] : static_cast<unsigned short>(0);
    if (p.with_zeros) record[2 * per + in] = in_range ? p.zeros[e][at] & 15 : 8;
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

// What is taken from the unpacked pairs, in both halves: the magic number plus the zero; and for the
// nibbles left four bits up in FP16 the same of (1024 + 16 q) / 16, -(64 + zero). `zeros`: the zeros of
// outputs l / 4 (low byte) and l / 4 + 8.
template <bool kBf16, int kHalf>
struct Q4Zero {
  unsigned ones, sixteens;
  __device__ __forceinline__ explicit Q4Zero(unsigned zeros) {
    ones = __byte_perm(zeros, kBf16 ? 0x43434343u : 0x64646464u, kHalf ? 0x4141 : 0x4040);
    sixteens = __byte_perm(zeros << 4, 0xd4d4d4d4u, kHalf ? 0x4141 : 0x4040);  // a step of 1 is 16 units in the last place
  }
};

// The eight nibbles of a word as four pairs q - zero, exact (whole numbers below 2048, below 256 in
// BF16), by a widely published method: a nibble put into the low mantissa bits of a fixed power of two makes the
// number power + q, without a conversion. FP16's ten mantissa bits leave room to take two of the four pairs without a shift.
__device__ __forceinline__ unsigned and_or(unsigned x, unsigned mask, unsigned add) {  // (x & mask) | add
  unsigned d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(x), "r"(mask), "r"(add));
  return d;
}

template <bool kBf16, typename Zero>
__device__ __forceinline__ void unpack8(unsigned w, const Zero& z, unsigned (&f)[4]) {
  constexpr unsigned kMagic = Q4Type<kBf16>::kMagic;
  if constexpr (kBf16) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const unsigned x = and_or(w >> (4 * v), 0x000f000fu, kMagic);
      asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(f[v]) : "r"(x), "r"(z.ones));
    }
  } else {
#pragma unroll
    for (int v = 0; v < 4; v += 2) {
      const unsigned u = v == 0 ? w : w >> 8;
      const unsigned x = and_or(u, 0x000f000fu, kMagic), y = and_or(u, 0x00f000f0u, kMagic);
      asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(f[v]) : "r"(x), "r"(z.ones));
      asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(f[v + 1]) : "r"(y), "r"(0x2c002c00u), "r"(z.sixteens));
    }
  }
}

// c = a b (first) or c += a b; `first` is known at compile time.
template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&c)[4], bool first, unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                         unsigned b1) {
  if constexpr (kBf16) {
    if (first)
      asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                   : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                   : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
      asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                   : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                   : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    if (first)
      asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                   : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                   : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
      asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                   : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                   : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

// As in the grouped product's epilogue (a NaN's ReLU is 0), with GELU through the full-range exponential.
__device__ __forceinline__ float q4_activate(float x, int act) {
  if (act == GG_ACT_RELU) return fmaxf(x, 0.0f);
  if (act == GG_ACT_GELU) return x / (1.0f + expf(-1.5957691216057308f * fmaf(0.044715f * x, x * x, x)));
  return x;
}

// Eight activations from `at` on, of which `have` exist (the others are zero), as four packed pairs. kLoad: 2
// where the rows are made up of aligned pairs, else 1.
template <int kLoad>
__device__ __forceinline__ uint4 load_units(const unsigned short* at, int have) {
  unsigned v[8];
#pragma unroll
  for (int i = 0; i < 8; i += kLoad) {
    if constexpr (kLoad == 2) v[i / 2] = i < have ? __ldg(reinterpret_cast<const unsigned*>(at) + i / 2) : 0u;
    else v[i] = i < have ? __ldg(at + i) : 0u;
  }
  if constexpr (kLoad == 2) return make_uint4(v[0], v[1], v[2], v[3]);
  else return make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
}

// `bytes` (a multiple of 16) from global to shared memory, counted on the mbarrier.
__device__ __forceinline__ void copy_bulk(uint32_t to, const void* from, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from),
               "r"(bytes), "r"(bar)
               : "memory");
}

// Whether a wait of the block's has run out. (At a constant address: one kept in a register, or a place ahead that a
// wait may change, spills in the loop: 64 rows on eight experts of 4096 x 14336 then take 84 us, 76 so.)
__shared__ int s_gave_up;

__device__ __forceinline__ bool gave_up() {
  int v;
  asm volatile("ld.shared.s32 %0, [%1];" : "=r"(v) : "r"(ptx::smem_addr(&s_gave_up)) : "memory");
  return v != 0;
}

// Waits for the copy of a stage, at most timeout_ns; where that runs out raises GG_STATUS_TIMEOUT_PRODUCER and
// waits as long again. If it has not come then, the block gives up: it starts no more copies (a copy is only ever
// started into a stage whose last one was seen), and goes through its ranges with what is in the stages, so that
// the barriers of its groups stay matched. Every copy under way still has its wait, a thousandth as long, before
// the block ends; those for copies that were not started run out as well.
__device__ __forceinline__ void wait_bounded(uint32_t bar, uint32_t parity, unsigned long long timeout_ns, int* status) {
  if (ptx::mbar_try_wait(bar, parity)) return;
  const unsigned long long limit = gave_up() ? timeout_ns / 1000 : timeout_ns;
  for (int again = 0; again < 2; ++again) {
    const uint64_t start = ptx::global_timer_ns();
    for (unsigned i = 0; ptx::global_timer_ns() - start <= limit && i <= 0x40000000u; ++i)
      if (ptx::mbar_try_wait_sleep(bar, parity, 1000u)) return;
    atomicOr(status, GG_STATUS_TIMEOUT_PRODUCER);
  }
  asm volatile("st.shared.s32 [%0], %1;" ::"r"(ptx::smem_addr(&s_gave_up)), "r"(1) : "memory");
}

// The kernel's work is cut into tasks: a tile (16 outputs) of a busy expert against a chunk of up to 8 kNT of
// its rows. A group of `splits` warps of a block takes a contiguous range of the tasks; each of its
// warps has a contiguous share of k, and they add their sums up in shared memory, in order. Ranges differ by
// at most one task, and the blocks that share an SM have neighbouring ones. A warp's blocks of a tile
// lie one after the other: it keeps two stages of up to kStageBlocks of them coming, one bulk copy each,
// started by its first lane as soon as the warp is through with a stage, whatever task comes next.
constexpr int kTaskCost = 2;
constexpr int kStageBlocks = 4;
constexpr int kStages = 2;
constexpr int kSumPitch = 20;  // floats per row of the warps' sums: no two lanes meet in a bank

// The busy experts, found from the counts by every block for itself.
struct Q4Work {
  int* expert;  // busy experts, in order
  int* row0;    // their first packed row
  int* rows;
  int* chunk0;  // their first chunk; one more entry: all chunks
  int* weight0; // the same of the weights of their chunks
  int splits, tasks, weight;
};

// A place in the sequence of tasks: expert by expert, tile by tile, in a tile chunk by chunk (those after the
// first find the weights in L2).
struct Q4Place {
  int cur, tile, chunk, chunks;  // busy expert, tile, chunk of the expert's chunks
  int left;                      // tasks left of the range, this one included
};

// What a task weighs when the ranges are cut: a chunk of more than 8 rows against one of up to 8 (64 rows on eight
// experts of 4096 x 14336, 3 to 14 each: 71 us with these, 78 with equal ones, 76 with 3 and 5).
constexpr int kWeight8 = 3, kWeight16 = 4;

// The weight of an expert's chunks: all but the last have 8 kNT rows.
template <int kNT>
__device__ __forceinline__ int chunks_weight(int rows) {
  constexpr int kFull = kNT == 1 ? kWeight8 : kWeight16;
  const int rest = rows % (8 * kNT);
  return rows / (8 * kNT) * kFull + (rest == 0 ? 0 : rest <= 8 ? kWeight8 : kWeight16);
}

// The first task that starts at or after a weight, as its number; the place of a number.
template <int kNT>
__device__ __forceinline__ int task_at(const Q4Work& w, int n_tiles, int weight, int* expert) {
  int cur = 0;
  while (w.weight0[cur + 1] * n_tiles <= weight) ++cur;
  *expert = cur;
  constexpr int kFull = kNT == 1 ? kWeight8 : kWeight16;
  const int chunks = w.chunk0[cur + 1] - w.chunk0[cur], per_tile = w.weight0[cur + 1] - w.weight0[cur];
  const int in = weight - w.weight0[cur] * n_tiles, tile = in / per_tile;
  return w.chunk0[cur] * n_tiles + tile * chunks + min(chunks, (in - tile * per_tile + kFull - 1) / kFull);
}

__device__ __forceinline__ Q4Place place_of(const Q4Work& w, int n_tiles, int task, int end, int cur) {
  Q4Place c{cur, 0, 0, 1, end - task};
  if (c.left <= 0) return c;
  while (w.chunk0[c.cur + 1] * n_tiles <= task) ++c.cur;
  c.chunks = w.chunk0[c.cur + 1] - w.chunk0[c.cur];
  const int in = task - w.chunk0[c.cur] * n_tiles;
  c.tile = in / c.chunks;
  c.chunk = in - c.tile * c.chunks;
  return c;
}

// To the next task; true where that is of another tile.
__device__ __forceinline__ bool advance(const Q4Work& w, int n_tiles, Q4Place& c) {
  if (--c.left <= 0) return false;
  if (++c.chunk < c.chunks) return false;
  c.chunk = 0;
  if (++c.tile == n_tiles) {
    c.tile = 0;
    ++c.cur;
    c.chunks = w.chunk0[c.cur + 1] - w.chunk0[c.cur];
  }
  return true;
}

template <bool kBf16, int kPer, bool kZeros, int kNT, int kLoad>
struct Q4Warp {
  static constexpr int kRecord = record_bytes(kPer, kZeros);
  static constexpr int kStageBytes = kStageBlocks * kRecord;
  const Q4Params& p;
  const Q4Work& work;
  const unsigned char* ring;  // this lane's 16 bytes of the first stage
  uint32_t ring_address, bars;  // the first stage and the stages' barriers as shared addresses
  int warp, lane;
  int share, kb0, run;  // the warp's share of k: blocks [kb0, kb0 + run)

  // The copies run ahead of the arithmetic with a place of their own.
  struct Ahead {
    Q4Place place;
    int left;                   // blocks of the task that are not under way
    const unsigned char* from;  // the next of them
  };
  __device__ __forceinline__ void enter(Ahead& c) const {
    c.left = c.place.left > 0 ? run : 0;
    if (c.left > 0)
      c.from = p.blocks + ((static_cast<int64_t>(work.expert[c.place.cur]) * p.n_tiles + c.place.tile) * p.k_blocks + kb0) * kRecord;
  }
  // Starts the copy of the next blocks into a stage.
  __device__ __forceinline__ void fetch(Ahead& c, int stage) const {
    if (c.left <= 0) return;
    const int blocks = min(kStageBlocks, c.left);
    if (lane == 0 && !gave_up()) {
      ptx::mbar_arrive_expect_tx(bars + 8 * stage, blocks * kRecord);
      copy_bulk(ring_address + stage * kStageBytes, c.from, blocks * kRecord, bars + 8 * stage);
    }
    c.from += blocks * kRecord;
    c.left -= blocks;
    if (c.left == 0) {
      advance(work, p.n_tiles, c.place);
      enter(c);
    }
  }

  // 16 outputs x 32 k (word i of the lane's pieces) against 8 rows: two products.
  static __device__ __forceinline__ unsigned word(const uint4& q, int i) {  // i is known at compile time
    return i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w;
  }
  static __device__ __forceinline__ void multiply(float (&part)[4], bool first, const unsigned (&f0)[4], const unsigned (&f1)[4],
                                                  const uint4& x) {
    mma16816<kBf16>(part, first, f0[0], f1[0], f0[1], f1[1], x.x, x.y);
    mma16816<kBf16>(part, false, f0[2], f1[2], f0[3], f1[3], x.z, x.w);
  }
  static __device__ __forceinline__ void scale_add(float (&acc)[4], const float2& s, const float (&part)[4]) {
    acc[0] = fmaf(s.x, part[0], acc[0]);
    acc[1] = fmaf(s.x, part[1], acc[1]);
    acc[2] = fmaf(s.y, part[2], acc[2]);
    acc[3] = fmaf(s.y, part[3], acc[3]);
  }

  // One block, 16 outputs x 128 k, against NT x 8 rows. at: this lane's first 16 bytes of the block; x: the
  // lane's activations of its four words; reload(i): called when word i is used.
  template <int NT, typename Reload>
  __device__ __forceinline__ void multiply_block(const unsigned char* at, const uint4 (&x)[4][NT], float (&acc)[NT][4],
                                                 const Reload& reload) const {
    const uint4 q0 = *reinterpret_cast<const uint4*>(at), q1 = *reinterpret_cast<const uint4*>(at + 512);
    const unsigned char* meta = at - 16 * lane + kBlockBytes;
    const int first = lane / 4 * kPer;
#pragma unroll
    for (int sub = 0; sub < kPer; ++sub) {
      unsigned zz = 0x0808u;
      if constexpr (kZeros) zz = reinterpret_cast<const unsigned short*>(meta + 32 * kPer)[first + sub];
      const Q4Zero<kBf16, 0> z0(zz);
      const Q4Zero<kBf16, 1> z1(zz);
      float part[NT][4];
#pragma unroll
      for (int i = sub * (4 / kPer); i < (sub + 1) * (4 / kPer); ++i) {
        unsigned f0[4], f1[4];
        unpack8<kBf16>(word(q0, i), z0, f0);
        unpack8<kBf16>(word(q1, i), z1, f1);
#pragma unroll
        for (int j = 0; j < NT; ++j) multiply(part[j], i == sub * (4 / kPer), f0, f1, x[i][j]);
        reload(i);
      }
      const float2 s = unpack2<Q4Type<kBf16>::kOut>(reinterpret_cast<const unsigned*>(meta)[first + sub]);
#pragma unroll
      for (int j = 0; j < NT; ++j) scale_add(acc[j], s, part[j]);
    }
  }

  // Where this lane's activations start, of column lane / 4 of each 8 rows and the warp's share of k; they
  // change with the expert and the chunk, not with the outputs.
  struct Rows {
    int row0 = -1;
    const unsigned short* at[kNT];
  };
  __device__ __forceinline__ void find_rows(int row0, int count, Rows& r) const {
    if (row0 == r.row0) return;
    r.row0 = row0;
#pragma unroll
    for (int j = 0; j < kNT; ++j) {
      // a column past the chunk's rows is computed and not stored: it reads the first row again
      int64_t row = row0 + (8 * j + lane / 4 < count ? 8 * j + lane / 4 : 0);
      if (p.row_tokens) row = __ldg(p.row_tokens + row);
      r.at[j] = (row >= 0 && row < p.a_rows ? static_cast<const unsigned short*>(p.a) + row * p.lda : p.no_row) + kBlockK * kb0 +
                8 * (lane % 4);
    }
  }

  // This warp's share of one task, then the group's sums and the outputs. `stage`, `parity`: of the next stage.
  template <int NT>
  __device__ __forceinline__ void compute(int e, int tile, int count, const Rows& r, Ahead& ahead, int& stage, uint32_t& parity,
                                          float* sums, int& flip) const {
    const int g = lane / 4, t4 = lane % 4;
    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[j][v] = 0.0f;
    const unsigned short* rows[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) rows[j] = r.at[j];
    int k_left = p.k - kBlockK * kb0;  // activations of a row from the block on
    // Eight activations of 32-k word i from rows[j] on; past k (checked where a word may reach it) zeros.
    const auto load = [&](int i, int j, auto check) {
      if constexpr (kLoad != 8) return load_units<kLoad>(rows[j] + 32 * i, k_left - 32 * i - 8 * t4);
      else if constexpr (check()) return __ldg(reinterpret_cast<const uint4*>(k_left > 32 * i + 8 * t4 ? rows[j] + 32 * i : p.no_row));
      else return __ldg(reinterpret_cast<const uint4*>(rows[j] + 32 * i));
    };
    // A block's words in registers, each read again, of the next block, as soon as it is used.
    uint4 x[4][NT];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) x[i][j] = load(i, j, std::true_type());
    // Blocks [b, b + count) of the stage, as one piece of code: their addresses are constants from two bases.
    const auto blocks_of = [&](const unsigned char* at, auto count, auto check) {
      constexpr int kCount = count();
#pragma unroll
      for (int b = 0; b < kCount; ++b)
        multiply_block<NT>(at + b * kRecord, x, acc, [&](int i) {
#pragma unroll
          for (int j = 0; j < NT; ++j) x[i][j] = load(4 * b + i + 4, j, check);
        });
      k_left -= kCount * kBlockK;
#pragma unroll
      for (int j = 0; j < NT; ++j) rows[j] += kCount * kBlockK;
    };
    constexpr int kTogether = kLoad == 8 ? 2 : 1;
    for (int left = run; left > 0; left -= kStageBlocks) {
      wait_bounded(bars + 8 * stage, parity, p.timeout_ns, p.status);
      const unsigned char* at = ring + stage * kStageBytes;
      int blocks = min(kStageBlocks, left);
      // The words ahead are of these blocks and the next: within k for all lanes, or else looked at (past the
      // warp's last block they may be another share's: not used).
      if constexpr (kLoad == 8) {
#pragma unroll 1
        for (; blocks >= kTogether && k_left >= (kTogether + 1) * kBlockK; blocks -= kTogether, at += kTogether * kRecord)
          blocks_of(at, std::integral_constant<int, kTogether>(), std::false_type());
      }
#pragma unroll 1
      for (; blocks > 0; --blocks, at += kRecord) blocks_of(at, std::integral_constant<int, 1>(), std::true_type());
      __syncwarp();  // all lanes are through with the stage
      fetch(ahead, stage);
      stage ^= 1;
      parity ^= stage == 0;
    }
    const int first = warp - share, id = 32 * share + lane;  // the group's first warp; the thread in the group
    const float* bias = p.bias ? p.bias[e] : nullptr;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if (8 * j >= count) break;  // the same for the whole group
      // [warp][row][output], in two buffers: a thread may still read the last one when another writes
      float* mine = sums + (flip * kQ4Warps + warp) * 8 * kSumPitch + 2 * t4 * kSumPitch + g;
      mine[0] = acc[j][0];
      mine[kSumPitch] = acc[j][1];
      mine[8] = acc[j][2];
      mine[kSumPitch + 8] = acc[j][3];
      if (work.splits > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + first / work.splits), "r"(32 * work.splits) : "memory");
      else __syncwarp();
      for (int i = id; i < 8 * kTileN; i += 32 * work.splits) {
        const int row = i / kTileN, o = kTileN * tile + i % kTileN;
        if (8 * j + row >= count || o >= p.n) continue;
        const float* from = sums + ((flip * kQ4Warps + first) * 8 + row) * kSumPitch + i % kTileN;
        float sum = 0.0f;
        for (int w = 0; w < work.splits; ++w) sum += from[w * 8 * kSumPitch];
        if (bias) sum += __ldg(bias + o);
        store_out_rt(p.output_type, p.d, static_cast<int64_t>(r.row0 + 8 * j + row) * p.ldd + o, q4_activate(sum, p.activation));
      }
      flip ^= 1;
    }
  }
};

// The busy experts and the split, by one warp. False: the counts are not valid.
template <int kNT>
__device__ __forceinline__ bool find_work(const Q4Params& p, Q4Work& w, int lane) {
  constexpr int most_rows = 8 * kNT;
  int busy = 0, chunks = 0, weights = 0;
  int64_t row = 0;
  bool bad = false;
  for (int e0 = 0; e0 < p.experts; e0 += 32) {
    const int e = e0 + lane;
    const int rows = e >= p.experts ? 0 : p.rows ? p.rows[e] : p.capacity_rows;
    bad |= rows < 0;
    const int mine = max(0, rows);
    int64_t upto = mine;
    const int counted = min(mine, p.capacity_rows);
    int chunk = (counted + most_rows - 1) / most_rows, weight = chunks_weight<kNT>(counted);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, upto, d);
      const int cu = __shfl_up_sync(0xffffffffu, chunk, d), wu = __shfl_up_sync(0xffffffffu, weight, d);
      if (lane >= d) upto += up, chunk += cu, weight += wu;
    }
    const unsigned has = __ballot_sync(0xffffffffu, mine > 0);
    const int at = busy + __popc(has & ((1u << lane) - 1u));
    if (mine > 0) {
      w.expert[at] = e;
      w.rows[at] = mine;
      w.row0[at] = static_cast<int>(min(static_cast<int64_t>(p.capacity_rows), row + upto - mine));
      w.chunk0[at + 1] = chunks + chunk;
      w.weight0[at + 1] = weights + weight;
    }
    busy += __popc(has);
    row += __shfl_sync(0xffffffffu, upto, 31);
    chunks += __shfl_sync(0xffffffffu, chunk, 31);
    weights += __shfl_sync(0xffffffffu, weight, 31);
    // a sum past the rows there are is refused below; stopping here keeps the sums from overflowing
    if (row > p.capacity_rows) break;
  }
  if (lane == 0) w.chunk0[0] = w.weight0[0] = 0;
  bad = __any_sync(0xffffffffu, bad) || row > p.capacity_rows || (p.row_tokens == nullptr && row > p.a_rows);
  w.tasks = bad ? 0 : chunks * p.n_tiles;
  w.weight = weights * p.n_tiles;
  // The split whose longest group is done first: its tasks times a share's blocks and what a task costs besides
  // (its sums and outputs, about kTaskCost blocks). One warp takes about as long for a block whether all or
  // half of an SM's warps are busy, so few whole shares beat many with a short last round: 896 tasks of 32
  // blocks take 13.3 us in two shares, 14.7 in eight.
  const float warps = static_cast<float>(kQ4Warps * gridDim.x);
  float least = INFINITY;
  w.splits = 1;
  for (int splits = 1; splits <= kQ4Warps && splits <= p.k_blocks; splits *= 2) {
    const float longest = ceilf(__fdividef(static_cast<float>(w.tasks) * splits, warps));
    const float cost = longest * (static_cast<float>((p.k_blocks + splits - 1) / splits) + kTaskCost);
    if (cost < least) least = cost, w.splits = splits;
  }
  return !bad;
}

// kPer: groups per 128-k block (1, 2 or 4). kNT: most rows of an expert worked on together, in eights. kLoad:
// elements of the activations read at a time: 8 (aligned rows, k a multiple of 8), 2 or 1.
template <bool kBf16, int kPer, bool kZeros, int kNT, int kLoad>
__global__ void __launch_bounds__(kQ4Threads, 2) q4_kernel(const __grid_constant__ Q4Params p) {
  using Warp = Q4Warp<kBf16, kPer, kZeros, kNT, kLoad>;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int s_plan[3];
  const int tid = static_cast<int>(threadIdx.x), warp = tid / 32, lane = tid % 32;
  float* sums = reinterpret_cast<float*>(smem + kQ4Warps * kStages * Warp::kStageBytes);
  __shared__ uint64_t s_bars[kQ4Warps][kStages];
  Q4Work work;
  work.expert = reinterpret_cast<int*>(sums + 2 * kQ4Warps * 8 * kSumPitch);
  work.row0 = work.expert + p.experts;
  work.rows = work.row0 + p.experts;
  work.chunk0 = work.rows + p.experts;
  work.weight0 = work.chunk0 + p.experts + 1;
  if (tid < kQ4Warps * kStages) {
    ptx::mbar_init(ptx::smem_addr(&s_bars[0][0] + tid), 1);
    ptx::fence_mbar_init();
  }
  if (tid == 0) s_gave_up = 0;
  chained_begin();
  if (warp == 0) {
    const bool good = find_work<kNT>(p, work, lane);
    if (lane == 0) {
      s_plan[0] = work.splits, s_plan[1] = work.tasks, s_plan[2] = work.weight;
      if (!good && blockIdx.x == 0) atomicOr(p.status, GG_STATUS_BAD_ROWS);
    }
  }
  __syncthreads();
  work.splits = s_plan[0], work.tasks = s_plan[1], work.weight = s_plan[2];

  // the group's range: blocks b, b + SMs, ... (which share an SM) are neighbours
  const int per_sm = gridDim.x % p.sms == 0 ? gridDim.x / p.sms : 0;
  const int rank = per_sm ? blockIdx.x % p.sms * per_sm + blockIdx.x / p.sms : blockIdx.x;
  const int groups = gridDim.x * (kQ4Warps / work.splits), group = rank * (kQ4Warps / work.splits) + warp / work.splits;
  // Rounded alike for the end of one range and the start of the next; the last ends with the tasks. Where all
  // tasks weigh the same the weights are the tasks.
  const int total = kNT == 1 ? work.tasks : work.weight;
  const float share_of = __fdividef(static_cast<float>(total), static_cast<float>(groups));
  int cur = 0, other;
  const auto start = [&](int g, int* at) {
    const int weight = __float2int_rz(g * share_of);
    if (work.tasks == 0 || g == groups || weight >= total) return work.tasks;
    if constexpr (kNT == 1) return weight;
    else return task_at<kNT>(work, p.n_tiles, weight, at);
  };
  const int begin = start(group, &cur), end = start(group + 1, &other);
  Q4Place place = place_of(work, p.n_tiles, begin, end, cur);

  const int share = warp % work.splits, kb0 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * share / work.splits);
  const unsigned char* ring = smem + warp * kStages * Warp::kStageBytes;
  const Warp w{p, work, ring + 16 * lane, ptx::smem_addr(ring), ptx::smem_addr(s_bars[warp]), warp, lane, share, kb0,
               static_cast<int>(static_cast<int64_t>(p.k_blocks) * (share + 1) / work.splits) - kb0};
  typename Warp::Ahead ahead{place, 0, nullptr};
  w.enter(ahead);
  for (int i = 0; i < kStages; ++i) w.fetch(ahead, i);
  int stage = 0, flip = 0;
  uint32_t parity = 0;
  typename Warp::Rows rows;
  for (; place.left > 0; advance(work, p.n_tiles, place)) {
    const int most = 8 * kNT, row0 = work.row0[place.cur] + most * place.chunk;
    const int count = min(most, work.rows[place.cur] - most * place.chunk);
    const int e = work.expert[place.cur];
    w.find_rows(row0, count, rows);
    if (kNT == 1 || count <= 8) w.template compute<1>(e, place.tile, count, rows, ahead, stage, parity, sums, flip);
    else w.template compute<kNT>(e, place.tile, count, rows, ahead, stage, parity, sums, flip);
  }
}

template <int kPer, bool kZeros>
size_t q4_smem(int experts) {
  return static_cast<size_t>(kQ4Warps) * kStages * kStageBlocks * record_bytes(kPer, kZeros) + 2 * kQ4Warps * 8 * kSumPitch * sizeof(float) +
         (5 * static_cast<size_t>(experts) + 2) * sizeof(int);
}

// The variants of a run, by the most rows any expert can have: 8, whose registers let the compiler order the block
// more freely, or 16 at a time (32 at a time, in spilled registers, took 34 us where two chunks of 16, the second from
// L2, take 30); and by the units in which the activations are read: 8, 2 or single elements, the last 8 rows at
// a time only (the loads of 16 rows start a task too slowly: 19 rows of k 257 took 7.2 us, 5.2 so).
enum Q4Variant { kQ4Single8, kQ4Pairs8, kQ4Pairs16, kQ4Rows8, kQ4Rows16, kQ4Variants };

template <typename F>
void with_variant(int v, F f) {
  using std::integral_constant;
  if (v == kQ4Single8) f(integral_constant<int, 1>(), integral_constant<int, 1>());
  else if (v == kQ4Pairs8) f(integral_constant<int, 1>(), integral_constant<int, 2>());
  else if (v == kQ4Pairs16) f(integral_constant<int, 2>(), integral_constant<int, 2>());
  else if (v == kQ4Rows8) f(integral_constant<int, 1>(), integral_constant<int, 8>());
  else f(integral_constant<int, 2>(), integral_constant<int, 8>());
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
  void* block = nullptr;  // blocks of weights | bias table | status | a row of zeros | the caller's pointers
  gg::Q4Params params{};
  bool bf16 = false, zeros = false;
  int per_block = 1, device = 0;
  int grid[gg::kQ4Variants] = {};  // resident blocks of each variant
  size_t smem = 0;
};

extern "C" {

int gg_q4_plan_create(const gg_q4_problem* problem, void* stream, gg_q4_plan** out) {
  if (!out) return cudaErrorInvalidValue;
  *out = nullptr;
  if (!problem) return cudaErrorInvalidValue;
  const gg_q4_problem& q = *problem;
  if (q.experts < 1 || q.experts > GG_Q4_MAX_EXPERTS || q.n < 1 || q.k < 1 || q.ldq < q.k / 2 + q.k % 2 || !q.q || !q.scales ||
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
  const int record = gg::record_bytes(per_block, q.zeros != nullptr);
  const size_t bias_at = up(blocks * record);
  const size_t status_at = up(bias_at + E * sizeof(void*));
  const size_t no_row_at = up(status_at + sizeof(int));
  const size_t tables_at = up(no_row_at + static_cast<size_t>(q.k) * 2);  // the caller's pointers, read once
  const size_t bytes = tables_at + 3 * E * sizeof(void*);

  gg_q4_plan* plan = new (std::nothrow) gg_q4_plan();
  if (!plan) return cudaErrorMemoryAllocation;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const void* tables[3 * GG_Q4_MAX_EXPERTS];
  for (size_t e = 0; e < E; ++e) {
    tables[e] = q.q[e];
    tables[E + e] = q.scales[e];
    tables[2 * E + e] = q.zeros ? q.zeros[e] : nullptr;
  }
  int device = 0, sms = 0, per_sm[gg::kQ4Variants] = {};
  size_t smem = 0;
  cudaError_t st = cudaGetDevice(&device);
  if (st == cudaSuccess) st = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (st == cudaSuccess)
    gg::with_q4(q.input_type == GG_INPUT_BF16, per_block, q.zeros != nullptr, [&](auto b, auto n, auto z) {
      smem = gg::q4_smem<n(), z()>(q.experts);
      for (int v = 0; v < gg::kQ4Variants && st == cudaSuccess; ++v)
        gg::with_variant(v, [&](auto nt, auto load) {
          const auto kernel = gg::q4_kernel<b(), n(), z(), nt(), load()>;
          st = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(gg::q4_smem<n(), z()>(GG_Q4_MAX_EXPERTS)));
          if (st == cudaSuccess) st = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm[v], kernel, gg::kQ4Threads, smem);
        });
    });
  if (st == cudaSuccess) st = cudaMalloc(&plan->block, bytes);
  if (st != cudaSuccess) {
    delete plan;
    return st;
  }
  unsigned char* base = static_cast<unsigned char*>(plan->block);
  st = cudaMemcpyAsync(base + tables_at, tables, 3 * E * sizeof(void*), cudaMemcpyHostToDevice, s);
  if (st == cudaSuccess && q.bias)
    st = cudaMemcpyAsync(base + bias_at, q.bias, E * sizeof(void*), cudaMemcpyHostToDevice, s);
  if (st == cudaSuccess) st = cudaMemsetAsync(base + status_at, 0, tables_at - status_at, s);
  if (st == cudaSuccess) {
    const unsigned char* const* table = reinterpret_cast<const unsigned char* const*>(base + tables_at);
    gg::Q4PackParams pk{table,   reinterpret_cast<const void* const*>(table + E), table + 2 * E, base,   q.experts, q.n,
                        q.k,     q.group, n_tiles, k_blocks, per_block, record, q.zeros != nullptr, q.ldq};
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
  p.blocks = base;
  p.sms = sms;
  p.bias = q.bias ? reinterpret_cast<const float* const*>(base + bias_at) : nullptr;
  p.status = reinterpret_cast<int*>(base + status_at);
  p.no_row = reinterpret_cast<const unsigned short*>(base + no_row_at);
  p.experts = q.experts;
  p.n = q.n;
  p.k = q.k;
  p.n_tiles = n_tiles;
  p.k_blocks = k_blocks;
  p.timeout_ns = gg::wait_limit_ns();
  p.output_type = q.output_type;
  p.activation = q.activation;
  plan->bf16 = q.input_type == GG_INPUT_BF16;
  plan->zeros = q.zeros != nullptr;
  plan->per_block = per_block;
  plan->device = device;
  for (int v = 0; v < gg::kQ4Variants; ++v) plan->grid[v] = std::max(1, sms * per_sm[v]);
  plan->smem = smem;
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
  p.a = a;
  p.lda = lda;
  p.a_rows = a_rows;
  p.row_tokens = row_tokens;
  p.rows = rows;
  p.d = d;
  p.ldd = ldd;
  p.capacity_rows = capacity_rows;
  // units that the rows' starts and their length are multiples of (a last unit past k would read other values)
  const auto made_of = [&](int unit) { return reinterpret_cast<uintptr_t>(a) % (2 * unit) == 0 && lda % unit == 0 && p.k % unit == 0; };
  const bool few = capacity_rows <= 8;
  const int variant = made_of(8)   ? (few ? gg::kQ4Rows8 : gg::kQ4Rows16)
                      : made_of(2) ? (few ? gg::kQ4Pairs8 : gg::kQ4Pairs16)
                                   : gg::kQ4Single8;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t st = gg::expect_device(plan->device);
  if (st != cudaSuccess) return st;
  gg::with_variant(variant, [&](auto nt, auto load) {
    // tasks and their weights are counted in an int: one task per tile of each chunk of rows, chunks at most this
    const int64_t chunks = std::min<int64_t>(capacity_rows, static_cast<int64_t>(capacity_rows) / (8 * nt()) + p.experts);
    const int64_t most = chunks * p.n_tiles;
    if (most > INT32_MAX / gg::kWeight16) {
      st = cudaErrorInvalidValue;
      return;
    }
    const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(plan->grid[variant], most)));
    gg::with_q4(plan->bf16, plan->per_block, plan->zeros, [&](auto b, auto n, auto z) {
      st = gg::launch_chained(gg::q4_kernel<b(), n(), z(), nt(), load()>, dim3(grid), gg::kQ4Threads, plan->smem, s, 1, p);
    });
  });
  return st;
}

int gg_q4_plan_status(gg_q4_plan* plan, int* status) {
  if (!plan || !plan->block) return cudaErrorInvalidDevicePointer;
  if (!status) return cudaErrorInvalidValue;
  cudaError_t st = gg::expect_device(plan->device);
  if (st == cudaSuccess) st = cudaDeviceSynchronize();
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
