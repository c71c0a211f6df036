// gg_wait.cuh -- bounded waits on mbarriers, shared by the kernels whose warps hand work to one another.
#pragma once

#include <cstdint>

#include "gg_ptx.cuh"

namespace gg {

// ---- bounded waits ---------------------------------------------------------------------------
static __device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status,
                                              unsigned long long timeout_ns, int code) {
  const uint64_t t0 = ptx::global_timer_ns();
  for (uint32_t i = 0;; ++i) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    if ((i & 31u) == 31u) {
      if (*abort_flag) return false;
      if (ptx::global_timer_ns() - t0 > timeout_ns || i > 0x40000000u) {
        *abort_flag = 1;
        atomicOr(status, code);
        return false;
      }
    }
  }
}

__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status,
                                           unsigned long long timeout_ns, int code) {
  if (ptx::mbar_try_wait(bar, parity)) return true;
  return wait_slow(bar, parity, abort_flag, status, timeout_ns, code);
}

// The same without a call, for code that holds more in registers than a call lets it keep, and for waits that are mostly short:
// the clock is first read after 32 tries (a read takes some 300 cycles, more than what is waited for).
// kCluster: what another CTA of the cluster wrote before it arrived is visible then.
template <bool kCluster = false>
__device__ __forceinline__ bool wait_phase_inline(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status,
                                                  unsigned long long timeout_ns, int code) {
  uint64_t t0 = 0;
  for (uint32_t i = 0;; ++i) {
    if (kCluster ? ptx::mbar_try_wait_cluster(bar, parity) : ptx::mbar_try_wait(bar, parity)) return true;
    if ((i & 31u) == 31u) {
      if (*abort_flag) return false;
      const uint64_t now = ptx::global_timer_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > timeout_ns || i > 0x40000000u) {
        *abort_flag = 1;
        atomicOr(status, code);
        return false;
      }
    }
  }
}

// The same for a wait that lasts as long as many steps of others do, so that no limit on one step bounds it: the limit starts
// anew whenever `progress` has changed, two words in shared memory that those who take the steps count up.
template <bool kCluster = false>
__device__ __forceinline__ bool wait_progress_inline(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status,
                                                     unsigned long long timeout_ns, int code, const volatile uint32_t* progress) {
  uint64_t t0 = 0;
  uint32_t seen = 0;
  for (uint32_t i = 0;; ++i) {
    if (kCluster ? ptx::mbar_try_wait_cluster(bar, parity) : ptx::mbar_try_wait(bar, parity)) return true;
    if ((i & 31u) == 31u) {
      if (*abort_flag) return false;
      const uint64_t now = ptx::global_timer_ns();
      const uint32_t at = progress[0] + progress[1];
      if (t0 == 0 || at != seen) t0 = now, seen = at, i = 31u;
      if (now - t0 > timeout_ns || i > 0x40000000u) {
        *abort_flag = 1;
        atomicOr(status, code);
        return false;
      }
    }
  }
}

// Drain wait used after an abort: ignores the abort flag, gives up after `limit_ns`.
__device__ __forceinline__ void wait_drain_inline(uint32_t bar, uint32_t parity, unsigned long long limit_ns) {
  const uint64_t t0 = ptx::global_timer_ns();
  while (!ptx::mbar_try_wait(bar, parity)) {
    if (ptx::global_timer_ns() - t0 > limit_ns) return;
  }
}
static __device__ __noinline__ void wait_drain(uint32_t bar, uint32_t parity, unsigned long long limit_ns) {
  wait_drain_inline(bar, parity, limit_ns);
}

}  // namespace gg
