// Bounded waits on mbarriers, for every kernel with roles: a wait that runs into its limit records which one it was and makes the
// other roles of its CTA give up, too, so that the kernel returns.
#pragma once
#include "ptx_sm100.cuh"

namespace sk {

constexpr long long kWaitLimitCycles = 1000000000ll;  // default: every mbarrier wait gives up after 1e9 SM cycles (0.5-0.8 s)

// device status codes: role * 16 + barrier kind
enum : int {
  kStProducerEmpty = 0x11,
  kStExpanderFull = 0x21, kStExpanderEmpty = 0x22,
  kStMmaLdFull = 0x31, kStMmaExFull = 0x32, kStMmaAccEmpty = 0x33,
  kStEpilogueAccFull = 0x41, kStEpilogueScales = 0x42,
  kStDrain = 0x51,
  kStStreamSlots = 0x61   // balanced-split decode kernel: host and device disagree on how a tile is cut (never expected)
};

struct WaitCtx {
  volatile int* abort_flag;  // shared memory
  int* status;               // global
  long long limit;           // SM cycles
};

// Slow path of a bounded wait (inlined: a real call inside a kernel that re-partitions registers with setmaxnreg
// does not compile); the fast path in wait_bounded is a single poll.
// The limit is counted on the SM clock (%globaltimer costs about a microsecond per read).
__device__ __forceinline__ bool wait_slow(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code,
                                          long long limit) {
  const long long t0 = clock64();
  for (uint32_t spins = 1;; ++spins) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((spins & 63u) == 0) {
      if (*abort_flag) return false;
      if (clock64() - t0 > limit) {
        *abort_flag = 1;
        atomicCAS(status, 0, code);
        return false;
      }
    }
  }
}
// Bounded wait.  Returns false if the limit expired here or in any other thread of the CTA.
__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity, const WaitCtx& ctx, int code) {
  if (mbar_try_wait(bar, parity)) return true;
  return wait_slow(bar, parity, ctx.abort_flag, ctx.status, code, ctx.limit);
}

// Bounded wait for two barriers: where both are complete already, as they mostly are, the two polls overlap and there is one
// branch.
__device__ __forceinline__ bool wait_bounded_two(uint32_t bar_a, uint32_t parity_a, uint32_t bar_b, uint32_t parity_b, const WaitCtx& ctx,
                                                 int code_a, int code_b) {
  long long t0 = 0;
  for (uint32_t spins = 0;; ++spins) {
    const bool a = mbar_try_wait(bar_a, parity_a), b = mbar_try_wait(bar_b, parity_b);
    if (a && b) return true;
    if ((spins & 63u) == 0) {
      if (spins == 0) t0 = clock64();
      if (*ctx.abort_flag) return false;
      if (clock64() - t0 > ctx.limit) {
        *ctx.abort_flag = 1;
        atomicCAS(ctx.status, 0, a ? code_b : code_a);
        return false;
      }
    }
  }
}

// Bounded wait for a role that is not on the critical path of a K block: sleeps between polls, so that it does not
// take issue slots and integer-pipe cycles from the warps that expand (the expansion saturates the integer pipe).
__device__ __forceinline__ bool wait_bounded_relaxed(uint32_t bar, uint32_t parity, const WaitCtx& ctx, int code,
                                                     unsigned sleep_ns) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  for (;;) {
    __nanosleep(sleep_ns);
    if (mbar_try_wait(bar, parity)) return true;
    if (*ctx.abort_flag) return false;
    if (clock64() - t0 > ctx.limit) {
      *ctx.abort_flag = 1;
      atomicCAS(ctx.status, 0, code);
      return false;
    }
  }
}

}  // namespace sk
