// Bounded waits of a kernel's roles on mbarriers. A wait that expires records an error in the caller's
// status word and raises the block's abort flag; every other role finds one or the other and drains.
#pragma once
#include "common.cuh"
#include "ptx.cuh"

namespace fga {

struct WaitCtx {
  int* status;
  unsigned long long timeout_ns;
  uint32_t abort_flag;  // shared address of this CTA's abort word
  bool dead;
};

__device__ __forceinline__ void report(WaitCtx& w, int code, int where, int detail) {
  if (atomicCAS(w.status, 0, code) == 0) {
    w.status[1] = where;
    w.status[2] = detail;
  }
  asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(w.abort_flag), "r"(1u) : "memory");
  w.dead = true;
}

__device__ __forceinline__ bool should_abort(WaitCtx& w) {
  uint32_t f;
  asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(f) : "r"(w.abort_flag) : "memory");
  if (f != 0 || ld_relaxed_sys_s32(w.status) != 0) {
    w.dead = true;
    return true;
  }
  return false;
}

// Bounded mbarrier wait. Returns false when the kernel is aborting.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, WaitCtx& w, int where) {
  if (w.dead) return false;
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  uint32_t it = 0;
  while (!mbar_try_wait(bar, parity)) {
    if ((++it & 0x3ff) == 0) {
      if (should_abort(w)) return false;
      if (globaltimer_ns() - t0 > w.timeout_ns) {
        report(w, kErrPipelineTimeout, where, static_cast<int>(bar));
        return false;
      }
    }
  }
  return true;
}

// The same with as little as possible in front of and inside the spin: what a role executes once per tile has
// to come from the instruction cache each time, beside the other roles' code.
__device__ __forceinline__ bool wait_small(uint32_t bar, uint32_t parity, WaitCtx& w, int where) {
  if (w.dead) return false;
  uint64_t since = 0;
#pragma unroll 1
  for (uint32_t it = 1;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if (__builtin_expect((it & 0x3ff) == 0, 0)) {
      if (should_abort(w)) return false;
      const uint64_t now = globaltimer_ns();
      if (since == 0) {
        since = now;
      } else if (now - since > w.timeout_ns) {
        report(w, kErrPipelineTimeout, where, static_cast<int>(bar));
        return false;
      }
    }
  }
}
// For a converged warp whose lanes must take the same way afterwards.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, WaitCtx& w, int where) {
  const bool ok = __all_sync(0xffffffffu, wait_small(bar, parity, w, where));
  w.dead = !ok;
  return ok;
}

}  // namespace fga
