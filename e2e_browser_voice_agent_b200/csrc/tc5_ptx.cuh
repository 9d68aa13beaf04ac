// Wrappers of the Blackwell instructions that the tensor-core kernels share: mbarriers with bounded waits, TMA loads,
// shared-memory matrix descriptors, tcgen05 fences, commits and TMEM loads.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace h2 {

// cuTensorMapEncodeTiled of the process's driver, nullptr without one (tc5.cu)
PFN_cuTensorMapEncodeTiled_v12000 tma_encode_fn();

namespace {

constexpr unsigned long long TIMEOUT_NS = 1000000000ull;

__device__ __forceinline__ uint32_t su32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t* b, unsigned n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(b)), "r"(n));
}
__device__ __forceinline__ void bar_expect(uint64_t* b, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(su32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(b)) : "memory");
}
// (with a suspend-time hint: a waiting thread sleeps in hardware until the phase completes, or at most ~20 us,
// instead of polling; polling warps crowd the shared-memory pipe that the working warps need)
__device__ __forceinline__ bool bar_try(uint64_t* b, unsigned parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(su32(b)), "r"(parity), "r"(20000u)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

struct Abort {
  volatile int* flag;  // shared: any role of the CTA raised it
  int* err;            // global: {code, CTA, role, 0}
};
__device__ __noinline__ void raise_abort(const Abort& a, int role) {
  if (atomicCAS(a.err, 0, 1) == 0) {
    a.err[1] = blockIdx.x;
    a.err[2] = role;
  }
  *a.flag = 1;
}
// bounded wait for the completion of the phase with this parity; false (abort raised) on expiry or abort
__device__ __forceinline__ bool wait_phase(uint64_t* b, unsigned parity, const Abort& a, int role) {
  if (bar_try(b, parity)) return true;
  const unsigned long long t0 = now_ns();
  for (unsigned it = 0;; it++) {
    if (bar_try(b, parity)) return true;
    if ((it & 3) == 3) {
      if (*a.flag) return false;
      if (now_ns() - t0 > TIMEOUT_NS) {
        raise_abort(a, role);
        return false;
      }
    }
  }
}
// the same for a whole warp: lane 0 polls (32 lanes polling one mbarrier serialize on it) and the warp follows;
// false on every lane if it failed
__device__ __forceinline__ bool wait_phase_warp(uint64_t* b, unsigned parity, const Abort& a, int role) {
  int ok = 1;
  if ((threadIdx.x & 31) == 0) ok = wait_phase(b, parity, a, role);
  ok = __shfl_sync(0xffffffffu, ok, 0);
  __syncwarp();
  return ok != 0;
}
// the same, ignoring the abort flag (teardown: copies or MMAs that were issued must complete)
__device__ __forceinline__ void drain_phase(uint64_t* b, unsigned parity) {
  const unsigned long long t0 = now_ns();
  while (!bar_try(b, parity))
    if (now_ns() - t0 > TIMEOUT_NS) return;
}

__device__ __forceinline__ void tma2d(void* dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          su32(dst)),
      "l"((uint64_t)map), "r"(c0), "r"(c1), "r"(su32(bar))
      : "memory");
}
__device__ __forceinline__ void bulk1d(void* dst, const void* src, unsigned bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(su32(dst)),
               "l"(src), "r"(bytes), "r"(su32(bar))
               : "memory");
}

// shared-memory matrix descriptors (tcgen05): start address, leading / stride byte offsets (16-byte units), version 1
__device__ __forceinline__ uint64_t desc_plain(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46);
}
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (1ull << 16) | ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46) |
         (2ull << 61);
}

__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(su32(bar))
               : "memory");
}
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 lanes x 16 columns of 32-bit words (lane = the thread's TMEM lane) into v[0..16)
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}

}  // namespace
}  // namespace h2
