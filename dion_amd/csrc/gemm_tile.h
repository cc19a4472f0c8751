// Pieces the MFMA kernels share (gemm_nt.hip, linear.hip): waits, fragment reads from LDS, host-known divisions.
#pragma once
#include <type_traits>

#include "common.h"

namespace dion {

#define LDS_PTR(p) ((__attribute__((address_space(3))) void*)(p))
#define GLB_PTR(p) ((const __attribute__((address_space(1))) void*)(p))

// s_waitcnt with only vmcnt constrained (gfx9 encoding: vmcnt[3:0] | expcnt[6:4] | lgkmcnt[11:8]
// | vmcnt_hi[15:14]).
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | 0x0F70);
}

// Compile-time loop: f(std::integral_constant<int, I>()) for I in [I0, N).
template <int I, int N, class F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    static_for<I + 1, N>(f);
  }
}

// Fragment wait: an asm statement that takes the fragments it guards as read-write operands, so that to
// the compiler they are (re)defined here and no use of them can be scheduled ahead of the wait.
template <int N>
__device__ __forceinline__ void frag_wait(bf16x8& a, bf16x8& b) {
  asm volatile("s_waitcnt lgkmcnt(%2)" : "+v"(a), "+v"(b) : "n"(N));
}
// 16-byte LDS read at addr + OFF, issued from assembly (the compiler does not know it is in flight: the
// matching frag_wait is what its consumers wait on).
template <int OFF>
__device__ __forceinline__ void lds_read16(bf16x8& dst, uint32_t addr) {
  static_assert(OFF >= 0 && OFF < 65536, "ds offset field");
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(dst) : "v"(addr), "n"(OFF));
}
// K-major fragment: two transposing reads, rows k..k+3 and k+4..k+7 of the tile (HI bytes apart)
template <int OFF, int HI>
__device__ __forceinline__ void lds_read_tr(bf16x8& dst, uint32_t addr) {
  static_assert(OFF >= 0 && OFF + HI < 65536, "ds offset field");
  typedef __attribute__((ext_vector_type(2))) unsigned u32x2;
  typedef __attribute__((ext_vector_type(4))) unsigned u32x4f;
  u32x2 lo, hi;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(lo) : "v"(addr), "n"(OFF));
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(hi) : "v"(addr), "n"(OFF + HI));
  const u32x4f v = {lo[0], lo[1], hi[0], hi[1]};
  dst = __builtin_bit_cast(bf16x8, v);
}

// Quotient and remainder by a divisor the host knows: inv = (2^32 - 1) / d gives the quotient or one less for x < 2^31.
__device__ __forceinline__ int div_known(int x, int d, uint32_t inv, int& rem) {
  int q = (int)__umulhi((uint32_t)x, inv);
  rem = x - q * d;
  if (rem >= d) {
    rem -= d;
    ++q;
  }
  return q;
}

// Workgroup barrier preceded by the counter waits the software pipeline needs: every LDS read
// this wave issued has returned (the ring slot they read is about to be refilled) and all but the
// newest VM_LEFT direct-to-LDS loads of this wave have landed.  The "memory" clobber keeps the
// compiler from moving LDS accesses across it.
template <int VM_LEFT>
__device__ __forceinline__ void pipeline_barrier() {
  static_assert(VM_LEFT >= 0 && VM_LEFT < 64, "vmcnt range");
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  // vmcnt = VM_LEFT, lgkmcnt = 0, expcnt unconstrained (gfx9 s_waitcnt encoding).
  __builtin_amdgcn_s_waitcnt((VM_LEFT & 0xF) | ((VM_LEFT >> 4) << 14) | 0x0070);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

}  // namespace dion
