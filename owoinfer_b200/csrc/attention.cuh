// Device helpers of the attention kernels: bounded waits, packed fp32 arithmetic, the hardware's exponential, 16-bit MMAs.
#pragma once

#include "common.cuh"

namespace b2 {

__device__ __forceinline__ std::uint64_t global_ns() {
  std::uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ bool wait_bar(std::uint32_t bar, std::uint32_t parity, volatile int* abort_word) {
  if (mbar_try_wait(bar, parity)) return true;
  const std::uint64_t t0 = global_ns();
  for (;;) {
    // A tight inner loop (test, branch); the abort word and the clock are looked at once per 256 tests.
#pragma unroll 1
    for (int i = 0; i < 256; ++i) {
      if (mbar_try_wait_hint(bar, parity)) return true;
    }
    if (*abort_word != 0) return false;
    if (global_ns() - t0 > 200000000ull) {
      *abort_word = 1;
      return false;
    }
  }
}

// The same for a whole converged warp with one answer, in as little code as that takes.
__device__ __forceinline__ bool warp_wait_bar(std::uint32_t bar, std::uint32_t parity, volatile int* abort_word) {
  if (__builtin_expect(__all_sync(0xffffffffu, mbar_try_wait(bar, parity)), 1)) return true;
  const std::uint64_t t0 = global_ns();
#pragma unroll 1
  while (!__all_sync(0xffffffffu, mbar_try_wait_hint(bar, parity))) {
    if (__any_sync(0xffffffffu, *abort_word != 0 || global_ns() - t0 > 200000000ull)) {
      *abort_word = 1;
      return false;
    }
  }
  return true;
}

// The same for a role with slack (the TMA and MMA warps share their scheduler with softmax warps): sleeps between tests so
// that waiting costs next to no issue slots.
template <int kSleepNs>
__device__ __forceinline__ bool wait_bar_relaxed(std::uint32_t bar, std::uint32_t parity, volatile int* abort_word) {
  if (mbar_try_wait(bar, parity)) return true;
  const std::uint64_t t0 = global_ns();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i) {
      __nanosleep(kSleepNs);
      if (mbar_try_wait(bar, parity)) return true;
    }
    if (*abort_word != 0) return false;
    if (global_ns() - t0 > 200000000ull) {
      *abort_word = 1;
      return false;
    }
  }
}

// Packed fp32 pairs (one instruction for two lanes of work): d = a * b + c and d = a + b on (x, y) pairs.
__device__ __forceinline__ std::uint64_t pack2(float x, float y) {
  std::uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack2(std::uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ std::uint64_t fma2(std::uint64_t a, std::uint64_t b, std::uint64_t c) {
  std::uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ std::uint64_t add2(std::uint64_t a, std::uint64_t b) {
  std::uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ std::uint64_t mul2(std::uint64_t a, std::uint64_t b) {
  std::uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// D[tmem] (+)= A[smem] * B[smem] for bf16 or fp16 operands, one thread issues.
__device__ __forceinline__ void umma_f16(std::uint32_t d_tmem, std::uint64_t a_desc, std::uint64_t b_desc,
                                          std::uint32_t idesc, std::uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The same with A in tensor memory: row r of A is lane r, two values to a 32-bit column in K order (K = 16 is eight columns).
__device__ __forceinline__ void umma_f16_ts(std::uint32_t d_tmem, std::uint32_t a_tmem, std::uint64_t b_desc,
                                            std::uint32_t idesc, std::uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Both for a CTA pair (see umma_i8_pair): 128 rows of A and of D in each CTA, half of B's N in each; issued by the pair's leader only.
__device__ __forceinline__ void umma_f16_pair(std::uint32_t d_tmem, std::uint64_t a_desc, std::uint64_t b_desc,
                                              std::uint32_t idesc, std::uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_f16_ts_pair(std::uint32_t d_tmem, std::uint32_t a_tmem, std::uint64_t b_desc,
                                                 std::uint32_t idesc, std::uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrive on an mbarrier of a CTA of the cluster for what tcgen05 fences order, tensor memory that is read or written: ordinary
// memory goes along at CTA scope only. (With release.cluster every such arrival waits some 900 clocks for the warp's other accesses.)
__device__ __forceinline__ void mbar_arrive_tensor(std::uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// 4-D tiled TMA load global -> shared, completion on an mbarrier of this CTA.
__device__ __forceinline__ void tma_load_4d(std::uint32_t dst, const CUtensorMap* map, std::uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<std::uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(std::uint32_t dst, const CUtensorMap* map, std::uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<std::uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// The same with completion on an mbarrier that may live in the peer CTA of the pair (shared::cluster address).
__device__ __forceinline__ void tma_load_4d_pair(std::uint32_t dst, const CUtensorMap* map, std::uint32_t bar_cluster_addr, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<std::uint64_t>(map)), "r"(bar_cluster_addr), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ uint4 ld_shared(std::uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared(std::uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

}  // namespace b2
