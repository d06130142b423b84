// Device helpers of the sequence kernels: packed fp32 arithmetic, parked waits,
// matrix instructions, and CTA pairs (tcgen05 cta_group::2): two CTAs of a
// cluster work on one 256-row tile.  Each holds its half of both operands and of the
// accumulator; the even CTA issues the matrix instructions for both.
#pragma once

#include "common.cuh"

namespace tgcm {

// Bounded wait that sleeps: a thread whose phase is not over is suspended by the
// hardware for up to 100 us a try instead of asking again at once, so waiting
// warps leave the issue slots to the ones that compute.
__device__ __forceinline__ bool mbar_park(uint64_t* bar, uint32_t parity, int* err, int code) {
  const uint32_t addr = smem_u32(bar);
  if (mbar_try_wait(addr, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(addr), "r"(parity), "r"(100000u)
        : "memory");
    if (ok) return true;
    if (global_timer_ns() - t0 > kWaitBudgetNs) {
      record_error(err, code);
      return false;
    }
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}


__device__ __forceinline__ uint32_t pair_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void pair_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Address of a barrier of the even CTA, in the cluster's shared window.
__device__ __forceinline__ uint32_t leader_addr(const void* p) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
  return a;
}

// Orders nothing but this CTA's own accesses: a release at cluster scope would
// wait for every global store in flight (1000 to 2000 cycles in an epilogue).
// What the arrival hands over is read from TMEM, which tcgen05's fences order.
__device__ __forceinline__ void arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}

// 2-D tiled load into this CTA's shared memory that completes on the leader's barrier.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}

__device__ __forceinline__ void pair_tmem_alloc(uint32_t* dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)),
               "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// Completion of the issued pair instructions arrives on `bar` of both CTAs.
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

// Matrix descriptors (128-byte swizzle, rows of 128 bytes in groups of eight,
// 1024 bytes apart) as their two words.  The upper one is a constant and the
// lower one moves by an addition from step to step: the issuing warp has a few
// dozen cycles for an instruction, less than it takes to build a descriptor anew.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);

// lead: bytes between 64-value chunks of an MN-major operand (K-major: ignored).
__device__ __forceinline__ uint32_t desc_lo(uint32_t smem_addr, uint32_t lead = 16) {
  return ((smem_addr >> 4) & 0x3FFFu) | ((lead >> 4) << 16);
}
// Steps of 16 along the reduction: within a K-major row (four to a 64-value
// chunk, `rows` rows each), or 16 rows down an MN-major tile.
__device__ __forceinline__ constexpr uint32_t step_k(int rows, int k) { return (k >> 2) * rows * 8 + (k & 3) * 2; }
__device__ __forceinline__ constexpr uint32_t step_mn(int k) { return k * 128; }

#define TGCM_UMMA(NAME, GROUP)                                                                                     \
  __device__ __forceinline__ void NAME(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc,              \
                                       uint32_t accumulate) {                                                      \
    asm volatile(                                                                                                  \
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"                                                              \
        "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"                                                       \
        "setp.ne.b32 p, %4, 0;\n\t"                                                                                \
        "tcgen05.mma.cta_group::" #GROUP ".kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(tmem_d),                     \
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHi)                                            \
        : "memory");                                                                                               \
  }
TGCM_UMMA(umma_ss, 1)        // one CTA
TGCM_UMMA(pair_umma_ss, 2)   // both CTAs of a pair
#undef TGCM_UMMA

// A from TMEM (one CTA).
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHi)
      : "memory");
}

// Start of a kernel's work: waits until the kernel before it in the stream has ended and its
// writes are seen, then lets the next one's blocks come in beside this one's.  Before this
// call a block touches nothing but its own shared memory, tensor memory and parameters.
__device__ __forceinline__ void after_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// One lane of a converged warp, the same one every time.
__device__ __forceinline__ bool elect_lane() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is != 0;
}

// 32 lanes x 32 columns of 32 bits, one row to a thread.
__device__ __forceinline__ void tmem_ld_32x32b_x32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

}  // namespace tgcm
