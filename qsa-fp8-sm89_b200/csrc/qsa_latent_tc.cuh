// PTX wrappers of the latent cache's tensor-core kernels, beside those of
// qsa_common.cuh: barriers and bounded waits, tensor-memory stores, and the
// matrix instructions with A in tensor memory.
#pragma once

#include "qsa_common.cuh"

namespace qsa {

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void bar_sync(int id, int count) {
  asm volatile("bar.sync %0, %1;\n" ::"r"(id), "r"(count) : "memory");
}
// Named-barrier vote of count threads: true when pred holds in any of them.
__device__ __forceinline__ bool bar_vote(int id, int count, bool pred) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, %2, %3, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"((uint32_t)pred), "r"(id), "r"(count)
      : "memory");
  return r != 0u;
}

// Bounded wait: false once `tries` looks at the barrier have not seen the phase end. A
// look that finds nothing took 4 us where a whole warp looks (the instruction itself
// waits) and 0.1 us where one lane of a warp does. It is this short because it stands in
// so many places. (A look with a time to sleep wakes up to 2 us after its barrier.) A wait
// is for one step of the work, some microseconds; one that may take longer counts its
// looks anew with each step.
__device__ __forceinline__ bool wait_tries(uint64_t* bar, uint32_t parity, uint32_t tries) {
#pragma unroll 1
  for (uint32_t i = 0; !mbar_try_wait(bar, parity); ++i)
    if (i >= tries) return false;
  return true;
}
// Tries that a limit in ns allows: they take a tenth of it to four times as long.
__device__ __forceinline__ uint32_t tries_of(uint64_t limit_ns) { return (uint32_t)(limit_ns / 1024 < 0x7fffffffu ? limit_ns / 1024 : 0x7fffffffu); }

// Descriptors of 128-byte swizzled operands whose 8-row groups lie 1024 bytes
// apart: the high words are all the same, the low word is the address in 16-byte
// steps (and the step between 128-byte columns where an operand has several).
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t column_step = 16) {
  return ((saddr >> 4) & 0x3FFF) | (column_step >> 4) << 16;
}

// The same for an operand without swizzle: 8 rows of 16 bytes side by side, the
// next 8 rows 128 bytes on, the next 16 bytes of the rows `column_step` on.
constexpr uint32_t kDescHighPlain = (128u >> 4) | (1u << 14);

// D[tmem] (+)= A B with A in tensor memory (ts) or shared memory (ss), B in shared
// memory. A whole warp calls these, with the same arguments, and one lane issues: the
// operands then stay in uniform registers, and a product takes 40 cycles to issue
// instead of 50 (64 rows of B at most; with 128 the product itself takes 64).
__device__ __forceinline__ void mma_f8_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p, e;\nelect.sync _|e, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n"
      ".reg .b64 bd;\nmov.b64 bd, {%2, %5};\n"
      "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], bd, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc),
      "r"(accumulate), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_f8_ss_plain_a(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p, e;\nelect.sync _|e, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n"
      ".reg .b64 ad, bd;\nmov.b64 ad, {%1, %6};\nmov.b64 bd, {%2, %5};\n"
      "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], ad, bd, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc),
      "r"(accumulate), "n"(kDescHigh), "n"(kDescHighPlain)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p, e;\nelect.sync _|e, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n"
      ".reg .b64 ad, bd;\nmov.b64 ad, {%1, %5};\nmov.b64 bd, {%2, %5};\n"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc),
      "r"(accumulate), "n"(kDescHigh)
      : "memory");
}
// With a power of two for each row of A and of B (exponent + 127, a byte for each 32
// values of K, four to a word): rows 32 c + l of an operand have theirs in lane l of
// column c, the same in every quarter of the lanes. The byte is named by idesc.
__device__ __forceinline__ void mma_mxf8_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t a_scales, uint32_t b_scales,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p, e;\nelect.sync _|e, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n"
      ".reg .b64 ad, bd;\nmov.b64 ad, {%1, %5};\nmov.b64 bd, {%2, %5};\n"
      "@e tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], ad, bd, %3, [%6], [%7], p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc),
      "r"(accumulate), "n"(kDescHigh), "r"(a_scales), "r"(b_scales)
      : "memory");
}
// Arrives once on `bar` when every product that the warp issued so far is done.
__device__ __forceinline__ void warp_commit(uint64_t* bar) {
  asm volatile(
      "{\n.reg .pred e;\nelect.sync _|e, 0xffffffff;\n"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar))
      : "memory");
}

// The same for a pair of CTAs (a cluster of two): the even one issues. Each holds its
// 128 of the 256 rows of A and D, and half of B's columns (its N is the instruction's
// over two), all at the same addresses.
__device__ __forceinline__ void pair_mma_f16_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p, e;\nelect.sync _|e, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n"
      ".reg .b64 bd;\nmov.b64 bd, {%2, %5};\n"
      "@e tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], bd, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc),
      "r"(accumulate), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void pair_mma_f16_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p, e;\nelect.sync _|e, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n"
      ".reg .b64 ad, bd;\nmov.b64 ad, {%1, %5};\nmov.b64 bd, {%2, %5};\n"
      "@e tcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc),
      "r"(accumulate), "n"(kDescHigh)
      : "memory");
}
// Arrives on the barrier at this address in both CTAs.
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
  asm volatile(
      "{\n.reg .pred e;\nelect.sync _|e, 0xffffffff;\n"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}\n" ::"r"(smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t smem_of(const void* at, uint32_t rank) {  // the address in another CTA of the cluster
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(smem_u32(at)), "r"(rank));
  return r;
}
// Arrivals and waits between the CTAs of a cluster.
__device__ __forceinline__ void cluster_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
// Orders nothing but what tcgen05 fences do, as tensor memory needs: the release above
// takes 500 cycles and more.
__device__ __forceinline__ void cluster_arrive_relaxed(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool cluster_wait_tries(uint64_t* bar, uint32_t parity, uint32_t tries) {
#pragma unroll 1
  for (uint32_t i = 0;; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
    if (i >= tries) return false;
  }
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_alloc(uint32_t* at, uint32_t columns) {  // a warp of each CTA
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(at)), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_free(uint32_t taddr, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(taddr), "r"(columns) : "memory");
}

// Instruction descriptor of kind::f16, A and B both bf16 or both f16, FP32 accumulator.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool bf16, bool b_mn_major) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn_major ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// Instruction descriptor of kind::mxf8f6f4, E4M3 A and B, scales of 8 exponent bits;
// B's byte of a scale word is added as byte << 4.
__host__ __device__ constexpr uint32_t idesc_mxf8(int m, int n, bool a_mn_major, bool b_mn_major) {
  return ((a_mn_major ? 1u : 0u) << 15) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (1u << 23) |
         ((uint32_t)(m >> 4) << 24);
}

// Consecutive 32-bit columns of a thread's lane.
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
               : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
               : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&v)[2]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1,%2};\n" ::"r"(taddr), "r"(v[0]), "r"(v[1]) : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&v)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3])
               : "memory");
}
// Two runs of 32 consecutive columns, loaded and waited for in one asm statement, so
// that no instruction can touch the destination registers before the data has arrived.
__device__ __forceinline__ void tmem_ld_2x32_wait(uint32_t a, uint32_t b, float (&x)[32], float (&y)[32]) {
  uint32_t r[64];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(a), "r"(b)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(r[i]), y[i] = __uint_as_float(r[32 + i]);
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

// Of a chain of dependent launches: lets the next kernel start, and waits for
// all of the one before (nothing where the launch was an ordinary one).
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }
__device__ __forceinline__ void wait_for_prerequisites() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

// The largest of three.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
  return r;
}

}  // namespace qsa
