// Tensor cores of sm_100a (tcgen05): tensor memory, descriptors, products.
#pragma once

#include "async.cuh"

namespace tw {

// ---- tensor memory: 128 lanes x 512 columns of 32 bits per SM; address = lane << 16 | column
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t columns) {  // a whole warp
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   smem_addr(slot)),
               "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t columns) {  // the same warp
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns)
               : "memory");
}

// Order of tensor-memory accesses and products against barriers between threads.
__device__ __forceinline__ void tmem_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tmem_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// The same, for the values of one tmem_ld32: what uses them comes after.
__device__ __forceinline__ void tmem_wait_ld(float (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]),
        "+f"(r[7]), "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]),
        "+f"(r[14]), "+f"(r[15]), "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]),
        "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]), "+f"(r[24]), "+f"(r[25]),
        "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31])
      :: "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// 32 columns of the warp's 32 lanes: thread l gets lane l (+ the warp's first lane).
__device__ __forceinline__ void tmem_ld32(float (&r)[32], uint32_t tmem) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]),
        "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]),
        "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]),
        "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]),
        "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(tmem));
}
__device__ __forceinline__ void tmem_st32(uint32_t tmem, const uint32_t (&u)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(tmem),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]),
      "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]),
      "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]), "r"(u[20]), "r"(u[21]),
      "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]),
      "r"(u[29]), "r"(u[30]), "r"(u[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t tmem, const uint32_t (&u)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(tmem),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]),
      "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]),
      "r"(u[15])
      : "memory");
}

// ---- products: 16-bit operands, 32-bit accumulators, M = 128
// Shared-memory operand in 128-byte rows, 16-byte columns XORed by row % 8
// (8-row groups of 1024 bytes, which begin on 1024-byte boundaries).
//   rows along M or N, K contiguous: 8-row groups `group` bytes apart
//   rows along K, M or N contiguous: 8-row groups `group` bytes apart along K,
//     blocks of 64 elements `block` bytes apart along M or N
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t block, uint32_t group) {
  return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)((block >> 4) & 0x3fff) << 16) |
         ((uint64_t)((group >> 4) & 0x3fff) << 32) | (1ull << 46) | (2ull << 61);
}

// Instruction descriptor of a 128 x N product; b_rows_k: B's rows run along K.
__host__ __device__ constexpr uint32_t product_desc(bool bf16, int n, bool b_rows_k) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_rows_k ? 1u << 16 : 0u) |
         ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

// D (+)= A B, one 16-deep step, issued by one thread.
__device__ __forceinline__ void mma_smem(uint32_t d, uint64_t a, uint64_t b, uint32_t desc,
                                         bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(desc), "r"((uint32_t)add)
      : "memory");
}
// The same with A in tensor memory (two 16-bit values per column).
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t desc,
                                         bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(desc), "r"((uint32_t)add)
      : "memory");
}
// The barrier gets an arrival when this thread's products so far are done.
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_addr(bar))
      : "memory");
}

// ---- pairs of 32-bit floats in one instruction
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t x, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}


// The largest of three.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x of a pair on the FMA pipe, for x <= 126 (below -126: 2^-126; NaN: NaN): n = x
// rounded to a whole number by adding 1.5 * 2^23, 2^(x - n) on [-1/2, 1/2] by the
// polynomial of degree 4 with the smallest largest relative error there (Remez
// exchange; 2.7e-6 with its roundings), times 2^n put together from its bits.
__device__ __forceinline__ void ex2_fma(uint64_t x2, float& e0, float& e1) {
  float x0, x1;
  unpair(x2, x0, x1);
  x2 = pair(max_nan(x0, -126.f), max_nan(x1, -126.f));
  const uint64_t round = pair(12582912.f, 12582912.f), back = pair(-12582912.f, -12582912.f);
  const uint64_t r = add2(x2, round);
  const uint64_t f = fma2(add2(r, back), pair(-1.f, -1.f), x2);
  uint64_t p = pair(0x1.3997d6p-7f, 0x1.3997d6p-7f);
  p = fma2(p, f, pair(0x1.ca1440p-5f, 0x1.ca1440p-5f));
  p = fma2(p, f, pair(0x1.ec06dap-3f, 0x1.ec06dap-3f));
  p = fma2(p, f, pair(0x1.62e0dcp-1f, 0x1.62e0dcp-1f));
  p = fma2(p, f, pair(0x1.ffffe8p-1f, 0x1.ffffe8p-1f));
  float r0, r1;
  unpair(r, r0, r1);
  p = mul2(p, pair(__int_as_float((__float_as_int(r0) << 23) + 0x3f800000),
                   __int_as_float((__float_as_int(r1) << 23) + 0x3f800000)));
  unpair(p, e0, e1);
}

// Registers of a warpgroup's threads, all of which run this.
template <int kRegs> __device__ __forceinline__ void grow_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs> __device__ __forceinline__ void shrink_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

}  // namespace tw
