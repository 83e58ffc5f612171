// tcgen05 products of 16-bit operands and packed fp32 arithmetic, for the
// grouped-query kernels.
#pragma once

#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "dsv4b_ptx.cuh"

namespace dsv4b {

__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(r));
  return r != 0;
}

// A SWIZZLE_128B operand's descriptor: its low word, and the high one, the
// same for all (8 rows of 128 bytes after another).
constexpr uint32_t kSw128High = (1024 >> 4) | (1u << 14) | (2u << 29);  // SBO, version, swizzle
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t lbo) {
  return ((saddr >> 4) & 0x3FFFu) | ((lbo >> 4) << 16);
}

// D[tmem] (+)= A[smem] * B[smem], 16-bit operands, fp32 sums; descriptors as
// their low words and a common high one.
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t high, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(high), "r"(idesc), "r"(accumulate));
}
// The same with A from TMEM.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t high, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(high), "r"(idesc), "r"(accumulate));
}

// The instruction descriptor of [128 x n] from 16-bit operands, A K-major.
template <typename T>
__host__ __device__ constexpr uint32_t idesc_of(int n, bool b_mn_major) {
  constexpr uint32_t types = (1u << 7) | (1u << 10);  // A, B: bf16 (0: fp16)
  return std::is_same_v<T, __half> ? (idesc_bf16_f32(128, n, false, b_mn_major) & ~types)
                                   : idesc_bf16_f32(128, n, false, b_mn_major);
}

// Two fp32 at once (Blackwell's packed forms; each half an ordinary fp32 operation).
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

}  // namespace dsv4b
