// kvattn_mma.cuh -- warp matrix instructions and the result's store, for the kernels of attention that
// keep their sums in registers (kvattn.cu, kvattn_one.cu).
#pragma once

#include "kvattn.cuh"

namespace ex {

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two neighbouring outputs of a row whose sums are o and weight l.  A row that sees nothing is 0; one
// that sees only scores of -inf is 0/0, as its softmax is.
template <typename T>
__device__ __forceinline__ void store_out(const AttnArgs& a, long long at, float o0, float o1, float l, bool sees) {
  const float r = 1.0f / l;
  o0 = sees ? o0 * r : 0.0f;
  o1 = sees ? o1 * r : 0.0f;
  if (a.out_f32)
    *reinterpret_cast<float2*>(static_cast<float*>(a.out) + at) = make_float2(o0, o1);
  else
    *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + at) = pack16<T>(o0, o1);
}

}  // namespace ex
