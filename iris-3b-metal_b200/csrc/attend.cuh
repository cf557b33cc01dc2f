// Device helpers that the text side's attention kernels share (window.cu, prefix.cu):
// 16-bit operand types, exponentials, mma.sync with its shared-memory loads.
#pragma once

#include "common.cuh"

namespace iris {
namespace attend {

template <typename T>
struct IsHalf { static constexpr bool value = false; };
template <>
struct IsHalf<__half> { static constexpr bool value = true; };

template <typename T>
IRIS_DEVICE float2 unpack2(uint32_t v);
template <>
IRIS_DEVICE float2 unpack2<__nv_bfloat16>(uint32_t v) { return unpack_bf16x2(v); }
template <>
IRIS_DEVICE float2 unpack2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
template <typename T>
IRIS_DEVICE uint32_t pack2(float a, float b);
template <>
IRIS_DEVICE uint32_t pack2<__nv_bfloat16>(float a, float b) { return pack_bf16x2(a, b); }
template <>
IRIS_DEVICE uint32_t pack2<__half>(float a, float b) { return pack_f16x2(a, b); }

constexpr float RESCALE = 8.0f;  // the running maximum is kept until a row exceeds it by 2^8

IRIS_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
IRIS_DEVICE float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Bits [0, n) of a 32-bit word, n of any value.
IRIS_DEVICE uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

template <typename T>
IRIS_DEVICE void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (IsHalf<T>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
IRIS_DEVICE void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
IRIS_DEVICE void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16 bytes global -> shared, or 16 zero bytes
IRIS_DEVICE void copy16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}

IRIS_DEVICE void store_remote(uint32_t at, float2 v) {  // another CTA's shared memory (map_to_cta)
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(v.x), "f"(v.y) : "memory");
}

}  // namespace attend
}  // namespace iris
