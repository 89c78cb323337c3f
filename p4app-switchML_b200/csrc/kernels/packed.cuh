// Vectors in registers: 8 neighbouring values as they lie in memory, and arithmetic on two fp32 numbers at once.
#ifndef SWITCHML_PACKED_CUH_
#define SWITCHML_PACKED_CUH_

#include <cuda_bf16.h>

namespace switchml {
namespace kernels {

// Two fp32 operations in one instruction (sm_100's f32x2): half the instructions to issue. ptxas makes one operation with
// one rounding of a product and a sum, as it does for single numbers.
struct Pair {
  unsigned long long w;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(w) : "f"(x), "f"(y)); }
  __device__ __forceinline__ explicit Pair(float x) : Pair(x, x) {}
  __device__ __forceinline__ float2 Both() const {
    float2 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(w));
    return v;
  }
};
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.w) : "l"(a.w), "l"(b.w));
  return r;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.w) : "l"(a.w), "l"(b.w));
  return r;
}
__device__ __forceinline__ Pair Fma(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.w) : "l"(a.w), "l"(b.w), "l"(c.w));
  return r;
}
__device__ __forceinline__ float Sum(Pair p) {
  const float2 v = p.Both();
  return v.x + v.y;
}

// 8 values of a lane that are neighbours in memory, as they lie there.
template <class T> struct Packed;
template <> struct Packed<float> {
  unsigned w[8];
  __device__ __forceinline__ float At(int i) const { return __uint_as_float(w[i]); }
};
template <> struct Packed<__nv_bfloat16> {
  unsigned w[4];
  __device__ __forceinline__ float At(int i) const { return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16); }
};
template <int kWords> __device__ __forceinline__ void LoadWords(const void* from, unsigned (&w)[kWords]) {
  if constexpr (kWords == 8) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(from));
  } else if constexpr (kWords == 4) {
    asm volatile("ld.global.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(from));
  } else if constexpr (kWords == 2) {
    asm volatile("ld.global.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(from));
  } else {
    asm volatile("ld.global.b32 %0, [%1];" : "=r"(w[0]) : "l"(from));
  }
}
// Only where left > 0, else zeros: without a branch.
template <int kWords> __device__ __forceinline__ void LoadWordsIf(int left, const void* from, unsigned (&w)[kWords]) {
#pragma unroll
  for (int i = 0; i < kWords; i++) w[i] = 0;
  if constexpr (kWords == 8) {
    asm volatile("{.reg .pred p; setp.gt.s32 p, %9, 0; @p ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];}"
                 : "+r"(w[0]), "+r"(w[1]), "+r"(w[2]), "+r"(w[3]), "+r"(w[4]), "+r"(w[5]), "+r"(w[6]), "+r"(w[7])
                 : "l"(from), "r"(left));
  } else if constexpr (kWords == 4) {
    asm volatile("{.reg .pred p; setp.gt.s32 p, %5, 0; @p ld.global.v4.b32 {%0,%1,%2,%3}, [%4];}"
                 : "+r"(w[0]), "+r"(w[1]), "+r"(w[2]), "+r"(w[3]) : "l"(from), "r"(left));
  } else if constexpr (kWords == 2) {
    asm volatile("{.reg .pred p; setp.gt.s32 p, %3, 0; @p ld.global.v2.b32 {%0,%1}, [%2];}"
                 : "+r"(w[0]), "+r"(w[1]) : "l"(from), "r"(left));
  } else {
    asm volatile("{.reg .pred p; setp.gt.s32 p, %2, 0; @p ld.global.b32 %0, [%1];}" : "+r"(w[0]) : "l"(from), "r"(left));
  }
}
template <int kWords> __device__ __forceinline__ void StoreWords(void* to, const unsigned (&w)[kWords]) {
  if constexpr (kWords == 8) {
    asm volatile("st.global.v8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};"
                 :: "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "l"(to) : "memory");
  } else if constexpr (kWords == 4) {
    asm volatile("st.global.v4.b32 [%4], {%0,%1,%2,%3};" :: "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "l"(to) : "memory");
  } else if constexpr (kWords == 2) {
    asm volatile("st.global.v2.b32 [%2], {%0,%1};" :: "r"(w[0]), "r"(w[1]), "l"(to) : "memory");
  } else {
    asm volatile("st.global.b32 [%1], %0;" :: "r"(w[0]), "l"(to) : "memory");
  }
}

}  // namespace kernels
}  // namespace switchml
#endif  // SWITCHML_PACKED_CUH_
