// Packed single-precision arithmetic of sm_100 (two floats per instruction).
#pragma once

#include <stdint.h>

namespace fp4t {

// Two floats in one 64-bit register pair, worked on by one instruction; Pack<1> is one float with the
// same interface.
template <int W>
struct Pack {
  uint64_t v;
  static __device__ __forceinline__ Pack of(const float* p) {
    Pack r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(p[0]), "f"(p[1]));
    return r;
  }
  static __device__ __forceinline__ Pack all(float x) {
    const float t[2] = {x, x};
    return of(t);
  }
  __device__ __forceinline__ void to(float* p) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(p[0]), "=f"(p[1]) : "l"(v)); }
  __device__ __forceinline__ float sum() const {
    float t[2];
    to(t);
    return t[0] + t[1];
  }
};
template <>
struct Pack<1> {
  float v;
  static __device__ __forceinline__ Pack of(const float* p) { return Pack{p[0]}; }
  static __device__ __forceinline__ Pack all(float x) { return Pack{x}; }
  __device__ __forceinline__ void to(float* p) const { p[0] = v; }
  __device__ __forceinline__ float sum() const { return v; }
};
__device__ __forceinline__ Pack<2> mul(Pack<2> a, Pack<2> b) {
  Pack<2> r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pack<2> fma(Pack<2> a, Pack<2> b, Pack<2> c) {
  Pack<2> r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Pack<1> mul(Pack<1> a, Pack<1> b) { return Pack<1>{a.v * b.v}; }
__device__ __forceinline__ Pack<1> fma(Pack<1> a, Pack<1> b, Pack<1> c) { return Pack<1>{fmaf(a.v, b.v, c.v)}; }
__device__ __forceinline__ Pack<2> add(Pack<2> a, Pack<2> b) {
  Pack<2> r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

}  // namespace fp4t
