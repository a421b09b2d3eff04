// Two float32 lanes in one instruction (sm_100a's .f32x2 forms), rounded like the scalar ones.
#pragma once
#include <stdint.h>

namespace atlas {

struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 f2_get(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 operator-(F2 a, F2 b) {
  F2 r;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
// bf16 pair (low half first) <-> float32 pair
__device__ __forceinline__ F2 bf2_unpack(uint32_t h) { return f2(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u)); }
__device__ __forceinline__ uint32_t bf2_pack(F2 a) {
  const float2 x = f2_get(a);
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(x.y), "f"(x.x));
  return r;
}
// the upper halves of both: rounded toward zero
__device__ __forceinline__ uint32_t bf2_cut(F2 a) {
  const float2 x = f2_get(a);
  return __byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x7632);
}

}  // namespace atlas
