// Two floats in a register pair: one instruction of sm_100a works on both.
//
// a * b + c written with the operators may become one fused multiply-add.  Where the
// product has to be rounded by itself, addRounded adds: a multiply-add by a `one` that
// the assembler cannot see to be 1.
#ifndef MLUOP_B200_CORE_PAIR_CUH_
#define MLUOP_B200_CORE_PAIR_CUH_

#include <cuda_runtime.h>

#include "core/convert.cuh"

namespace mluop {

struct Two {
  unsigned long long v;
};
__device__ __forceinline__ Two two(float lo, float hi) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 split(Two t) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(t.v));
  return r;
}
__device__ __forceinline__ Two operator+(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two addRounded(Two a, Two b, float one) {
  Two r;
  asm("{\n.reg .b64 o;\nmov.b64 o, {%3, %3};\nfma.rn.f32x2 %0, %1, o, %2;\n}" : "=l"(r.v) : "l"(a.v), "l"(b.v), "f"(one));
  return r;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// A thread's VEC consecutive values as pairs; VEC is a 16-byte vector of T, or 1 (then the pair's second half is idle).
// The words stay in registers: an array of T seen as pairs would be put into local memory.
template <typename T, int VEC>
struct Values;
template <typename T>
struct Values<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T *p) { v = *p; }
  __device__ __forceinline__ Two pair(int) const { return two(toFloat(v), 0.0f); }
  static __device__ __forceinline__ void store(T *p, const Two (&t)[1]) { *p = fromFloat<T>(split(t[0]).x); }
  static __device__ __forceinline__ void storeZero(T *p) { *p = fromFloat<T>(0.0f); }
};
struct Vector16 {
  uint4 q;
  __device__ __forceinline__ unsigned word(int i) const { return i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w; }
  __device__ __forceinline__ void load(const void *p) { q = *static_cast<const uint4 *>(p); }
  static __device__ __forceinline__ void storeZero(void *p) { *static_cast<uint4 *>(p) = make_uint4(0u, 0u, 0u, 0u); }
};
template <>
struct Values<float, 4> : Vector16 {
  __device__ __forceinline__ Two pair(int j) const { return two(__uint_as_float(word(2 * j)), __uint_as_float(word(2 * j + 1))); }
  static __device__ __forceinline__ void store(float *p, const Two (&t)[2]) {
    const float2 a = split(t[0]), b = split(t[1]);
    *reinterpret_cast<float4 *>(p) = make_float4(a.x, a.y, b.x, b.y);
  }
};
template <>
struct Values<__half, 8> : Vector16 {
  __device__ __forceinline__ Two pair(int j) const {
    const unsigned w = word(j);
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
    return two(f.x, f.y);
  }
  static __device__ __forceinline__ unsigned pack(Two t) {
    const float2 f = split(t);
    const __half2 h = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const unsigned *>(&h);
  }
  static __device__ __forceinline__ void store(__half *p, const Two (&t)[4]) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack(t[0]), pack(t[1]), pack(t[2]), pack(t[3]));
  }
};
template <>
struct Values<__nv_bfloat16, 8> : Vector16 {
  __device__ __forceinline__ Two pair(int j) const {
    const unsigned w = word(j);
    return two(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ unsigned pack(Two t) {
    const float2 f = split(t);
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const unsigned *>(&h);
  }
  static __device__ __forceinline__ void store(__nv_bfloat16 *p, const Two (&t)[4]) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack(t[0]), pack(t[1]), pack(t[2]), pack(t[3]));
  }
};

}  // namespace mluop

#endif  // MLUOP_B200_CORE_PAIR_CUH_
