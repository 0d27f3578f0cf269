// Rows of fp32, bf16 or fp16 values, eight at a time, for the kernels in which
// bytes count: values stay in the stored type until they are used.
#pragma once
#include "common.cuh"

namespace moe {

template <typename T>
MOE_D T from_float(float v);
template <>
MOE_D float from_float<float>(float v) { return v; }
template <>
MOE_D __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
MOE_D __half from_float<__half>(float v) { return __float2half_rn(v); }
template <typename T>
MOE_D float widen(T v) { return static_cast<float>(v); }

// Eight columns of a row as they are stored: 16-byte accesses when VEC (whole
// and aligned), else one element at a time, `n` of them present.
template <typename T>
struct alignas(16) Eight {
  T v[8];
};
template <typename T, bool VEC>
MOE_D void load8(const T* p, int n, Eight<T>& e) {
  if (VEC) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      reinterpret_cast<uint4*>(e.v)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) e.v[i] = i < n ? p[i] : from_float<T>(0.0f);
  }
}
template <typename T, bool VEC>
MOE_D void store8(T* p, int n, const Eight<T>& e) {
  if (VEC) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(e.v)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = e.v[i];
  }
}
template <typename T>
MOE_D void clear8(Eight<T>& e) {
#pragma unroll
  for (int i = 0; i < 8; ++i) e.v[i] = from_float<T>(0.0f);
}

// Two fp32 values in one instruction (packed operations of sm_100).
MOE_D float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
MOE_D float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n .reg .b64 w, x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 w, {%6, %7};\n"
      " fma.rn.f32x2 z, x, y, w;\n mov.b64 {%0, %1}, z;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

}  // namespace moe
