// Elements of f32, bf16 or f16 as f32 values, one at a time or eight (16 or 32 bytes) at a time.
#ifndef SEE_CUDA_VEC_TYPES_CUH_
#define SEE_CUDA_VEC_TYPES_CUH_

#include <cuda_runtime.h>

#include <cstdint>

namespace see::k {

struct Bf16 { uint16_t bits; };
struct F16 { uint16_t bits; };

__device__ __forceinline__ float ToF32(float v) { return v; }
__device__ __forceinline__ float ToF32(Bf16 v) { return __uint_as_float(static_cast<uint32_t>(v.bits) << 16); }
__device__ __forceinline__ float ToF32(F16 v) {
  float f;
  asm("cvt.f32.f16 %0, %1;" : "=f"(f) : "h"(v.bits));
  return f;
}
template <typename T> __device__ __forceinline__ T FromF32(float v);   // to nearest, ties to even
template <> __device__ __forceinline__ float FromF32<float>(float v) { return v; }
template <> __device__ __forceinline__ Bf16 FromF32<Bf16>(float v) {
  Bf16 r;
  asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r.bits) : "f"(v));
  return r;
}
template <> __device__ __forceinline__ F16 FromF32<F16>(float v) {
  F16 r;
  asm("cvt.rn.f16.f32 %0, %1;" : "=h"(r.bits) : "f"(v));
  return r;
}
template <typename T> __device__ __forceinline__ uint32_t Pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t Pack2<Bf16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <> __device__ __forceinline__ uint32_t Pack2<F16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <typename T> __device__ __forceinline__ void Unpack2(uint32_t v, float& lo, float& hi) {
  T a, b;
  a.bits = static_cast<uint16_t>(v);
  b.bits = static_cast<uint16_t>(v >> 16);
  lo = ToF32(a);
  hi = ToF32(b);
}

template <> __device__ __forceinline__ void Unpack2<Bf16>(uint32_t v, float& lo, float& hi) {
  lo = __uint_as_float(v << 16);
  hi = __uint_as_float(v & 0xFFFF0000u);
}

template <typename T> __device__ __forceinline__ void Load8(const T* p, float* v) {
  const uint4 r = *reinterpret_cast<const uint4*>(p);
  Unpack2<T>(r.x, v[0], v[1]);
  Unpack2<T>(r.y, v[2], v[3]);
  Unpack2<T>(r.z, v[4], v[5]);
  Unpack2<T>(r.w, v[6], v[7]);
}
template <> __device__ __forceinline__ void Load8<float>(const float* p, float* v) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename T> __device__ __forceinline__ void Store8(T* p, const float* v) {
  *reinterpret_cast<uint4*>(p) = make_uint4(Pack2<T>(v[0], v[1]), Pack2<T>(v[2], v[3]), Pack2<T>(v[4], v[5]), Pack2<T>(v[6], v[7]));
}
template <> __device__ __forceinline__ void Store8<float>(float* p, const float* v) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

}  // namespace see::k

#endif  // SEE_CUDA_VEC_TYPES_CUH_
