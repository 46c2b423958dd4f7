// elem.cuh — element types of the multi-type kernels (fp32, bf16, fp16):
// conversion to and from fp32 and 16-byte vectors of them. Conversions to 16
// bits round to nearest even.
#pragma once
#include <cuda_fp16.h>

#include "kt_common.cuh"

namespace kt {
namespace elem {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// Elements of a 16-byte vector.
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

__device__ __forceinline__ void unpack(const uint4& r, float (&f)[4]) {
  f[0] = __uint_as_float(r.x);
  f[1] = __uint_as_float(r.y);
  f[2] = __uint_as_float(r.z);
  f[3] = __uint_as_float(r.w);
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  // bf16 is the upper half of an fp32
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T>
__device__ __forceinline__ void unpack_vec(const uint4& r, float (&f)[kVec<T>]) {
  if constexpr (sizeof(T) == 4) {
    unpack(r, f);
  } else {
    const float2 a = unpack2<T>(r.x), b = unpack2<T>(r.y), c = unpack2<T>(r.z), d = unpack2<T>(r.w);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
    f[4] = c.x; f[5] = c.y; f[6] = d.x; f[7] = d.y;
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack_vec(const float (&f)[kVec<T>]) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  } else {
    return make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
  }
}

// Two fp32 operations by one instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  return (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
}
__device__ __forceinline__ float2 halves(uint64_t v) {
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
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
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// A 16-byte piece as pairs of fp32, and back.
template <typename T>
__device__ __forceinline__ void unpack_pairs(const uint4& r, uint64_t (&f)[kVec<T> / 2]) {
  float v[kVec<T>];
  unpack_vec<T>(r, v);
#pragma unroll
  for (int j = 0; j < kVec<T> / 2; ++j) f[j] = pair(v[2 * j], v[2 * j + 1]);
}
template <typename T>
__device__ __forceinline__ uint4 pack_pairs(const uint64_t (&f)[kVec<T> / 2]) {
  float v[kVec<T>];
#pragma unroll
  for (int j = 0; j < kVec<T> / 2; ++j) {
    const float2 h = halves(f[j]);
    v[2 * j] = h.x;
    v[2 * j + 1] = h.y;
  }
  return pack_vec<T>(v);
}

// Read-only 16-byte load of data used once (not kept in L1).
__device__ __forceinline__ uint4 ld_once16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// A value that the compiler takes for a new one: what is computed from it is
// not kept in registers across the rows. (Only a row's first and last piece need
// those computations, and holding them for all pieces costs more registers than
// the data.)
__device__ __forceinline__ int opaque(int v) {
  asm volatile("" : "+r"(v));
  return v;
}

// Elements between the 16-byte boundary at or below `p` and `p`.
template <typename T>
__host__ __device__ __forceinline__ int misalign(const void* p) {
  return (int)((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
}

// One value of a weight vector whose type is known at run time.
__device__ __forceinline__ float ld_weight(const void* p, int dtype, int64_t i) {
  if (dtype == KT_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == KT_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}

__device__ __forceinline__ void st_weight(void* p, int dtype, int64_t i, float v) {
  if (dtype == KT_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else if (dtype == KT_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<float*>(p)[i] = v;
}

inline int size_of(int dtype) { return dtype == KT_F32 ? 4 : (dtype == KT_BF16 || dtype == KT_F16) ? 2 : 0; }
inline bool aligned_to(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }

}  // namespace elem
}  // namespace kt
