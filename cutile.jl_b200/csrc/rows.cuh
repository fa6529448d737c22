// Rows of f32, f16 or bf16 that start at any element, read and written as the 16-byte vectors that they touch.
//
// Vector v of a row covers elements v * V - off ... v * V - off + V - 1, where V elements make 16 bytes and off is the row's distance
// from the vector boundary before it: vectors are aligned whatever the row is, and only the first and last one may be partly outside.  What
// is outside is not read (it reads as -inf) and not written.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

namespace ctb {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T>
__device__ __forceinline__ void unpack_row(const uint4& q, float (&f)[16 / sizeof(T)]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
  } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack_row(const float (&f)[16 / sizeof(T)]) {
  uint32_t w[4];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(f[i]);
  } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A vector of -inf.
template <typename T>
__device__ __forceinline__ uint4 empty_row_vec() {
  const uint32_t w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  return make_uint4(w, w, w, w);
}

// Element i of vector v is an element of the row.
template <int V>
__device__ __forceinline__ bool in_row(int off, int n, int v, int i) {
  const int e = v * V - off + i;
  return e >= 0 && e < n;
}

// KEEP: the row is read again, from L2.
template <typename T, bool KEEP = false>
__device__ __forceinline__ uint4 load_row_vec(const T* src, int off, int n, int v) {
  constexpr int V = 16 / (int)sizeof(T);
  const int e0 = v * V - off;
  if (e0 >= 0 && e0 + V <= n) {
    const uint4* p = reinterpret_cast<const uint4*>(src + e0);
    return KEEP ? __ldcg(p) : __ldcs(p);
  }
  uint4 q = empty_row_vec<T>();
  T* f = reinterpret_cast<T*>(&q);
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (e0 + i >= 0 && e0 + i < n) f[i] = src[e0 + i];
  return q;
}
// aligned: the row that is written lies off elements behind a vector boundary, like the one that was read.
template <typename T>
__device__ __forceinline__ void store_row_vec(T* dst, int off, int n, int v, const float (&f)[16 / sizeof(T)], bool aligned) {
  constexpr int V = 16 / (int)sizeof(T);
  const int e0 = v * V - off;
  if (aligned && e0 >= 0 && e0 + V <= n) {
    __stcs(reinterpret_cast<uint4*>(dst + e0), pack_row<T>(f));
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (e0 + i >= 0 && e0 + i < n) dst[e0 + i] = from_float<T>(f[i]);
}

// Two f32 operations in one instruction.
__device__ __forceinline__ float2 add_pair(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul_pair(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma_pair(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 w, x, y, z;\n\tmov.b64 w, {%2, %3};\n\tmov.b64 x, {%4, %5};\n\tmov.b64 y, {%6, %7};\n\tfma.rn.f32x2 z, w, x, y;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

}  // namespace ctb
