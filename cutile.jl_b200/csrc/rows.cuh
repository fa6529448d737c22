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
// A vector of -inf.
template <typename T>
__device__ __forceinline__ uint4 empty_row_vec() {
  const uint32_t w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  return make_uint4(w, w, w, w);
}

// A 32-bit word of a row is one f32 or two 16-bit elements.  Larger of two words, element by element; a number where one of them is NaN.
template <typename T>
__device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (sizeof(T) == 4) asm("max.f32 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else if constexpr (std::is_same<T, __half>::value) asm("max.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// The elements of a 16-bit word.
template <typename T>
__device__ __forceinline__ float2 word_pair(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// The larger element of a word.
template <typename T>
__device__ __forceinline__ float word_max(uint32_t w) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(w);
  else {
    const float2 f = word_pair<T>(w);
    return fmaxf(f.x, f.y);
  }
}

__device__ __forceinline__ double sum_lanes(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Two f32 values in a 64-bit register, and operations that take one instruction for both.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 halves(Pair a) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(a));
  return f;
}
__device__ __forceinline__ float sum_of(Pair a) {
  const float2 f = halves(a);
  return f.x + f.y;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ Pair exp2_pair(Pair t) {
  const float2 f = halves(t);
  float a, b;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(f.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(f.y));
  return pair(a, b);
}

// Pair i of a vector's elements.
template <typename T>
__device__ __forceinline__ Pair vec_pair(const uint32_t (&w)[4], int i) {
  if constexpr (sizeof(T) == 4) return pair(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
  else {
    const float2 f = word_pair<T>(w[i]);
    return pair(f.x, f.y);
  }
}
template <typename T>
__device__ __forceinline__ void put_pair(uint32_t (&w)[4], int i, Pair d) {
  const float2 f = halves(d);
  if constexpr (sizeof(T) == 4) {
    w[2 * i] = __float_as_uint(f.x);
    w[2 * i + 1] = __float_as_uint(f.y);
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(f.x, f.y);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
}

// A row and the vectors [v0, v1) of it.
template <typename T>
struct Range {
  static constexpr int V = 16 / (int)sizeof(T);
  const T* src;
  int off, n, v0, v1;

  __device__ __forceinline__ bool has(int v, int i) const {  // element i of vector v is one of the row
    const int e = v * V - off + i;
    return e >= 0 && e < n;
  }
  // Vectors [v, v + count) lie wholly inside of the row and the range.
  __device__ __forceinline__ bool inside(int v, int count) const {
    return (v > 0 || off == 0) && v + count <= v1 && (v + count) * V - off <= n;
  }
  __device__ __forceinline__ const uint4* at(int v) const { return reinterpret_cast<const uint4*>(src - off) + v; }
};

// A vector that may be partly outside of the row; -inf there, and beyond the range.
template <typename T>
__device__ __noinline__ uint4 load_edge(const T* src, int off, int n, int v) {
  constexpr int V = 16 / (int)sizeof(T);
  const uint4 empty = empty_row_vec<T>();
  alignas(uint4) T f[V];  // read as one vector below
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = v * V - off + i;
    f[i] = e >= 0 && e < n ? src[e] : reinterpret_cast<const T*>(&empty)[0];
  }
  return *reinterpret_cast<const uint4*>(f);
}
template <typename T>
__device__ __forceinline__ uint4 load_vec(const Range<T>& r, int v) {
  if (v >= r.v1) return empty_row_vec<T>();
  if (r.inside(v, 1)) return __ldcs(r.at(v));
  return load_edge<T>(r.src, r.off, r.n, v);
}
// Writes a vector to a row that starts like r; what is outside of the row is left as it is.
template <typename T>
__device__ __noinline__ void store_edge(T* dst, int off, int n, int v, uint4 q) {
  constexpr int V = 16 / (int)sizeof(T);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = v * V - off + i;
    if (e >= 0 && e < n) dst[e] = reinterpret_cast<const T*>(&q)[i];
  }
}

}  // namespace ctb
