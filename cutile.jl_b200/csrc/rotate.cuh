// Rotary positions: the angles of a few tokens in shared memory, and rows packed again.
#pragma once
#include "rows.cuh"

namespace ctb {

__device__ __forceinline__ long long index_at(const void* p, bool wide, int64_t i) {
  return wide ? __ldg(static_cast<const long long*>(p) + i) : (long long)__ldg(static_cast<const int*>(p) + i);
}

// n / d for n < 2^31 and 1 <= d < 2^31 by a multiplication (Granlund and Montgomery, Division by Invariant Integers using Multiplication, 1994):
// with 2^(s - 1) < d <= 2^s and m = floor(2^32 (2^s - d) / d) + 1, n / d = (n + (m n >> 32)) >> s.
struct Divisor {
  uint32_t d, m, s;
  Divisor() = default;
  explicit Divisor(uint32_t by) : d(by), s(0) {
    while ((1ull << s) < d) ++s;
    m = (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (n + __umulhi(n, m)) >> s; }
};

// scale * (cos, sin) of position * frequency.  The product and its reduction to half a turn are in f64, the latter by 2 pi in two
// numbers: an f32 angle of a far position (1e6 radians) has no digits left behind the point.  sincospif then takes half turns in [-1, 1], where
// its argument is off by 2^-25 at most.
__device__ __forceinline__ float2 turn(long long position, double frequency, float scale) {
  const double a = (double)position * frequency, n = rint(a * 0.15915494309189535);
  const double r = fma(n, -2.4492935982947064e-16, fma(n, -6.283185307179586, a));
  float s, c;
  sincospif((float)(r * 0.3183098861837907), &s, &c);
  return make_float2(c * scale, s * scale);
}

// The angles of a few tokens in shared memory.  Threads take neighbouring runs of 2^step_log2 pairs and read the k-th and (k + 1)-th pair of
// their runs at the same time, so these lie together, as (cos, cos, sin, sin), next to those of the other runs.  A step of 1: (cos, sin).
struct AngleTable {
  int pairs, step_log2, runs;  // runs << step_log2 = pairs
  Divisor by_pairs;
  AngleTable() = default;
  AngleTable(int pairs, int step_log2) : pairs(pairs), step_log2(step_log2), runs(pairs >> step_log2), by_pairs(pairs ? pairs : 1) {}
  __device__ __forceinline__ void fill(float* table, const void* positions, bool wide, int64_t t0, int tokens, const double* frequencies,
                                       float scale, bool inverse, int thread, int threads) const {
    for (int i = thread; i < tokens * pairs; i += threads) {
      const int t = by_pairs(i), pair = i - t * pairs;
      const float2 a = turn(index_at(positions, wide, t0 + t), __ldg(frequencies + pair), scale);
      const int run = pair >> step_log2, k = pair - (run << step_log2);
      float* to = table + 2 * t * pairs + (step_log2 == 0 ? 2 * pair : ((k >> 1) * runs + run) * 4 + (k & 1));
      to[0] = a.x;
      to[step_log2 == 0 ? 1 : 2] = inverse ? -a.y : a.y;
    }
  }
};
// Pairs 2 i and 2 i + 1 of a run, step > 1; table: of the token.
struct TwoAngles {
  Pair cos, sin;
};
__device__ __forceinline__ TwoAngles angles_of(const float* table, int runs, int run, int i) {
  const float4 a = reinterpret_cast<const float4*>(table)[i * runs + run];
  return {pair(a.x, a.y), pair(a.z, a.w)};
}
__device__ __forceinline__ Pair minus(Pair a) { return a ^ 0x8000000080000000ull; }

// Words 2 i and 2 i + 1 of interleaved pairs in 16 bits, or a vector's two pairs in f32, as (x, x) and (y, y), and back.
template <typename T>
__device__ __forceinline__ void split_pairs(const uint32_t (&w)[4], int i, Pair& x, Pair& y) {
  if constexpr (sizeof(T) == 4) {
    x = pair(__uint_as_float(w[0]), __uint_as_float(w[2]));
    y = pair(__uint_as_float(w[1]), __uint_as_float(w[3]));
  } else {
    const float2 a = word_pair<T>(w[2 * i]), b = word_pair<T>(w[2 * i + 1]);
    x = pair(a.x, b.x);
    y = pair(a.y, b.y);
  }
}
template <typename T>
__device__ __forceinline__ void join_pairs(uint32_t (&w)[4], int i, Pair x, Pair y) {
  const float2 a = halves(x), b = halves(y);
  put_pair<T>(w, 2 * i, pair(a.x, b.x));
  put_pair<T>(w, 2 * i + 1, pair(a.y, b.y));
}

}  // namespace ctb
