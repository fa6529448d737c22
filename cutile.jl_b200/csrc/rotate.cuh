// Rotary positions: the angles of a few tokens in shared memory, and rows packed again.
#pragma once
#include "rows.cuh"

namespace ctb {

__device__ __forceinline__ long long index_at(const void* p, bool wide, int64_t i) {
  return wide ? __ldg(static_cast<const long long*>(p) + i) : (long long)__ldg(static_cast<const int*>(p) + i);
}

// scale * (cos, sin) of position * frequency.  The product and its reduction to a turn are in f64: an f32 angle of a far position
// (1e6 radians) has no digits left behind the point.  sincospif then takes half turns in [-1, 1], where its argument is off by
// 2^-25 at most.
__device__ __forceinline__ float2 turn(long long position, double frequency, float scale) {
  double t = (double)position * (frequency * 0.15915494309189535);  // turns
  t -= rint(t);
  float s, c;
  sincospif((float)(2.0 * t), &s, &c);
  return make_float2(c * scale, s * scale);
}

// Threads that work on neighbouring runs of `step` pairs read the k-th pair of their runs at the same time: it lies next to its like.
struct AngleTable {
  int pairs, step, runs;  // runs = ceil(pairs / step)
  __host__ __device__ int size() const { return step * runs; }
  __device__ __forceinline__ int at(int run, int k) const { return k * runs + run; }
  __device__ __forceinline__ void fill(float2* table, const void* positions, bool wide, int64_t t0, int tokens, const double* frequencies,
                                       float scale, bool inverse, int thread, int threads) const {
    for (int i = thread; i < tokens * pairs; i += threads) {
      const int t = i / pairs, pair = i - t * pairs;
      float2 a = turn(index_at(positions, wide, t0 + t), __ldg(frequencies + pair), scale);
      if (inverse) a.y = -a.y;
      table[t * size() + at(pair / step, pair % step)] = a;
    }
  }
};

template <typename T>
__device__ __forceinline__ uint4 pack_row(const float (&f)[16 / sizeof(T)]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 8 / (int)sizeof(T); ++i) put_pair<T>(w, i, pair(f[2 * i], f[2 * i + 1]));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace ctb
