// Heads turned by the angles of their tokens: what a CTA of ctb_rope does, and one of ctb_kv_write with queries.
#pragma once
#include <algorithm>

#include "rotate.cuh"

namespace ctb {

constexpr int kRopeThreads = 256;

struct RopeSide {
  const void* src;
  void* dst;
  int64_t src_b, dst_b;
  int src_s, src_h, dst_s, dst_h, heads;
};
struct RopeParams {
  RopeSide side[2];
  const void* positions;
  const double* frequencies;
  AngleTable table;
  Divisor by_seq, by_token, by_units;  // units of a token, of a head
  int64_t units_all;
  int span;  // units of a CTA
  int tokens, q_heads, dim, turned, wide, interleaved, inverse;
  float scale;
};

// V: elements of a vector (16 bytes), or 1 where something does not lie on the 16-byte grid.  A unit of a head is V pairs (two
// vectors, or with interleaved pairs two neighbouring ones), or for what is only copied two vectors.  A thread asks for its U units, then
// takes its share of the CTA's angles, and turns the units behind the barrier.
template <typename T, int V, int U>
__device__ __forceinline__ void rope_cta(const RopeParams& p, int cta, float* angles) {
  using Vec = std::conditional_t<V == 1, T, uint4>;
  const int64_t unit0 = (int64_t)cta * p.span;
  const int t0 = (int)(unit0 / p.by_token.d);
  const uint32_t local0 = (uint32_t)(unit0 - (int64_t)t0 * p.by_token.d), n = (uint32_t)min((int64_t)p.span, p.units_all - unit0);
  Vec x[U], y[U];
  T* to[U];
  int at[U], run[U], e0[U], e1[U];  // angles of the unit's token (-1: none) and run, the first elements of its vectors
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const uint32_t i = threadIdx.x + k * blockDim.x;
    to[k] = nullptr;
    if (i >= n) continue;
    const uint32_t t = p.by_token(local0 + i), r = local0 + i - t * p.by_token.d, h = p.by_units(r), u = r - h * p.by_units.d;
    const bool second = (int)h >= p.q_heads;
    const RopeSide& s = p.side[second];
    const int head = second ? h - p.q_heads : h;
    const int token = t0 + t, b = p.by_seq(token), place = token - b * (int)p.by_seq.d;
    const T* src = static_cast<const T*>(s.src) + (b * s.src_b + (int64_t)place * s.src_s + (int64_t)head * s.src_h);
    to[k] = static_cast<T*>(s.dst) + (b * s.dst_b + (int64_t)place * s.dst_s + (int64_t)head * s.dst_h);
    const bool turned = (int)u < p.turned;
    at[k] = turned ? (int)t * 2 * p.table.pairs : -1;
    run[k] = u;
    e0[k] = !turned ? 2 * p.table.pairs + (u - p.turned) * 2 * V : p.interleaved ? u * 2 * V : u * V;
    e1[k] = turned && !p.interleaved ? p.table.pairs + u * V : e0[k] + V;
    if constexpr (V == 1) {
      x[k] = src[e0[k]];
      y[k] = e1[k] < p.dim ? src[e1[k]] : T(0.f);
    } else {
      x[k] = __ldcs(reinterpret_cast<const uint4*>(src + e0[k]));
      y[k] = e1[k] < p.dim ? __ldcs(reinterpret_cast<const uint4*>(src + e1[k])) : make_uint4(0, 0, 0, 0);
    }
  }
  const int tokens = (int)p.by_token(local0 + n - 1) + 1;
  p.table.fill(angles, p.positions, p.wide, t0, tokens, p.frequencies, p.scale, p.inverse, threadIdx.x, blockDim.x);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < U; ++k) {
    if (!to[k]) continue;
    if (at[k] >= 0) {
      const float* table = angles + at[k];
      if constexpr (V == 1) {
        const float a = to_float(x[k]), b = to_float(y[k]), c = table[2 * run[k]], d = table[2 * run[k] + 1];
        x[k] = from_float<T>(a * c - b * d);
        y[k] = from_float<T>(a * d + b * c);
      } else {
        uint32_t a[4] = {x[k].x, x[k].y, x[k].z, x[k].w}, b[4] = {y[k].x, y[k].y, y[k].z, y[k].w};
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          const TwoAngles t = angles_of(table, p.turned, run[k], i);
          auto turned = [&](Pair& u, Pair& v) {
            const Pair first = fma2(v, minus(t.sin), mul2(u, t.cos));
            v = fma2(v, t.cos, mul2(u, t.sin));
            u = first;
          };
          Pair u, v;
          if (p.interleaved) {
            uint32_t (&w)[4] = i < V / 4 ? a : b;
            split_pairs<T>(w, i % (V / 4), u, v);
            turned(u, v);
            join_pairs<T>(w, i % (V / 4), u, v);
          } else {
            u = vec_pair<T>(a, i);
            v = vec_pair<T>(b, i);
            turned(u, v);
            put_pair<T>(a, i, u);
            put_pair<T>(b, i, v);
          }
        }
        x[k] = make_uint4(a[0], a[1], a[2], a[3]);
        y[k] = make_uint4(b[0], b[1], b[2], b[3]);
      }
    }
    *reinterpret_cast<Vec*>(to[k] + e0[k]) = x[k];
    if (e1[k] < p.dim) *reinterpret_cast<Vec*>(to[k] + e1[k]) = y[k];
  }
}

// Units, tokens and the CTAs' share of them.  Returns the number of CTAs; threads and the bytes of their angles.
template <int V, int U>
int64_t rope_shares(RopeParams& p, int* threads, size_t* smem) {
  const int pairs = p.table.pairs, heads = p.side[0].heads + p.side[1].heads;
  p.turned = pairs / V;
  p.table = AngleTable(pairs, V == 8 ? 3 : V == 4 ? 2 : 0);
  const int units = p.turned + (p.dim - 2 * pairs + 2 * V - 1) / (2 * V);
  const int64_t per_token = (int64_t)units * heads;
  p.by_units = Divisor(units);
  p.by_token = Divisor((uint32_t)per_token);
  p.units_all = p.tokens * per_token;
  // Whole tokens where one fits: their angles are worked out once.
  const int64_t most = kRopeThreads * U;
  p.span = (int)(most >= per_token ? most / per_token * per_token : most);
  *threads = (p.span + 32 * U - 1) / (32 * U) * 32;
  *smem = std::max<int64_t>(p.span / per_token + (p.span % per_token != 0), 1 + (per_token > most)) * 2 * pairs * sizeof(float);
  return (p.units_all + p.span - 1) / p.span;
}

}  // namespace ctb
