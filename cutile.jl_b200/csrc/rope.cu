// Rotary positions (ctb_rope): pairs of elements of every head turned by the angle of their token.
//
// What bounds it is HBM: every element is read and written once, for three operations.  The angles are the only arithmetic of note (an f64
// product, a reduction and a sincospif, about 60 instructions), and all heads of a token share them: a CTA takes a run of heads, asks for
// them, works out the angles of their tokens, a thread each, into shared memory while they come, and turns them.
#include <math.h>

#include <algorithm>

#include "ctx.h"
#include "ptx.cuh"
#include "rotate.cuh"

using namespace ctb;
using namespace ctb_internal;

namespace {

constexpr int kMaxThreads = 256;

struct Side {
  const void* src;
  void* dst;
  int src_b, src_s, src_h, dst_b, dst_s, dst_h;
};
struct Params {
  Side side[2];
  const void* positions;
  const double* frequencies;
  AngleTable table;
  Divisor by_seq, by_token, by_units;  // units of a token, of a head
  int64_t units_all;
  int span;  // units of a CTA
  int tokens, seq, q_heads, dim, turned, wide, interleaved, inverse;
  float scale;
};

// V: elements of a vector (16 bytes), or 1 where something does not lie on the 16-byte grid.  A unit of a head is V pairs (two
// vectors, or with interleaved pairs two neighbouring ones), or for what is only copied two vectors.  A thread asks for its U units, then
// takes its share of the CTA's angles, and turns the units behind the barrier.
template <typename T, int V, int U>
__global__ void __launch_bounds__(kMaxThreads, 4) rope_kernel(const Params p) {
  using Vec = std::conditional_t<V == 1, T, uint4>;
  extern __shared__ __align__(16) float angles[];
  const int64_t unit0 = (int64_t)blockIdx.x * p.span;
  const int t0 = (int)(unit0 / p.by_token.d);
  const uint32_t local0 = (uint32_t)(unit0 - (int64_t)t0 * p.by_token.d), n = (uint32_t)min((int64_t)p.span, p.units_all - unit0);
  grid_dependency_sync();
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
    const Side& s = p.side[second];
    const int head = second ? h - p.q_heads : h;
    const int token = t0 + t, b = p.by_seq(token), place = token - b * (int)p.by_seq.d;
    const T* src = static_cast<const T*>(s.src) + ((int64_t)b * s.src_b + (int64_t)place * s.src_s + (int64_t)head * s.src_h);
    to[k] = static_cast<T*>(s.dst) + ((int64_t)b * s.dst_b + (int64_t)place * s.dst_s + (int64_t)head * s.dst_h);
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

template <typename T, int V, int U>
int launch(cudaStream_t st, Params p) {
  const int64_t per_token = p.by_token.d;
  // Whole tokens where one fits: their angles are worked out once.
  p.span = (int)(kMaxThreads * U >= per_token ? kMaxThreads * U / per_token * per_token : kMaxThreads * U);
  const int threads = (p.span + 32 * U - 1) / (32 * U) * 32;
  const int64_t grid = (p.units_all + p.span - 1) / p.span, tokens = std::max<int64_t>(p.span / per_token, 1) + (p.span % per_token != 0);  // that a CTA has units of
  if (grid > INT32_MAX) return fail(CTB_UNSUPPORTED, "ctb_rope: shape too large");
  const size_t smem = tokens * 2 * p.table.pairs * sizeof(float);
  auto kern = rope_kernel<T, V, U>;
  launch_kernel(kern, (unsigned)grid, threads, smem, st, 0, p);
  CTB_CHECK_LAUNCH("ctb_rope launch");
  return CTB_OK;
}

template <typename T>
int launch(ctb_ctx* ctx, cudaStream_t st, Params p, int heads, bool vectors) {
  constexpr int V = 16 / (int)sizeof(T);
  const int v = vectors ? V : 1, pairs = p.table.pairs;
  p.turned = pairs / v;
  p.table = AngleTable(pairs, v == 8 ? 3 : v == 4 ? 2 : 0);
  const int units = p.turned + (p.dim - 2 * pairs + 2 * v - 1) / (2 * v);
  p.by_units = Divisor(units);
  p.by_token = Divisor(units * heads);
  p.units_all = (int64_t)p.tokens * units * heads;
  const bool many = p.units_all >= (int64_t)kMaxThreads * 2 * 4 * ctx->sm_count;  // two units per thread still give every SM four CTAs
  if (vectors) return many ? launch<T, V, 2>(st, p) : launch<T, V, 1>(st, p);
  return many ? launch<T, 1, 2>(st, p) : launch<T, 1, 1>(st, p);
}

}  // namespace

namespace ctb_internal {

int check_turned_in_place(const char* who, const void* in, const int64_t* in_strides, const void* out, const int64_t* out_strides,
                          const int64_t* extents, int64_t D, int64_t elem_size) {
  int64_t in_last = D, out_last = D;
  bool same = in == out;
  for (int i = 0; i < 3; ++i) {
    const int64_t n = extents[i] - 1;
    if (n == 0) continue;
    if (in_strides[i] < 0 || out_strides[i] < 0) return fail(CTB_BAD_ARG, "%s: negative strides", who);
    if (out_strides[i] < D) return fail(CTB_BAD_ARG, "%s: the rows of a result overlap", who);
    if (in_strides[i] > INT64_MAX / 64 / n || out_strides[i] > INT64_MAX / 64 / n) return fail(CTB_UNSUPPORTED, "%s: strides too large", who);
    in_last += n * in_strides[i];
    out_last += n * out_strides[i];
    same &= in_strides[i] == out_strides[i];
  }
  const uintptr_t a = (uintptr_t)in, b = (uintptr_t)out;
  if (same || a + in_last * elem_size <= b || b + out_last * elem_size <= a) return CTB_OK;
  return fail(CTB_BAD_ARG, "%s: a result must lie where its rows lie or not overlap them", who);
}

}  // namespace ctb_internal

extern "C" int ctb_rope(ctb_ctx* ctx, void* stream, void* q_out, const void* q, void* k_out, const void* k, const void* positions,
                        int position_bits, const double* frequencies, int64_t batch, int64_t seq, int64_t q_heads, int64_t k_heads,
                        int64_t D, int64_t rotary, const int64_t* strides, int interleaved, int inverse, float scale, int dtype) {
  CTB_CHECK_CTX(ctx);
  CurrentDevice on(ctx);
  if (!strides) return fail(CTB_BAD_ARG, "ctb_rope: no strides");
  if (batch < 0 || seq < 0 || q_heads <= 0 || k_heads < 0 || D <= 0) return fail(CTB_BAD_ARG, "ctb_rope: non-positive dimension");
  if (rotary <= 0 || rotary % 2 || rotary > D) return fail(CTB_BAD_ARG, "ctb_rope: rotary must be even and between 2 and the head's dimension");
  if (position_bits != 32 && position_bits != 64) return fail(CTB_BAD_ARG, "ctb_rope: positions are 32- or 64-bit");
  if (dtype != CTB_F32 && dtype != CTB_F16 && dtype != CTB_BF16) return fail(CTB_UNSUPPORTED, "ctb_rope: f32, f16 and bf16 are implemented");
  if (!isfinite(scale)) return fail(CTB_BAD_ARG, "ctb_rope: scale is not finite");
  if (D > 4096 || q_heads + k_heads > 65536 || seq > INT32_MAX || (seq && batch > INT32_MAX / seq))
    return fail(CTB_UNSUPPORTED, "ctb_rope: shape too large");
  if (batch * seq == 0) return CTB_OK;
  CTB_CHECK_DEV(q); CTB_CHECK_DEV(q_out); CTB_CHECK_DEV(positions); CTB_CHECK_DEV(frequencies);
  if (k_heads) { CTB_CHECK_DEV(k); CTB_CHECK_DEV(k_out); }
  Params p = {};
  const int64_t size = dtype == CTB_F32 ? 4 : 2, V = 16 / size;
  bool vectors = rotary % (2 * V) == 0 && D % V == 0;
  for (int i = 0; i < (k_heads ? 2 : 1); ++i) {
    const int64_t* s = strides + 6 * i;
    for (int j = 0; j < 6; ++j)
      if (s[j] > INT32_MAX) return fail(CTB_UNSUPPORTED, "ctb_rope: strides too large");
    p.side[i] = Side{i ? k : q, i ? k_out : q_out, (int)s[3], (int)s[4], (int)s[5], (int)s[0], (int)s[1], (int)s[2]};
    const int64_t extents[3] = {batch, seq, i ? k_heads : q_heads};
    const int r = check_turned_in_place("ctb_rope", p.side[i].src, s + 3, p.side[i].dst, s, extents, D, size);
    if (r) return r;
    vectors &= (uintptr_t)p.side[i].src % 16 == 0 && (uintptr_t)p.side[i].dst % 16 == 0;
    for (int j = 0; j < 6; ++j) vectors &= extents[j % 3] == 1 || s[j] % V == 0;
  }
  p.positions = positions;
  p.frequencies = frequencies;
  p.tokens = (int)(batch * seq);
  p.by_seq = Divisor((uint32_t)seq);
  p.seq = (int)seq; p.q_heads = (int)q_heads; p.table.pairs = (int)(rotary / 2); p.dim = (int)D;
  p.wide = position_bits == 64; p.interleaved = interleaved != 0; p.inverse = inverse != 0;
  p.scale = scale;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int heads = (int)(q_heads + k_heads);
  if (dtype == CTB_F32) return launch<float>(ctx, st, p, heads, vectors);
  if (dtype == CTB_F16) return launch<__half>(ctx, st, p, heads, vectors);
  return launch<__nv_bfloat16>(ctx, st, p, heads, vectors);
}
