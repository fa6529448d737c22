// Rotary positions (ctb_rope): pairs of elements of every head turned by the angle of their token.
//
// What bounds it is HBM: every element is read and written once, for three operations.  The angles are the only arithmetic of note (an f64
// product, a reduction and a sincospif, about 60 instructions), and all heads of a token share them: a CTA takes a few tokens, works out their
// angles once, a thread each, into shared memory, and then walks over the tokens' heads.
#include <math.h>

#include <algorithm>

#include "ctx.h"
#include "ptx.cuh"
#include "rotate.cuh"

using namespace ctb;
using namespace ctb_internal;

namespace {

constexpr int kThreads = 256, kMaxPairs = 2048;  // angles of a CTA

struct Side {
  const void* src;
  void* dst;
  int64_t src_b, src_s, src_h, dst_b, dst_s, dst_h;
};
struct Params {
  Side side[2];
  const void* positions;
  const double* frequencies;
  int64_t tokens;
  AngleTable table;
  int seq, q_heads, heads, pairs, dim, turned, units, per_cta, wide, interleaved, inverse;
  float scale;
};

// V: elements of a vector (16 bytes), or 1 where something does not lie on the 16-byte grid.  A unit of a head is V pairs (two
// vectors, or with interleaved pairs two neighbouring ones), or for what is only copied two vectors.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) rope_kernel(const Params p) {
  __shared__ float2 angles[kMaxPairs];
  const int64_t t0 = (int64_t)blockIdx.x * p.per_cta;
  const int tokens = (int)min((int64_t)p.per_cta, p.tokens - t0);
  grid_dependency_sync();
  p.table.fill(angles, p.positions, p.wide, t0, tokens, p.frequencies, p.scale, p.inverse, threadIdx.x, kThreads);
  __syncthreads();
  const int per_token = p.heads * p.units;
  for (int i = threadIdx.x; i < tokens * per_token; i += kThreads) {
    const int t = i / per_token, r = i - t * per_token, h = r / p.units, u = r - h * p.units;
    const bool second = h >= p.q_heads;
    const Side& s = p.side[second];
    const int head = second ? h - p.q_heads : h;
    const int64_t token = t0 + t, b = token / p.seq, n = token - b * p.seq;
    const T* src = static_cast<const T*>(s.src) + b * s.src_b + n * s.src_s + head * s.src_h;
    T* dst = static_cast<T*>(s.dst) + b * s.dst_b + n * s.dst_s + head * s.dst_h;
    const float2* a = angles + t * p.table.size();
    auto angle = [&](int k) { return a[p.table.at(u, k)]; };  // of pair u * V + k
    const bool turned = u < p.turned;
    // the unit's two vectors
    int e0, e1;
    if (!turned) {
      e0 = 2 * p.pairs + (u - p.turned) * 2 * V;
      e1 = e0 + V;
    } else if (p.interleaved) {
      e0 = u * 2 * V;
      e1 = e0 + V;
    } else {
      e0 = u * V;
      e1 = p.pairs + u * V;
    }
    if constexpr (V == 1) {
      float x = to_float(src[e0]), y = e1 < p.dim ? to_float(src[e1]) : 0.f;
      if (turned) {
        const float2 cs = angle(0);
        const float x1 = x * cs.x - y * cs.y, y1 = x * cs.y + y * cs.x;
        dst[e0] = from_float<T>(x1);
        dst[e1] = from_float<T>(y1);
      } else {
        dst[e0] = src[e0];
        if (e1 < p.dim) dst[e1] = src[e1];
      }
    } else {
      uint4 q0 = __ldcs(reinterpret_cast<const uint4*>(src + e0));
      uint4 q1 = e1 < p.dim ? __ldcs(reinterpret_cast<const uint4*>(src + e1)) : make_uint4(0, 0, 0, 0);
      if (turned) {
        float x[V], y[V];
        unpack_row<T>(q0, x);
        unpack_row<T>(q1, y);
        if (p.interleaved) {
#pragma unroll
          for (int k = 0; k < V; k += 2) {
            const float2 c0 = angle(k / 2), c1 = angle(V / 2 + k / 2);
            const float x0 = x[k] * c0.x - x[k + 1] * c0.y, y0 = y[k] * c1.x - y[k + 1] * c1.y;
            x[k + 1] = x[k] * c0.y + x[k + 1] * c0.x;
            y[k + 1] = y[k] * c1.y + y[k + 1] * c1.x;
            x[k] = x0;
            y[k] = y0;
          }
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const float2 cs = angle(k);
            const float x0 = x[k] * cs.x - y[k] * cs.y;
            y[k] = x[k] * cs.y + y[k] * cs.x;
            x[k] = x0;
          }
        }
        q0 = pack_row<T>(x);
        q1 = pack_row<T>(y);
      }
      *reinterpret_cast<uint4*>(dst + e0) = q0;
      if (e1 < p.dim) *reinterpret_cast<uint4*>(dst + e1) = q1;
    }
  }
}

template <typename T>
int launch(ctb_ctx* ctx, cudaStream_t st, Params p, bool vectors) {
  constexpr int V = 16 / (int)sizeof(T);
  const int v = vectors ? V : 1;
  p.turned = p.pairs / v;
  p.table = AngleTable{p.pairs, v, p.turned};
  p.units = p.turned + (p.dim - 2 * p.pairs + 2 * v - 1) / (2 * v);
  p.per_cta = (int)std::max<int64_t>(1, std::min<int64_t>(kMaxPairs / p.pairs, p.tokens / (ctx->sm_count * 8)));
  const int64_t grid = (p.tokens + p.per_cta - 1) / p.per_cta;
  if (grid > INT32_MAX) return fail(CTB_UNSUPPORTED, "ctb_rope: shape too large");
  launch_kernel(vectors ? rope_kernel<T, V> : rope_kernel<T, 1>, (unsigned)grid, kThreads, 0, st, 0, p);
  CTB_CHECK_LAUNCH("ctb_rope launch");
  return CTB_OK;
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
  if (D > 4096 || q_heads + k_heads > 65536 || seq > INT32_MAX || (seq && batch > INT64_MAX / seq))
    return fail(CTB_UNSUPPORTED, "ctb_rope: shape too large");
  if (batch * seq == 0) return CTB_OK;
  CTB_CHECK_DEV(q); CTB_CHECK_DEV(q_out); CTB_CHECK_DEV(positions); CTB_CHECK_DEV(frequencies);
  if (k_heads) { CTB_CHECK_DEV(k); CTB_CHECK_DEV(k_out); }
  Params p = {};
  const int64_t size = dtype == CTB_F32 ? 4 : 2, V = 16 / size;
  bool vectors = rotary % (2 * V) == 0 && D % V == 0;
  for (int i = 0; i < (k_heads ? 2 : 1); ++i) {
    const int64_t* s = strides + 6 * i;
    p.side[i] = Side{i ? k : q, i ? k_out : q_out, s[3], s[4], s[5], s[0], s[1], s[2]};
    const int64_t extents[3] = {batch, seq, i ? k_heads : q_heads};
    const int r = check_turned_in_place("ctb_rope", p.side[i].src, s + 3, p.side[i].dst, s, extents, D, size);
    if (r) return r;
    vectors &= (uintptr_t)p.side[i].src % 16 == 0 && (uintptr_t)p.side[i].dst % 16 == 0;
    for (int j = 0; j < 6; ++j) vectors &= extents[j % 3] == 1 || s[j] % V == 0;
  }
  p.positions = positions;
  p.frequencies = frequencies;
  p.tokens = batch * seq;
  p.seq = (int)seq; p.q_heads = (int)q_heads; p.heads = (int)(q_heads + k_heads); p.pairs = (int)(rotary / 2); p.dim = (int)D;
  p.wide = position_bits == 64; p.interleaved = interleaved != 0; p.inverse = inverse != 0;
  p.scale = scale;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == CTB_F32) return launch<float>(ctx, st, p, vectors);
  if (dtype == CTB_F16) return launch<__half>(ctx, st, p, vectors);
  return launch<__nv_bfloat16>(ctx, st, p, vectors);
}
