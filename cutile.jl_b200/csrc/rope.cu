// Rotary positions (ctb_rope): pairs of elements of every head turned by the angle of their token.
//
// What bounds it is HBM: every element is read and written once, for three operations.  The angles are the only arithmetic of note (an f64
// product, a reduction and a sincospif, about 60 instructions), and all heads of a token share them: a CTA takes the heads of a few tokens (or
// a part of one's), asks for them, works out the angles, a thread each, into shared memory while they come, and turns them.  16384 tokens
// of 32 + 8 heads of 128 in bf16 (336 MB) 51.4 us, the copy rate; interleaved pairs 55, f32 52 (its 8192 tokens are as many bytes), 80
// dimensions 18 for a floor of 13 (a head is ten vectors, five units); 8 tokens 1.6 us.  Small CTAs count, as they hide each other's barrier:
// 512 threads 61 us; CTAs that begin within a token, and so work out more angles than they need, 55; four heads per thread, which
// share what is read of the angles, 64 (83 registers).
#include <math.h>

#include <algorithm>

#include "ctx.h"
#include "ptx.cuh"
#include "rope.cuh"

using namespace ctb;
using namespace ctb_internal;

namespace {

template <typename T, int V, int U>
__global__ void __launch_bounds__(kRopeThreads, 4) rope_kernel(const RopeParams p) {
  extern __shared__ __align__(16) float angles[];
  grid_dependency_sync();
  rope_cta<T, V, U>(p, blockIdx.x, angles);
}

template <typename T, int V, int U>
int launch(cudaStream_t st, RopeParams p) {
  int threads;
  size_t smem;
  const int64_t grid = rope_shares<V, U>(p, &threads, &smem);
  if (grid > INT32_MAX) return fail(CTB_UNSUPPORTED, "ctb_rope: shape too large");
  launch_kernel(rope_kernel<T, V, U>, (unsigned)grid, threads, smem, st, 0, p);
  CTB_CHECK_LAUNCH("ctb_rope launch");
  return CTB_OK;
}

template <typename T>
int launch(ctb_ctx* ctx, cudaStream_t st, const RopeParams& p, bool vectors) {
  constexpr int V = 16 / (int)sizeof(T);
  // two units per thread where that still gives every SM four CTAs
  const int64_t elements = (int64_t)p.tokens * (p.side[0].heads + p.side[1].heads) * p.dim;
  const bool many = elements >= 2ll * (vectors ? V : 1) * kRopeThreads * 2 * 4 * ctx->sm_count;
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
    if (in_strides[i] > INT64_MAX / 64 / n || out_strides[i] > INT64_MAX / 64 / n) return fail(CTB_UNSUPPORTED, "%s: strides too large", who);
    in_last += n * in_strides[i];
    out_last += n * out_strides[i];
    same &= in_strides[i] == out_strides[i];
  }
  // In the order of their strides, the rows of a dimension lie behind all that one of them has.
  int64_t reach = D;
  bool seen[3] = {};
  for (int step = 0; step < 3; ++step) {
    int next = -1;
    for (int i = 0; i < 3; ++i)
      if (!seen[i] && extents[i] > 1 && (next < 0 || out_strides[i] < out_strides[next])) next = i;
    if (next < 0) break;
    if (out_strides[next] < reach) return fail(CTB_BAD_ARG, "%s: the rows of a result overlap", who);
    seen[next] = true;
    reach += (extents[next] - 1) * out_strides[next];
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
  RopeParams p = {};
  const int64_t size = dtype == CTB_F32 ? 4 : 2, V = 16 / size;
  bool vectors = rotary % (2 * V) == 0 && D % V == 0;
  for (int i = 0; i < (k_heads ? 2 : 1); ++i) {
    const int64_t extents[3] = {batch, seq, i ? k_heads : q_heads};
    int64_t s[6];
    for (int j = 0; j < 6; ++j) {
      s[j] = extents[j % 3] == 1 ? 0 : strides[6 * i + j];
      if (j % 3 && s[j] > INT32_MAX) return fail(CTB_UNSUPPORTED, "ctb_rope: strides too large");
    }
    p.side[i] = RopeSide{i ? k : q, i ? k_out : q_out, s[3], s[0], (int)s[4], (int)s[5], (int)s[1], (int)s[2], (int)extents[2]};
    const int r = check_turned_in_place("ctb_rope", p.side[i].src, s + 3, p.side[i].dst, s, extents, D, size);
    if (r) return r;
    vectors &= (uintptr_t)p.side[i].src % 16 == 0 && (uintptr_t)p.side[i].dst % 16 == 0;
    for (int j = 0; j < 6; ++j) vectors &= s[j] % V == 0;
  }
  p.positions = positions;
  p.frequencies = frequencies;
  p.tokens = (int)(batch * seq);
  p.by_seq = Divisor((uint32_t)seq);
  p.q_heads = (int)q_heads; p.table.pairs = (int)(rotary / 2); p.dim = (int)D;
  p.wide = position_bits == 64; p.interleaved = interleaved != 0; p.inverse = inverse != 0;
  p.scale = scale;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == CTB_F32) return launch<float>(ctx, st, p, vectors);
  if (dtype == CTB_F16) return launch<__half>(ctx, st, p, vectors);
  return launch<__nv_bfloat16>(ctx, st, p, vectors);
}
