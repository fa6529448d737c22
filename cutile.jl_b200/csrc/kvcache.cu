// The paged key-value cache: writing new tokens to it (turned by their positions and rounded to 8 bits on the way) and reading sequences back.
//
// Reading is bound by HBM: 4 x 4096 tokens of 8 heads of 128 from e4m3 (101 MB) 15.2 us, the copy rate.
// Writing: by HBM in 16 bits (10240 tokens with 32 + 8 + 8 heads of 128 in bf16, 252 MB, 48 us for 38), by the issue of instructions in 8
// (in e4m3 51 us for 35; int8, keys and values alone, without angles, 20 for 10: a row's maximum, two products and a Newton step per
// element, and the codes, 180 instructions per 256 elements); few tokens by latencies (64: 2.3 us).  A row (one head of one token) is the
// work of D / 8 neighbouring lanes, eight elements each, so that its largest magnitude is found by a few shuffles and its pairs (i, i +
// rotary / 2) meet by one.  Slower: all kinds of rows in the same warps (84 to 98 us for the 51), CTAs that walk over the tokens and ask a
// round ahead (96: registers), one group of rows per warp (110).
#include <math.h>

#include <algorithm>

#include "ctx.h"
#include "ptx.cuh"
#include "rope.cuh"

using namespace ctb;
using namespace ctb_internal;

namespace {

constexpr int kThreads = 256;       // of a CTA that reads
constexpr int kMaxWarps = 8;        // of one that writes
static_assert(kMaxWarps * 32 == kRopeThreads, "CTAs of both kinds in one launch");
constexpr float kSmallest = 7.888609052210118e-31f;  // 2^-100: rows below it are zeros in 8 bits

enum Store { Same = 0, E4M3 = 1, I8 = 2 };

struct Cache {
  void *k, *v;
  float *ks, *vs;
  int64_t k_page, v_page, ks_page, vs_page;
  int kv_heads, page_log2, pages;
};
Cache cache_of(const ctb_kv_cache* c) {
  Cache d = {c->k, c->v, c->k_scale, c->v_scale, c->k_page_stride, c->v_page_stride, c->k_scale_page_stride, c->v_scale_page_stride,
             (int)c->kv_heads, 0, (int)c->pages};
  while ((1ll << d.page_log2) < c->page_size) ++d.page_log2;
  return d;
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint32_t w;
  asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\tmov.b32 %0, {l, h};\n\t}"
      : "=r"(w)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return w;
}
__device__ __forceinline__ uint32_t i8x4(float a, float b, float c, float d) {  // 1.5 2^23 + x has x, rounded, in its low bits
  const float m = 12582912.f;
  const uint32_t u = __byte_perm(__float_as_uint(a + m), __float_as_uint(b + m), 0x0040);
  const uint32_t w = __byte_perm(__float_as_uint(c + m), __float_as_uint(d + m), 0x0040);
  return __byte_perm(u, w, 0x5410);
}

enum Kind { Query = 0, Key = 1, Value = 2 };
struct Side {
  const void* src;
  void* dst;           // of queries, or pages
  float* scales;
  int64_t page, scale_page;
  int t_stride, h_stride, heads, tasks;  // tasks of a token
};
struct WriteParams {
  Side side[3];
  const void *slots, *positions;
  const double* frequencies;
  int64_t tokens, places;  // places: of the cache
  int qo_t, qo_h, page_log2;
  AngleTable table;
  Divisor by_token;  // tasks of a token
  int span;          // tokens of a CTA; 0: parts of tokens
  int pairs, wide_slots, wide_positions, interleaved, vectors;  // pairs: 0 without angles
  float scale;
  int rope_vectors, ctas, period;  // CTAs with tasks, one in `period`; the others turn queries
  RopeParams rope;
};

// The largest magnitude of 8 elements, NaN where there is one.
__device__ __forceinline__ float peak_of(const Pair (&x)[4]) {
  float peak = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = halves(x[i]);
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(peak) : "f"(peak), "f"(f.x), "f"(f.y));
  }
  return peak;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// A warp's task is U groups of 32 / (D / 8) neighbouring heads of one token's queries, keys or values: it asks for them, takes its
// share of the CTA's angles and slots while they come, and behind the barrier turns all of them by the angles that it reads once.
// U > 1: many tokens, whose queries are other CTAs' of the same launch, in between: turning them is bound by HBM, rounding to codes by the
// issue of instructions.
template <typename T, int D, int STORE, int U>
__global__ void __launch_bounds__(kMaxWarps * 32, U == 1 ? 1 : 4) kv_write_kernel(const WriteParams p, int* status) {
  constexpr int L = D / 8, kRows = 32 / L;  // lanes of a row, rows of a group
  extern __shared__ __align__(16) float angles[];
  __shared__ long long places[kMaxWarps];
  int cta = blockIdx.x;
  if constexpr (U > 1) {
    if (cta >= p.ctas * p.period || cta % p.period) {
      grid_dependency_sync();
      cta -= cta >= p.ctas * p.period ? p.ctas : cta / p.period + 1;
      if (p.rope_vectors) rope_cta<T, 8, 2>(p.rope, cta, angles);
      else rope_cta<T, 1, 2>(p.rope, cta, angles);
      return;
    }
    cta /= p.period;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = kMaxWarps, chunk = lane & (L - 1), e0 = chunk * 8;
  const int per_token = p.by_token.d;
  const int64_t task0 = (int64_t)cta * (p.span ? p.span * per_token : warps), t0 = p.span ? (int64_t)cta * p.span : task0 / per_token;
  const int local0 = (int)(task0 - t0 * per_token);
  const int n = (int)min((int64_t)(p.span ? p.span * per_token : warps), p.tokens * per_token - task0);  // tasks of the CTA
  const int i = min(warp, n - 1), token = p.by_token(local0 + i);
  const bool busy = warp < n;
  int r = local0 + i - token * per_token;
  const int queries = p.side[Query].tasks, keys = p.side[Key].tasks;
  const int kind = r < queries ? Query : r < queries + keys ? Key : Value;
  r -= kind == Query ? 0 : kind == Key ? queries : queries + keys;
  const Side& side = p.side[kind];
  const int head0 = r * (kRows * U) + lane / L, heads = busy ? side.heads : 0;  // the lane's heads: head0 + k kRows
  grid_dependency_sync();
  const T* src = static_cast<const T*>(side.src) + ((t0 + token) * side.t_stride + (int64_t)head0 * side.h_stride) + e0;
  const int64_t next_src = (int64_t)kRows * side.h_stride;
  uint4 asked[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    asked[k] = make_uint4(0, 0, 0, 0);
    if (head0 + k * kRows >= heads) continue;
    if (p.vectors) asked[k] = __ldcs(reinterpret_cast<const uint4*>(src + k * next_src));
    else {
      alignas(16) T x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = src[k * next_src + j];
      asked[k] = *reinterpret_cast<const uint4*>(x);
    }
  }
  const int tokens = (int)p.by_token(local0 + n - 1) + 1;
  if (p.pairs) p.table.fill(angles, p.positions, p.wide_positions, t0, tokens, p.frequencies, p.scale, false, threadIdx.x, blockDim.x);
  for (int t = threadIdx.x; t < tokens; t += blockDim.x) {
    const long long slot = index_at(p.slots, p.wide_slots, t0 + t);
    const bool bad = slot < 0 || slot > p.places;
    if (bad) atomicMax(status, (int)DEV_BAD_INDEX);
    places[t] = bad ? -1 : slot - 1;
  }
  __syncthreads();
  if (!busy) return;

  const float* table = angles + token * 2 * p.pairs;
  const bool turns = p.pairs && kind != Value, mine = turns && e0 < 2 * p.pairs;  // the lane's elements are turned
  const bool halves_apart = !p.interleaved && p.pairs % 8 == 0, side_by_side = p.interleaved && p.table.step_log2 == 2;
  const int half = p.pairs / 8;
  const bool second = chunk >= half;
  const int other = mine ? (second ? lane - half : lane + half) : lane;
  TwoAngles a[4];
  if (mine && (halves_apart || side_by_side)) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (halves_apart || j < 2) a[j] = angles_of(table, p.table.runs, halves_apart && second ? chunk - half : chunk, j);
    if (halves_apart && !second) {  // x cos - y sin, and y cos + x sin
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j].sin = minus(a[j].sin);
    }
  }
  // Turns the eight elements w of a row; x has them in f32.
  auto turn_row = [&](int k, uint32_t (&w)[4], Pair (&x)[4]) {
    if (halves_apart) {  // a pair's other elements are another lane's eight
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = __shfl_sync(0xffffffffu, w[j], other);
      if (mine) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = fma2(vec_pair<T>(o, j), a[j].sin, mul2(x[j], a[j].cos));
      }
    } else if (side_by_side) {
      if (mine) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          Pair u, v;
          split_pairs<T>(w, j, u, v);
          const float2 f = halves(fma2(v, minus(a[j].sin), mul2(u, a[j].cos))), g = halves(fma2(v, a[j].cos, mul2(u, a[j].sin)));
          x[2 * j] = pair(f.x, g.x);
          x[2 * j + 1] = pair(f.y, g.y);
        }
      }
    } else {
      if (mine && head0 + k * kRows < heads) {  // element by element
        const T* row = src + k * next_src - e0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float f[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int e = e0 + 2 * j + h;
            const bool later = p.interleaved ? e & 1 : e >= p.pairs;
            const int at = p.interleaved ? e >> 1 : later ? e - p.pairs : e;
            f[h] = to_float(reinterpret_cast<const T*>(w)[2 * j + h]);
            if (e >= 2 * p.pairs) continue;
            const float y = to_float(row[p.interleaved ? e ^ 1 : later ? at : e + p.pairs]);
            f[h] = f[h] * table[2 * at] + (later ? y : -y) * table[2 * at + 1];
          }
          x[j] = pair(f[0], f[1]);
        }
      }
      __syncwarp();  // queries in place: what other lanes read here is written below
    }
    if (mine) {
#pragma unroll
      for (int j = 0; j < 4; ++j) put_pair<T>(w, j, x[j]);
    }
  };
  if (U == 1 && kind == Query) {
    T* to = static_cast<T*>(side.dst) + ((t0 + token) * p.qo_t + (int64_t)head0 * p.qo_h) + e0;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      uint32_t w[4] = {asked[k].x, asked[k].y, asked[k].z, asked[k].w};
      Pair x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = vec_pair<T>(w, j);
      turn_row(k, w, x);
      if (head0 + k * kRows >= heads) continue;
      const uint4 words = make_uint4(w[0], w[1], w[2], w[3]);
      if (p.vectors) *reinterpret_cast<uint4*>(to + (int64_t)k * kRows * p.qo_h) = words;
      else {
#pragma unroll
        for (int j = 0; j < 8; ++j) to[(int64_t)k * kRows * p.qo_h + j] = reinterpret_cast<const T*>(&words)[j];
      }
    }
    return;
  }
  const long long place = places[token];
  if (place < 0) return;
  const int64_t page = place >> p.page_log2;
  const int row0 = (head0 << p.page_log2) + (int)(place & ((1 << p.page_log2) - 1)), next_row = kRows << p.page_log2;
  const int64_t to = page * side.page + (int64_t)row0 * D + e0;
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const bool live = head0 + k * kRows < heads;
    uint32_t w[4] = {asked[k].x, asked[k].y, asked[k].z, asked[k].w};
    Pair x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = vec_pair<T>(w, j);
    if (turns) turn_row(k, w, x);
    const int64_t at = to + (int64_t)k * next_row * D;
    if constexpr (STORE == Same) {
      if (live) *reinterpret_cast<uint4*>(static_cast<T*>(side.dst) + at) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      constexpr float kMost = STORE == I8 ? 127.f : 448.f;
      float peak = peak_of(x);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) peak = max_nan(peak, __shfl_xor_sync(0xffffffffu, peak, o));
      if (!live) continue;
      // x c / a (and a / c) with a Newton step behind the product with a reciprocal: quotients that are numbers of f32 come out as they are,
      // so ties are ties
      const bool fine = peak >= kSmallest && peak < INFINITY;
      const float pre = peak > 1.2676506e30f ? 5.9604645e-8f : 1.f;  // beyond 2^100 in units of 2^24: x c is finite
      const float top = peak * pre, inv = rcp_approx_ftz(top), most = pre * kMost;
      const Pair inv2 = pair(inv, inv), top2 = pair(-top, -top), most2 = pair(most, most);
      float y[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const Pair m = mul2(x[j], most2), z = mul2(m, inv2);
        const float2 f = halves(fma2(fma2(z, top2, m), inv2, z));
        y[2 * j] = f.x;
        y[2 * j + 1] = f.y;
      }
      uint2 codes;
      if constexpr (STORE == I8) codes = make_uint2(i8x4(y[0], y[1], y[2], y[3]), i8x4(y[4], y[5], y[6], y[7]));
      else codes = make_uint2(e4m3x4(y[0], y[1], y[2], y[3]), e4m3x4(y[4], y[5], y[6], y[7]));
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(side.dst) + at) = fine ? codes : make_uint2(0, 0);
      if (chunk == 0) {
        const float scale = peak * (1.f / kMost);
        side.scales[page * side.scale_page + row0 + k * next_row] = fine ? fmaf(fmaf(-scale, kMost, peak), 1.f / kMost, scale) : peak < kSmallest ? 0.f : peak;
      }
    }
  }
}

struct ReadParams {
  Cache cache;
  void *K, *V;
  const int32_t *table, *lengths;
  int64_t table_ld;
  int batch, seq, width, blocks;  // blocks of kReadTokens tokens of a head
};
constexpr int kReadTokens = 64;

template <int STORE>
__device__ __forceinline__ void values8(uint2 w, float scale, float (&x)[8]) {
  const uint32_t u[2] = {w.x, w.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (STORE == E4M3) {
      uint32_t lo, hi;
      asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(u[i]));
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
      x[4 * i] = a.x; x[4 * i + 1] = a.y; x[4 * i + 2] = b.x; x[4 * i + 3] = b.y;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * i + j] = (float)(int8_t)(u[i] >> (8 * j));
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] *= scale;
}

template <typename T, int D, int STORE>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const ReadParams p, int* status) {
  constexpr int L = D / 8, kRows = kThreads / L, kTurns = kReadTokens / kRows;  // rows at a time, times
  const int chunk = threadIdx.x % L;
  grid_dependency_sync();
  const int64_t pair = blockIdx.x / p.blocks;  // sequence and head
  const int first = (int)(blockIdx.x - pair * p.blocks) * kReadTokens;
  const int b = (int)(pair / p.cache.kv_heads), head = (int)(pair - (int64_t)b * p.cache.kv_heads);
  const int n = __ldg(p.lengths + b);
  const int64_t most = (int64_t)p.width << p.cache.page_log2;
  bool bad = n < 0 || n > most;
  const int len = (int)min((int64_t)max(n, 0), most);
  using Raw = std::conditional_t<STORE == Same, uint4, uint2>;
  Raw w[kTurns][2];
  float scale[kTurns][2];
  bool hole[kTurns];
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int at = first + i * kRows + threadIdx.x / L;
    hole[i] = bad && (n < 0 || at >= len);
    w[i][0] = w[i][1] = Raw{};
    scale[i][0] = scale[i][1] = 0.f;
    if (at >= len || at >= p.seq) continue;
    const int id = __ldg(p.table + b * p.table_ld + (at >> p.cache.page_log2));
    if ((unsigned)(id - 1) >= (unsigned)p.cache.pages) {
      hole[i] = true;
      continue;
    }
    const int64_t row = ((int64_t)head << p.cache.page_log2) + (at & ((1 << p.cache.page_log2) - 1)), page = id - 1;
    constexpr int E = STORE == Same ? 2 : 1;
    w[i][0] = __ldcs(reinterpret_cast<const Raw*>(static_cast<const char*>(p.cache.k) + (page * p.cache.k_page + row * D + chunk * 8) * E));
    w[i][1] = __ldcs(reinterpret_cast<const Raw*>(static_cast<const char*>(p.cache.v) + (page * p.cache.v_page + row * D + chunk * 8) * E));
    if constexpr (STORE != Same) {
      scale[i][0] = __ldg(p.cache.ks + page * p.cache.ks_page + row);
      scale[i][1] = __ldg(p.cache.vs + page * p.cache.vs_page + row);
    }
  }
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int at = first + i * kRows + threadIdx.x / L;
    if (at >= p.seq) continue;
    bad |= hole[i];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      uint4 out;
      if (hole[i]) out = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
      else if constexpr (STORE == Same) out = w[i][s];
      else {
        float x[8];
        values8<STORE>(w[i][s], scale[i][s], x);
        uint32_t u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) put_pair<T>(u, j, ctb::pair(x[2 * j], x[2 * j + 1]));
        out = make_uint4(u[0], u[1], u[2], u[3]);
      }
      __stcs(reinterpret_cast<uint4*>(static_cast<T*>(s ? p.V : p.K) + (pair * p.seq + at) * D) + chunk, out);
    }
  }
  if (bad && chunk == 0) atomicMax(status, (int)DEV_BAD_INDEX);
}

// The kernel for the types and the head's size of a call.
template <template <typename, int, int> class F, typename... A>
int by_type(int dtype, int64_t D, int store, A&&... args) {
  auto size = [&](auto t, auto s) {
    using T = decltype(t);
    constexpr int STORE = decltype(s)::value;
    return D == 64 ? F<T, 64, STORE>::run(args...) : F<T, 128, STORE>::run(args...);
  };
  auto type = [&](auto s) { return dtype == CTB_F16 ? size(__half(), s) : size(__nv_bfloat16(), s); };
  if (store == CTB_E4M3) return type(std::integral_constant<int, E4M3>());
  if (store == CTB_I8) return type(std::integral_constant<int, I8>());
  return type(std::integral_constant<int, Same>());
}
template <typename T, int D, int STORE>
struct Write {
  template <int U>
  static int launch(ctb_ctx* ctx, cudaStream_t st, WriteParams p) {
    int64_t per_token = 0, queries = 0;
    int threads = kMaxWarps * 32;
    size_t rope_smem = 0;
    if (U > 1 && p.side[Query].heads) {
      queries = p.rope_vectors ? rope_shares<8, 2>(p.rope, &threads, &rope_smem) : rope_shares<1, 2>(p.rope, &threads, &rope_smem);
      p.side[Query].heads = 0;
    }
    for (Side& s : p.side) {
      s.tasks = (s.heads + 256 / D * U - 1) / (256 / D * U);
      per_token += s.tasks;
    }
    p.by_token = Divisor((uint32_t)per_token);
    p.span = (int)std::min<int64_t>(kMaxWarps / per_token, p.tokens);
    const int64_t ctas = p.span ? (p.tokens + p.span - 1) / p.span : (p.tokens * per_token + kMaxWarps - 1) / kMaxWarps;
    if (ctas + queries > INT32_MAX) return fail(CTB_UNSUPPORTED, "ctb_kv_write: shape too large");
    p.ctas = (int)ctas;
    p.period = (int)((ctas + queries) / ctas);
    // a CTA has parts of at most two tokens where it cannot have a whole one
    const size_t smem = std::max(rope_smem, (size_t)(p.span ? p.span : 2) * 2 * p.pairs * sizeof(float));
    launch_kernel(kv_write_kernel<T, D, STORE, U>, (unsigned)(ctas + queries), kMaxWarps * 32, smem, st, 0, p, ctx->dev_status);
    CTB_CHECK_LAUNCH("ctb_kv_write launch");
    return CTB_OK;
  }
  static int run(ctb_ctx* ctx, cudaStream_t st, const WriteParams& p) {
    const int64_t heads = p.side[Query].heads + p.side[Key].heads + p.side[Value].heads;
    // four groups per warp (two where a token's keys have no more) where that still gives every SM 16 warps
    if (p.tokens * heads * D < 256ll * 4 * 16 * ctx->sm_count) return launch<1>(ctx, st, p);
    return p.side[Key].heads * D > 256 * 2 ? launch<4>(ctx, st, p) : launch<2>(ctx, st, p);
  }
};
template <typename T, int D, int STORE>
struct Read {
  static int run(ctb_ctx* ctx, cudaStream_t st, unsigned grid, const ReadParams& p) {
    launch_kernel(kv_read_kernel<T, D, STORE>, grid, kThreads, 0, st, 0, p, ctx->dev_status);
    CTB_CHECK_LAUNCH("ctb_kv_read launch");
    return CTB_OK;
  }
};

int check_types(const char* who, const ctb_kv_cache* cache, int dtype) {
  if (dtype != CTB_F16 && dtype != CTB_BF16) return fail(CTB_UNSUPPORTED, "%s: f16 and bf16 are implemented", who);
  if (cache->dtype != dtype && cache->dtype != CTB_E4M3 && cache->dtype != CTB_I8)
    return fail(CTB_BAD_ARG, "%s: a cache of 16-bit elements takes and gives elements of its own type", who);
  return CTB_OK;
}

}  // namespace

namespace ctb_internal {

int check_kv_cache(const char* who, const ctb_kv_cache* c) {
  if (!c) return fail(CTB_BAD_ARG, "%s: null cache", who);
  if (c->dtype != CTB_F16 && c->dtype != CTB_BF16 && c->dtype != CTB_E4M3 && c->dtype != CTB_I8)
    return fail(CTB_UNSUPPORTED, "%s: a cache has elements of f16, bf16, e4m3 or int8", who);
  const bool bytes = c->dtype == CTB_E4M3 || c->dtype == CTB_I8;
  if (c->head_dim != 64 && c->head_dim != 128) return fail(CTB_UNSUPPORTED, "%s: head dimensions 64 and 128 are implemented", who);
  if (!is_pow2(c->page_size) || c->page_size < 16 || c->page_size > 1024)
    return fail(CTB_UNSUPPORTED_TILE, "%s: page_size must be a power of two from 16 to 1024", who);
  if (c->pages <= 0 || c->kv_heads <= 0) return fail(CTB_BAD_ARG, "%s: non-positive dimension of the cache", who);
  if (c->pages > INT32_MAX / 2 || c->kv_heads > 65536) return fail(CTB_UNSUPPORTED, "%s: the cache is too large", who);
  if (!is_device_ptr(c->k) || !is_device_ptr(c->v) || (bytes && (!is_device_ptr(c->k_scale) || !is_device_ptr(c->v_scale))))
    return fail(CTB_BAD_ARG, "%s: an array of the cache is not a device pointer", who);
  if (!bytes && (c->k_scale || c->v_scale)) return fail(CTB_BAD_ARG, "%s: a cache of 16-bit elements has no scales", who);
  const int64_t rows = c->kv_heads * c->page_size, size = bytes ? 1 : 2;
  for (const int64_t s : {c->k_page_stride, c->v_page_stride})
    if (c->pages > 1 && (s < rows * c->head_dim || s > INT64_MAX / 8 / c->pages)) return fail(CTB_BAD_ARG, "%s: bad page stride", who);
  for (const int64_t s : {c->k_scale_page_stride, c->v_scale_page_stride})
    if (bytes && c->pages > 1 && (s < rows || s > INT64_MAX / 8 / c->pages)) return fail(CTB_BAD_ARG, "%s: bad page stride of the scales", who);
  if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16 || (c->pages > 1 && (c->k_page_stride * size % 16 || c->v_page_stride * size % 16)))
    return fail(CTB_BAD_ALIGN, "%s: pages of the cache must be 16-byte aligned", who);
  return CTB_OK;
}

}  // namespace ctb_internal

extern "C" int ctb_kv_write(ctb_ctx* ctx, void* stream, const ctb_kv_cache* cache, const void* slots, int slot_bits, void* q_out,
                            const void* q, const void* k, const void* v, const int64_t* strides, const void* positions, int position_bits,
                            const double* frequencies, int64_t tokens, int64_t heads, int64_t rotary, int interleaved, float scale, int dtype) {
  CTB_CHECK_CTX(ctx);
  CurrentDevice on(ctx);
  int r = check_kv_cache("ctb_kv_write", cache);
  if (r) return r;
  if ((r = check_types("ctb_kv_write", cache, dtype))) return r;
  if (!strides) return fail(CTB_BAD_ARG, "ctb_kv_write: no strides");
  if (tokens < 0 || heads < 0) return fail(CTB_BAD_ARG, "ctb_kv_write: negative dimension");
  if (slot_bits != 32 && slot_bits != 64) return fail(CTB_BAD_ARG, "ctb_kv_write: slots are 32- or 64-bit");
  if (frequencies) {
    if (rotary <= 0 || rotary % 2 || rotary > cache->head_dim)
      return fail(CTB_BAD_ARG, "ctb_kv_write: rotary must be even and between 2 and the head's dimension");
    if (position_bits != 32 && position_bits != 64) return fail(CTB_BAD_ARG, "ctb_kv_write: positions are 32- or 64-bit");
    if (!isfinite(scale)) return fail(CTB_BAD_ARG, "ctb_kv_write: scale is not finite");
  } else if (heads) {
    return fail(CTB_BAD_ARG, "ctb_kv_write: queries come with positions and frequencies");
  }
  if (tokens > INT32_MAX || heads + 2 * cache->kv_heads > 1 << 20) return fail(CTB_UNSUPPORTED, "ctb_kv_write: shape too large");
  if (tokens == 0) return CTB_OK;
  CTB_CHECK_DEV(slots); CTB_CHECK_DEV(k); CTB_CHECK_DEV(v);
  if (frequencies) { CTB_CHECK_DEV(positions); CTB_CHECK_DEV(frequencies); }
  int64_t s[8];  // none along what has one element
  for (int i = 0; i < 8; ++i) {
    s[i] = (i & 1 ? (i < 4 ? heads : cache->kv_heads) : tokens) == 1 ? 0 : strides[i];
    if ((heads || i >= 4) && (s[i] < 0 || s[i] > INT32_MAX)) return fail(CTB_UNSUPPORTED, "ctb_kv_write: strides too large");
  }
  if (heads) {
    CTB_CHECK_DEV(q); CTB_CHECK_DEV(q_out);
    const int64_t extents[3] = {1, tokens, heads}, out[3] = {0, s[0], s[1]}, in[3] = {0, s[2], s[3]};
    if ((r = check_turned_in_place("ctb_kv_write", q, in, q_out, out, extents, cache->head_dim, 2))) return r;
  }
  WriteParams p = {};
  p.side[Query] = Side{q, q_out, nullptr, 0, 0, (int)s[2], (int)s[3], (int)heads, 0};
  p.side[Key] = Side{k, cache->k, cache->k_scale, cache->k_page_stride, cache->k_scale_page_stride, (int)s[4], (int)s[5], (int)cache->kv_heads, 0};
  p.side[Value] = Side{v, cache->v, cache->v_scale, cache->v_page_stride, cache->v_scale_page_stride, (int)s[6], (int)s[7], (int)cache->kv_heads, 0};
  p.slots = slots; p.positions = positions; p.frequencies = frequencies;
  p.tokens = tokens;
  p.places = cache->pages * cache->page_size;
  p.qo_t = (int)s[0]; p.qo_h = (int)s[1];
  while ((1ll << p.page_log2) < cache->page_size) ++p.page_log2;
  p.pairs = frequencies ? (int)(rotary / 2) : 0;
  // runs of pairs that lie in the eight elements of a lane; where those would not all be full, single ones
  const int step_log2 = interleaved ? 2 : 3;
  p.table = AngleTable(p.pairs, p.pairs % (1 << step_log2) ? 0 : step_log2);
  p.wide_slots = slot_bits == 64; p.wide_positions = position_bits == 64; p.interleaved = interleaved != 0;
  p.scale = scale;
  p.vectors = (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && (!heads || ((uintptr_t)q % 16 == 0 && (uintptr_t)q_out % 16 == 0));
  for (int i = heads ? 0 : 4; i < 8; ++i) p.vectors &= s[i] % 8 == 0;
  if (heads) {
    p.rope.side[0] = RopeSide{q, q_out, 0, 0, p.side[Query].t_stride, p.side[Query].h_stride, p.qo_t, p.qo_h, (int)heads};
    p.rope.positions = positions; p.rope.frequencies = frequencies;
    p.rope.table.pairs = p.pairs;
    p.rope.by_seq = Divisor((uint32_t)tokens);
    p.rope.tokens = (int)tokens; p.rope.q_heads = (int)heads; p.rope.dim = (int)cache->head_dim;
    p.rope.wide = p.wide_positions; p.rope.interleaved = p.interleaved; p.rope.scale = scale;
    p.rope_vectors = p.vectors && rotary % 16 == 0;
  }
  return by_type<Write>(dtype, cache->head_dim, cache->dtype, ctx, static_cast<cudaStream_t>(stream), p);
}

extern "C" int ctb_kv_read(ctb_ctx* ctx, void* stream, void* K, void* V, const ctb_kv_cache* cache, const int32_t* page_table,
                           const int32_t* lengths, int64_t batch, int64_t seq, int64_t table_width, int64_t table_stride, int dtype) {
  CTB_CHECK_CTX(ctx);
  CurrentDevice on(ctx);
  int r = check_kv_cache("ctb_kv_read", cache);
  if (r) return r;
  if ((r = check_types("ctb_kv_read", cache, dtype))) return r;
  if (batch < 0 || seq < 0 || table_width < 0) return fail(CTB_BAD_ARG, "ctb_kv_read: negative dimension");
  const int64_t blocks = (seq + kReadTokens - 1) / kReadTokens;
  if (seq > 1 << 28 || table_width > 1 << 28 || (batch && blocks * cache->kv_heads > INT32_MAX / batch))
    return fail(CTB_UNSUPPORTED, "ctb_kv_read: shape too large");
  if (batch == 0 || seq == 0) return CTB_OK;
  CTB_CHECK_DEV(K); CTB_CHECK_DEV(V); CTB_CHECK_DEV(lengths);
  if (table_width) CTB_CHECK_DEV(page_table);
  if (table_stride < table_width && batch > 1) return fail(CTB_BAD_ARG, "ctb_kv_read: rows of the page table overlap");
  if ((uintptr_t)K % 16 || (uintptr_t)V % 16) return fail(CTB_BAD_ALIGN, "ctb_kv_read: K and V must be 16-byte aligned");
  ReadParams p = {};
  p.cache = cache_of(cache);
  p.K = K; p.V = V; p.table = page_table; p.lengths = lengths; p.table_ld = table_stride;
  p.batch = (int)batch; p.seq = (int)seq; p.width = (int)table_width; p.blocks = (int)blocks;
  return by_type<Read>(dtype, cache->head_dim, cache->dtype, ctx, static_cast<cudaStream_t>(stream), (unsigned)(blocks * batch * cache->kv_heads), p);
}
