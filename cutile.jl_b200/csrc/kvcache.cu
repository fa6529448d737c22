// The paged key-value cache: writing new tokens to it (turned by their positions and rounded to 8 bits on the way) and reading sequences back.
//
// What bounds both is HBM.  A row (one head of one token) is the work of D / 8 neighbouring lanes, eight elements each, so that its
// largest magnitude is found by a few shuffles and its pairs (i, i + rotary / 2) meet by one.
#include <math.h>

#include <algorithm>

#include "ctx.h"
#include "ptx.cuh"
#include "rotate.cuh"

using namespace ctb;
using namespace ctb_internal;

namespace {

constexpr int kThreads = 256;
constexpr float kSmallest = 7.888609052210118e-31f;  // 2^-100: rows below it are zeros in 8 bits

enum Store { Same = 0, E4M3 = 1, I8 = 2 };

struct Cache {
  void *k, *v;
  float *ks, *vs;
  int64_t k_page, v_page, ks_page, vs_page, tokens;  // tokens: pages * page_size
  int kv_heads, page_log2, pages;
};
Cache cache_of(const ctb_kv_cache* c) {
  Cache d = {c->k, c->v, c->k_scale, c->v_scale, c->k_page_stride, c->v_page_stride, c->k_scale_page_stride, c->v_scale_page_stride,
             c->pages * c->page_size, (int)c->kv_heads, 0, (int)c->pages};
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

struct WriteParams {
  Cache cache;
  const void *slots, *q, *k, *v, *positions;
  void* q_out;
  const double* frequencies;
  int qo_t, qo_h, q_t, q_h, k_t, k_h, v_t, v_h;
  int64_t rows_all;
  AngleTable table;
  Divisor by_token;  // rows of a token: of queries, keys, values
  int q_heads, pairs, wide_slots, wide_positions, interleaved, vectors;  // q_heads: 0 without queries; pairs: 0 without angles
  float scale;
};

// A warp has U groups of 32 / (D / 8) neighbouring rows: it asks for them, takes its share of the CTA's angles and slots while they come, and
// stores them behind the barrier.
template <typename T, int D, int STORE, int U>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const WriteParams p, int* status) {
  constexpr int L = D / 8, kRows = kThreads / L;  // lanes of a row, rows at a time
  constexpr int kMaxTokens = kRows * U / 2 + 1;   // a token has two rows at least
  __shared__ __align__(16) float angles[kMaxTokens * D];
  __shared__ long long places[kMaxTokens];
  const int lane = threadIdx.x & 31, chunk = lane & (L - 1), e0 = chunk * 8;
  const int64_t row0 = (int64_t)blockIdx.x * (kRows * U), t0 = row0 / p.by_token.d;
  const uint32_t local0 = (uint32_t)(row0 - t0 * p.by_token.d), n = (uint32_t)min((int64_t)(kRows * U), p.rows_all - row0);
  const int kv_heads = p.cache.kv_heads;
  grid_dependency_sync();
  uint4 asked[U];
  int token_of[U], row_of[U];  // -1: none
  auto rows_of = [&](int k, const void*& base, int& head, int& t_stride, int& h_stride) {  // the array that row k is in
    const int r = row_of[k];
    const bool key = r < p.q_heads + kv_heads;
    head = r - (key ? p.q_heads : p.q_heads + kv_heads);
    base = key ? p.k : p.v;
    t_stride = key ? p.k_t : p.v_t;
    h_stride = key ? p.k_h : p.v_h;
    if (r < p.q_heads) {
      head = r;
      base = p.q;
      t_stride = p.q_t;
      h_stride = p.q_h;
    }
  };
  auto source = [&](int k) {
    const void* base;
    int head, t_stride, h_stride;
    rows_of(k, base, head, t_stride, h_stride);
    return static_cast<const T*>(base) + (t0 * t_stride + (int64_t)token_of[k] * t_stride + (int64_t)head * h_stride);
  };
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const uint32_t i = k * kRows + threadIdx.x / L;
    asked[k] = make_uint4(0, 0, 0, 0);
    token_of[k] = 0;
    row_of[k] = -1;
    if (i >= n) continue;
    token_of[k] = p.by_token(local0 + i);
    row_of[k] = (int)(local0 + i) - token_of[k] * (int)p.by_token.d;
    const T* src = source(k);
    if (p.vectors) asked[k] = __ldcs(reinterpret_cast<const uint4*>(src + e0));
    else {
      alignas(16) T x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = src[e0 + j];
      asked[k] = *reinterpret_cast<const uint4*>(x);
    }
  }
  const int tokens = (int)p.by_token(local0 + n - 1) + 1;
  if (p.pairs) p.table.fill(angles, p.positions, p.wide_positions, t0, tokens, p.frequencies, p.scale, false, threadIdx.x, kThreads);
  for (int t = threadIdx.x; t < tokens; t += kThreads) {
    const long long slot = index_at(p.slots, p.wide_slots, t0 + t);
    const bool bad = slot < 0 || slot > p.cache.tokens;
    if (bad) atomicMax(status, (int)DEV_BAD_INDEX);
    places[t] = bad ? -1 : slot - 1;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int t = token_of[k], r = row_of[k];
    const bool live = r >= 0, query = r < p.q_heads, value = r >= p.q_heads + kv_heads;
    const int head = query ? r : value ? r - p.q_heads - kv_heads : r - p.q_heads;
    const long long place = places[t];
    const bool stored = live && !query && place >= 0;
    uint32_t w[4] = {asked[k].x, asked[k].y, asked[k].z, asked[k].w};
    Pair x[4];  // the elements in f32, for 8 bits
    const bool turned = live && !value && e0 < 2 * p.pairs;
    const float* table = angles + t * 2 * p.pairs;
    if (p.pairs) {
      if (p.interleaved || p.pairs % 8 == 0) {
        // with pairs (i, i + pairs), a pair's other elements are another lane's eight
        const int half = p.pairs / 8;
        const bool second = chunk >= half;
        uint32_t o[4];
        if (!p.interleaved) {
          const int other = turned ? (second ? lane - half : lane + half) : lane;
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = __shfl_sync(0xffffffffu, w[i], other) ^ (second ? 0u : 0x80008000u);
        }
        if (turned) {
          if (!p.interleaved) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const TwoAngles a = angles_of(table, p.table.runs, second ? chunk - half : chunk, i);
              x[i] = fma2(vec_pair<T>(o, i), a.sin, mul2(vec_pair<T>(w, i), a.cos));
            }
          } else if (p.table.step == 4) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const TwoAngles a = angles_of(table, p.table.runs, chunk, i);
              Pair u, v;
              split_pairs<T>(w, i, u, v);
              const float2 f = halves(fma2(v, minus(a.sin), mul2(u, a.cos))), g = halves(fma2(v, a.cos, mul2(u, a.sin)));
              x[2 * i] = pair(f.x, g.x);
              x[2 * i + 1] = pair(f.y, g.y);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              x[i] = vec_pair<T>(w, i);
              if (e0 + 2 * i < 2 * p.pairs) {
                const float2 f = halves(x[i]);
                const float c = table[e0 + 2 * i], d = table[e0 + 2 * i + 1];
                x[i] = pair(f.x * c - f.y * d, f.x * d + f.y * c);
              }
            }
          }
        }
      } else {
        if (turned) {
          const T* src = source(k);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float f[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int e = e0 + 2 * i + j;
              const bool second = e >= p.pairs;
              const int at = second ? e - p.pairs : e;
              f[j] = to_float(reinterpret_cast<const T*>(&asked[k])[2 * i + j]);
              if (e >= 2 * p.pairs) continue;
              const float y = to_float(src[second ? at : e + p.pairs]);
              f[j] = f[j] * table[2 * at] + (second ? y : -y) * table[2 * at + 1];
            }
            x[i] = pair(f[0], f[1]);
          }
        }
        __syncwarp();  // queries in place: what other lanes read here is written below
      }
      if (turned) {
#pragma unroll
        for (int i = 0; i < 4; ++i) put_pair<T>(w, i, x[i]);
      }
    }
    const uint4 words = make_uint4(w[0], w[1], w[2], w[3]);
    if (live && query) {
      T* to = static_cast<T*>(p.q_out) + (t0 * p.qo_t + (int64_t)t * p.qo_t + (int64_t)head * p.qo_h) + e0;
      if (p.vectors) *reinterpret_cast<uint4*>(to) = words;
      else {
#pragma unroll
        for (int j = 0; j < 8; ++j) to[j] = reinterpret_cast<const T*>(&words)[j];
      }
    }
    if (!__any_sync(0xffffffffu, stored)) continue;
    const int64_t page = place >> p.cache.page_log2;
    const int64_t row = (head << p.cache.page_log2) + (int)(place & ((1 << p.cache.page_log2) - 1));
    if constexpr (STORE == Same) {
      if (stored) {
        T* to = static_cast<T*>(value ? p.cache.v : p.cache.k) + page * (value ? p.cache.v_page : p.cache.k_page) + row * D + e0;
        *reinterpret_cast<uint4*>(to) = words;
      }
    } else {
      constexpr float kMost = STORE == I8 ? 127.f : 448.f;
      if (!turned) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = vec_pair<T>(w, i);
      }
      float peak = 0.f;  // NaN where there is one
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = halves(x[i]);
        asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(peak) : "f"(peak), "f"(f.x), "f"(f.y));
      }
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) asm("max.NaN.f32 %0, %1, %2;" : "=f"(peak) : "f"(peak), "f"(__shfl_xor_sync(0xffffffffu, peak, o)));
      if (stored) {
        const bool fine = peak >= kSmallest && peak < INFINITY;
        // x c / a with one Newton step behind the product with 1 / a: a quotient that is a number of f32 comes out as it is, so ties are ties
        const float pre = peak > 1.2676506e30f ? 5.9604645e-8f : 1.f;  // beyond 2^100 in units of 2^24: x c is finite
        const float a = peak * pre, inv = fine ? __frcp_rn(a) : 0.f, most = pre * kMost;
        const Pair inv2 = pair(inv, inv), a2 = pair(-a, -a), most2 = pair(most, most);
        float y[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const Pair m = mul2(x[i], most2), z = mul2(m, inv2);
          const float2 f = halves(fma2(fma2(z, a2, m), inv2, z));
          y[2 * i] = fine ? f.x : 0.f;
          y[2 * i + 1] = fine ? f.y : 0.f;
        }
        uint2 codes;
        if constexpr (STORE == I8) codes = make_uint2(i8x4(y[0], y[1], y[2], y[3]), i8x4(y[4], y[5], y[6], y[7]));
        else codes = make_uint2(e4m3x4(y[0], y[1], y[2], y[3]), e4m3x4(y[4], y[5], y[6], y[7]));
        uint8_t* to = static_cast<uint8_t*>(value ? p.cache.v : p.cache.k) + page * (value ? p.cache.v_page : p.cache.k_page) + row * D + e0;
        *reinterpret_cast<uint2*>(to) = codes;
        if (chunk == 0)
          (value ? p.cache.vs : p.cache.ks)[page * (value ? p.cache.vs_page : p.cache.ks_page) + row] = peak < kSmallest ? 0.f : __fdiv_rn(peak, kMost);
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
  static int launch(ctb_ctx* ctx, cudaStream_t st, const WriteParams& p) {
    constexpr int kRows = kThreads / (D / 8) * U;
    const int64_t grid = (p.rows_all + kRows - 1) / kRows;
    if (grid > INT32_MAX) return fail(CTB_UNSUPPORTED, "ctb_kv_write: shape too large");
    launch_kernel(kv_write_kernel<T, D, STORE, U>, (unsigned)grid, kThreads, 0, st, 0, p, ctx->dev_status);
    CTB_CHECK_LAUNCH("ctb_kv_write launch");
    return CTB_OK;
  }
  static int run(ctb_ctx* ctx, cudaStream_t st, const WriteParams& p) {
    const int64_t ctas = p.rows_all / (kThreads / (D / 8));
    return ctas >= 4ll * ctx->sm_count ? launch<4>(ctx, st, p) : launch<1>(ctx, st, p);  // four groups per warp still give every SM a CTA
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
  if (heads) {
    CTB_CHECK_DEV(q); CTB_CHECK_DEV(q_out);
    const int64_t extents[3] = {1, tokens, heads}, out[3] = {0, strides[0], strides[1]}, in[3] = {0, strides[2], strides[3]};
    if ((r = check_turned_in_place("ctb_kv_write", q, in, q_out, out, extents, cache->head_dim, 2))) return r;
  }
  WriteParams p = {};
  p.cache = cache_of(cache);
  p.slots = slots; p.q = q; p.k = k; p.v = v; p.positions = positions; p.q_out = q_out; p.frequencies = frequencies;
  for (int i = 0; i < 8; ++i)
    if (strides[i] < 0 || strides[i] > INT32_MAX) return fail(CTB_UNSUPPORTED, "ctb_kv_write: strides too large");
  p.qo_t = (int)strides[0]; p.qo_h = (int)strides[1]; p.q_t = (int)strides[2]; p.q_h = (int)strides[3];
  p.k_t = (int)strides[4]; p.k_h = (int)strides[5]; p.v_t = (int)strides[6]; p.v_h = (int)strides[7];
  const int64_t rows = heads + 2 * cache->kv_heads;
  p.q_heads = (int)heads;
  p.by_token = Divisor((uint32_t)rows);
  p.rows_all = tokens * rows;
  p.pairs = frequencies ? (int)(rotary / 2) : 0;
  // runs of pairs that lie in the eight elements of a lane; where those would not all be full, single ones
  const int step = interleaved ? 4 : 8;
  p.table = p.pairs % step ? AngleTable{p.pairs, 1, p.pairs} : AngleTable{p.pairs, step, p.pairs / step};
  p.wide_slots = slot_bits == 64; p.wide_positions = position_bits == 64; p.interleaved = interleaved != 0;
  p.scale = scale;
  p.vectors = (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && (!heads || ((uintptr_t)q % 16 == 0 && (uintptr_t)q_out % 16 == 0));
  for (int i = heads ? 0 : 4; i < 8; ++i) p.vectors &= strides[i] % 8 == 0;
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
