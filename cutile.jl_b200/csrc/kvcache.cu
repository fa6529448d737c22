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

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxTokens = 16;  // of a CTA that writes
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
  int64_t qo_t, qo_h, q_t, q_h, k_t, k_h, v_t, v_h, tokens;
  AngleTable table;
  int q_heads, rows, pairs, per_cta, wide_slots, wide_positions, interleaved, vectors;  // q_heads: 0 without queries; pairs: 0 without angles
  float scale;
};

template <typename T, int D, int STORE>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const WriteParams p, int* status) {
  constexpr int L = D / 8, kRows = 32 / L;  // lanes of a row, rows of a warp
  __shared__ float2 angles[kMaxTokens * (D / 2 + 8)];
  __shared__ long long places[kMaxTokens];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, chunk = lane & (L - 1), e0 = chunk * 8;
  const int64_t t0 = (int64_t)blockIdx.x * p.per_cta;
  const int tokens = (int)min((int64_t)p.per_cta, p.tokens - t0);
  grid_dependency_sync();
  if (p.pairs)
    p.table.fill(angles, p.positions, p.wide_positions, t0, tokens, p.frequencies, p.scale, false, threadIdx.x, kThreads);
  if (threadIdx.x < tokens) {
    const long long slot = index_at(p.slots, p.wide_slots, t0 + threadIdx.x);
    const bool bad = slot < 0 || slot > p.cache.tokens;
    if (bad) atomicMax(status, (int)DEV_BAD_INDEX);
    places[threadIdx.x] = bad ? -1 : slot - 1;
  }
  __syncthreads();
  const int all = tokens * p.rows;
  for (int i0 = warp * kRows; i0 < all; i0 += kWarps * kRows) {
    const int i = i0 + lane / L;
    const bool live = i < all;
    const int t = live ? i / p.rows : 0, r = live ? i - t * p.rows : 0;
    const bool query = r < p.q_heads, value = r >= p.q_heads + p.cache.kv_heads;
    const int head = query ? r : value ? r - p.q_heads - p.cache.kv_heads : r - p.q_heads;
    const long long place = places[t];
    const bool wanted = live && (query || place >= 0);
    const T* src = query ? static_cast<const T*>(p.q) + (t0 + t) * p.q_t + head * p.q_h
                         : value ? static_cast<const T*>(p.v) + (t0 + t) * p.v_t + head * p.v_h
                                 : static_cast<const T*>(p.k) + (t0 + t) * p.k_t + head * p.k_h;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (wanted) {
      if (p.vectors) w = __ldcs(reinterpret_cast<const uint4*>(src + e0));
      else {
        alignas(16) T x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = src[e0 + j];
        w = *reinterpret_cast<const uint4*>(x);
      }
    }
    float x[8];
    unpack_row<T>(w, x);
    const bool turned = !value && e0 < 2 * p.pairs;
    const float2* a = angles + t * p.table.size();
    if (p.pairs && p.interleaved) {
      if (turned) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (e0 + 2 * j < 2 * p.pairs) {
            const float2 cs = a[p.table.at(chunk, j)];
            const float y = x[2 * j] * cs.x - x[2 * j + 1] * cs.y;
            x[2 * j + 1] = x[2 * j] * cs.y + x[2 * j + 1] * cs.x;
            x[2 * j] = y;
          }
      }
    } else if (p.pairs && p.pairs % 8 == 0) {  // the pair's other elements are another lane's eight
      const int half = p.pairs / 8;
      const bool second = chunk >= half;
      const int other = turned ? (second ? lane - half : lane + half) : lane;
      const uint4 o = make_uint4(__shfl_sync(0xffffffffu, w.x, other), __shfl_sync(0xffffffffu, w.y, other),
                                 __shfl_sync(0xffffffffu, w.z, other), __shfl_sync(0xffffffffu, w.w, other));
      if (turned) {
        float y[8];
        unpack_row<T>(o, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 cs = a[p.table.at(second ? chunk - half : chunk, j)];
          x[j] = x[j] * cs.x + (second ? y[j] * cs.y : -y[j] * cs.y);
        }
      }
    } else if (p.pairs) {
      if (turned && wanted) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int e = e0 + j;
          if (e >= 2 * p.pairs) continue;
          const bool second = e >= p.pairs;
          const int pair = second ? e - p.pairs : e;
          const float2 cs = a[p.table.at(pair / p.table.step, pair % p.table.step)];
          const float y = to_float(src[second ? pair : e + p.pairs]);
          x[j] = x[j] * cs.x + (second ? y * cs.y : -y * cs.y);
        }
      }
      __syncwarp();  // queries in place: what other lanes read here is written below
    }
    if (turned) w = pack_row<T>(x);
    if (query) {
      if (live) {
        T* to = static_cast<T*>(p.q_out) + (t0 + t) * p.qo_t + head * p.qo_h + e0;
        if (p.vectors) *reinterpret_cast<uint4*>(to) = w;
        else {
#pragma unroll
          for (int j = 0; j < 8; ++j) to[j] = reinterpret_cast<const T*>(&w)[j];
        }
      }
    }
    const int64_t page = place >> p.cache.page_log2;
    const int64_t row = ((int64_t)head << p.cache.page_log2) + (place & ((1 << p.cache.page_log2) - 1));
    if constexpr (STORE == Same) {
      if (wanted && !query) {
        T* to = static_cast<T*>(value ? p.cache.v : p.cache.k) + page * (value ? p.cache.v_page : p.cache.k_page) + row * D + e0;
        *reinterpret_cast<uint4*>(to) = w;
      }
    } else {
      constexpr float kMost = STORE == I8 ? 127.f : 448.f;
      uint32_t top = 0;  // magnitudes as whole numbers: NaN is above infinity
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (wanted && !query) {
        const float peak = __uint_as_float(top);
        const bool fine = peak >= kSmallest && peak < INFINITY;
        // x c / a with one Newton step behind the product with 1 / a: a quotient that is a number of f32 comes out as it is, so ties are ties
        const float pre = peak > 1.2676506e30f ? 5.9604645e-8f : 1.f;  // beyond 2^100 in units of 2^24: x c is finite
        const float a = peak * pre, inv = fine ? __frcp_rn(a) : 0.f;
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float n = x[j] * pre * kMost, z = n * inv;
          y[j] = fine ? fmaf(fmaf(-z, a, n), inv, z) : 0.f;
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
        out = pack_row<T>(x);
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
  static int run(ctb_ctx* ctx, cudaStream_t st, unsigned grid, const WriteParams& p) {
    launch_kernel(kv_write_kernel<T, D, STORE>, grid, kThreads, 0, st, 0, p, ctx->dev_status);
    CTB_CHECK_LAUNCH("ctb_kv_write launch");
    return CTB_OK;
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
  p.qo_t = strides[0]; p.qo_h = strides[1]; p.q_t = strides[2]; p.q_h = strides[3];
  p.k_t = strides[4]; p.k_h = strides[5]; p.v_t = strides[6]; p.v_h = strides[7];
  p.tokens = tokens;
  p.q_heads = (int)heads;
  p.rows = (int)(heads + 2 * cache->kv_heads);
  p.pairs = frequencies ? (int)(rotary / 2) : 0;
  const int step = interleaved ? 4 : 8;
  p.table = AngleTable{p.pairs, step, (p.pairs + step - 1) / step};
  p.wide_slots = slot_bits == 64; p.wide_positions = position_bits == 64; p.interleaved = interleaved != 0;
  p.scale = scale;
  p.vectors = (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && (!heads || ((uintptr_t)q % 16 == 0 && (uintptr_t)q_out % 16 == 0));
  for (int i = heads ? 0 : 4; i < 8; ++i) p.vectors &= strides[i] % 8 == 0;
  p.per_cta = (int)std::max<int64_t>(1, std::min<int64_t>(kMaxTokens, tokens / (ctx->sm_count * 8)));
  return by_type<Write>(dtype, cache->head_dim, cache->dtype, ctx, static_cast<cudaStream_t>(stream), (unsigned)((tokens + p.per_cta - 1) / p.per_cta),
                        p);
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
