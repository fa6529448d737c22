// Attention of one new token per sequence over a paged key-value cache: o = sum_j p_j v_j / sum_j p_j, p_j = exp(c q.k_j), for every
// query head, with the heads of a group as rows of one operand.
//
// What bounds it is HBM: every stored key and value is read once, 2 D bytes times the element's size, against 4 D operations per row.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "ctx.h"
#include "ptx.cuh"

using namespace ctb;
using namespace ctb_internal;

namespace {

enum Store { F16 = 0, BF16 = 1, E4M3 = 2, I8 = 3 };

constexpr int kMaxBatch = 4096;  // sequences of a launch (their prefix sums lie in shared memory)
constexpr int kMinTiles = 2;     // of a warp, where there is that much work
// Exponents' reference (in powers of two): it moves once a score stands kLazy above the largest that it knows.  What goes to f16 is lifted
// by kLift, so that the largest is at most 2^(kLazy + kLift + 1) and what f16 pairs cannot tell from 0 is 2^-(25 + kLift) of it.
constexpr int kLazy = 6, kLift = 8;

struct Params {
  const void *Q, *K, *V;
  const float *Ks, *Vs;
  void* Out;
  float* lse;
  const int32_t *table, *lengths;
  int64_t q_seq, q_head, k_page, v_page, ks_page, vs_page, table_ld;
  int batch, heads, kv_heads, group, row_tiles, width, page_log2, pages;
  int q_bf16;
  float scale_log2;
  float* part;        // [CTA][first, last item of its range][rows x D, maxima, sums]
  unsigned* tickets;  // per CTA: parts left of the item that begins in its range and ends in another's
};

template <int STORE, int D_, int NT_>
struct Shape {
  static constexpr int D = D_, NT = NT_;
  static constexpr bool kBytes = STORE >= E4M3;
  static constexpr int kRow = D * (kBytes ? 1 : 2);  // bytes of a key's row
  static constexpr int KC = kRow / 64;               // 16-byte chunks that a lane has of a key's row
  static constexpr int KT = 256 / kRow;              // groups of 16 keys in a tile: K and V of a tile are 4 KB each
  static constexpr int VW = kRow / 32;               // 32-bit words that a lane has of a value's row
  static constexpr int MT = D / 16;                  // instructions along the dimensions of O
  static constexpr int QW = D / 8;                   // words that a lane has of a query row
  static constexpr int R = 8 * NT;
  static constexpr int kWarps = NT == 1 ? 12 : 8, kThreads = kWarps * 32;
  static constexpr int kPitch = D + 4;               // floats between rows of partial results in shared memory
  static constexpr int kSlotFloats = R * kPitch + 2 * R;
  static constexpr int kPartFloats = R * D + 2 * R;
  static constexpr size_t kSmem = sizeof(float) * 2 * kWarps * kSlotFloats + sizeof(unsigned) * (kMaxBatch + 1);
};

__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 load8(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
template <bool BF>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {  // of an 8 x 8 matrix of 16-bit elements
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <bool BF>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// Two codes (the bytes of a 16-bit half of w) as f16: both types are exact in it.
template <int STORE>
__device__ __forceinline__ void codes4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (STORE == E4M3) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {  // 0x6400 + u is the f16 1024 + u; u = code + 128
    w ^= 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1152
    const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off), y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}
__device__ __forceinline__ float max_over_keys(float v) {  // over the lanes that hold the same rows
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float sum_over_keys(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}
__device__ __forceinline__ float from_minus_inf(float m) { return m == -INFINITY ? 0.f : m; }

// Range of a worker among `workers` that share out `n` tiles, and the worker that has tile x.
__device__ __forceinline__ unsigned first_tile(unsigned w, unsigned n, unsigned workers) {
  return (unsigned)((unsigned long long)w * n / workers);
}
__device__ __forceinline__ unsigned worker_of(unsigned x, unsigned n, unsigned workers) {
  return (unsigned)((((unsigned long long)x + 1) * workers - 1) / n);
}

// A tile: the sequence, the row of heads, and the keys.
struct Cursor {
  int b, head, rt, key, len;  // head: of the keys and values
};

template <int STORE, int D, int NT>
__global__ void __launch_bounds__(Shape<STORE, D, NT>::kThreads, 1) fmha_paged_kernel(const Params p, int* status) {
  using S = Shape<STORE, D, NT>;
  constexpr int KC = S::KC, KT = S::KT, VW = S::VW, MT = S::MT, QW = S::QW, R = S::R, kWarps = S::kWarps, kThreads = S::kThreads;
  constexpr int kTileKeys = 16 * KT;
  constexpr bool BF = STORE == BF16;
  constexpr float kAbove = STORE == F16 ? kLift : 0;  // what the known largest score stands above m
  extern __shared__ __align__(16) float smem[];
  float* slots = smem;  // [warp][first, last item of its range][R rows, maxima, sums]
  unsigned* prefix = reinterpret_cast<unsigned*>(smem + 2 * kWarps * S::kSlotFloats);
  __shared__ unsigned warp_sum[kWarps], seg_lo[2 * kWarps], seg_hi[2 * kWarps];
  __shared__ int seg_item[2 * kWarps];
  __shared__ int last_s[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  grid_dependency_sync();

  // ---- tiles before every sequence
  const int most = p.width << p.page_log2;
  const unsigned per_tile = (unsigned)p.kv_heads * p.row_tiles;
  {
    const int per = (p.batch + kThreads - 1) / kThreads, b0 = tid * per, b1 = min(p.batch, b0 + per);
    auto tiles = [&](int b) {
      const int n = min(max(__ldg(p.lengths + b), 0), most);
      return (unsigned)((n + kTileKeys - 1) / kTileKeys) * per_tile;
    };
    unsigned sum = 0;
    for (int b = b0; b < b1; ++b) sum += tiles(b);
    unsigned up = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned v = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += v;
    }
    if (lane == 31) warp_sum[warp] = up;
    if (tid < 2 * kWarps) seg_item[tid] = -1;
    __syncthreads();
    unsigned before = up - sum;
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
    for (int b = b0; b < b1; ++b) {
      prefix[b] = before;
      before += tiles(b);
    }
    if (tid == kThreads - 1) prefix[p.batch] = before;
    __syncthreads();
  }
  const unsigned total = prefix[p.batch];
  // sequences without keys
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    const int n = __ldg(p.lengths + b);
    if (min(n, most) > 0) continue;
    if (n != 0 && tid == 0) atomicMax(status, (int)DEV_BAD_INDEX);
    uint32_t* out = static_cast<uint32_t*>(p.Out) + (int64_t)b * p.heads * (D / 2);
    for (int i = tid; i < p.heads * (D / 2); i += kThreads) out[i] = n != 0 ? 0x7fff7fffu : 0u;
    if (p.lse)
      for (int i = tid; i < p.heads; i += kThreads) p.lse[(int64_t)b * p.heads + i] = n != 0 ? NAN : -INFINITY;
  }
  if (total == 0) return;
  const unsigned all = gridDim.x * kWarps, workers = min(all, (total + kMinTiles - 1) / kMinTiles);
  const unsigned me = blockIdx.x * kWarps + warp;
  auto range_of = [&](unsigned w) { return first_tile(min(w, workers), total, workers); };
  const unsigned lo = range_of(me), hi = range_of(me + 1);

  auto write_row = [&](int b, int head, int row, int d, const float (&v)[8]) {  // eight dimensions of a head of the group
    uint16_t* out = static_cast<uint16_t*>(p.Out) + ((int64_t)b * p.heads + (int64_t)head * p.group + row) * D + d;
    uint4 w;
    if (p.q_bf16) w = make_uint4(pack2<true>(v[0], v[1]), pack2<true>(v[2], v[3]), pack2<true>(v[4], v[5]), pack2<true>(v[6], v[7]));
    else w = make_uint4(pack2<false>(v[0], v[1]), pack2<false>(v[2], v[3]), pack2<false>(v[4], v[5]), pack2<false>(v[6], v[7]));
    *reinterpret_cast<uint4*>(out) = w;
  };
  auto write_lse = [&](int b, int head, int row, float m, float l) {
    if (p.lse) p.lse[(int64_t)b * p.heads + (int64_t)head * p.group + row] = (m + log2f(l)) * 0.6931471805599453f;
  };

  if (lo < hi) {
    const int page_keys = 1 << p.page_log2;
    bool seen_bad = false;
    auto length_of = [&](int b) { return min(__ldg(p.lengths + b), most); };
    auto next = [&](Cursor& t) {
      t.key += kTileKeys;
      if (t.key < t.len) return;
      t.key = 0;
      if (++t.rt < p.row_tiles) return;
      t.rt = 0;
      if (++t.head < p.kv_heads) return;
      t.head = 0;
      do ++t.b;
      while (t.b < p.batch && (t.len = length_of(t.b)) <= 0);
    };
    auto page_ids = [&](const Cursor& t, int (&id)[KT]) {
#pragma unroll
      for (int s = 0; s < KT; ++s) {
        const int key = t.key + 16 * s;
        id[s] = key < t.len ? __ldg(p.table + (int64_t)t.b * p.table_ld + (key >> p.page_log2)) : 0;
      }
    };
    // the page that is read for an id: the first one where there is none
    auto page = [&](int id) { return (unsigned)(id - 1) < (unsigned)p.pages ? id - 1 : 0; };
    auto load_k = [&](const Cursor& t, const int (&id)[KT], uint4 (&k)[KT][2][KC], float (&ks)[KT][2]) {
#pragma unroll
      for (int s = 0; s < KT; ++s) {
        const int key = t.key + 16 * s;
        if (KT > 1 && key >= t.len) continue;
        const int64_t row = ((int64_t)t.head << p.page_log2) + (key & (page_keys - 1)) + g;
        const char* src = static_cast<const char*>(p.K) + (page(id[s]) * p.k_page + row * D) * (S::kBytes ? 1 : 2) + c * 16;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < KC; ++i) k[s][h][i] = load16(src + h * 8 * S::kRow + i * 64);
        if constexpr (S::kBytes) {
          const float* sc = p.Ks + page(id[s]) * p.ks_page + row;
          ks[s][0] = __ldg(sc);
          ks[s][1] = __ldg(sc + 8);
        }
      }
    };
    // keys 2c, 2c + 1, 2c + 8, 2c + 9 of each sixteen; a word has the dimensions that stand in it
    auto load_v = [&](const Cursor& t, const int (&id)[KT], uint32_t (&v)[KT][4][VW], float (&vs)[KT][2]) {
#pragma unroll
      for (int s = 0; s < KT; ++s) {
        const int key = t.key + 16 * s;
        const int64_t row = ((int64_t)t.head << p.page_log2) + (key & (page_keys - 1));
        const char* src = static_cast<const char*>(p.V) + (page(id[s]) * p.v_page + row * D) * (S::kBytes ? 1 : 2);
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const int j = 2 * c + (h & 1) + 8 * (h >> 1);
          const bool live = key + j < t.len;  // rows behind the last key may hold anything: 0 x NaN is NaN
          const char* at = src + j * S::kRow;
          if constexpr (S::kRow == 64) {
            const uint2 w = live ? load8(at + g * 8) : make_uint2(0, 0);
            v[s][h][0] = w.x;
            v[s][h][1] = w.y;
          } else {
#pragma unroll
            for (int l = 0; l < S::kRow / 128; ++l) {
              const uint4 w = live ? load16(at + g * 16 + l * 128) : make_uint4(0, 0, 0, 0);
              v[s][h][4 * l] = w.x;
              v[s][h][4 * l + 1] = w.y;
              v[s][h][4 * l + 2] = w.z;
              v[s][h][4 * l + 3] = w.w;
            }
          }
        }
        if constexpr (S::kBytes) {
          const float* sc = p.Vs + page(id[s]) * p.vs_page + row + g;
          vs[s][0] = key + g < t.len ? __ldg(sc) : 0.f;
          vs[s][1] = key + g + 8 < t.len ? __ldg(sc + 8) : 0.f;
        }
      }
    };
    // first dimension of instruction j's pair in this lane
    auto dim_of = [&](int j) {
      if constexpr (S::kRow == 256) return (j >> 2) * 64 + g * 8 + 2 * (j & 3);
      else return g * (D / 8) + 2 * j;
    };

    Cursor now;  // the tile at hand
    {
      int a = 0, z = p.batch - 1;  // the sequence that has tile lo: the last one that begins at or before it and has keys
      while (a < z) {
        const int mid = (a + z + 1) >> 1;
        if (prefix[mid] <= lo) a = mid;
        else z = mid - 1;
      }
      now.b = a;
      now.len = length_of(a);
      const unsigned tiles = (unsigned)(now.len + kTileKeys - 1) / kTileKeys, at = lo - prefix[a], item = at / tiles;
      now.head = item / p.row_tiles;
      now.rt = item - now.head * p.row_tiles;
      now.key = (int)(at - item * tiles) * kTileKeys;
    }
    Cursor ahead = now;  // the tile whose keys are asked for
    int id[KT], id1[KT];
    uint4 k[KT][2][KC];
    float ks[KT][2] = {};
    page_ids(ahead, id1);
    load_k(ahead, id1, k, ks);
    next(ahead);
    int id2[KT] = {};
    if (lo + 1 < hi) page_ids(ahead, id2);

    for (unsigned x = lo; x < hi;) {
      // ---- an item or the part of it that is this warp's
      const int b = now.b, head = now.head, rt = now.rt, len = now.len;
      const unsigned tiles = (unsigned)(len + kTileKeys - 1) / kTileKeys;
      const unsigned item_lo = x - (unsigned)now.key / kTileKeys, item_hi = item_lo + tiles, end = min(hi, item_hi);
      bool bad = __ldg(p.lengths + b) > most;
      const int rows = p.group - rt * R;  // live rows, at least one
      uint32_t q[NT][QW];
      float mult[NT][2];  // score in powers of two of the rows 2c, 2c + 1
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int row = n * 8 + g;
        const bool live = row < rows;
        const uint16_t* src = static_cast<const uint16_t*>(p.Q) + (int64_t)b * p.q_seq + ((int64_t)head * p.group + rt * R + (live ? row : 0)) * p.q_head;
        constexpr int kDims = S::kBytes ? 16 : 8;  // of a chunk
#pragma unroll
        for (int i = 0; i < KC; ++i)
#pragma unroll
          for (int h = 0; h < kDims / 8; ++h) {
            const uint4 w = live ? __ldg(reinterpret_cast<const uint4*>(src + (i * 4 + c) * kDims + 8 * h)) : make_uint4(0, 0, 0, 0);
            const int at = (i * kDims / 8 + h) * 4;
            q[n][at] = w.x;
            q[n][at + 1] = w.y;
            q[n][at + 2] = w.z;
            q[n][at + 3] = w.w;
          }
        float factor = 1.f;
        if constexpr (S::kBytes) {
          // bf16 queries as f16 times a power of two that brings the row's largest element to 2^8: elements of at least 2^-25 of
          // that stay exact, smaller ones are off by 2^-33 of it at most
          if (p.q_bf16) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < QW; ++i) top = max(top, max(q[n][i] & 0x7fffu, (q[n][i] >> 16) & 0x7fffu));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = (int)(top >> 7);  // the exponent's field
            factor = e == 255 || top == 0 ? 1.f : __uint_as_float((uint32_t)min(254 - e + 8, 254) << 23);
#pragma unroll
            for (int i = 0; i < QW; ++i) {
              const float2 f = unpack2<true>(q[n][i]);
              q[n][i] = pack2<false>(f.x * factor, f.y * factor);
            }
          }
        }
        const float mine = p.scale_log2 / factor;
        mult[n][0] = __shfl_sync(0xffffffffu, mine, 8 * c);
        mult[n][1] = __shfl_sync(0xffffffffu, mine, 8 * c + 4);
      }
      float o[MT][NT][4], m[NT][2], ref[NT][2], l[NT][2], unit[NT][2], peak[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          m[n][r] = -INFINITY;
          ref[n][r] = l[n][r] = peak[n][r] = 0.f;
          unit[n][r] = 1.f;
        }
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[j][n][e] = 0.f;

      for (; x < end; ++x) {
#pragma unroll
        for (int s = 0; s < KT; ++s) {
          id[s] = id1[s];
          id1[s] = id2[s];
          bad |= now.key + 16 * s < len && (unsigned)(id[s] - 1) >= (unsigned)p.pages;
        }
        uint32_t v[KT][4][VW];
        float vs[KT][2] = {};
        load_v(now, id, v, vs);
        float sc[KT][NT][4];
#pragma unroll
        for (int s = 0; s < KT; ++s)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[s][n][e] = 0.f;
#pragma unroll
            for (int i = 0; i < KC; ++i) {
              const uint32_t w0[4] = {k[s][0][i].x, k[s][0][i].y, k[s][0][i].z, k[s][0][i].w};
              const uint32_t w1[4] = {k[s][1][i].x, k[s][1][i].y, k[s][1][i].z, k[s][1][i].w};
              if constexpr (S::kBytes) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  uint32_t a0, a1, a2, a3;
                  codes4<STORE>(w0[j], a0, a2);
                  codes4<STORE>(w1[j], a1, a3);
                  mma<false>(sc[s][n], a0, a1, a2, a3, q[n][8 * i + 2 * j], q[n][8 * i + 2 * j + 1]);
                }
              } else {
#pragma unroll
                for (int j = 0; j < 2; ++j)
                  mma<BF>(sc[s][n], w0[2 * j], w1[2 * j], w0[2 * j + 1], w1[2 * j + 1], q[n][4 * i + 2 * j], q[n][4 * i + 2 * j + 1]);
              }
            }
          }
        float ks_now[KT][2];
#pragma unroll
        for (int s = 0; s < KT; ++s) {
          ks_now[s][0] = ks[s][0];
          ks_now[s][1] = ks[s][1];
        }
        if (x + 1 < hi) {
          load_k(ahead, id1, k, ks);
          next(ahead);
          if (x + 2 < hi) page_ids(ahead, id2);
        }
        // ---- scores in powers of two; e = 0, 1: key g, rows 2c, 2c + 1; e = 2, 3: key g + 8
        bool grown = false;
#pragma unroll
        for (int s = 0; s < KT; ++s)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float t = sc[s][n][e] * mult[n][e & 1];
              if constexpr (S::kBytes) t *= ks_now[s][e >> 1];
              if (now.key + kTileKeys > len && now.key + 16 * s + g + 8 * (e >> 1) >= len) t = -INFINITY;
              sc[s][n][e] = t;
              grown |= t > m[n][e & 1] + (kAbove + kLazy);
            }
        grown = __any_sync(0xffffffffu, grown);
        if (grown) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float top = -INFINITY;
#pragma unroll
              for (int s = 0; s < KT; ++s) top = fmaxf(top, fmaxf(sc[s][n][r], sc[s][n][r + 2]));
              const float m_new = fmaxf(m[n][r], max_over_keys(top) - kAbove);
              ref[n][r] = from_minus_inf(m_new);
              const float alpha = ex2_approx_ftz(m[n][r] - ref[n][r]);
              m[n][r] = m_new;
              l[n][r] *= alpha;
              peak[n][r] *= alpha;
#pragma unroll
              for (int j = 0; j < MT; ++j) {
                o[j][n][r] *= alpha;
                o[j][n][r + 2] *= alpha;
              }
            }
        }
#pragma unroll
        for (int s = 0; s < KT; ++s)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float w = ex2_approx_ftz(sc[s][n][e] - ref[n][e & 1]);
              l[n][e & 1] += w;
              sc[s][n][e] = S::kBytes ? w * vs[s][e >> 1] : w;
            }
        if constexpr (S::kBytes) {
          // A probability times its value's scale goes to f16 in units of (about) the largest so far: scales differ from key to key by
          // any factor.
          bool off = grown;
#pragma unroll
          for (int s = 0; s < KT; ++s)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) off |= sc[s][n][e] > (1 << kLazy) * peak[n][e & 1];
          if (__any_sync(0xffffffffu, off)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                float top = peak[n][r];
#pragma unroll
                for (int s = 0; s < KT; ++s) top = fmaxf(top, fmaxf(sc[s][n][r], sc[s][n][r + 2]));
                top = max_over_keys(top);
                peak[n][r] = top;
                const int e = (int)(__float_as_uint(top) >> 23);
                const float u = top > 0.f && e < 255 ? __uint_as_float((uint32_t)min(max(254 + kLift - e, 1), 253) << 23) : unit[n][r];
                const float f = u / unit[n][r];
                unit[n][r] = u;
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                  o[j][n][r] *= f;
                  o[j][n][r + 2] *= f;
                }
              }
          }
#pragma unroll
          for (int s = 0; s < KT; ++s)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) sc[s][n][e] *= unit[n][e & 1];
        }
        // ---- O += V P, probabilities as two 16-bit numbers
#pragma unroll
        for (int s = 0; s < KT; ++s) {
          uint32_t hi_[NT][2], lo_[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float a = sc[s][n][2 * h], z = sc[s][n][2 * h + 1];
              const uint32_t w = pack2<BF>(a, z);
              const float2 f = unpack2<BF>(w);
              hi_[n][h] = transposed(w);
              lo_[n][h] = transposed(pack2<BF>(a - f.x, z - f.y));
            }
          if constexpr (S::kBytes) {
#pragma unroll
            for (int i = 0; i < VW; ++i) {  // four dimensions
              uint32_t a[2][4];
              codes4<STORE>(__byte_perm(v[s][0][i], v[s][1][i], 0x5140), a[0][0], a[0][1]);
              codes4<STORE>(__byte_perm(v[s][2][i], v[s][3][i], 0x5140), a[0][2], a[0][3]);
              codes4<STORE>(__byte_perm(v[s][0][i], v[s][1][i], 0x7362), a[1][0], a[1][1]);
              codes4<STORE>(__byte_perm(v[s][2][i], v[s][3][i], 0x7362), a[1][2], a[1][3]);
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  mma<false>(o[2 * i + h][n], a[h][0], a[h][1], a[h][2], a[h][3], hi_[n][0], hi_[n][1]);
                  mma<false>(o[2 * i + h][n], a[h][0], a[h][1], a[h][2], a[h][3], lo_[n][0], lo_[n][1]);
                }
            }
          } else {
#pragma unroll
            for (int i = 0; i < VW; ++i) {  // two dimensions
              const uint32_t a0 = __byte_perm(v[s][0][i], v[s][1][i], 0x5410), a1 = __byte_perm(v[s][0][i], v[s][1][i], 0x7632);
              const uint32_t a2 = __byte_perm(v[s][2][i], v[s][3][i], 0x5410), a3 = __byte_perm(v[s][2][i], v[s][3][i], 0x7632);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma<BF>(o[i][n], a0, a1, a2, a3, hi_[n][0], hi_[n][1]);
                mma<BF>(o[i][n], a0, a1, a2, a3, lo_[n][0], lo_[n][1]);
              }
            }
          }
        }
        next(now);
      }
      // ---- leaving the item
      seen_bad |= bad;
      const bool whole = item_lo >= lo && item_hi <= hi;
      const int slot = warp * 2 + (item_lo <= lo ? 0 : 1);
      float* mine = slots + slot * S::kSlotFloats;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float sum = bad ? NAN : sum_over_keys(l[n][r]);
          const int row = n * 8 + 2 * c + r;
          const float f = (whole ? 1.f / sum : 1.f) / unit[n][r];
#pragma unroll
          for (int j = 0; j < MT; j += 4) {
            float d[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              d[2 * i] = o[j + i][n][r] * f;
              d[2 * i + 1] = o[j + i][n][r + 2] * f;
            }
            if (whole) {
              if (row < rows) write_row(b, head, rt * R + row, dim_of(j), d);
            } else {
              float4* at = reinterpret_cast<float4*>(mine + row * S::kPitch + dim_of(j));
              at[0] = make_float4(d[0], d[1], d[2], d[3]);
              at[1] = make_float4(d[4], d[5], d[6], d[7]);
            }
          }
          if (g == 0) {
            if (whole) {
              if (row < rows) write_lse(b, head, rt * R + row, m[n][r], sum);
            } else {
              mine[R * S::kPitch + row] = m[n][r];
              mine[R * S::kPitch + R + row] = sum;
            }
          }
        }
      if (!whole && lane == 0) {
        seg_item[slot] = (b * p.kv_heads + head) * p.row_tiles + rt;
        seg_lo[slot] = item_lo;
        seg_hi[slot] = item_hi;
      }
    }
    if (seen_bad && lane == 0) atomicMax(status, (int)DEV_BAD_INDEX);
  }
  __syncthreads();

  // ---- items that several warps had
  const unsigned cta_lo = range_of(blockIdx.x * kWarps), cta_hi = range_of((blockIdx.x + 1) * kWarps);
  // The parts in slots [s0, s1) (those that are marked), added in ascending order: to the output, or to a part of the item in memory.
  auto join = [&](int s0, int s1, int item, float* part) {
    const int rt = item % p.row_tiles, pair = item / p.row_tiles, head = pair % p.kv_heads, b = pair / p.kv_heads;
    const int rows = min(R, p.group - rt * R);
    for (int i = tid; i < rows * (D / 8); i += kThreads) {
      const int row = i / (D / 8), d = (i - row * (D / 8)) * 8;
      float M = -INFINITY, L = 0.f, acc[8] = {};
      for (int s = s0; s < s1; ++s)
        if (seg_item[s] >= 0) M = fmaxf(M, slots[s * S::kSlotFloats + R * S::kPitch + row]);
      const float ref = from_minus_inf(M);
      for (int s = s0; s < s1; ++s) {
        if (seg_item[s] < 0) continue;
        const float* from = slots + s * S::kSlotFloats;
        const float f = ex2_approx_ftz(from[R * S::kPitch + row] - ref);
        const float4 u = *reinterpret_cast<const float4*>(from + row * S::kPitch + d), w = *reinterpret_cast<const float4*>(from + row * S::kPitch + d + 4);
        L += from[R * S::kPitch + R + row] * f;
        acc[0] += u.x * f; acc[1] += u.y * f; acc[2] += u.z * f; acc[3] += u.w * f;
        acc[4] += w.x * f; acc[5] += w.y * f; acc[6] += w.z * f; acc[7] += w.w * f;
      }
      if (part) {
        float4* to = reinterpret_cast<float4*>(part + row * D + d);
        to[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        to[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
        if (d == 0) {
          part[R * D + row] = M;
          part[R * D + R + row] = L;
        }
      } else {
        const float inv = 1.f / L;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] *= inv;
        write_row(b, head, rt * R + row, d, acc);
        if (d == 0) write_lse(b, head, rt * R + row, M, L);
      }
    }
  };
  int shared_item[2] = {-1, -1};  // of several CTAs: the first and the last of the range
  unsigned shared_lo[2] = {}, shared_hi[2] = {};
  for (int s = 0; s < 2 * kWarps;) {
    const int item = seg_item[s];
    int z = s + 1;
    if (item >= 0) {
      while (z < 2 * kWarps && (seg_item[z] < 0 || seg_item[z] == item)) ++z;
      const bool inside = seg_lo[s] >= cta_lo && seg_hi[s] <= cta_hi;
      const int which = seg_lo[s] < cta_lo ? 0 : 1;
      join(s, z, item, inside ? nullptr : p.part + ((int64_t)blockIdx.x * 2 + which) * S::kPartFloats);
      if (!inside) {
        shared_item[which] = item;
        shared_lo[which] = seg_lo[s];
        shared_hi[which] = seg_hi[s];
      }
    }
    s = z;
  }
  if (shared_item[0] < 0 && shared_item[1] < 0) return;
  __syncthreads();
  if (tid < 2) {
    last_s[tid] = 0;
    const int which = tid;
    if (shared_item[which] >= 0) {
      const unsigned c0 = worker_of(shared_lo[which], total, workers) / kWarps, c1 = worker_of(shared_hi[which] - 1, total, workers) / kWarps;
      __threadfence();
      last_s[which] = atomicInc(&p.tickets[c0], c1 - c0) == c1 - c0;  // back to zero by the last
      __threadfence();
    }
  }
  __syncthreads();
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (!last_s[which]) continue;
    // warp w takes the parts c0 + w, c0 + w + kWarps, ...; a lane has eight (D = 64: four) rows' share of the dimensions
    const int c0 = worker_of(shared_lo[which], total, workers) / kWarps, c1 = worker_of(shared_hi[which] - 1, total, workers) / kWarps;
    auto part_of = [&](int i) { return p.part + ((int64_t)i * 2 + (i == c0 ? 1 : 0)) * S::kPartFloats; };
    constexpr int kVecs = R * D / 4 / 32;  // of a lane; vector i is number i * 32 + lane
    const int row = lane & (R - 1);
    float M = -INFINITY, L = 0.f;
    for (int i = c0 + warp; i <= c1; i += kWarps) M = fmaxf(M, __ldcg(part_of(i) + R * D + row));
    const float ref = from_minus_inf(M);
    float4 acc[kVecs];
#pragma unroll
    for (int e = 0; e < kVecs; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    const int rows = min(R, p.group - shared_item[which] % p.row_tiles * R);
    for (int i = c0 + warp; i <= c1; i += kWarps) {
      const float* from = part_of(i);
      const float f = ex2_approx_ftz(__ldcg(from + R * D + row) - ref);
      L += __ldcg(from + R * D + R + row) * f;
#pragma unroll
      for (int e = 0; e < kVecs; ++e) {
        const int at = e * 32 + lane, r = at / (D / 4);
        const float fr = __shfl_sync(0xffffffffu, f, r);
        if (r < rows) {
          const float4 u = __ldcg(reinterpret_cast<const float4*>(from) + at);
          acc[e].x += u.x * fr; acc[e].y += u.y * fr; acc[e].z += u.z * fr; acc[e].w += u.w * fr;
        }
      }
    }
    __syncthreads();  // the slots are free
    float* mine = slots + warp * S::kSlotFloats;
#pragma unroll
    for (int e = 0; e < kVecs; ++e) {
      const int at = e * 32 + lane, r = at / (D / 4);
      *reinterpret_cast<float4*>(mine + r * S::kPitch + (at - r * (D / 4)) * 4) = acc[e];
    }
    if (lane < R) {
      mine[R * S::kPitch + lane] = M;
      mine[R * S::kPitch + R + lane] = L;
    }
    if (tid < 2 * kWarps) seg_item[tid] = tid < kWarps ? 0 : -1;
    __syncthreads();
    join(0, kWarps, shared_item[which], nullptr);
  }
}

template <int STORE, int D, int NT>
int launch(ctb_ctx* ctx, cudaStream_t st, Params p, int64_t batch) {
  using S = Shape<STORE, D, NT>;
  static_assert(S::kSmem <= 227 * 1024, "shared memory of a CTA");
  p.row_tiles = (p.group + S::R - 1) / S::R;
  // of a sequence, at most; one where the page table is empty
  const int64_t tiles = std::max<int64_t>(1, (((int64_t)p.width << p.page_log2) + 16 * S::KT - 1) / (16 * S::KT) * p.kv_heads * p.row_tiles);
  if (tiles > INT32_MAX) return fail(CTB_UNSUPPORTED, "ctb_fmha_paged: a sequence has too many keys");
  const int64_t chunk = std::min<int64_t>(kMaxBatch, INT32_MAX / tiles);
  if ((size_t)ctx->sm_count * 2 * S::kPartFloats * sizeof(float) > kSlotBytes || ctx->sm_count > kTickets)
    return fail(CTB_UNSUPPORTED, "ctb_fmha_paged: more SMs than the split over keys has scratch for");
  auto kern = fmha_paged_kernel<STORE, D, NT>;
  cudaError_t e = allow_smem(kern, S::kSmem);
  if (e != cudaSuccess) return cuda_fail(e, "ctb_fmha_paged: shared memory opt-in");
  const StreamScratch scratch(ctx, st);
  if (!scratch.data) return fail(CTB_CUDA_ERROR, "ctb_fmha_paged: no scratch for the split over keys");
  p.part = scratch.data;
  p.tickets = scratch.tickets;
  for (int64_t b = 0; b < batch; b += chunk) {
    Params q = p;
    q.batch = (int)std::min(chunk, batch - b);
    q.Q = static_cast<const uint16_t*>(p.Q) + b * p.q_seq;
    q.Out = static_cast<uint16_t*>(p.Out) + b * p.heads * D;
    q.lse = p.lse ? p.lse + b * p.heads : nullptr;
    q.table = p.table + b * p.table_ld;
    q.lengths = p.lengths + b;
    const int64_t most = (tiles * q.batch + (int64_t)S::kWarps * kMinTiles - 1) / ((int64_t)S::kWarps * kMinTiles);
    launch_kernel(kern, (unsigned)std::min<int64_t>(most, ctx->sm_count), S::kThreads, S::kSmem, st, 0, q, ctx->dev_status);
    CTB_CHECK_LAUNCH("ctb_fmha_paged launch");
  }
  return CTB_OK;
}

template <int STORE>
int pick(ctb_ctx* ctx, cudaStream_t st, const Params& p, int64_t batch, int64_t D) {
  const bool small = p.group <= 8;
  if (D == 64) return small ? launch<STORE, 64, 1>(ctx, st, p, batch) : launch<STORE, 64, 2>(ctx, st, p, batch);
  return small ? launch<STORE, 128, 1>(ctx, st, p, batch) : launch<STORE, 128, 2>(ctx, st, p, batch);
}

}  // namespace

extern "C" int ctb_fmha_paged(ctb_ctx* ctx, void* stream, void* Out, float* lse, const void* Q, const ctb_kv_cache* cache,
                              const int32_t* page_table, const int32_t* lengths, int64_t batch, int64_t heads, int64_t q_seq_stride,
                              int64_t q_head_stride, int64_t table_width, int64_t table_stride, float qk_scale, int dtype) {
  CTB_CHECK_CTX(ctx);
  CurrentDevice on(ctx);
  int r = check_kv_cache("ctb_fmha_paged", cache);
  if (r) return r;
  if (batch < 0 || heads <= 0 || table_width < 0) return fail(CTB_BAD_ARG, "ctb_fmha_paged: non-positive dimension");
  if (heads % cache->kv_heads)
    return fail(CTB_BAD_ARG, "ctb_fmha_paged: heads (%lld) is not a multiple of kv_heads (%lld)", (long long)heads, (long long)cache->kv_heads);
  if (dtype != CTB_F16 && dtype != CTB_BF16) return fail(CTB_UNSUPPORTED, "ctb_fmha_paged: queries are f16 or bf16");
  if (cache->dtype != dtype && cache->dtype != CTB_E4M3 && cache->dtype != CTB_I8)
    return fail(CTB_BAD_ARG, "ctb_fmha_paged: a cache of 16-bit elements has the type of the queries");
  if (!isfinite(qk_scale)) return fail(CTB_BAD_ARG, "ctb_fmha_paged: qk_scale is not finite");
  const int64_t D = cache->head_dim, page = cache->page_size;
  if (heads > 65536 || table_width * page > (1 << 28) || table_width > (1 << 28))
    return fail(CTB_UNSUPPORTED, "ctb_fmha_paged: shape too large");
  if (batch == 0) return CTB_OK;
  CTB_CHECK_DEV(Q); CTB_CHECK_DEV(Out); CTB_CHECK_DEV(lengths);
  if (lse) CTB_CHECK_DEV(lse);
  if (table_width) CTB_CHECK_DEV(page_table);
  if (table_stride < table_width && batch > 1) return fail(CTB_BAD_ARG, "ctb_fmha_paged: rows of the page table overlap");
  if ((uintptr_t)Q % 16 || (uintptr_t)Out % 16 || q_seq_stride % 8 || q_head_stride % 8)
    return fail(CTB_BAD_ALIGN, "ctb_fmha_paged: Q and Out must be 16-byte aligned and the strides of Q multiples of 8 elements");
  Params p = {};
  p.Q = Q; p.Out = Out; p.lse = lse;
  p.K = cache->k; p.V = cache->v; p.Ks = cache->k_scale; p.Vs = cache->v_scale;
  p.table = page_table; p.lengths = lengths;
  p.q_seq = q_seq_stride; p.q_head = q_head_stride; p.table_ld = table_stride;
  p.k_page = cache->k_page_stride; p.v_page = cache->v_page_stride;
  p.ks_page = cache->k_scale_page_stride; p.vs_page = cache->v_scale_page_stride;
  p.heads = (int)heads; p.kv_heads = (int)cache->kv_heads; p.group = (int)(heads / cache->kv_heads);
  p.width = (int)table_width; p.pages = (int)cache->pages;
  while ((1ll << p.page_log2) < page) ++p.page_log2;
  p.q_bf16 = dtype == CTB_BF16;
  p.scale_log2 = qk_scale * 1.4426950408889634f;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (cache->dtype) {
    case CTB_F16: return pick<F16>(ctx, st, p, batch, D);
    case CTB_BF16: return pick<BF16>(ctx, st, p, batch, D);
    case CTB_E4M3: return pick<E4M3>(ctx, st, p, batch, D);
    default: return pick<I8>(ctx, st, p, batch, D);
  }
}
