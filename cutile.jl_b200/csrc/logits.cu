// Operators over rows of logits for sm_100a: log probabilities of given tokens with entropy and top alternatives, distillation from
// a teacher's top logits, and their gradients.
//
// With z = x / temperature, all of them rest on the maximum and the sum of exponentials of a row,
//   lse = log sum_v e^z_v = z_max + log s,   s = sum_v e^(z_v - z_max),
// which one pass over the row finds (a running reference per thread; a common one where the threads meet):
//   log p_v  = (z_v - z_max) - log s
//   entropy  = -sum_v p_v log p_v = log s - w / s,   w = sum_v e^(z_v - z_max) (z_v - z_max)
// and nothing of the row is kept.  A forward pass reads every logit once and writes a few numbers per row; a gradient reads every
// logit once more and writes as much.  HBM bounds both; what there is to compute per element (one ex2 and a handful of f32 operations,
// for 16-bit logits 11 issue slots in the time that HBM takes for an element) has to stay below that.
#include <float.h>

#include <algorithm>
#include <type_traits>

#include "ctx.h"
#include "ptx.cuh"
#include "rows.cuh"

using namespace ctb;
using namespace ctb_internal;

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 4;               // vectors of 16 bytes per thread and tile
constexpr int kTile = kThreads * kUnroll;  // vectors
constexpr int kMaxTop = 32;
constexpr int kMaxEntries = kThreads;    // of a teacher's list
constexpr int kCand = 1024;
constexpr int kMaxParts = 32;
constexpr int kPlainPerSm = 5, kTopPerSm = 4, kDistillPerSm = 4, kBackwardPerSm = 4;  // CTAs on an SM
constexpr int kMostHoles = 512 * 1024;  // elements of a part that have a bit (in two sets) in shared memory
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Exponents (base 2) are held above this where they are multiplied by their power, which is 0 there: 0 * -inf would be NaN.
constexpr float kLowest = -16384.f;
// A thread's reference follows its maximum only when an element is 2^kSlack above it: powers up to 2^kSlack are harmless in f32.
constexpr float kSlack = 64.f;
constexpr float kFar = 1e30f;  // rows with a maximum beyond +-kFar (masked as a whole, or infinite) are summed in another way

// ------------------------------------------------------------------ the best k of a row
// One pass, every element compared with a threshold that at least k earlier elements reach:
//   - The threads' running maxima, taken over groups of four threads, are 64 maxima of disjoint parts of what has been read.  The k-th
//     largest of them is reached by at least k elements, and few more (24 of 8192 for k = 20), so an element that is read later and is not
//     above it cannot be one of the best k: k earlier ones (lower indices) precede it in the order by value, then index.
//   - The first tile gives the first threshold; it is taken again when 2, 4, 8... tiles have been read.  What is above goes to a
//     list in shared memory, about 24 (k = 20) for every doubling.
//   - Elements of the first tile that EQUAL its threshold may belong to the best k, but only if fewer than k are above it in the whole
//     row; they are then the lowest-numbered ones of the first tile, and are looked up there (rows that are masked but for a few
//     elements, rows of equal values).
//   - A list that overflows (rows in ascending order) is made again by a radix search for the k-th value, which reads the row
//     four times more.
struct Best {
  float group[64];
  float theta;
  int count, count2;
  int warp_n[kWarps];
  int bin, above;
  float value[kCand], value2[kCand];
  int index[kCand], index2[kCand];
  float out_value[kMaxTop];
  int out_index[kMaxTop];
};

// The k-th largest of the 64 group maxima; the whole CTA.
__device__ __forceinline__ float group_threshold(float mine, int k, Best& b) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float g = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
  g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 2));
  const int i = warp * 8 + (lane >> 2);
  if ((lane & 3) == 0) b.group[i] = g;
  __syncthreads();
  int rank = 0;  // among a quarter of the groups per lane
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int o = (lane & 3) * 16 + j;
    const float v = b.group[o];
    rank += v > g || (v == g && o < i);
  }
  rank += __shfl_xor_sync(0xffffffffu, rank, 1);
  rank += __shfl_xor_sync(0xffffffffu, rank, 2);
  if (rank == k - 1 && (lane & 3) == 0) b.theta = g;
  __syncthreads();
  return b.theta;
}

// Writes the best k of the n listed elements to out_*, in order; what is missing gets index -1.  The whole CTA; the list is complete and
// visible.
__device__ void select_list(int n, int k, Best& b) {
  const int tid = threadIdx.x;
  const float* value = b.value;
  const int* index = b.index;
  if (tid < kMaxTop) b.out_index[tid] = -1;
  if (tid == 0) b.count2 = 0;
  if (n > 64) {  // thinned out first, or ranking each against all others would take longest
    float mine = -INFINITY;
    for (int i = tid; i < n; i += kThreads) mine = fmaxf(mine, b.value[i]);
    const float theta = group_threshold(mine, k, b);
    for (int i = tid; i < n; i += kThreads)
      if (b.value[i] >= theta) {
        const int at = atomicAdd(&b.count2, 1);
        b.value2[at] = b.value[i];
        b.index2[at] = b.index[i];
      }
    value = b.value2;
    index = b.index2;
    __syncthreads();
    n = b.count2;
  } else {
    __syncthreads();
  }
  for (int i = tid; i < n; i += kThreads) {
    const float v = value[i];
    const int id = index[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += value[j] > v || (value[j] == v && index[j] < id);
    if (rank < k) {
      b.out_value[rank] = v;
      b.out_index[rank] = id;
    }
  }
  __syncthreads();
}

// Adds the first `need` elements that equal `value`, in the order of their indices, to the `have` listed ones; returns how many are listed.
template <typename T>
__device__ int append_equal(const Range<T>& r, float value, int have, int need, Best& b) {
  constexpr int V = 16 / (int)sizeof(T);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int base = r.v0; need > 0 && base < r.v1; base += kThreads) {
    const int v = base + tid;
    unsigned match = 0;
    float f[V];
    if (v < r.v1) {
      unpack_row<T>(load_vec(r, v), f);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (f[i] == value && r.has(v, i)) match |= 1u << i;
    }
    const int mine = __popc(match);
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) b.warp_n[warp] = upto;
    __syncthreads();
    int at = upto - mine, total = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) at += b.warp_n[w];
      total += b.warp_n[w];
    }
    for (; match && at < need; match &= match - 1, ++at) {
      b.value[have + at] = value;
      b.index[have + at] = v * V - r.off + __ffs(match) - 1;
    }
    have += min(total, need);
    need -= min(total, need);
    __syncthreads();
  }
  return have;
}

// f32 bits in the order of the values; both zeros alike.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// Makes the list anew: the k-th largest value bit by bit, from counts of eight bits at a time.  Returns how many are listed.
template <typename T>
__device__ int radix_list(const Range<T>& r, int k, Best& b) {
  constexpr int V = 16 / (int)sizeof(T);
  const int tid = threadIdx.x;
  int* hist = b.index2;  // 256 counters
  uint32_t prefix = 0, mask = 0;
  int want = k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    hist[tid] = 0;
    __syncthreads();
    for (int v = r.v0 + tid; v < r.v1; v += kThreads) {
      float f[V];
      unpack_row<T>(load_vec(r, v), f);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint32_t key = order_key(f[i]);
        if (f[i] == f[i] && r.has(v, i) && (key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1);
      }
    }
    __syncthreads();
    if (tid == 0) {
      int bin = 255, above = 0;
      while (bin > 0 && above + hist[bin] < want) above += hist[bin--];
      b.bin = bin;
      b.above = above;
    }
    __syncthreads();
    prefix |= (uint32_t)b.bin << shift;
    mask |= 255u << shift;
    want -= b.above;
    __syncthreads();
  }
  const float kth = key_value(prefix);
  if (tid == 0) b.count = 0;
  __syncthreads();
  for (int v = r.v0 + tid; v < r.v1; v += kThreads) {
    float f[V];
    unpack_row<T>(load_vec(r, v), f);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (f[i] > kth) {  // fewer than k
        const int at = atomicAdd(&b.count, 1);
        b.value[at] = f[i];
        b.index[at] = v * V - r.off + i;
      }
  }
  __syncthreads();
  return append_equal(r, kth, b.count, want, b);
}

// ------------------------------------------------------------------ sums of a row
template <typename T>
__device__ __forceinline__ void load_tile(uint4 (&q)[kUnroll], const Range<T>& r, int v, bool keep) {
  const int tid = threadIdx.x;
  if (r.inside(v, kTile)) {
    const uint4* p = r.at(v) + tid;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) q[u] = keep ? __ldcg(p + u * kThreads) : __ldcs(p + u * kThreads);
  } else {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) q[u] = load_vec(r, v + u * kThreads + tid);
  }
}

// A thread's share of s = sum 2^(x c - m2) and w = sum 2^(x c - m2) (x c - m2), with c = log2(e) / temperature: one fused multiply-add gives
// an exponent with one rounding, whatever the magnitude of x, and the rounding of c is that of a temperature, the same for the whole row.
// Masked elements (-inf) would make w NaN (0 * -inf): with ENTROPY words are raised to a floor whose power is 0.  Valid for rows whose
// maximum is `plain`; the others take slow_sums.
template <typename T, bool ENTROPY>
struct Sums {
  [[maybe_unused]] static constexpr uint32_t kFloor = sizeof(T) == 4 ? 0xf149f2cau : std::is_same<T, __half>::value ? 0xfbfffbffu : 0xf14af14au;
  // -1e30 (bf16: the next one below), -65504
  float m2 = 0.f, limit = -FLT_MAX;  // elements above limit move the reference
  uint32_t top = empty_row_vec<T>().x;
  float2 s = make_float2(0.f, 0.f), w = make_float2(0.f, 0.f);

  static __device__ __forceinline__ bool plain(float maximum, float c) {
    if (!(maximum <= kFar && maximum >= -0.1f * kFar)) return false;
    return !(ENTROPY && std::is_same<T, __half>::value) || (maximum + 65504.f) * c > 256.f;
  }
  // Returns the largest element of the tile.
  __device__ __forceinline__ float add(const uint4 (&q)[kUnroll], float c) {
    uint32_t all = 0;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t a = max_word<T, true>(max_word<T, true>(q[u].x, q[u].y), max_word<T, true>(q[u].z, q[u].w));
      all = u == 0 ? a : max_word<T, true>(all, a);
    }
    top = max_word<T, true>(top, all);
    const float t = word_max<T>(all);
    if (t > limit) {
      const float x = fminf(fmaxf(t, -kFar), kFar), to = x * c, d = fmaxf(fminf(m2 - to, 0.f), kLowest), r = ex2_approx_ftz(d);
      if constexpr (ENTROPY) {
        w.x = r * fmaf(s.x, d, w.x);
        w.y = r * fmaf(s.y, d, w.y);
      }
      s.x *= r;
      s.y *= r;
      m2 = to;
      limit = x + kSlack / c;
    }
    const float2 cc = make_float2(c, c), minus = make_float2(-m2, -m2);
    float2 ts = make_float2(0.f, 0.f), tw = ts;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      uint32_t word[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
      if constexpr (ENTROPY)
#pragma unroll
        for (int i = 0; i < 4; ++i) word[i] = max_word<T, false>(word[i], kFloor);
#pragma unroll
      for (int i = 0; i < 8 / (int)sizeof(T); ++i) {
        const float2 t2 = fma_pair(vec_pair<T>(word, i), cc, minus);
        const float2 e = make_float2(ex2_approx_ftz(t2.x), ex2_approx_ftz(t2.y));
        ts = add_pair(ts, e);
        if constexpr (ENTROPY) tw = fma_pair(e, t2, tw);
      }
    }
    s = add_pair(s, ts);
    if constexpr (ENTROPY) w = add_pair(w, tw);
    return t;
  }
  // The warp's (maximum, s, w), the sums relative to that maximum.
  __device__ __forceinline__ float3 over_warp(float c) const {
    const float most = warp_max(word_max<T>(top)), to = fminf(fmaxf(most, -kFar), kFar);
    const float d = fminf(fmaf(-to, c, m2), 1.f), r = ex2_approx_ftz(d), sum = s.x + s.y;  // a thread without elements has m2 = sum = 0
    return make_float3(most, warp_sum(sum * r), ENTROPY ? warp_sum(r * fmaf(sum, fmaxf(d, kLowest), w.x + w.y)) : 0.f);
  }
};

// Listed elements of a range: a bit for each element from vector v0 on, or nothing.
template <typename T>
__device__ __forceinline__ unsigned hole_bits(const unsigned* holes, int v) {  // of the range's vector v
  if constexpr (sizeof(T) == 4) return holes[v >> 3] >> (v & 7) * 4 & 15;
  else return reinterpret_cast<const unsigned char*>(holes)[v];
}
template <typename T>
__device__ __forceinline__ void mask_holes(uint4& q, unsigned bits) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      if (bits >> i & 1) w[i] = 0xff800000u;
    } else {
      const uint32_t low = empty_row_vec<T>().x;
      if (bits >> 2 * i & 1) w[i] = (w[i] & 0xffff0000u) | (low & 0xffffu);
      if (bits >> 2 * i & 2) w[i] = (w[i] & 0xffffu) | (low & 0xffff0000u);
    }
  }
}

// The sums of a warp's threads relative to a maximum that is not `plain`, from differences (x - maximum).
template <typename T>
__device__ __noinline__ float2 slow_sums(const Range<T>& r, const unsigned* holes, float maximum, float c) {
  constexpr int V = 16 / (int)sizeof(T);
  float s = 0.f, w = 0.f;
  for (int v = r.v0 + (int)threadIdx.x; v < r.v1; v += kThreads) {
    uint4 q = load_vec(r, v);
    if (holes) mask_holes<T>(q, hole_bits<T>(holes, v - r.v0));
    float f[V];
    unpack_row<T>(q, f);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float t = (f[i] - maximum) * c, e = ex2_approx_ftz(t);
      s += e;
      w = fmaf(e, fmaxf(t, kLowest), w);
    }
  }
  return make_float2(warp_sum(s), warp_sum(w));
}

// (s, w) of the eight warps, each relative to its own maximum and held by lanes w, w + 8, ..., relative to the maximum of them all.
__device__ __forceinline__ float2 join(float maximum, float s, float w, float most, float c) {
  const float d = (maximum - most) * c, r = ex2_approx_ftz(d);
  float a = s * r, b = r * fmaf(s, fmaxf(d, kLowest), w);
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  return make_float2(a, b);
}
// The same for the records of a row's parts, whose maxima are finite; one per lane.
__device__ __forceinline__ float2 join_parts(float4 record, float most, float c) {
  const float d = (record.x - most) * c, r = ex2_approx_ftz(d);
  return make_float2(warp_sum(record.y * r), warp_sum(r * fmaf(record.y, fmaxf(d, kLowest), record.z)));
}
__device__ __forceinline__ float red_max(const float (&v)[kWarps]) {
  float m = v[0];
#pragma unroll
  for (int i = 1; i < kWarps; ++i) m = fmaxf(m, v[i]);
  return m;
}

__device__ __forceinline__ long long load_id(const void* p, long long i, int bits) {
  return bits == 64 ? static_cast<const long long*>(p)[i] : static_cast<const int*>(p)[i];
}
__device__ __forceinline__ float load_value(const void* p, long long i, int dtype) {
  if (dtype == CTB_F32) return static_cast<const float*>(p)[i];
  if (dtype == CTB_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __uint_as_float((uint32_t) static_cast<const unsigned short*>(p)[i] << 16);
}
template <typename T>
__device__ __forceinline__ Range<T> range_of(const void* x, long long ld, int n, long long row, int part, int per) {
  constexpr int V = 16 / (int)sizeof(T);
  Range<T> r;
  r.src = static_cast<const T*>(x) + row * ld;
  r.off = (int)(((uintptr_t)r.src & 15) / sizeof(T));
  r.n = n;
  const int nvec = (r.off + n + V - 1) / V;
  r.v0 = min(nvec, part * per);
  r.v1 = min(nvec, r.v0 + per);
  return r;
}

// What the kernels below have in common: the logits, and how their rows are cut.
struct Rows {
  const void* x;
  long long ld;
  int n, rows, parts, per;  // per: vectors of a part
  float c, temperature;     // c = log2(e) / temperature
  int* status;
  float* scratch;           // records of the parts: maximum, s, w, -, then the best values and their indices
  unsigned* tickets;        // a counter per row
};
// Floats of a part's record.
__host__ __device__ constexpr int record_floats(int top) { return 4 + (2 * top + 3) / 4 * 4; }

// ------------------------------------------------------------------ log probabilities, forward
struct Logprobs : Rows {
  const void* tokens;
  int token_bits, top;
  float *logprobs, *entropy, *lse, *top_logprobs;
  int* top_ids;
};

// A CTA takes (row, part) after (row, part).  Rows are cut into parts where there are fewer rows than room for CTAs; the CTA that
// finishes a row's last part puts the parts together.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, TOP ? kTopPerSm : kPlainPerSm) logprobs_kernel(const __grid_constant__ Logprobs p) {
  __shared__ float red[2][3][kWarps];
  __shared__ int last;
  __shared__ typename std::conditional<TOP, Best, int>::type best_store;
  Best& best = reinterpret_cast<Best&>(best_store);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dependency_sync();
  const long long items = (long long)p.rows * p.parts;
  auto token_of = [&](long long at) { return at < items && p.tokens ? load_id(p.tokens, at / p.parts, p.token_bits) : -1ll; };
  long long next_token = token_of(blockIdx.x);
  int turn = 0;
  for (long long at = blockIdx.x; at < items; at += gridDim.x) {
    const long long row = at / p.parts, token = next_token;
    const int part = (int)(at - row * p.parts);
    next_token = token_of(at + gridDim.x);
    if (token == 0) {
      if (part == 0) {
        if (tid == 0) {
          if (p.logprobs) p.logprobs[row] = 0.f;
          if (p.entropy) p.entropy[row] = 0.f;
          if (p.lse) p.lse[row] = 0.f;
        }
        if (TOP && tid < p.top) {
          p.top_logprobs[row * p.top + tid] = 0.f;
          p.top_ids[row * p.top + tid] = 0;
        }
      }
      continue;
    }
    const Range<T> r = range_of<T>(p.x, p.ld, p.n, row, part, p.per);
    Sums<T, true> sums;
    float theta = -INFINITY;
    if constexpr (TOP) {
      if (tid == 0) best.count = 0;  // ahead of the barriers of the first threshold
    }
    int tile = 0;
#pragma unroll 1
    for (int v = r.v0; v < r.v1 || tile == 0; v += kTile, ++tile) {
      uint4 q[kUnroll];
      load_tile(q, r, v, false);
      const float most = sums.add(q, p.c);
      if constexpr (TOP) {
        if (tile == 0) theta = group_threshold(word_max<T>(sums.top), p.top, best);
        if (most > theta) {
#pragma unroll
          for (int u = 0; u < kUnroll; ++u) {
            constexpr int V = 16 / (int)sizeof(T);
            float f[V];
            unpack_row<T>(q[u], f);
            const int e0 = (v + u * kThreads + tid) * V - r.off;
#pragma unroll
            for (int i = 0; i < V; ++i)
              if (f[i] > theta) {
                const int pos = atomicAdd(&best.count, 1);
                if (pos < kCand) {
                  best.value[pos] = f[i];
                  best.index[pos] = e0 + i;
                }
              }
          }
        }
        if (tile > 0 && (tile & (tile + 1)) == 0 && v + kTile < r.v1) theta = group_threshold(word_max<T>(sums.top), p.top, best);
      }
    }

    float(&mine)[3][kWarps] = red[turn++ & 1];
    {
      const float3 of_warp = sums.over_warp(p.c);
      if (lane == 0) {
        mine[0][warp] = of_warp.x;
        mine[1][warp] = of_warp.y;
        mine[2][warp] = of_warp.z;
      }
    }
    __syncthreads();
    float top_max = red_max(mine[0]);
    const bool plain = Sums<T, true>::plain(top_max, p.c);
    if (!plain) {
      top_max = fmaxf(top_max, -FLT_MAX);
      const float2 of_warp = slow_sums(r, nullptr, top_max, p.c);
      if (lane == 0) {
        mine[1][warp] = of_warp.x;
        mine[2][warp] = of_warp.y;
      }
      __syncthreads();
    }
    if constexpr (TOP) {
      int n = best.count;
      if (n > kCand) {
        n = radix_list(r, p.top, best);
      } else if (n < p.top) {
        // theta of the first tile: with fewer than k above it, it is also the last one
        Range<T> first = r;
        first.v1 = min(r.v1, r.v0 + kTile);
        n = append_equal(first, theta, n, p.top - n, best);
      }
      select_list(n, p.top, best);
    }
    float2 sum = make_float2(0.f, 0.f);
    if (warp == 0) {
      const int w = lane & 7;
      sum = join(plain ? mine[0][w] : top_max, mine[1][w], mine[2][w], top_max, p.c);
    }

    bool finish = true;
    if (p.parts > 1) {
      const int stride = record_floats(p.top);
      float* record = p.scratch + at * stride;
      if (tid == 0) *reinterpret_cast<float4*>(record) = make_float4(top_max, sum.x, sum.y, 0.f);
      if constexpr (TOP) {
        if (tid < p.top) {
          const int id = best.out_index[tid];
          record[4 + tid] = id >= 0 ? best.out_value[tid] : -INFINITY;
          reinterpret_cast<int*>(record)[4 + p.top + tid] = id;
        }
      }
      if (warp == 0) {  // it alone has written
        __threadfence();
        __syncwarp();
        if (lane == 0) last = atomicInc(p.tickets + row, p.parts - 1) == (unsigned)p.parts - 1;
      }
      __syncthreads();
      finish = last;
      if (finish) {
        __threadfence();
        const float* all = p.scratch + row * p.parts * stride;
        const float4 one = lane < p.parts ? __ldcg(reinterpret_cast<const float4*>(all + (long long)lane * stride))
                                          : make_float4(-FLT_MAX, 0.f, 0.f, 0.f);
        top_max = warp_max(one.x);
        sum = join_parts(one, top_max, p.c);
        if constexpr (TOP) {
          if (tid == 0) best.count = 0;
          __syncthreads();
          for (int i = tid; i < p.parts * p.top; i += kThreads) {
            const float* rec = all + (long long)(i / p.top) * stride + 4 + i % p.top;
            const int id = __ldcg(reinterpret_cast<const int*>(rec) + p.top);
            if (id >= 0) {
              const int pos = atomicAdd(&best.count, 1);
              best.value[pos] = __ldcg(rec);
              best.index[pos] = id;
            }
          }
          __syncthreads();
          select_list(best.count, p.top, best);
        }
      }
      __syncthreads();  // `last` has been read
    }

    if (finish && warp == 0) {
      const float log_sum = logf(sum.x);
      if (lane == 0) {
        if (p.lse) p.lse[row] = top_max / p.temperature + log_sum;
        if (p.entropy) p.entropy[row] = log_sum - kLn2 * (sum.y / sum.x);
        if (p.logprobs) {
          float lp = NAN;
          if (token < 0 || token > p.n) atomicMax(p.status, DEV_BAD_INDEX);
          else lp = (to_float(r.src[token - 1]) - top_max) / p.temperature - log_sum;
          p.logprobs[row] = lp;
        }
      }
      if constexpr (TOP) {
        if (lane < p.top) {
          const int id = best.out_index[lane];
          p.top_logprobs[row * p.top + lane] = id >= 0 ? (best.out_value[lane] - top_max) / p.temperature - log_sum : NAN;
          p.top_ids[row * p.top + lane] = id + 1;
        }
      }
    }
  }
}

// ------------------------------------------------------------------ gradients
// d = p (a + b t), t = log2 p, over vectors of a row; KEPT: they are in L2.
template <typename T, bool ENTROPY>
__device__ __forceinline__ void stream_gradient(const Range<T>& r, T* dst, float c, float lse2, float a, float b) {
  const int tid = threadIdx.x;
  const bool aligned = ((uintptr_t)(dst - r.off) & 15) == 0;
  const float2 cc = make_float2(c, c), minus = make_float2(-lse2, -lse2), aa = make_float2(a, a), bb = make_float2(b, b);
#pragma unroll 1
  for (int v = r.v0; v < r.v1; v += kTile) {
    uint4 q[kUnroll];
    load_tile(q, r, v, false);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      uint32_t word[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
      for (int i = 0; i < 8 / (int)sizeof(T); ++i) {
        float2 t = fma_pair(vec_pair<T>(word, i), cc, minus);
        float2 e = make_float2(ex2_approx_ftz(t.x), ex2_approx_ftz(t.y));
        if constexpr (ENTROPY) {
          t = make_float2(fmaxf(t.x, kLowest), fmaxf(t.y, kLowest));
          e = mul_pair(e, fma_pair(bb, t, aa));
        } else {
          e = mul_pair(e, aa);
        }
        put_pair<T>(word, i, e);
      }
      q[u] = make_uint4(word[0], word[1], word[2], word[3]);
    }
    if (aligned && r.inside(v, kTile)) {
      uint4* to = reinterpret_cast<uint4*>(dst - r.off) + v + tid;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) __stcs(to + u * kThreads, q[u]);
    } else {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int at = v + u * kThreads + tid;
        if (at >= r.v1) continue;
        if (aligned && r.inside(at, 1)) __stcs(reinterpret_cast<uint4*>(dst - r.off) + at, q[u]);
        else store_edge<T>(dst, r.off, r.n, at, q[u]);
      }
    }
  }
}
// Zeros over vectors of a row, by `threads` threads of which this is the i-th.
template <typename T>
__device__ __noinline__ void stream_zeros(const Range<T>& r, T* dst, int i, int threads) {
  const bool aligned = ((uintptr_t)(dst - r.off) & 15) == 0;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int v = r.v0 + i; v < r.v1; v += threads) {
    if (aligned && r.inside(v, 1)) __stcs(reinterpret_cast<uint4*>(dst - r.off) + v, zero);
    else store_edge<T>(dst, r.off, r.n, v, zero);
  }
}

// Gradient at what a teacher lists: g (all p - sum of the q of this id), once per id.  Thread j has entry j and its logit x.
template <typename T>
__device__ __forceinline__ void patch_entries(T* dst, const int* entry, const float* q, int entries, float x, float c, float lse2, float g,
                                              float all, long long lo, long long hi) {
  const int j = threadIdx.x;
  if (j >= entries) return;
  const int id = entry[j];
  if (id <= lo || id > hi) return;
  float sum = 0.f;
  for (int i = 0; i < entries; ++i)
    if (entry[i] == id) {
      if (i < j) return;
      sum += q[i];
    }
  dst[id - 1] = from_float<T>(g * (all * ex2_approx_ftz(fmaf(x, c, -lse2)) - sum));
}

// ------------------------------------------------------------------ distillation, forward, and the gradient at once
struct Distill : Rows {
  const void* ids;
  int id_bits, entries;
  const void* values;
  int values_dtype;
  const float* teacher_lse;
  float *loss, *saved;
  // with the gradient
  const float* d_loss;
  void* dx;
  long long ld_dx;
};

__device__ __forceinline__ double sum_lanes(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double max_lanes(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The teacher's side of a row, in f64: what its list leaves over is a difference from one.
struct Lesson {
  long long at;              // row * parts + part; -1: no more
  double terms, all, norm;   // sum q (log q - z), sum q
  float listed_max, listed;  // what the student gives to the listed ids, each once: maximum, sum of powers relative to it
  int entry[kMaxEntries];    // ids, 0: unused
  float q[kMaxEntries], x[kMaxEntries];
};

__device__ __forceinline__ void bar_stream() { asm volatile("bar.sync 1, 256;" ::: "memory"); }  // the streaming warps alone
static_assert(kThreads == 256, "bar_stream names the number of threads");

// Eight warps stream rows; a ninth one prepares the teacher's side of the next row meanwhile (loads that depend on loads, f64
// exponentials), so that a row ends with one barrier and a handful of operations.  HOLES: teacher_lse is given; what the teacher lists is left out of
// the row's sum by a bit per element and added apart, since the rest's probability from a difference would lose all digits where it
// is small.  GRAD: the same CTA reads the row again, from L2, and writes the gradient.
template <typename T, bool GRAD, bool HOLES>
__global__ void __launch_bounds__(kThreads + 32, kDistillPerSm) distill_kernel(const __grid_constant__ Distill p) {
  constexpr int V = 16 / (int)sizeof(T);
  extern __shared__ __align__(16) unsigned hole_store[];  // HOLES: two sets of bits
  __shared__ Lesson lessons[3];
  __shared__ double power[kMaxEntries];  // the ninth warp's
  __shared__ float red[2][3][kWarps];
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hole_words = HOLES ? (p.per * V + 31) / 32 : 0;
  if constexpr (HOLES)
    for (int i = tid; i < 2 * hole_words; i += kThreads + 32) hole_store[i] = 0;
  grid_dependency_sync();
  const long long items = (long long)p.rows * p.parts;
  long long at = (long long)blockIdx.x - gridDim.x;

  // Ninth warp: the next row that is not padding, or -1; results of padding rows are written on the way.
  auto prepare = [&](Lesson& l) {
    for (;;) {
      at += gridDim.x;
      if (at >= items) {
        if (lane == 0) l.at = -1;
        return;
      }
      const long long row = at / p.parts;
      const int part = (int)(at - row * p.parts);
      const T* src = static_cast<const T*>(p.x) + row * p.ld;
      bool used = false, bad = false;
      double most = -INFINITY;
      for (int j = lane; j < p.entries; j += 32) {
        const long long id = load_id(p.ids, row * p.entries + j, p.id_bits);
        const double u = (double)load_value(p.values, row * p.entries + j, p.values_dtype) / (double)p.temperature;
        const bool out = id < 0 || id > p.n;
        bad |= out;
        used |= id != 0;
        l.entry[j] = out ? 0 : (int)id;
        power[j] = u;
        if (id) most = fmax(most, u);
      }
      used = __any_sync(0xffffffffu, used);
      bad = __any_sync(0xffffffffu, bad);
      if (!used || bad) {
        if (part == 0) {
          if (lane == 0) {
            if (bad) atomicMax(p.status, DEV_BAD_INDEX);
            p.loss[row] = bad ? NAN : 0.f;
            reinterpret_cast<float4*>(p.saved)[row] = make_float4(0.f, 0.f, 0.f, 0.f);
          }
          if constexpr (GRAD)
            stream_zeros<T>(range_of<T>(p.x, p.ld, p.n, row, 0, p.per), static_cast<T*>(p.dx) + row * p.ld_dx, lane, 32);
        }
        continue;
      }
      __syncwarp();
      float x_most = -INFINITY;
      for (int j = lane; j < p.entries; j += 32) {
        const int id = l.entry[j];
        const float x = id ? to_float(src[id - 1]) : -INFINITY;
        l.x[j] = x;
        x_most = fmaxf(x_most, x);
      }
      double sum = 1, norm;
      if constexpr (HOLES) {
        norm = p.teacher_lse[row];
      } else {
        most = max_lanes(most);
        sum = 0;
        for (int j = lane; j < p.entries; j += 32)
          if (l.entry[j]) sum += exp(power[j] - most);
        norm = most + log(sum_lanes(sum));
      }
      double all = 0, terms = 0;
      for (int j = lane; j < p.entries; j += 32) {
        if (l.entry[j] == 0) continue;
        const double log_q = power[j] - norm, q = exp(log_q);
        if (q != 0) terms += q * (log_q - (double)l.x[j] / (double)p.temperature);
        all += q;
        l.q[j] = (float)q;
      }
      all = sum_lanes(all);
      terms = sum_lanes(terms);
      float listed = 0.f;
      if constexpr (HOLES) {
        x_most = fmaxf(warp_max(x_most), -FLT_MAX);
        for (int j = lane; j < p.entries; j += 32) {
          const int id = l.entry[j];
          bool again = id == 0;
          for (int i = 0; i < j; ++i) again |= l.entry[i] == id;
          if (!again) listed += ex2_approx_ftz((l.x[j] - x_most) * p.c);
        }
        listed = warp_sum(listed);
      }
      if (lane == 0) {
        l.at = at;
        l.terms = terms;
        l.all = all;
        l.norm = norm;
        l.listed_max = x_most;
        l.listed = listed;
      }
      return;
    }
  };
  // Ninth warp: sets or clears the bits of a lesson's entries in its part.
  auto punch = [&](const Lesson& l, unsigned* holes, bool set) {
    if (l.at < 0) return;
    const long long row = l.at / p.parts;
    const Range<T> r = range_of<T>(p.x, p.ld, p.n, row, (int)(l.at - row * p.parts), p.per);
    for (int j = lane; j < p.entries; j += 32) {
      const int id = l.entry[j];
      const long long e = (long long)id - 1 + r.off - (long long)r.v0 * V;
      if (id == 0 || e < 0 || e >= (long long)(r.v1 - r.v0) * V) continue;
      if (set) atomicOr(holes + (e >> 5), 1u << (e & 31));
      else holes[e >> 5] = 0;
    }
    __syncwarp();
  };

  if (warp == kWarps) {
    prepare(lessons[0]);
    __syncwarp();
    if constexpr (HOLES) punch(lessons[0], hole_store, true);
  }
  __syncthreads();
  for (int turn = 0;; ++turn) {
    const Lesson& l = lessons[turn % 3];
    if (l.at < 0) break;
    const long long row = l.at / p.parts;
    const int part = (int)(l.at - row * p.parts);
    const Range<T> r = range_of<T>(p.x, p.ld, p.n, row, part, p.per);
    const unsigned* holes = HOLES ? hole_store + (turn & 1) * hole_words : nullptr;
    float(&mine)[3][kWarps] = red[turn & 1];
    if (warp == kWarps) {
      // The row before this one has been summed, and its bits lie where the next row's go.
      unsigned* next_holes = hole_store + (~turn & 1) * hole_words;
      if constexpr (HOLES)
        if (turn > 0) punch(lessons[(turn + 2) % 3], next_holes, false);
      prepare(lessons[(turn + 1) % 3]);
      __syncwarp();
      if constexpr (HOLES) punch(lessons[(turn + 1) % 3], next_holes, true);
    } else {
      Sums<T, false> sums;
#pragma unroll 1
      for (int v = r.v0; v < r.v1; v += kTile) {
        uint4 q[kUnroll];
        load_tile(q, r, v, GRAD);
        if constexpr (HOLES)
#pragma unroll
          for (int u = 0; u < kUnroll; ++u) {
            const int of = v - r.v0 + u * kThreads + tid;
            const unsigned bits = of < r.v1 - r.v0 ? hole_bits<T>(holes, of) : 0u;
            if (bits) mask_holes<T>(q[u], bits);
          }
        (void)sums.add(q, p.c);
      }
      const float3 of_warp = sums.over_warp(p.c);
      if (lane == 0) {
        mine[0][warp] = of_warp.x;
        mine[1][warp] = of_warp.y;
      }
    }
    __syncthreads();
    if (warp == kWarps) continue;

    float top_max = red_max(mine[0]);
    const bool plain = Sums<T, false>::plain(top_max, p.c);
    if (!plain) {
      top_max = fmaxf(top_max, -FLT_MAX);
      const float2 of_warp = slow_sums(r, holes, top_max, p.c);
      if (lane == 0) mine[1][warp] = of_warp.x;
      bar_stream();
    }
    float sum = join(plain ? mine[0][lane & 7] : top_max, mine[1][lane & 7], 0.f, top_max, p.c).x;
    bool finish = true;
    if (p.parts > 1) {
      float* record = p.scratch + l.at * record_floats(0);
      if (tid == 0) {
        *reinterpret_cast<float4*>(record) = make_float4(top_max, sum, 0.f, 0.f);
        __threadfence();
        last = atomicInc(p.tickets + row, p.parts - 1) == (unsigned)p.parts - 1;
      }
      bar_stream();
      finish = last;
      if (finish) {
        __threadfence();
        const float4 one = lane < p.parts ? __ldcg(reinterpret_cast<const float4*>(p.scratch + (row * p.parts + lane) * record_floats(0)))
                                          : make_float4(-FLT_MAX, 0.f, 0.f, 0.f);
        top_max = warp_max(one.x);
        sum = join_parts(one, top_max, p.c).x;
      }
      bar_stream();  // `last` has been read
    }
    if (!finish) continue;
    float total = sum, rest = sum, all = 1.f, outside = 1.f;
    if constexpr (HOLES) {
      const float both = fmaxf(top_max, l.listed_max);
      rest = sum * ex2_approx_ftz((top_max - both) * p.c);
      total = rest + l.listed * ex2_approx_ftz((l.listed_max - both) * p.c);
      top_max = both;
      const double left = l.all > 1 ? 0 : 1 - l.all;
      all = (float)(l.all + left);
      outside = rest == 0.f ? all : (float)(l.all + left - left * ((double)total / (double)rest));
    }
    if (tid == 0) {
      const double log_total = log((double)total), lse = (double)top_max / (double)p.temperature + log_total;
      double loss = l.terms + l.all * lse;
      if constexpr (HOLES) {
        const double left = l.all > 1 ? 0 : 1 - l.all;
        if (left != 0) loss += left * (log(left) - (log((double)rest) - log_total));
      }
      // (lse, outside, all, norm) with teacher_lse; else outside and all are 1, and the norm keeps 48 bits: (lse, low part, -1, norm)
      const float high = (float)l.norm;
      p.loss[row] = (float)loss;
      reinterpret_cast<float4*>(p.saved)[row] = HOLES ? make_float4((float)lse, outside, all, high)
                                                      : make_float4((float)lse, (float)(l.norm - (double)high), -1.f, high);
    }
    if constexpr (GRAD) {  // one part
      T* dst = static_cast<T*>(p.dx) + row * p.ld_dx;
      const float g = p.d_loss[row] / p.temperature;
      const float lse2 = fmaf(top_max, p.c, log2f(total));
      stream_gradient<T, false>(r, dst, p.c, lse2, g * outside, 0.f);
      bar_stream();
      patch_entries<T>(dst, l.entry, l.q, p.entries, tid < p.entries ? l.x[tid] : 0.f, p.c, lse2, g, all, 0, p.n);
    }
  }
}

// ------------------------------------------------------------------ backward
struct Backward {
  const void* x;
  void* dx;
  long long ld, ld_dx;
  int n, rows, parts, per;
  float c, temperature;
  int* status;
  // log probabilities
  const void* tokens;
  int token_bits, top;
  const float *lse, *entropy, *d_logprobs, *d_entropy, *d_top;
  const int* top_ids;
  // distillation
  const void* ids;
  int id_bits, entries;
  const void* values;
  int values_dtype;
  const float *saved, *d_loss;
};

// Gradient of the log probabilities, the entropy and the alternatives of a row:
//   dx_v = 1/temperature [ sum of the gradients that meet at v - p_v (G + g_H (log p_v + H)) ],  G = the sum of all but g_H
// and of the distillation loss (DISTILL): g/temperature p_v outside, or g/temperature (all p_v - q_v) where the teacher lists v.
// A CTA takes part after part; the few places that a gradient meets directly are written behind the part's stream.
template <typename T, bool DISTILL>
__global__ void __launch_bounds__(kThreads, kBackwardPerSm) logits_backward_kernel(const __grid_constant__ Backward p) {
  constexpr int V = 16 / (int)sizeof(T);
  __shared__ int entry[kMaxEntries];
  __shared__ float weight[kMaxEntries];
  const int tid = threadIdx.x, lane = tid & 31;
  grid_dependency_sync();
  const long long items = (long long)p.rows * p.parts;
  for (long long at = blockIdx.x; at < items; at += gridDim.x) {
    const long long row = at / p.parts;
    const Range<T> r = range_of<T>(p.x, p.ld, p.n, row, (int)(at - row * p.parts), p.per);
    T* dst = static_cast<T*>(p.dx) + row * p.ld_dx;
    const long long lo = max(0ll, (long long)r.v0 * V - r.off), hi = min((long long)p.n, (long long)r.v1 * V - r.off);  // ids (lo, hi] lie in this part
    if constexpr (!DISTILL) {
      const long long token = p.tokens ? load_id(p.tokens, row, p.token_bits) : -1;
      const bool bad = p.tokens && (token < 0 || token > p.n);
      if (token == 0 || bad) {
        if (bad && tid == 0) atomicMax(p.status, DEV_BAD_INDEX);
        stream_zeros<T>(r, dst, tid, kThreads);
        continue;
      }
      const float g0 = p.d_logprobs ? p.d_logprobs[row] : 0.f, gh = p.d_entropy ? p.d_entropy[row] : 0.f;
      const float h = p.d_entropy ? p.entropy[row] : 0.f, lse2 = p.lse[row] * kLog2e;
      float all = lane < p.top ? p.d_top[row * p.top + lane] : 0.f;
      all = g0 + warp_sum(all);
      // entries: the alternatives, then the token
      const int entries = p.top + (p.d_logprobs ? 1 : 0);
      __syncthreads();
      if (tid < entries) {
        long long id = tid < p.top ? p.top_ids[row * p.top + tid] : token;
        if (id < 0 || id > p.n) {
          atomicMax(p.status, DEV_BAD_INDEX);
          id = 0;
        }
        entry[tid] = (int)id;
        weight[tid] = tid < p.top ? p.d_top[row * p.top + tid] : g0;
      }
      __syncthreads();
      const int id = tid < entries ? entry[tid] : 0;
      const float x = id > lo && id <= hi ? to_float(r.src[id - 1]) : 0.f;
      const float a = -(all + gh * h) / p.temperature, b = -gh * kLn2 / p.temperature;
      __syncthreads();  // dst may be the logits themselves
      if (p.d_entropy) stream_gradient<T, true>(r, dst, p.c, lse2, a, b);
      else stream_gradient<T, false>(r, dst, p.c, lse2, a, 0.f);
      __syncthreads();
      if (id > lo && id <= hi) {
        float g = 0.f;
        bool again = false;
        for (int i = 0; i < entries; ++i)
          if (entry[i] == id) {
            again |= i < tid;
            g += weight[i];
          }
        const float t = fmaf(x, p.c, -lse2);
        if (!again) dst[id - 1] = from_float<T>(g / p.temperature + ex2_approx_ftz(t) * fmaf(b, fmaxf(t, kLowest), a));
      }
    } else {
      const float4 saved = reinterpret_cast<const float4*>(p.saved)[row];
      if (saved.z == 0.f) {
        stream_zeros<T>(r, dst, tid, kThreads);
        continue;
      }
      const bool whole = saved.z < 0.f;  // the teacher's list is all of its distribution
      const float outside = whole ? 1.f : saved.y, all = whole ? 1.f : saved.z;
      const double norm = (double)saved.w + (whole ? (double)saved.y : 0.);
      const float g = p.d_loss[row] / p.temperature, lse2 = saved.x * kLog2e;
      __syncthreads();
      if (tid < p.entries) {
        long long id = load_id(p.ids, row * p.entries + tid, p.id_bits);
        if (id < 0 || id > p.n) {
          atomicMax(p.status, DEV_BAD_INDEX);
          id = 0;
        }
        entry[tid] = (int)id;
        weight[tid] = (float)exp((double)load_value(p.values, row * p.entries + tid, p.values_dtype) / (double)p.temperature - norm);
      }
      __syncthreads();
      const int id = tid < p.entries ? entry[tid] : 0;
      const float x = id > lo && id <= hi ? to_float(r.src[id - 1]) : 0.f;
      __syncthreads();  // dst may be the logits themselves
      stream_gradient<T, false>(r, dst, p.c, lse2, g * outside, 0.f);
      __syncthreads();
      patch_entries<T>(dst, entry, weight, p.entries, x, p.c, lse2, g, all, lo, hi);
    }
  }
}

// ------------------------------------------------------------------ host side
int elem_size(int dtype) { return dtype == CTB_F32 ? 4 : 2; }

int check_rows(const char* who, const void* x, int64_t V, int64_t T, int64_t ld, float temperature, int dtype) {
  if (dtype != CTB_F32 && dtype != CTB_F16 && dtype != CTB_BF16) return fail(CTB_BAD_ARG, "%s: dtype must be CTB_F32, CTB_F16 or CTB_BF16", who);
  if (V <= 0 || T < 0 || V > INT32_MAX - 64 || T > INT32_MAX) return fail(CTB_BAD_ARG, "%s: bad shape V=%lld T=%lld", who, (long long)V, (long long)T);
  if (ld < V) return fail(CTB_BAD_ARG, "%s: leading dimension smaller than V", who);
  if (!(temperature >= 1e-6f && temperature <= 1e6f)) return fail(CTB_BAD_ARG, "%s: temperature must lie between 1e-6 and 1e6", who);
  if (T == 0) return CTB_OK;
  if (!is_device_ptr(x)) return fail(CTB_BAD_ARG, "%s: logits is not a device pointer", who);
  if ((uintptr_t)x % elem_size(dtype)) return fail(CTB_BAD_ALIGN, "%s: logits must be aligned to their element size", who);
  return CTB_OK;
}
// d_logits may be the logits themselves; rows of the two must not overlap in any other way.
int check_gradient(const char* who, const void* x, void* dx, int64_t V, int64_t T, int64_t ld, int64_t ld_dx, int dtype) {
  const int64_t b = elem_size(dtype);
  if (ld_dx < V) return fail(CTB_BAD_ARG, "%s: leading dimension of d_logits smaller than V", who);
  if (!is_device_ptr(dx)) return fail(CTB_BAD_ARG, "%s: d_logits is not a device pointer", who);
  if ((uintptr_t)dx % b) return fail(CTB_BAD_ALIGN, "%s: d_logits must be aligned to their element size", who);
  return check_in_place(who, x, ld, dx, ld_dx, V, T, b);
}
#define CTB_CHECK_PTR(who, p)                                                                  \
  do {                                                                                         \
    if (!is_device_ptr(p)) return fail(CTB_BAD_ARG, "%s: argument %s is not a device pointer", who, #p); \
  } while (0)

// Parts of a row in a forward pass, and vectors per part: as many parts as bring work to every place for a CTA, none below one tile.
void cut_rows(int64_t places, int64_t rows, int64_t nvec, int64_t least, int most, int* parts, int* per) {
  int64_t n = rows >= places ? 1 : places / rows;
  n = std::min<int64_t>(n, (nvec + kTile - 1) / kTile);
  n = std::min<int64_t>(std::max(n, least), most);
  int64_t v = (nvec + n - 1) / n;
  v = (v + 31) / 32 * 32;
  *per = (int)v;
  *parts = (int)((nvec + v - 1) / v);
}

// Launches a forward kernel: rows whole or in parts.  `most` parts at most; holes: of the bits per element that a part may have in shared
// memory.
template <typename T, typename P>
int launch_forward(ctb_ctx* ctx, cudaStream_t st, P p, void (*kernel)(P), int threads, int per_sm, int top, bool whole, bool holes, const char* who) {
  constexpr int V = 16 / (int)sizeof(T);
  const int64_t nvec = (p.n + V - 1) / V + 1;  // a row that starts off a vector boundary touches one more
  int most = kMaxParts;
  if (p.rows > kTickets || whole) most = 1;
  else most = std::max<int>(1, std::min<int64_t>(most, kStreamScratchBytes / sizeof(float) / record_floats(top) / p.rows));
  if (top) most = std::min(most, kCand / top);
  cut_rows(per_sm * ctx->sm_count, p.rows, nvec, holes ? (nvec * V + kMostHoles - 1) / kMostHoles : 1, most, &p.parts, &p.per);
  auto go = [&] {
    const size_t smem = holes ? 2 * 4 * (((size_t)p.per * V + 31) / 32) : 0;
    if (holes) {
      if ((int64_t)p.per * V > kMostHoles + 1024)
        return fail(CTB_UNSUPPORTED, "%s: with teacher_lse, %d rows of %d elements are too long", who, p.rows, p.n);
      cudaError_t e = allow_smem(kernel, 2 * (kMostHoles + 1024) / 8);
      if (e != cudaSuccess) return cuda_fail(e, who);
    }
    int fit = per_sm;  // more shared memory may leave room for fewer
    if (holes) cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kernel, threads, smem);
    const int grid = (int)std::min<int64_t>((int64_t)p.rows * p.parts, (int64_t)std::max(1, std::min(fit, per_sm)) * ctx->sm_count);
    launch_kernel(kernel, grid, threads, smem, st, 0, p);
    CTB_CHECK_LAUNCH(who);
    return (int)CTB_OK;
  };
  if (p.parts > 1) {
    StreamScratch scratch(ctx, st);
    if (scratch.data) {
      p.scratch = scratch.data;
      p.tickets = scratch.tickets;
      return go();
    }
    p.parts = 1;
    p.per = (int)((nvec + 31) / 32 * 32);
  }
  return go();
}

template <typename T>
int launch_logprobs(ctb_ctx* ctx, cudaStream_t st, const Logprobs& p, const char* who) {
  return launch_forward<T>(ctx, st, p, p.top ? logprobs_kernel<T, true> : logprobs_kernel<T, false>, kThreads, p.top ? kTopPerSm : kPlainPerSm, p.top, false,
                           false, who);
}
template <typename T>
int launch_distill(ctb_ctx* ctx, cudaStream_t st, const Distill& p, const char* who) {
  const bool grad = p.dx, holes = p.teacher_lse;
  auto kernel = grad ? holes ? distill_kernel<T, true, true> : distill_kernel<T, true, false>
                     : holes ? distill_kernel<T, false, true> : distill_kernel<T, false, false>;
  return launch_forward<T>(ctx, st, p, kernel, kThreads + 32, kDistillPerSm, 0, grad, holes, who);
}
template <typename F>
int by_type(int dtype, F f) {
  if (dtype == CTB_F32) return f(float());
  if (dtype == CTB_F16) return f(__half());
  return f(__nv_bfloat16());
}

template <typename T, bool DISTILL>
int launch_backward(ctb_ctx* ctx, cudaStream_t st, Backward p, const char* who) {
  constexpr int V = 16 / (int)sizeof(T);
  const int64_t nvec = (p.n + V - 1) / V + 1;
  // parts of at most four tiles, and of one where that spreads the work over more SMs
  const int64_t tiles = p.rows * ((nvec + kTile - 1) / kTile);
  const int64_t want = tiles >= 16ll * ctx->sm_count ? 4 : 1;
  const int64_t parts = (nvec + want * kTile - 1) / (want * kTile);
  p.per = (int)(((nvec + parts - 1) / parts + 31) / 32 * 32);
  p.parts = (int)((nvec + p.per - 1) / p.per);
  const int grid = (int)std::min<int64_t>((int64_t)p.rows * p.parts, (int64_t)kBackwardPerSm * ctx->sm_count);
  launch_kernel(logits_backward_kernel<T, DISTILL>, grid, kThreads, 0, st, 0, p);
  CTB_CHECK_LAUNCH(who);
  return CTB_OK;
}
int check_bits(const char* who, int bits) {
  return bits == 32 || bits == 64 ? CTB_OK : fail(CTB_BAD_ARG, "%s: ids must be 32- or 64-bit integers", who);
}

int check_teacher(const char* who, const void* ids, int id_bits, const void* values, int values_dtype, int entries) {
  if (int s = check_bits(who, id_bits)) return s;
  if (entries < 1 || entries > kMaxEntries) return fail(CTB_UNSUPPORTED, "%s: a teacher's list has 1 to %d entries, not %d", who, kMaxEntries, entries);
  if (values_dtype != CTB_F32 && values_dtype != CTB_F16 && values_dtype != CTB_BF16)
    return fail(CTB_BAD_ARG, "%s: teacher_values must be CTB_F32, CTB_F16 or CTB_BF16", who);
  CTB_CHECK_PTR(who, ids);
  CTB_CHECK_PTR(who, values);
  return CTB_OK;
}

}  // namespace

extern "C" int ctb_token_logprobs(ctb_ctx* ctx, void* stream, const void* logits, const void* tokens, int token_bits, float* logprobs,
                                  float* entropy, float* lse, float* top_logprobs, int32_t* top_ids, int64_t V, int64_t T, int64_t ld,
                                  int top, float temperature, int dtype) {
  const char* who = "ctb_token_logprobs";
  CTB_CHECK_CTX(ctx);
  CurrentDevice current(ctx);
  if (int s = check_rows(who, logits, V, T, ld, temperature, dtype)) return s;
  if (top < 0 || top > kMaxTop || top > V)
    return fail(top > kMaxTop ? CTB_UNSUPPORTED : CTB_BAD_ARG, "%s: top must lie between 0 and min(%d, V), got %d", who, kMaxTop, top);
  if ((tokens != nullptr) != (logprobs != nullptr)) return fail(CTB_BAD_ARG, "%s: tokens and logprobs come together", who);
  if (int s = tokens ? check_bits(who, token_bits) : CTB_OK) return s;
  if (T == 0) return CTB_OK;
  if (tokens) CTB_CHECK_PTR(who, tokens);
  if (logprobs) CTB_CHECK_PTR(who, logprobs);
  if (entropy) CTB_CHECK_PTR(who, entropy);
  if (lse) CTB_CHECK_PTR(who, lse);
  if (top) {
    CTB_CHECK_PTR(who, top_logprobs);
    CTB_CHECK_PTR(who, top_ids);
  }
  Logprobs p = {};
  p.x = logits; p.ld = ld; p.n = (int)V; p.rows = (int)T;
  p.c = (float)(1.4426950408889634 / (double)temperature);
  p.temperature = temperature;
  p.status = ctx->dev_status;
  p.tokens = tokens; p.token_bits = token_bits; p.top = top;
  p.logprobs = logprobs; p.entropy = entropy; p.lse = lse; p.top_logprobs = top_logprobs; p.top_ids = top_ids;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_type(dtype, [&](auto t) { return launch_logprobs<decltype(t)>(ctx, st, p, who); });
}

extern "C" int ctb_token_logprobs_bwd(ctb_ctx* ctx, void* stream, void* d_logits, const void* logits, const void* tokens, int token_bits,
                                      const float* lse, const float* entropy, const float* d_logprobs, const float* d_entropy,
                                      const int32_t* top_ids, const float* d_top_logprobs, int64_t V, int64_t T, int64_t ld_out, int64_t ld,
                                      int top, float temperature, int dtype) {
  const char* who = "ctb_token_logprobs_bwd";
  CTB_CHECK_CTX(ctx);
  CurrentDevice current(ctx);
  if (int s = check_rows(who, logits, V, T, ld, temperature, dtype)) return s;
  if (!d_top_logprobs) top = 0;
  if (top < 0 || top > kMaxTop || top > V)
    return fail(top > kMaxTop ? CTB_UNSUPPORTED : CTB_BAD_ARG, "%s: top must lie between 0 and min(%d, V), got %d", who, kMaxTop, top);
  if (d_logprobs && !tokens) return fail(CTB_BAD_ARG, "%s: d_logprobs without tokens", who);
  if (int s = tokens ? check_bits(who, token_bits) : CTB_OK) return s;
  if (T == 0) return CTB_OK;
  if (int s = check_gradient(who, logits, d_logits, V, T, ld, ld_out, dtype)) return s;
  CTB_CHECK_PTR(who, lse);
  if (tokens) CTB_CHECK_PTR(who, tokens);
  if (d_logprobs) CTB_CHECK_PTR(who, d_logprobs);
  if (d_entropy) {
    CTB_CHECK_PTR(who, d_entropy);
    CTB_CHECK_PTR(who, entropy);
  }
  if (top) {
    CTB_CHECK_PTR(who, top_ids);
    CTB_CHECK_PTR(who, d_top_logprobs);
  }
  Backward p = {};
  p.x = logits; p.dx = d_logits; p.ld = ld; p.ld_dx = ld_out; p.n = (int)V; p.rows = (int)T;
  p.c = (float)(1.4426950408889634 / (double)temperature);
  p.temperature = temperature;
  p.status = ctx->dev_status;
  p.tokens = tokens; p.token_bits = token_bits; p.top = top;
  p.lse = lse; p.entropy = entropy; p.d_logprobs = d_logprobs; p.d_entropy = d_entropy; p.d_top = d_top_logprobs; p.top_ids = top_ids;
  return by_type(dtype, [&](auto t) { return launch_backward<decltype(t), false>(ctx, static_cast<cudaStream_t>(stream), p, who); });
}

static int distill_forward(const char* who, ctb_ctx* ctx, void* stream, const void* logits, const void* teacher_ids, int id_bits,
                           const void* teacher_values, int values_dtype, const float* teacher_lse, float* loss, float* saved,
                           const float* d_loss, void* d_logits, int64_t V, int64_t T, int64_t ld_out, int64_t ld, int entries,
                           float temperature, int dtype) {
  if (int s = check_rows(who, logits, V, T, ld, temperature, dtype)) return s;
  if (T == 0) return CTB_OK;
  if (int s = check_teacher(who, teacher_ids, id_bits, teacher_values, values_dtype, entries)) return s;
  if (teacher_lse) CTB_CHECK_PTR(who, teacher_lse);
  CTB_CHECK_PTR(who, loss);
  CTB_CHECK_PTR(who, saved);
  if ((uintptr_t)saved % 16) return fail(CTB_BAD_ALIGN, "%s: saved must be 16-byte aligned", who);
  Distill p = {};
  p.x = logits; p.ld = ld; p.n = (int)V; p.rows = (int)T;
  p.c = (float)(1.4426950408889634 / (double)temperature);
  p.temperature = temperature;
  p.status = ctx->dev_status;
  p.ids = teacher_ids; p.id_bits = id_bits; p.entries = entries; p.values = teacher_values; p.values_dtype = values_dtype;
  p.teacher_lse = teacher_lse; p.loss = loss; p.saved = saved;
  p.d_loss = d_loss; p.dx = d_logits; p.ld_dx = ld_out;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_type(dtype, [&](auto t) { return launch_distill<decltype(t)>(ctx, st, p, who); });
}

extern "C" int ctb_distill_fwd(ctb_ctx* ctx, void* stream, const void* logits, const void* teacher_ids, int id_bits,
                               const void* teacher_values, int values_dtype, const float* teacher_lse, float* loss, float* saved,
                               int64_t V, int64_t T, int64_t ld, int entries, float temperature, int dtype) {
  CTB_CHECK_CTX(ctx);
  CurrentDevice current(ctx);
  return distill_forward("ctb_distill_fwd", ctx, stream, logits, teacher_ids, id_bits, teacher_values, values_dtype, teacher_lse, loss, saved,
                         nullptr, nullptr, V, T, 0, ld, entries, temperature, dtype);
}

static int distill_backward(const char* who, ctb_ctx* ctx, void* stream, void* d_logits, const void* logits, const void* teacher_ids,
                            int id_bits, const void* teacher_values, int values_dtype, const float* saved, const float* d_loss, int64_t V,
                            int64_t T, int64_t ld_out, int64_t ld, int entries, float temperature, int dtype) {
  Backward p = {};
  p.x = logits; p.dx = d_logits; p.ld = ld; p.ld_dx = ld_out; p.n = (int)V; p.rows = (int)T;
  p.c = (float)(1.4426950408889634 / (double)temperature);
  p.temperature = temperature;
  p.status = ctx->dev_status;
  p.ids = teacher_ids; p.id_bits = id_bits; p.entries = entries; p.values = teacher_values; p.values_dtype = values_dtype;
  p.saved = saved; p.d_loss = d_loss;
  return by_type(dtype, [&](auto t) { return launch_backward<decltype(t), true>(ctx, static_cast<cudaStream_t>(stream), p, who); });
}

extern "C" int ctb_distill_bwd(ctb_ctx* ctx, void* stream, void* d_logits, const void* logits, const void* teacher_ids, int id_bits,
                               const void* teacher_values, int values_dtype, const float* saved, const float* d_loss, int64_t V, int64_t T,
                               int64_t ld_out, int64_t ld, int entries, float temperature, int dtype) {
  const char* who = "ctb_distill_bwd";
  CTB_CHECK_CTX(ctx);
  CurrentDevice current(ctx);
  if (int s = check_rows(who, logits, V, T, ld, temperature, dtype)) return s;
  if (T == 0) return CTB_OK;
  if (int s = check_gradient(who, logits, d_logits, V, T, ld, ld_out, dtype)) return s;
  if (int s = check_teacher(who, teacher_ids, id_bits, teacher_values, values_dtype, entries)) return s;
  CTB_CHECK_PTR(who, saved);
  CTB_CHECK_PTR(who, d_loss);
  if ((uintptr_t)saved % 16) return fail(CTB_BAD_ALIGN, "%s: saved must be 16-byte aligned", who);
  return distill_backward(who, ctx, stream, d_logits, logits, teacher_ids, id_bits, teacher_values, values_dtype, saved, d_loss, V, T, ld_out,
                          ld, entries, temperature, dtype);
}

extern "C" int ctb_distill_fwd_bwd(ctb_ctx* ctx, void* stream, void* d_logits, const void* logits, const void* teacher_ids, int id_bits,
                                   const void* teacher_values, int values_dtype, const float* teacher_lse, float* loss, float* saved,
                                   const float* d_loss, int64_t V, int64_t T, int64_t ld_out, int64_t ld, int entries, float temperature,
                                   int dtype) {
  const char* who = "ctb_distill_fwd_bwd";
  CTB_CHECK_CTX(ctx);
  CurrentDevice current(ctx);
  if (int s = check_rows(who, logits, V, T, ld, temperature, dtype)) return s;
  if (T == 0) return CTB_OK;
  if (int s = check_gradient(who, logits, d_logits, V, T, ld, ld_out, dtype)) return s;
  CTB_CHECK_PTR(who, d_loss);
    // One kernel where there are rows enough to give every SM its own, else the two halves, which cut rows into parts.
  if (T >= 2 * ctx->sm_count && !(teacher_lse && V > kMostHoles))
    return distill_forward(who, ctx, stream, logits, teacher_ids, id_bits, teacher_values, values_dtype, teacher_lse, loss, saved, d_loss,
                           d_logits, V, T, ld_out, ld, entries, temperature, dtype);
  if (int s = distill_forward(who, ctx, stream, logits, teacher_ids, id_bits, teacher_values, values_dtype, teacher_lse, loss, saved, nullptr,
                              nullptr, V, T, 0, ld, entries, temperature, dtype))
    return s;
  return distill_backward(who, ctx, stream, d_logits, logits, teacher_ids, id_bits, teacher_values, values_dtype, saved, d_loss, V, T, ld_out,
                          ld, entries, temperature, dtype);
}
