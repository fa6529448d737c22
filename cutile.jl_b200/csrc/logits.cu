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
#include <atomic>
#include <type_traits>

#include "ctx.h"
#include "ptx.cuh"
#include "rows.cuh"

using namespace ctb;
using namespace ctb_internal;

namespace {

constexpr int kThreads = 256;            // that stream
constexpr int kWarps = kThreads / 32;
constexpr int kAllThreads = kThreads + 32;  // and the clerk
constexpr int kUnroll = 4;               // vectors of 16 bytes per thread and tile
constexpr int kTile = kThreads * kUnroll;  // vectors
constexpr int kMaxTop = 32;
constexpr int kMaxEntries = kThreads;    // of a teacher's list
constexpr int kCand = 1024;
template <bool TOP>
constexpr int kLogprobsPerSm = TOP ? 3 : 5;  // CTAs on an SM
constexpr int kDistillPerSm = 4;
template <bool DISTILL>
constexpr int kBackwardPerSm = DISTILL ? 4 : 5;
constexpr int kMostHoles = 512 * 1024;  // elements of a part that have a bit (in two sets) in shared memory
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Exponents (base 2) are held above this where they are multiplied by their power, which is 0 there: 0 * -inf would be NaN.
constexpr float kLowest = -16384.f;
// A thread's reference follows its maximum only when an element is 2^kSlack above it.
constexpr float kSlack = 4.f;
constexpr float kFar = 1e30f;  // rows with a maximum beyond +-kFar (masked as a whole, or infinite) are summed in another way

__device__ __forceinline__ void bar_stream() { asm volatile("bar.sync 1, 256;" ::: "memory"); }      // the streaming threads
__device__ __forceinline__ void bar_row() { asm volatile("bar.sync 2, 288;" ::: "memory"); }         // and the clerk
static_assert(kThreads == 256, "the barriers name the numbers of threads");

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

// The k-th largest of the 64 group maxima; all streaming threads.
__device__ __forceinline__ float group_threshold(float mine, int k, Best& b) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float g = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
  g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 2));
  const int i = warp * 8 + (lane >> 2);
  if ((lane & 3) == 0) b.group[i] = g;
  bar_stream();
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
  bar_stream();
  return b.theta;
}

// Writes the best k of the n listed elements to out_*, in order; what is missing gets index -1.  All streaming threads; the list is
// complete and visible.
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
    bar_stream();
    n = b.count2;
  } else {
    bar_stream();
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
  bar_stream();
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
    bar_stream();
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
    bar_stream();
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
    bar_stream();
    for (int v = r.v0 + tid; v < r.v1; v += kThreads) {
      float f[V];
      unpack_row<T>(load_vec(r, v), f);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint32_t key = order_key(f[i]);
        if (f[i] == f[i] && r.has(v, i) && (key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1);
      }
    }
    bar_stream();
    if (tid == 0) {
      int bin = 255, above = 0;
      while (bin > 0 && above + hist[bin] < want) above += hist[bin--];
      b.bin = bin;
      b.above = above;
    }
    bar_stream();
    prefix |= (uint32_t)b.bin << shift;
    mask |= 255u << shift;
    want -= b.above;
    bar_stream();
  }
  const float kth = key_value(prefix);
  if (tid == 0) b.count = 0;
  bar_stream();
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
  bar_stream();
  return append_equal(r, kth, b.count, want, b);
}

// ------------------------------------------------------------------ sums of a row
// Exponents t = x c - m2, with c = log2(e) / temperature: one fused multiply-add gives them with one rounding, whatever the magnitude of x, and
// the rounding of c is that of a temperature, the same for the whole row.
//
// A thread's share of s = sum 2^t and w = sum 2^t t.  Its reference m2 follows its maximum, or t 2^t of a likely element would carry a
// rounding that the entropy, a difference of two such sums, shows.  Masked elements (-inf) make w NaN (0 * -inf); the tile's share is
// then taken again with exponents held above kLowest.  Valid for rows whose maximum is `plain`; the others take slow_sums.
template <typename T>
struct Sums {
  float m2 = 0.f, limit = -FLT_MAX;  // elements above limit move the reference
  uint32_t top = empty_row_vec<T>().x;
  Pair s = pair(0.f, 0.f), w = pair(0.f, 0.f);

  static __device__ __forceinline__ bool plain(float maximum) { return maximum <= kFar && maximum >= -kFar; }
  __device__ __forceinline__ void move(float t, float c) {
    const float x = fminf(fmaxf(t, -kFar), kFar), to = x * c, d = fmaxf(fminf(m2 - to, 0.f), kLowest), r = ex2_approx_ftz(d);
    const Pair rr = pair(r, r);
    w = mul2(rr, fma2(s, pair(d, d), w));
    s = mul2(rr, s);
    m2 = to;
    limit = x + kSlack / c;
  }
  // Returns the largest element of the tile.
  __device__ __forceinline__ float add(const uint4 (&q)[kUnroll], float c) {
    uint32_t all = 0;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t a = max_word<T>(max_word<T>(q[u].x, q[u].y), max_word<T>(q[u].z, q[u].w));
      all = u == 0 ? a : max_word<T>(all, a);
    }
    top = max_word<T>(top, all);
    const float most = word_max<T>(all);
    if (most > limit) move(most, c);
    const Pair cc = pair(c, c), minus = pair(-m2, -m2);
    Pair ts = pair(0.f, 0.f), tw = ts;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t word[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
      for (int i = 0; i < 8 / (int)sizeof(T); ++i) {
        const Pair t = fma2(vec_pair<T>(word, i), cc, minus), e = exp2_pair(t);
        ts = add2(ts, e);
        tw = fma2(e, t, tw);
      }
    }
    s = add2(s, ts);
    if (sum_of(tw) != sum_of(tw)) tw = pair((again(q[0], m2, c) + again(q[1], m2, c)) + (again(q[2], m2, c) + again(q[3], m2, c)), 0.f);
    w = add2(w, tw);
    return most;
  }
  static __device__ __noinline__ float again(uint4 q, float m2, float c) {
    static_assert(kUnroll == 4, "add() calls this for each vector of a tile");
    float f[16 / sizeof(T)], a = 0.f;
    unpack_row<T>(q, f);
#pragma unroll
    for (int i = 0; i < 16 / (int)sizeof(T); ++i) {
      const float t = fmaf(f[i], c, -m2);
      a = fmaf(ex2_approx_ftz(t), fmaxf(t, kLowest), a);
    }
    return a;
  }
  // One element more.
  __device__ __forceinline__ void add_one(float x, float c) {
    const T e = from_float<T>(x);
    top = max_word<T>(top, sizeof(T) == 4 ? __float_as_uint(x) : 0x10001u * *reinterpret_cast<const unsigned short*>(&e));
    if (x > limit) move(x, c);
    const float t = fmaf(x, c, -m2), v = ex2_approx_ftz(t);
    s = add2(s, pair(v, 0.f));
    w = add2(w, pair(v * fmaxf(t, kLowest), 0.f));
  }
  // The warp's (maximum, s, w), the sums relative to that maximum.
  __device__ __forceinline__ float3 over_warp(float c) const {
    const float most = warp_max(word_max<T>(top)), to = fminf(fmaxf(most, -kFar), kFar);
    const float d = fminf(fmaf(-to, c, m2), 1.f), r = ex2_approx_ftz(d), sum = sum_of(s);  // a thread without elements has m2 = sum = 0
    return make_float3(most, warp_sum(sum * r), warp_sum(r * fmaf(sum, fmaxf(d, kLowest), sum_of(w))));
  }
};

// s alone, for the warp: the reference is the largest element of the warp's first tile that has one above -inf, and stays.  What is
// more than 2^127 above it, or all of it below f32, shows as a sum that is not finite and positive; the row then takes slow_sums.
template <typename T>
struct LeanSums {
  float ref = -INFINITY, m2 = 0.f;  // m2 = ref c
  Pair s = pair(0.f, 0.f);

  __device__ __forceinline__ void add(const uint4 (&q)[kUnroll], float c) {
    if (ref == -INFINITY) {  // the same in the whole warp
      float most = -INFINITY;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        most = max_nan(most, max_nan(max_nan(word_nan<T>(q[u].x), word_nan<T>(q[u].y)), max_nan(word_nan<T>(q[u].z), word_nan<T>(q[u].w))));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (most == -INFINITY) return;
      ref = fminf(fmaxf(most, -kFar), kFar);  // of NaN: any number, the sum will be NaN
      m2 = ref * c;
    }
    const Pair cc = pair(c, c), minus = pair(-m2, -m2);
    Pair ts = pair(0.f, 0.f);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t word[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
      for (int i = 0; i < 8 / (int)sizeof(T); ++i) ts = add2(ts, exp2_pair(fma2(vec_pair<T>(word, i), cc, minus)));
    }
    s = add2(s, ts);
  }
  // One element more of each lane (-inf: none).
  __device__ __forceinline__ void add_one(float x, float c) {
    uint4 q[kUnroll] = {empty_row_vec<T>(), empty_row_vec<T>(), empty_row_vec<T>(), empty_row_vec<T>()};
    const T e = from_float<T>(x);
    q[0].x = sizeof(T) == 4 ? __float_as_uint(x) : (q[0].x & 0xffff0000u) | *reinterpret_cast<const unsigned short*>(&e);
    add(q, c);
  }
  // The warp's (reference, s), s relative to that reference.
  __device__ __forceinline__ float2 over_warp(float c) const {
    const float sum = warp_sum(sum_of(s));
    return make_float2(ref, ref == -INFINITY ? 0.f : sum * ex2_approx_ftz(fmaf(-ref, c, m2)));
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

// (maximum, s, w) of a range whose sums above are not valid, relative to its maximum, from differences (x - maximum); without the elements
// that the `entries` ids name.  All streaming threads; `red` is theirs.
template <typename T>
__device__ __noinline__ float3 slow_sums(const Range<T>& r, const int* entry, int entries, float c, float (&red)[3][kWarps]) {
  constexpr int V = 16 / (int)sizeof(T);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float most = -FLT_MAX, s = 0.f, w = 0.f;
  for (int pass = 0; pass < 2; ++pass) {
    for (int v = r.v0 + tid; v < r.v1; v += kThreads) {
      uint4 q = load_vec(r, v);
      unsigned bits = 0;
      for (int j = 0; j < entries; ++j) {
        const int i = entry[j] - 1 + r.off - v * V;
        if (entry[j] && i >= 0 && i < V) bits |= 1u << i;
      }
      if (bits) mask_holes<T>(q, bits);
      float f[V];
      unpack_row<T>(q, f);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (pass == 0) {
          most = fmaxf(most, f[i]);
        } else {
          const float t = (f[i] - most) * c, e = ex2_approx_ftz(t);
          s += e;
          w = fmaf(e, fmaxf(t, kLowest), w);
        }
      }
    }
    bar_stream();  // red has been read
    if (pass == 0) {
      most = warp_max(most);
      if (lane == 0) red[0][warp] = most;
    } else {
      s = warp_sum(s);
      w = warp_sum(w);
      if (lane == 0) {
        red[1][warp] = s;
        red[2][warp] = w;
      }
    }
    bar_stream();
    if (pass == 0) {
      for (int i = 0; i < kWarps; ++i) most = fmaxf(most, red[0][i]);
    }
  }
  s = w = 0.f;
  for (int i = 0; i < kWarps; ++i) {
    s += red[1][i];
    w += red[2][i];
  }
  return make_float3(most, s, w);
}

// (s, w) of up to 8 or 16 sets of sums, held by lanes i, i + 8 (16), ..., each relative to a maximum of its own, relative to `most`.
// apart: of the set's maximum below `most`, in units of log2.
template <int OF>
__device__ __forceinline__ float2 join(float apart, float s, float w) {
  const float r = ex2_approx_ftz(apart);
  float a = s * r, b = r * fmaf(s, fmaxf(apart, kLowest), w);
#pragma unroll
  for (int o = OF / 2; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  return make_float2(a, b);
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
// What the kernels below have in common: the logits, and how their rows are cut.
struct Rows {
  const void* x;
  long long ld;
  int n, rows, parts, per;  // per: vectors of a part
  int cluster;              // the parts of a row are the CTAs of a cluster, which meet; else they have nothing to do with each other
  float c, temperature;     // c = log2(e) / temperature
  int* status;
};
// The (row, part) of an item.
__device__ __forceinline__ long long row_of(const Rows& p, long long item) { return p.cluster ? item : item / p.parts; }
__device__ __forceinline__ int part_of(const Rows& p, long long item) {
  return p.cluster ? (int)cluster_ctarank() : (int)(item - item / p.parts * p.parts);
}
template <typename T>
__device__ __forceinline__ Range<T> range_of(const Rows& p, long long item) {
  constexpr int V = 16 / (int)sizeof(T);
  Range<T> r;
  r.src = static_cast<const T*>(p.x) + row_of(p, item) * p.ld;
  r.off = (int)(((uintptr_t)r.src & 15) / sizeof(T));
  r.n = p.n;
  const int nvec = (r.off + p.n + V - 1) / V;
  r.v0 = (int)min((long long)nvec, (long long)part_of(p, item) * p.per);
  r.v1 = min(nvec, r.v0 + p.per);
  return r;
}

// ------------------------------------------------------------------ rows through a CTA
// A CTA takes row after row, or parts of rows, with two roles:
//   stream   eight warps read the row, four vectors of 16 bytes per thread at a time; five CTAs on an SM keep HBM busy while one of them
//            computes or ends a row (a ring of bulk copies ahead of the warps was no faster: what it saved in waiting it took in
//            instructions, 10.7 per element instead of 7.4, for its barriers)
//   clerk    a warp prepares the next row: whether it is padding, what the operator needs besides its logits (loads that
//            depend on loads, f64 exponentials), so that a row ends with one barrier and a handful of operations
// The row's first and last elements, up to a vector boundary, are loaded one by one.
//
// Where a row is cut into parts whose sums have to meet, the parts are the CTAs of a cluster: they send their sums to each other's
// shared memory.  Few rows are spread over the GPU that way.
constexpr int kMaxCluster = 16;

// Whole vectors of a range, [a, b), and the elements before and behind them.
struct Inner {
  int a, b, head, tail;
  template <typename T>
  __device__ __forceinline__ explicit Inner(const Range<T>& r) {
    constexpr int V = Range<T>::V;
    const int nvec = (r.off + r.n + V - 1) / V;
    a = r.v0;
    head = 0;
    if (r.off > 0 && r.v0 == 0 && r.v1 > 0) {
      a = 1;
      head = min(r.n, V - r.off);
    }
    b = r.v1;
    if (r.v1 == nvec && nvec * V - r.off > r.n) --b;
    b = max(a, b);
    tail = r.v1 == nvec && r.v1 > r.v0 ? r.n - (b * V - r.off) : 0;
    if (tail < 0) tail = 0;  // all of the row lies before its first vector boundary
  }
};
// The element that thread tid < 16 holds: of the head (tid < 8) or the tail, or -1.
template <typename T>
__device__ __forceinline__ int edge_index(const Range<T>& r, const Inner& in, int tid) {
  if (tid < in.head) return tid;
  if (tid >= 8 && tid - 8 < in.tail) return r.n - in.tail + tid - 8;
  return -1;
}

// A streaming thread's vectors of the tile at v; beyond the range -inf.  KEEP: the row is read again, from L2.
template <typename T, bool KEEP = false>
__device__ __forceinline__ void load_tile(uint4 (&q)[kUnroll], const Range<T>& r, const Inner& in, int v) {
  const int tid = threadIdx.x;
  const uint4* p = r.at(v) + tid;
  if (v + kTile <= in.b) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) q[u] = KEEP ? __ldcg(p + u * kThreads) : __ldcs(p + u * kThreads);
  } else {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) q[u] = v + tid + u * kThreads < in.b ? (KEEP ? __ldcg(p + u * kThreads) : __ldcs(p + u * kThreads)) : empty_row_vec<T>();
  }
}

// Sums of a row's parts in the shared memory of every CTA of the cluster, for even and odd meetings.  A peer sends to the meeting after
// the next one only when this CTA has sent to the next, that is, has read this one.
struct Meeting {
  float4 part[2][kMaxCluster];
  uint64_t bar[2];
  volatile int abort;  // a wait ran out: no further message or wait
};

// The frame of the kernels below.  Op has
//   Lesson                     what the clerk prepares; .at is the item, -1 behind the last one; .zero: its gradient is 0 and its logits are not read
//   prepare(lesson, item)      the clerk: false for padding whose results it has written
//   before(turn, lessons), after(turn, lessons)             the clerk, before and after a lesson is made
//   stream(turn, lesson, range, inner)                      the streaming threads, up to the row's barrier
//   finish(turn, lesson, range, inner)                      the streaming threads behind it
template <typename T, typename Op>
__device__ __forceinline__ void run_rows(const Rows& p, Op& op, typename Op::Lesson* lessons, Meeting* meeting) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool cluster = p.cluster && p.parts > 1;
  if (cluster) {
    if (tid == 0) {
      for (int i = 0; i < 2; ++i) mbar_init(&meeting->bar[i], 1);
      meeting->abort = 0;
      fence_mbar_init();
    }
    __syncthreads();
    cluster_arrive();  // the peers' shared memory and barriers exist
    cluster_wait();
  } else {
    __syncthreads();
  }
  grid_dependency_sync();
  const long long items = p.cluster ? p.rows : (long long)p.rows * p.parts;
  if (warp == kWarps) {
    const int step = p.cluster ? gridDim.x / p.parts : gridDim.x;
    long long at = (long long)(p.cluster ? blockIdx.x / p.parts : blockIdx.x) - step;
    for (int turn = -1;; ++turn) {  // while row `turn` streams, the next one is prepared
      if (turn >= 0 && lessons[turn % 3].at < 0) break;
      typename Op::Lesson& l = lessons[(turn + 1) % 3];
      op.before(turn + 1, lessons);
      __syncwarp();
      if (lane == 0) l.zero = false;
      do at += step;
      while (at < items && !op.prepare(l, at));
      if (lane == 0) l.at = at < items ? at : -1;
      __syncwarp();
      op.after(turn + 1, lessons);
      __syncwarp();
      bar_row();
    }
  } else {
    bar_row();
    for (int turn = 0;; ++turn) {
      const typename Op::Lesson& l = lessons[turn % 3];
      if (l.at < 0) break;
      const Range<T> r = range_of<T>(p, l.at);
      const Inner in(r);
      op.stream(turn, l, r, in);
      bar_row();
      op.finish(turn, l, r, in);
    }
  }
  if (cluster) {  // no peer sends any more, and what they have sent is there unless a wait ran out
    __syncthreads();
    cluster_arrive_relaxed();
    cluster_wait();
    let_copies_land(&meeting->abort);
  }
}

// Sends (maximum, s, w) of this CTA's part to its row's CTAs; warp 0.  extra: bytes that come besides.
__device__ __forceinline__ void send_part(const Rows& p, Meeting& m, int turn, float3 mine, uint32_t extra) {
  const int lane = threadIdx.x & 31;
  if (m.abort) return;
  __syncwarp();
  if (lane == 0) mbar_expect_tx(&m.bar[turn & 1], p.parts * (uint32_t)sizeof(float4) + extra);
  if (lane < p.parts) send4_to_cta(&m.part[turn & 1][cluster_ctarank()], make_float4(mine.x, mine.y, mine.z, 0.f), &m.bar[turn & 1], lane);
}
// Waits for all parts; a warp.
__device__ __forceinline__ void await_parts(const Rows& p, Meeting& m, int turn) {
  if (m.abort) return;
  __syncwarp();
  if ((threadIdx.x & 31) == 0) (void)mbar_wait<true>(&m.bar[turn & 1], (turn >> 1) & 1, p.status, DEV_TIMEOUT_TMA, &m.abort);
  __syncwarp();
  (void)mbar_try_wait<true>(&m.bar[turn & 1], (turn >> 1) & 1);  // every lane acquires what the peers sent
}
// (maximum, s, w) of all parts, in all lanes of a warp.
__device__ __forceinline__ float3 join_parts(const Rows& p, const Meeting& m, int turn) {
  const int i = threadIdx.x & (kMaxCluster - 1);
  const float4 one = i < p.parts ? m.part[turn & 1][i] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
  float most = one.x;
#pragma unroll
  for (int o = kMaxCluster / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  most = fmaxf(most, -FLT_MAX);
  const float2 sum = join<kMaxCluster>((one.x - most) * p.c, one.y, one.z);
  return make_float3(most, sum.x, sum.y);
}

// ------------------------------------------------------------------ log probabilities, forward
struct Logprobs : Rows {
  const void* tokens;
  int token_bits, top;
  float *logprobs, *entropy, *lse, *top_logprobs;
  int* top_ids;
};
struct LogprobsLesson {
  long long at, token;
  float x;  // the token's logit
  bool zero;
};
struct Lists {  // of the parts, in the first CTA of a row
  float2 entry[2][kMaxCluster * kMaxTop];
};

template <typename T, bool TOP>
struct LogprobsOp {
  using Lesson = LogprobsLesson;
  const Logprobs& p;
  Best& best;
  Lists& lists;
  float (&red)[2][3][kWarps];
  Meeting& meeting;
  float theta;

  __device__ __forceinline__ void before(int, const Lesson*) {}
  __device__ __forceinline__ void after(int, const Lesson*) {}
  __device__ __forceinline__ bool prepare(Lesson& l, long long row) {
    const int lane = threadIdx.x & 31;
    const long long token = p.tokens ? load_id(p.tokens, row, p.token_bits) : -1;
    if (token != 0) {
      if (lane == 0) {
        l.token = token;
        l.x = token > 0 && token <= p.n ? to_float((static_cast<const T*>(p.x) + row * p.ld)[token - 1]) : 0.f;
      }
      return true;
    }
    if (p.parts == 1 || cluster_ctarank() == 0) {
      if (lane == 0) {
        if (p.logprobs) p.logprobs[row] = 0.f;
        if (p.entropy) p.entropy[row] = 0.f;
        if (p.lse) p.lse[row] = 0.f;
      }
      if (TOP && lane < p.top) {
        p.top_logprobs[row * p.top + lane] = 0.f;
        p.top_ids[row * p.top + lane] = 0;
      }
    }
    return false;
  }

  __device__ __forceinline__ void list(float x, int index) {
    if (x > theta) {
      const int pos = atomicAdd(&best.count, 1);
      if (pos < kCand) {
        best.value[pos] = x;
        best.index[pos] = index;
      }
    }
  }
  __device__ __forceinline__ void stream(int turn, const Lesson&, const Range<T>& r, const Inner& in) {
    constexpr int V = Range<T>::V;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, edge = edge_index(r, in, tid);
    const float x = edge >= 0 ? to_float(r.src[edge]) : 0.f;
    Sums<T> sums;
    if constexpr (TOP) {
      if (tid == 0) best.count = 0;  // ahead of the barriers of the first threshold
      theta = -INFINITY;
      if (edge >= 0 && tid < 8) sums.add_one(x, p.c);
    }
    int tile = 0;
#pragma unroll 1
    for (int v = in.a; v < in.b || (TOP && tile == 0); v += kTile, ++tile) {
      uint4 q[kUnroll];
      float most = -INFINITY;
      if (v < in.b) {
        load_tile(q, r, in, v);
        most = sums.add(q, p.c);
      }
      if constexpr (TOP) {
        if (tile == 0) {
          theta = group_threshold(word_max<T>(sums.top), p.top, best);
          if (edge >= 0 && tid < 8) list(x, edge);
        }
        if (most > theta) {
#pragma unroll
          for (int u = 0; u < kUnroll; ++u) {
            float f[V];
            unpack_row<T>(q[u], f);
            const int e0 = (v + u * kThreads + tid) * V - r.off;
#pragma unroll
            for (int i = 0; i < V; ++i) list(f[i], e0 + i);
          }
        }
        if (tile > 0 && (tile & (tile + 1)) == 0 && v + kTile < in.b) theta = group_threshold(word_max<T>(sums.top), p.top, best);
      }
    }
    if (edge >= 0 && (!TOP || tid >= 8)) {
      sums.add_one(x, p.c);
      if constexpr (TOP) list(x, edge);
    }
    const float3 of_warp = sums.over_warp(p.c);
    if (lane == 0) {
      red[turn & 1][0][warp] = of_warp.x;
      red[turn & 1][1][warp] = of_warp.y;
      red[turn & 1][2][warp] = of_warp.z;
    }
  }
  __device__ __forceinline__ void finish(int turn, const Lesson& l, const Range<T>& r, const Inner& in) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float(&mine)[3][kWarps] = red[turn & 1];
    const long long row = l.at;
    float3 sum = make_float3(red_max(mine[0]), 0.f, 0.f);
    if (!Sums<T>::plain(sum.x)) {
      sum = slow_sums(r, nullptr, 0, p.c, mine);
    } else if (warp == 0) {
      const float2 s = join<kWarps>((mine[0][lane & 7] - sum.x) * p.c, mine[1][lane & 7], mine[2][lane & 7]);
      sum = make_float3(sum.x, s.x, s.y);
    }
    if constexpr (TOP) {
      int n = best.count;
      if (n > kCand) {
        n = radix_list(r, p.top, best);
      } else if (n < p.top) {
        // theta of the first tile: with fewer than k above it, it is also the last one
        Range<T> first = r;
        first.v1 = min(r.v1, in.a + kTile);
        n = append_equal(first, theta, n, p.top - n, best);
      }
      select_list(n, p.top, best);
    }
    if (p.parts > 1) {
      const int rank = cluster_ctarank();
      if (warp == 0) {
        send_part(p, meeting, turn, sum, TOP && rank == 0 ? p.parts * p.top * (uint32_t)sizeof(float2) : 0);
        if (TOP && lane < p.top && !meeting.abort)
          send_to_cta(&lists.entry[turn & 1][rank * p.top + lane], best.out_value[lane], __int_as_float(best.out_index[lane]),
                      &meeting.bar[turn & 1], 0);
      }
      if (warp == 0 || (TOP && rank == 0)) {
        await_parts(p, meeting, turn);
        sum = join_parts(p, meeting, turn);
      }
      if (rank != 0) return;
      if constexpr (TOP) {
        if (tid == 0) best.count = 0;
        bar_stream();
        for (int i = tid; i < p.parts * p.top; i += kThreads) {
          const float2 e = lists.entry[turn & 1][i];
          const int id = __float_as_int(e.y);
          if (id >= 0) {
            const int pos = atomicAdd(&best.count, 1);
            best.value[pos] = e.x;
            best.index[pos] = id;
          }
        }
        bar_stream();
        select_list(best.count, p.top, best);
      }
    }
    if (warp == 0) {
      const float log_sum = logf(sum.y);
      if (lane == 0) {
        if (p.lse) p.lse[row] = sum.x / p.temperature + log_sum;
        if (p.entropy) p.entropy[row] = log_sum - kLn2 * (sum.z / sum.y);
        if (p.logprobs) {
          const bool bad = l.token < 0 || l.token > p.n;
          if (bad) atomicMax(p.status, DEV_BAD_INDEX);
          p.logprobs[row] = bad ? NAN : (l.x - sum.x) / p.temperature - log_sum;
        }
      }
      if (TOP && lane < p.top) {
        const int id = best.out_index[lane];
        p.top_logprobs[row * p.top + lane] = id >= 0 ? (best.out_value[lane] - sum.x) / p.temperature - log_sum : NAN;
        p.top_ids[row * p.top + lane] = id + 1;
      }
    }
  }
};
template <typename T, bool TOP>
__global__ void __launch_bounds__(kAllThreads, kLogprobsPerSm<TOP>) logprobs_kernel(const __grid_constant__ Logprobs p) {
  __shared__ Meeting meeting;
  __shared__ LogprobsLesson lessons[3];
  __shared__ float red[2][3][kWarps];
  __shared__ typename std::conditional<TOP, Best, int>::type best;
  __shared__ typename std::conditional<TOP, Lists, int>::type lists;
  LogprobsOp<T, TOP> op{p, reinterpret_cast<Best&>(best), reinterpret_cast<Lists&>(lists), red, meeting, 0.f};
  run_rows<T>(p, op, lessons, &meeting);
}

// ------------------------------------------------------------------ gradients
// d = p (a + b t), t = log2 p, over a range.
template <typename T, bool ENTROPY>
__device__ __forceinline__ void stream_gradient(const Range<T>& r, const Inner& in, T* dst, float c, float lse2, float a, float b) {
  const int tid = threadIdx.x, edge = edge_index(r, in, tid);
  const bool aligned = ((uintptr_t)(dst - r.off) & 15) == 0;
  const Pair cc = pair(c, c), minus = pair(-lse2, -lse2), aa = pair(a, a), bb = pair(b, b);
  const float x = edge >= 0 ? to_float(r.src[edge]) : 0.f;
#pragma unroll 1
  for (int v = in.a; v < in.b; v += kTile) {
    uint4 q[kUnroll];
    load_tile(q, r, in, v);
    uint4* to = reinterpret_cast<uint4*>(dst - r.off) + v + tid;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      uint32_t word[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
      for (int i = 0; i < 8 / (int)sizeof(T); ++i) {
        const Pair t = fma2(vec_pair<T>(word, i), cc, minus), e = exp2_pair(t);
        if constexpr (ENTROPY) {
          const float2 h = halves(t);
          put_pair<T>(word, i, mul2(e, fma2(bb, pair(fmaxf(h.x, kLowest), fmaxf(h.y, kLowest)), aa)));
        } else {
          put_pair<T>(word, i, mul2(e, aa));
        }
      }
      const uint4 d = make_uint4(word[0], word[1], word[2], word[3]);
      if (v + u * kThreads + tid < in.b) {
        if (aligned) __stcs(to + u * kThreads, d);
        else store_edge<T>(dst, r.off, r.n, v + u * kThreads + tid, d);
      }
    }
  }
  if (edge >= 0) {
    const float t = fmaf(x, c, -lse2), e = ex2_approx_ftz(t);
    dst[edge] = from_float<T>(ENTROPY ? e * fmaf(b, fmaxf(t, kLowest), a) : e * a);
  }
}
// Zeros over a range, by the streaming threads.
template <typename T>
__device__ __noinline__ void stream_zeros(const Range<T>& r, T* dst) {
  const bool aligned = ((uintptr_t)(dst - r.off) & 15) == 0;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int v = r.v0 + threadIdx.x; v < r.v1; v += kThreads) {
    if (aligned && r.inside(v, 1)) __stcs(reinterpret_cast<uint4*>(dst - r.off) + v, zero);
    else store_edge<T>(dst, r.off, r.n, v, zero);
  }
}

// Id of an entry if it lies in this range, else 0.
template <typename T>
__device__ __forceinline__ int in_range(const Range<T>& r, long long id) {
  const long long v = (id - 1 + r.off) / Range<T>::V;
  return id > 0 && v >= r.v0 && v < r.v1 ? (int)id : 0;
}
// Gradient at what a teacher lists: g (all p - sum of the q of this id), once per id.  Thread j has entry j; 0: unused or in another part.
template <typename T>
__device__ __forceinline__ void patch_entries(const Range<T>& r, T* dst, const int* entry, const float* q, const float* x, int entries, float c,
                                              float lse2, float g, float all) {
  const int j = threadIdx.x;
  if (j >= entries) return;
  const int id = entry[j];
  if (!in_range(r, id)) return;
  float sum = 0.f;
  for (int i = 0; i < entries; ++i)
    if (entry[i] == id) {
      if (i < j) return;
      sum += q[i];
    }
  dst[id - 1] = from_float<T>(g * (all * ex2_approx_ftz(fmaf(x[j], c, -lse2)) - sum));
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
struct DistillLesson {
  long long at;
  double terms, all, norm;   // sum q (log q - z), sum q
  float listed_max, listed;  // what the student gives to the listed ids, each once: maximum, sum of powers relative to it
  float g;                   // upstream gradient / temperature
  bool zero;
  int entry[kMaxEntries];    // ids, 0: unused
  float q[kMaxEntries], x[kMaxEntries];
};

// HOLES: teacher_lse is given; what the teacher lists is left out of the row's sum by a bit per element and added apart, since the rest's
// probability from a difference would lose all digits where it is small.  GRAD: the row is read a second time, out of L2, for the
// gradient.
template <typename T, bool GRAD, bool HOLES>
struct DistillOp {
  using Lesson = DistillLesson;
  static constexpr int V = Range<T>::V;
  const Distill& p;
  double (&power)[kMaxEntries];  // the clerk's
  float (&red)[2][3][kWarps];
  unsigned* holes;  // two sets of hole_words
  int hole_words;
  Meeting& meeting;
  int meetings;

  __device__ __forceinline__ bool prepare(Lesson& l, long long row) {
    const int lane = threadIdx.x & 31;
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
      if ((p.parts == 1 || cluster_ctarank() == 0) && lane == 0) {
        if (bad) atomicMax(p.status, DEV_BAD_INDEX);
        p.loss[row] = bad ? NAN : 0.f;
        reinterpret_cast<float4*>(p.saved)[row] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      if (GRAD && lane == 0) l.zero = true;
      return GRAD;
    }
    float x_most = -INFINITY;
    for (int j = lane; j < p.entries; j += 32) {
      const int id = l.entry[j];
      const float x = id ? to_float(src[id - 1]) : -INFINITY;
      l.x[j] = x;
      x_most = fmaxf(x_most, x);
    }
    double norm;
    if constexpr (HOLES) {
      norm = p.teacher_lse[row];
    } else {
      most = max_lanes(most);
      double sum = 0;
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
      __syncwarp();
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
      l.terms = terms;
      l.all = all;
      l.norm = norm;
      l.listed_max = x_most;
      l.listed = listed;
      if constexpr (GRAD) l.g = p.d_loss[row] / p.temperature;
    }
    return true;
  }
  // Sets or clears the bits of a lesson's entries in its part.
  __device__ __forceinline__ void punch(const Lesson& l, unsigned* set, bool on) {
    if (l.at < 0 || l.zero) return;
    const Range<T> r = range_of<T>(p, l.at);
    for (int j = threadIdx.x & 31; j < p.entries; j += 32) {
      const int id = in_range(r, l.entry[j]);
      if (id == 0) continue;
      const long long e = (long long)id - 1 + r.off - (long long)r.v0 * V;
      if (on) atomicOr(set + (e >> 5), 1u << (e & 31));
      else set[e >> 5] = 0;
    }
    __syncwarp();
  }
  // The row two before has been summed: its bits lie where the next row's go.
  __device__ __forceinline__ void before(int turn, const Lesson* lessons) {
    if constexpr (HOLES)
      if (turn >= 2) punch(lessons[(turn + 1) % 3], holes + (turn & 1) * hole_words, false);
  }
  __device__ __forceinline__ void after(int turn, const Lesson* lessons) {
    if constexpr (HOLES) punch(lessons[turn % 3], holes + (turn & 1) * hole_words, true);
  }

  __device__ __forceinline__ void stream(int turn, const Lesson& l, const Range<T>& r, const Inner& in) {
    if (GRAD && l.zero) return;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, edge = edge_index(r, in, tid);
    const unsigned* mine = holes + (turn & 1) * hole_words;
    float x = edge >= 0 ? to_float(r.src[edge]) : -INFINITY;
    LeanSums<T> sums;
#pragma unroll 1
    for (int v = in.a; v < in.b; v += kTile) {
      uint4 q[kUnroll];
      load_tile<T, GRAD>(q, r, in, v);
      if constexpr (HOLES)
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int of = v + u * kThreads + tid;
          const unsigned bits = of < in.b ? hole_bits<T>(mine, of - r.v0) : 0u;
          if (bits) mask_holes<T>(q[u], bits);
        }
      sums.add(q, p.c);
    }
    if (warp == 0 && in.head + in.tail > 0) {
      if (HOLES && edge >= 0) {
        const int e = edge + r.off - r.v0 * V;
        if (mine[e >> 5] >> (e & 31) & 1) x = -INFINITY;
      }
      sums.add_one(x, p.c);
    }
    const float2 of_warp = sums.over_warp(p.c);
    if (lane == 0) {
      red[turn & 1][0][warp] = of_warp.x;
      red[turn & 1][1][warp] = of_warp.y;
    }
  }
  __device__ __forceinline__ void finish(int turn, const Lesson& l, const Range<T>& r, const Inner& in) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long row = l.at;
    if (GRAD && l.zero) {
      stream_zeros<T>(r, static_cast<T*>(p.dx) + row * p.ld_dx);
      return;
    }
    float(&mine)[3][kWarps] = red[turn & 1];
    float3 sum;
    sum.x = red_max(mine[0]);
    sum.y = join<kWarps>((mine[0][lane & 7] - sum.x) * p.c, mine[1][lane & 7], 0.f).x;
    // A part of which nothing is left (all of it masked, or listed) counts as -inf, unless the row has no other.
    const bool nothing = sum.x == -INFINITY && p.parts > 1;
    if (!nothing && !(sum.y > 0.f && sum.y < INFINITY)) sum = slow_sums(r, l.entry, HOLES ? p.entries : 0, p.c, mine);
    if (nothing) sum.y = 0.f;
    if (p.parts > 1) {
      const int meet = meetings++;
      if (warp == 0) send_part(p, meeting, meet, make_float3(sum.x, sum.y, 0.f), 0);
      if (GRAD || warp == 0) {
        await_parts(p, meeting, meet);
        sum = join_parts(p, meeting, meet);
      }
    }
    if (!GRAD && warp != 0) return;
    float total = sum.y, rest = sum.y, all = 1.f, outside = 1.f;
    if constexpr (HOLES) {
      const float both = fmaxf(sum.x, l.listed_max);
      rest = sum.y * ex2_approx_ftz((sum.x - both) * p.c);
      total = rest + l.listed * ex2_approx_ftz((l.listed_max - both) * p.c);
      sum.x = both;
      const double left = l.all > 1 ? 0 : 1 - l.all;
      all = (float)(l.all + left);
      outside = rest == 0.f ? all : (float)(l.all + left - left * ((double)total / (double)rest));
    }
    if (tid == 0 && (p.parts == 1 || cluster_ctarank() == 0)) {
      const double log_total = log((double)total), lse = (double)sum.x / (double)p.temperature + log_total;
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
    if constexpr (GRAD) {
      T* dst = static_cast<T*>(p.dx) + row * p.ld_dx;
      int k;  // the logarithm's whole part joins the reference before it is rounded
      const float m = frexpf(total, &k), lse2 = fmaf(sum.x, p.c, (float)k) + log2f(m);
      stream_gradient<T, false>(r, in, dst, p.c, lse2, l.g * outside, 0.f);
      bar_stream();
      patch_entries<T>(r, dst, l.entry, l.q, l.x, p.entries, p.c, lse2, l.g, all);
    }
  }
};
template <typename T, bool GRAD, bool HOLES>
__global__ void __launch_bounds__(kAllThreads, kDistillPerSm) distill_kernel(const __grid_constant__ Distill p) {
  __shared__ Meeting meeting;
  __shared__ DistillLesson lessons[3];
  __shared__ double power[kMaxEntries];
  __shared__ float red[2][3][kWarps];
  extern __shared__ unsigned holes[];  // two sets
  const int hole_words = HOLES ? (p.per * Range<T>::V + 31) / 32 : 0;
  for (int i = threadIdx.x; i < 2 * hole_words; i += kAllThreads) holes[i] = 0;
  DistillOp<T, GRAD, HOLES> op{p, power, red, holes, hole_words, meeting, 0};
  run_rows<T>(p, op, lessons, &meeting);
}

// ------------------------------------------------------------------ backward
struct Backward : Rows {
  void* dx;
  long long ld_dx;
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

// A row's gradient is p (a + b log2 p) but where an entry (an alternative, the token, what the teacher lists) meets it.
template <int ENTRIES>
struct BackwardLesson {
  long long at;
  float lse2, a, b, all, g;
  int entries;
  bool zero;
  int entry[ENTRIES];
  float weight[ENTRIES], x[ENTRIES];
};

// Gradient of the log probabilities, the entropy and the alternatives of a row:
//   dx_v = 1/temperature [ sum of the gradients that meet at v - p_v (G + g_H (log p_v + H)) ],  G = the sum of all but g_H
// and of the distillation loss (DISTILL): g/temperature p_v outside, or g/temperature (all p_v - q_v) where the teacher lists v.
template <typename T, bool DISTILL, bool ENTROPY>
struct BackwardOp {
  using Lesson = BackwardLesson<DISTILL ? kMaxEntries : kMaxTop + 1>;
  const Backward& p;

  __device__ __forceinline__ void before(int, const Lesson*) {}
  __device__ __forceinline__ void after(int, const Lesson*) {}
  // dx may be the logits themselves: the entries' logits are read before their row is streamed.
  __device__ __forceinline__ void enter(Lesson& l, int j, long long id, float weight, const Range<T>& r) {
    if (id < 0 || id > p.n) {
      atomicMax(p.status, DEV_BAD_INDEX);
      id = 0;
    }
    const int mine = in_range(r, id);
    l.entry[j] = mine;
    l.weight[j] = weight;
    l.x[j] = mine ? to_float(r.src[mine - 1]) : 0.f;
  }
  __device__ __forceinline__ bool prepare(Lesson& l, long long item) {
    const int lane = threadIdx.x & 31;
    const long long row = row_of(p, item);
    const Range<T> r = range_of<T>(p, item);
    if constexpr (!DISTILL) {
      const long long token = p.tokens ? load_id(p.tokens, row, p.token_bits) : -1;
      const bool bad = p.tokens && (token < 0 || token > p.n);
      if (token == 0 || bad) {
        if (bad && lane == 0) atomicMax(p.status, DEV_BAD_INDEX);
        if (lane == 0) l.zero = true;
        return true;
      }
      const float g0 = p.d_logprobs ? p.d_logprobs[row] : 0.f, gh = ENTROPY ? p.d_entropy[row] : 0.f, h = ENTROPY ? p.entropy[row] : 0.f;
      const float gt = lane < p.top ? p.d_top[row * p.top + lane] : 0.f, all = g0 + warp_sum(gt);
      if (lane < p.top) enter(l, lane, p.top_ids[row * p.top + lane], gt, r);
      if (lane == 0) {
        if (p.d_logprobs) enter(l, p.top, token, g0, r);
        l.entries = p.top + (p.d_logprobs ? 1 : 0);
        l.lse2 = p.lse[row] * kLog2e;
        l.a = -(all + gh * h) / p.temperature;
        l.b = -gh * kLn2 / p.temperature;
      }
    } else {
      const float4 saved = reinterpret_cast<const float4*>(p.saved)[row];
      if (saved.z == 0.f) {
        if (lane == 0) l.zero = true;
        return true;
      }
      const bool whole = saved.z < 0.f;  // the teacher's list is all of its distribution
      const double norm = (double)saved.w + (whole ? (double)saved.y : 0.);
      for (int j = lane; j < p.entries; j += 32) {
        const double u = (double)load_value(p.values, row * p.entries + j, p.values_dtype) / (double)p.temperature;
        enter(l, j, load_id(p.ids, row * p.entries + j, p.id_bits), (float)exp(u - norm), r);
      }
      if (lane == 0) {
        l.g = p.d_loss[row] / p.temperature;
        l.entries = p.entries;
        l.lse2 = saved.x * kLog2e;
        l.a = l.g * (whole ? 1.f : saved.y);
        l.all = whole ? 1.f : saved.z;
      }
    }
    return true;
  }
  __device__ __forceinline__ void stream(int, const Lesson& l, const Range<T>& r, const Inner& in) {
    T* dst = static_cast<T*>(p.dx) + row_of(p, l.at) * p.ld_dx;
    if (l.zero) stream_zeros<T>(r, dst);
    else stream_gradient<T, ENTROPY>(r, in, dst, p.c, l.lse2, l.a, l.b);
  }
  __device__ __forceinline__ void finish(int, const Lesson& l, const Range<T>& r, const Inner&) {
    if (l.zero) return;
    T* dst = static_cast<T*>(p.dx) + row_of(p, l.at) * p.ld_dx;
    if constexpr (DISTILL) {
      patch_entries<T>(r, dst, l.entry, l.weight, l.x, l.entries, p.c, l.lse2, l.g, l.all);
    } else {
      const int j = threadIdx.x;
      if (j >= l.entries || l.entry[j] == 0) return;
      float g = 0.f;
      for (int i = 0; i < l.entries; ++i)
        if (l.entry[i] == l.entry[j]) {
          if (i < j) return;
          g += l.weight[i];
        }
      const float t = fmaf(l.x[j], p.c, -l.lse2);
      dst[l.entry[j] - 1] = from_float<T>(g / p.temperature + ex2_approx_ftz(t) * fmaf(l.b, fmaxf(t, kLowest), l.a));
    }
  }
};
template <typename T, bool DISTILL, bool ENTROPY>
__global__ void __launch_bounds__(kAllThreads, kBackwardPerSm<DISTILL>) logits_backward_kernel(const __grid_constant__ Backward p) {
  __shared__ typename BackwardOp<T, DISTILL, ENTROPY>::Lesson lessons[3];
  BackwardOp<T, DISTILL, ENTROPY> op{p};
  run_rows<T>(p, op, lessons, nullptr);
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

// Clusters of C CTAs of a kernel that run at once.
template <auto KERNEL>
int most_teams(ctb_ctx* ctx, int C, int per_sm, size_t smem, bool keep) {
  static std::atomic<int> cached[16][kMaxCluster + 1];
  std::atomic<int>& known = cached[ctx->device & 15][C];
  if (keep && known.load(std::memory_order_relaxed) > 0) return known.load(std::memory_order_relaxed);
  int n = 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctx->sm_count * per_sm / C * C);
  cfg.blockDim = dim3(kAllThreads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, KERNEL, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    n = 0;
  }
  if (keep && n > 0) known.store(n, std::memory_order_relaxed);
  return n;
}

// How the rows are cut: for the kernels whose parts meet, into the 1, 2, 4, 8 or 16 CTAs of a cluster.  Rows go over the teams in rounds;
// a round takes the time of its bytes at the rate of HBM, but no less than a part at the rate that a CTA reaches alone, and what begins
// and ends a row (`ends`, and a meeting).  Times in us, rates in bytes per us.
struct Cut {
  int parts, teams;
};
template <auto KERNEL>
Cut cut_rows(ctb_ctx* ctx, int64_t rows, int64_t row_bytes, int per_sm, int least, double ends) {
  constexpr double kAlone = 20e3, kAll = 6500e3, kMeeting = 1.0;
  Cut best = {0, 0};
  double best_time = 0;
  for (int C = 1; C <= kMaxCluster; C *= 2) {
    if (C < least) continue;
    if (row_bytes / C < 4096 && C > least) break;
    const int most = C == 1 ? ctx->sm_count * per_sm : most_teams<KERNEL>(ctx, C, per_sm, 0, true);
    if (most < 1) continue;
    const int teams = (int)std::min<int64_t>(rows, most);
    const double part = (double)row_bytes / C / kAlone + ends + (C > 1 ? kMeeting : 0.);
    const int64_t full = rows / teams, rest = rows % teams;
    const double time = (double)full * std::max((double)teams * (double)row_bytes / kAll, part) +
                        (rest ? std::max((double)rest * (double)row_bytes / kAll, part) : 0.);
    if (best.parts == 0 || time < best_time) {
      best = {C, teams};
      best_time = time;
    }
  }
  return best;
}

template <typename T>
int64_t vectors(const Rows& p) {  // of a row, wherever it starts
  constexpr int V = 16 / (int)sizeof(T);
  return (p.n + V - 1) / V + 1;
}
void cut_into(Rows& p, int64_t nvec, int64_t parts) {
  p.per = (int)(((nvec + parts - 1) / parts + 31) / 32 * 32);
  p.parts = (int)parts;
}
// Launches a forward kernel.  holes: two bits of shared memory for each element of a part.
template <auto KERNEL, typename T, typename P>
int launch_forward(ctb_ctx* ctx, cudaStream_t st, P p, int per_sm, bool holes, double ends, const char* who) {
  constexpr int V = 16 / (int)sizeof(T);
  const int64_t nvec = vectors<T>(p);
  p.cluster = 1;
  cudaError_t e = holes ? allow_smem(KERNEL, (kMostHoles + 1024) / 4) : cudaSuccess;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return cuda_fail(e, who);
  int least = 1;
  if (holes)
    while (least < kMaxCluster && nvec * V > (int64_t)least * kMostHoles) least *= 2;
  Cut cut = cut_rows<KERNEL>(ctx, p.rows, nvec * 16, per_sm, least, ends);
  if (cut.parts == 0) return fail(CTB_UNSUPPORTED, "%s: no room for a row's CTAs on this device", who);
  cut_into(p, nvec, cut.parts);
  size_t smem = 0;
  if (holes) {  // more shared memory may leave room for fewer
    if ((int64_t)p.per * V > kMostHoles + 1024) return fail(CTB_UNSUPPORTED, "%s: with teacher_lse, rows of %d elements are too long", who, p.n);
    smem = 2 * 4 * (((size_t)p.per * V + 31) / 32);
    int fit = 0;
    if (p.parts > 1) {
      fit = most_teams<KERNEL>(ctx, p.parts, per_sm, smem, false);
    } else {
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, KERNEL, kAllThreads, smem);
      fit *= ctx->sm_count;
    }
    cut.teams = std::max(1, std::min(cut.teams, fit));
  }
  launch_kernel(KERNEL, cut.teams * p.parts, kAllThreads, smem, st, p.parts, p);
  CTB_CHECK_LAUNCH(who);
  return CTB_OK;
}

template <typename T>
int launch_logprobs(ctb_ctx* ctx, cudaStream_t st, const Logprobs& p, const char* who) {
  return p.top ? launch_forward<logprobs_kernel<T, true>, T>(ctx, st, p, kLogprobsPerSm<true>, false, 3.0, who)
               : launch_forward<logprobs_kernel<T, false>, T>(ctx, st, p, kLogprobsPerSm<false>, false, 1.0, who);
}
template <typename T, bool GRAD>
int launch_distill(ctb_ctx* ctx, cudaStream_t st, const Distill& p, const char* who) {
  return p.teacher_lse ? launch_forward<distill_kernel<T, GRAD, true>, T>(ctx, st, p, kDistillPerSm, true, 2.5, who)
                       : launch_forward<distill_kernel<T, GRAD, false>, T>(ctx, st, p, kDistillPerSm, false, 2.5, who);
}
template <typename T, bool DISTILL>
int launch_backward(ctb_ctx* ctx, cudaStream_t st, Backward p, const char* who) {
  auto kernel = p.d_entropy ? logits_backward_kernel<T, DISTILL, !DISTILL> : logits_backward_kernel<T, DISTILL, false>;
  // Parts have nothing to do with each other: of at most four tiles, or one where that brings work to more places.
  const int64_t nvec = vectors<T>(p), places = (int64_t)kBackwardPerSm<DISTILL> * ctx->sm_count;
  const int64_t tiles = (nvec + kTile - 1) / kTile, each = p.rows * tiles >= 16 * places ? 4 : 1;
  cut_into(p, nvec, (tiles + each - 1) / each);
  launch_kernel(kernel, (int)std::min<int64_t>((int64_t)p.rows * p.parts, places), kAllThreads, 0, st, 0, p);
  CTB_CHECK_LAUNCH(who);
  return CTB_OK;
}
template <typename F>
int by_type(int dtype, F f) {
  if (dtype == CTB_F32) return f(float());
  if (dtype == CTB_F16) return f(__half());
  return f(__nv_bfloat16());
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
  p.x = logits; p.ld = ld; p.dx = d_logits; p.ld_dx = ld_out; p.n = (int)V; p.rows = (int)T;
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
  if (d_logits) return by_type(dtype, [&](auto t) { return launch_distill<decltype(t), true>(ctx, st, p, who); });
  return by_type(dtype, [&](auto t) { return launch_distill<decltype(t), false>(ctx, st, p, who); });
}

extern "C" int ctb_distill_fwd(ctb_ctx* ctx, void* stream, const void* logits, const void* teacher_ids, int id_bits,
                               const void* teacher_values, int values_dtype, const float* teacher_lse, float* loss, float* saved,
                               int64_t V, int64_t T, int64_t ld, int entries, float temperature, int dtype) {
  CTB_CHECK_CTX(ctx);
  CurrentDevice current(ctx);
  return distill_forward("ctb_distill_fwd", ctx, stream, logits, teacher_ids, id_bits, teacher_values, values_dtype, teacher_lse, loss, saved,
                         nullptr, nullptr, V, T, 0, ld, entries, temperature, dtype);
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
  Backward p = {};
  p.x = logits; p.ld = ld; p.dx = d_logits; p.ld_dx = ld_out; p.n = (int)V; p.rows = (int)T;
  p.c = (float)(1.4426950408889634 / (double)temperature);
  p.temperature = temperature;
  p.status = ctx->dev_status;
  p.ids = teacher_ids; p.id_bits = id_bits; p.entries = entries; p.values = teacher_values; p.values_dtype = values_dtype;
  p.saved = saved; p.d_loss = d_loss;
  return by_type(dtype, [&](auto t) { return launch_backward<decltype(t), true>(ctx, static_cast<cudaStream_t>(stream), p, who); });
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
    return distill_forward(who, ctx, stream, logits, teacher_ids, id_bits, teacher_values, values_dtype, teacher_lse, loss, saved, d_loss,
                         d_logits, V, T, ld_out, ld, entries, temperature, dtype);
}
