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
#include <limits.h>

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
constexpr int kMaxEntries = 256;         // of a teacher's list
constexpr int kCand = 1024;
constexpr int kPlainPerSm = 6, kTopPerSm = 4, kBackwardPerSm = 5, kBothPerSm = 4;  // CTAs on an SM
constexpr size_t kMostShared = 220 * 1024;  // dynamic shared memory of a CTA
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Exponents (base 2) are held above this where they are multiplied by their power, which is 0 there: 0 * -inf would be NaN.
constexpr float kLowest = -16384.f;
// A thread's reference follows its maximum only when an element is 2^kSlack above it.
constexpr float kSlack = 4.f;
// Beyond, the rounding of an exponent's reference is no small fraction (2^-4 here) of a power of two any more, or it overflows.
constexpr float kFar = 0x1p20f;

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
    __syncthreads();
    n = b.count2;
  } else {
    __syncthreads();
  }
  for (int i0 = 0; i0 < n; i0 += kThreads / 4) {  // four threads rank an element
    const int i = min(i0 + (tid >> 2), n - 1);
    const float v = value[i];
    const int id = index[i];
    int rank = 0;
#pragma unroll 4
    for (int j = tid & 3; j < n; j += 4) rank += value[j] > v || (value[j] == v && index[j] < id);
    rank += __shfl_xor_sync(0xffffffffu, rank, 1);
    rank += __shfl_xor_sync(0xffffffffu, rank, 2);
    if (rank < k && i == i0 + (tid >> 2)) {
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
// Exponents t = x c - m2, with c = log2(e) / temperature: one fused multiply-add gives them with one rounding, whatever the magnitude of x, and
// the rounding of c is that of a temperature, the same for the whole row.
//
// A thread's share of s = sum 2^t and, with ENTROPY, w = sum 2^t t.  Its reference follows its maximum, or t 2^t of a likely element would
// carry a rounding that the entropy, a difference of two such sums, shows.  Masked elements (-inf) make w NaN (0 * -inf): the tile's
// share is then taken again with exponents held above kLowest.  m2 is maximum c rounded, and t is off by what that lost, until the sums are
// put relative to the maximum itself.  Where m2 is beyond kFar (a small temperature, all that is left is masked by a number, infinities) that
// may be more than an exponent holds, and exponents are taken from differences, (x - maximum) c.
template <typename T, bool ENTROPY>
struct Sums {
  float ref = 0.f, m2 = 0.f, limit = -INFINITY;  // m2 = ref c; elements above limit move the reference
  uint32_t top = empty_row_vec<T>().x;
  Pair s = pair(0.f, 0.f), w = pair(0.f, 0.f);

  static __device__ __forceinline__ bool far(float m2) { return !(fabsf(m2) <= kFar); }
  __device__ __forceinline__ bool far() const { return far(m2); }
  // What the rounding of m2 has added to the exponents.
  static __device__ __forceinline__ float added(float ref, float m2, float c) { return far(m2) ? 0.f : fmaf(ref, c, -m2); }
  __device__ __forceinline__ void move(float x, float c) {
    const float to = __fmul_rn(x, c);  // rounded: as part of a fused m2 - x c it would not be what m2 becomes
    const float apart = (ref - x) * c - added(ref, m2, c) + added(x, to, c);  // m2 - to, but for what is far
    const float d = fmaxf(fminf(apart, 0.f), kLowest), r = ex2_approx_ftz(d);  // s = w = 0 until there is a reference
    const Pair rr = pair(r, r);
    if constexpr (ENTROPY) w = mul2(rr, fma2(s, pair(d, d), w));
    s = mul2(rr, s);
    ref = x;
    m2 = to;
    limit = x + kSlack / c;
  }
  // Returns the largest element.
  template <int N>
  __device__ __forceinline__ float add(const uint4 (&q)[N], float c) {
    uint32_t all = 0;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const uint32_t a = max_word<T>(max_word<T>(q[u].x, q[u].y), max_word<T>(q[u].z, q[u].w));
      all = u == 0 ? a : max_word<T>(all, a);
    }
    top = max_word<T>(top, all);
    const float most = word_max<T>(all);
    if (most > limit) move(most, c);
    const Pair cc = pair(c, c), minus = pair(-m2, -m2);
    Pair ts = pair(0.f, 0.f), tw = ts;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const uint32_t word[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
      for (int i = 0; i < 8 / (int)sizeof(T); ++i) {
        const Pair t = fma2(vec_pair<T>(word, i), cc, minus), e = exp2_pair(t);
        ts = add2(ts, e);
        if constexpr (ENTROPY) tw = fma2(e, t, tw);
      }
    }
    if (far() || (ENTROPY && sum_of(tw) != sum_of(tw))) {
      ts = tw = pair(0.f, 0.f);
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const float2 one = apart(q[u], ref, m2, c);
        ts = add2(ts, pair(one.x, 0.f));
        tw = add2(tw, pair(one.y, 0.f));
      }
    }
    s = add2(s, ts);
    if constexpr (ENTROPY) w = add2(w, tw);
    return most;
  }
  // (s, w) of a vector, exponents held above kLowest in w.
  static __device__ __noinline__ float2 apart(uint4 q, float ref, float m2, float c) {
    float f[16 / sizeof(T)], s = 0.f, w = 0.f;
    unpack_row<T>(q, f);
#pragma unroll
    for (int i = 0; i < 16 / (int)sizeof(T); ++i) {
      const float t = far(m2) ? (f[i] - ref) * c : fmaf(f[i], c, -m2), e = ex2_approx_ftz(t);
      s += e;
      w = fmaf(e, fmaxf(t, kLowest), w);
    }
    return make_float2(s, w);
  }
  // One element more.
  __device__ __forceinline__ void add_one(float x, float c) {
    const T e = from_float<T>(x);
    top = max_word<T>(top, sizeof(T) == 4 ? __float_as_uint(x) : 0x10001u * *reinterpret_cast<const unsigned short*>(&e));
    if (x > limit) move(x, c);
    const float t = far() ? (x - ref) * c : fmaf(x, c, -m2), v = ex2_approx_ftz(t);
    s = add2(s, pair(v, 0.f));
    if constexpr (ENTROPY) w = add2(w, pair(v * fmaxf(t, kLowest), 0.f));
  }
  // The warp's (maximum, s, w), the sums relative to that maximum.
  __device__ __forceinline__ float3 over_warp(float c) const {
    const float most = warp_max(word_max<T>(top));
    float d = (ref - most) * c - added(ref, m2, c);
    if (limit == -INFINITY) d = 0.f;  // nothing but masked elements, or NaN: its sums are 0, or NaN
    const float r = ex2_approx_ftz(d), sum = sum_of(s);
    return make_float3(most, warp_sum(sum * r), ENTROPY ? warp_sum(r * fmaf(sum, fmaxf(d, kLowest), sum_of(w))) : 0.f);
  }
};

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
// (maximum, s, w) of the warps' sums, in all lanes of a warp.
template <int W>
__device__ __forceinline__ float3 join_warps(const float (&red)[3][kWarps], float c) {
  const int w = threadIdx.x & (W - 1);
  float most = red[0][w];
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  most = fmaxf(most, -FLT_MAX);
  const float2 sum = join<W>((red[0][w] - most) * c, red[1][w], red[2][w]);
  return make_float3(most, sum.x, sum.y);
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
  float c, temperature;     // c = log2(e) / temperature
  int* status;
  float4* records;          // (maximum, s, w) of the parts of rows that warps have cut among them
  unsigned* tickets;        // a counter per row
};
template <typename T>
__device__ __forceinline__ Range<T> range_of(const Rows& p, long long row, int part) {
  constexpr int V = 16 / (int)sizeof(T);
  Range<T> r;
  r.src = static_cast<const T*>(p.x) + row * p.ld;
  r.off = (int)(((uintptr_t)r.src & 15) / sizeof(T));
  r.n = p.n;
  const int nvec = (r.off + p.n + V - 1) / V;
  r.v0 = (int)min((long long)nvec, (long long)part * p.per);
  r.v1 = min(nvec, r.v0 + p.per);
  return r;
}

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
// A bit per element of a warp's part, in the order in which the lanes take its vectors, kUnroll at a time; the last word: head, then tail.
__host__ __device__ constexpr int hole_words(int per, int elem) {
  const int words = (per + 32 * kUnroll - 1) / (32 * kUnroll) * kUnroll * (16 / elem);
  return (words > 256 ? words : 256) + 1;  // 256: the table in which equal ids meet
}
template <typename T>
__device__ __forceinline__ unsigned hole_bits(const unsigned* holes, int v) {  // of a lane's vectors from v on, v counted from the first inner one
  const int at = (v / (32 * kUnroll)) * 32 + (threadIdx.x & 31), u = v / 32 % kUnroll;
  if constexpr (sizeof(T) == 4) return reinterpret_cast<const unsigned short*>(holes)[at] >> 4 * u;
  else return holes[at] >> 8 * u;
}
template <typename T>
__device__ __forceinline__ void punch(const Range<T>& r, const Inner& in, int id, unsigned* holes, int words) {
  constexpr int V = Range<T>::V;
  const int e = id - 1 + r.off, v = e / V - in.a;
  int bit = (words - 1) * 32 + (e & (V - 1)) + (v < 0 ? 0 : 16);
  if (v >= 0 && e / V < in.b) bit = (((v / (32 * kUnroll)) * 32 + v % 32) * kUnroll + v / 32 % kUnroll) * V + (e & (V - 1));
  atomicOr(holes + (bit >> 5), 1u << (bit & 31));
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

// Calls f(q, v) for a thread's vectors, UNROLL at a time; v: the tile's first one.  What is left over comes one vector at a time, in
// the warps that have some of it; lanes beyond the end get -inf.  Lanes that took a rare branch in f would go on by
// themselves up to the next shuffle, behind the row: they meet before every tile (2220 x 100000 bf16: 110 -> 82 us).  W warps stream the row.  KEEP: it is read again,
// from L2.
template <typename T, int W, bool KEEP = false, int UNROLL = kUnroll, typename F>
__device__ __forceinline__ void each_tile(const Range<T>& r, const Inner& in, F f) {
  constexpr int kWide = W * 32;
  const int tid = threadIdx.x % kWide;
  const uint4* p = r.at(in.a) + tid;
  int v = in.a;
#pragma unroll 1
  for (; v + kWide * UNROLL <= in.b; v += kWide * UNROLL, p += kWide * UNROLL) {
    __syncwarp();
    uint4 q[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) q[u] = KEEP ? __ldcg(p + u * kWide) : __ldcs(p + u * kWide);
    f(q, v);
  }
#pragma unroll 1
  for (; v + (tid & ~31) < in.b; v += kWide, p += kWide) {
    __syncwarp();
    uint4 q[1] = {empty_row_vec<T>()};
    if (v + tid < in.b) q[0] = KEEP ? __ldcg(p) : __ldcs(p);
    f(q, v);
  }
}

// ------------------------------------------------------------------ rows cut among warps
// Where nothing but sums has to meet, a warp takes a part of a row (2 KB with few rows, 30 to 130 KB with thousands) after another, without a barrier and without a thought for the
// other warps of its CTA: (maximum, s, w) go to a record in scratch memory, and the warp that finishes a row's last part joins the
// records in their order and writes the results.  48 such warps on an SM keep 16-bit logits, whose exponentials keep the ex2 unit
// busy 55 % of the time, as close to HBM's rate as a loop without rows (2048 x 100003 bf16 80 us, 0.78 of the copy rate; 512 x 50001 f32 24.8); eight warps that meet at the end of every row left them at 78 %.
constexpr int kMaxParts = 256;
struct Items {  // of a warp (or, with W = 8, of the warps of a CTA, which share a part's tiles)
  const Rows& p;
  int parts;
  long long at, step, end;
  __device__ __forceinline__ explicit Items(const Rows& rows, int W = 1, int each = 0) : p(rows), parts(each ? each : rows.parts) {
    at = W == 1 ? (long long)blockIdx.x * kWarps + (threadIdx.x >> 5) : blockIdx.x;
    step = W == 1 ? (long long)gridDim.x * kWarps : gridDim.x;
    end = (long long)p.rows * parts;
  }
  __device__ __forceinline__ long long row(long long item) const { return parts == 1 ? item : item / parts; }
};
// A row's (maximum, s, w) from those of its parts.
__device__ __forceinline__ float3 gather_records(const float4* records, int parts, int size, float c) {
  const int lane = threadIdx.x & 31;
  float most = -FLT_MAX;
  for (int i = lane; i < parts; i += 32) most = fmaxf(most, __ldcg(&records[i * size].x));
  most = warp_max(most);
  float s = 0.f, w = 0.f;
  for (int i = lane; i < parts; i += 32) {
    const float4 one = __ldcg(records + i * size);
    const float d = (one.x - most) * c, r = ex2_approx_ftz(d);
    s = fmaf(one.y, r, s);
    w += r * fmaf(one.y, fmaxf(d, kLowest), one.z);
  }
  return make_float3(most, warp_sum(s), warp_sum(w));
}
// After a warp has summed a part: true for the row's last one, with the row's (maximum, s, w).
__device__ __forceinline__ bool join_records(const Rows& p, long long row, int part, float3& sum) {
  if (p.parts == 1) return true;
  float4* records = p.records + row * p.parts;
  unsigned order = 0;
  if ((threadIdx.x & 31) == 0) {
    __stcg(records + part, make_float4(sum.x, sum.y, sum.z, 0.f));
    __threadfence();
    order = atomicInc(p.tickets + row, p.parts - 1);
  }
  if (__shfl_sync(0xffffffffu, order, 0) != (unsigned)p.parts - 1) return false;
  __threadfence();
  sum = gather_records(records, p.parts, 1, p.c);
  return true;
}

// ------------------------------------------------------------------ log probabilities, forward
struct Logprobs : Rows {
  const void* tokens;
  int token_bits, top;
  float *logprobs, *entropy, *lse, *top_logprobs;
  int* top_ids;
};
// (x - most) / temperature; the difference by itself may be beyond f32.
__device__ __forceinline__ float scaled_apart(float x, float most, float temperature) { return 2 * ((0.5f * x - 0.5f * most) / temperature); }
__device__ __forceinline__ void write_results(const Logprobs& p, long long row, int token, float x, float3 sum) {
  if ((threadIdx.x & 31) != 0) return;
  const float log_sum = logf(sum.y);
  if (p.lse) p.lse[row] = sum.x / p.temperature + log_sum;
  if (p.entropy) p.entropy[row] = log_sum - kLn2 * (sum.z / sum.y);
  if (p.logprobs) {
    if (token < 0) atomicMax(p.status, DEV_BAD_INDEX);
    p.logprobs[row] = token < 0 ? NAN : scaled_apart(x, sum.x, p.temperature) - log_sum;
  }
}
// Token of a row: 0 for padding, -1 when it is out of range (or there are no tokens).
__device__ __forceinline__ int token_of(const Logprobs& p, long long row) {
  if (!p.tokens) return -1;
  const long long t = load_id(p.tokens, row, p.token_bits);
  return t < 0 || t > p.n ? -1 : (int)t;
}
__device__ __forceinline__ void write_padding(const Logprobs& p, long long row) {
  const int lane = threadIdx.x & 31;
  if (lane == 0) {
    if (p.logprobs) p.logprobs[row] = 0.f;
    if (p.entropy) p.entropy[row] = 0.f;
    if (p.lse) p.lse[row] = 0.f;
  }
  if (lane < p.top) {
    p.top_logprobs[row * p.top + lane] = 0.f;
    p.top_ids[row * p.top + lane] = 0;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, kPlainPerSm) logprobs_kernel(const __grid_constant__ Logprobs p) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const Items items(p);
  int tokens = 0;  // lane i: token of the i-th item of a batch of 32, and its logit
  float logits = 0.f;
  int n = 0;
  for (long long item = items.at; item < items.end; item += items.step, ++n) {
    if ((n & 31) == 0) {
      const long long mine = item + lane * items.step, row = items.row(mine);
      tokens = mine < items.end ? token_of(p, row) : 0;
      logits = tokens > 0 ? to_float((static_cast<const T*>(p.x) + row * p.ld)[tokens - 1]) : 0.f;
    }
    const long long row = items.row(item);
    const int part = (int)(item - row * p.parts), token = __shfl_sync(0xffffffffu, tokens, n & 31);
    const float x = __shfl_sync(0xffffffffu, logits, n & 31);
    if (token == 0) {
      if (part == 0) write_padding(p, row);
      continue;
    }
    const Range<T> r = range_of<T>(p, row, part);
    const Inner in(r);
    const int edge = edge_index(r, in, lane);
    const float at_edge = edge >= 0 ? to_float(r.src[edge]) : 0.f;
    Sums<T, true> sums;
    each_tile<T, 1>(r, in, [&](auto& q, int) { (void)sums.add(q, p.c); });
    if (edge >= 0) sums.add_one(at_edge, p.c);
    __syncwarp();
    float3 sum = sums.over_warp(p.c);
    if (join_records(p, row, part, sum)) write_results(p, row, token, x, sum);
  }
  grid_dependency_launch();
}

__device__ __forceinline__ void list_one(float value, int index, float theta, Best& best) {
  if (value > theta) {
    const int at = atomicAdd(&best.count, 1);
    if (at < kCand) {
      best.value[at] = value;
      best.index[at] = index;
    }
  }
}
// A call: in line it takes registers that the loop over tiles needs.
template <typename T>
__device__ __noinline__ void list_vector(uint4 q, int index, float theta, Best& best) {
  float f[16 / sizeof(T)];
  unpack_row<T>(q, f);
#pragma unroll
  for (int i = 0; i < 16 / (int)sizeof(T); ++i) list_one(f[i], index + i, theta, best);
}
// What a part leaves, in float4s: its sums, and a list of values and indices.
__host__ __device__ constexpr int record_size(int top) { return 1 + (top + 1) / 2; }

// With alternatives: rows, or parts of rows, a CTA each, whose threads meet for thresholds and lists.  The last CTA of a row joins the lists of
// its parts.  A list per warp, over parts of 16 KB, took twice as long: thresholds over so little are low, and choosing from lists is
// a chain of reductions.
template <typename T>
__global__ void __launch_bounds__(kThreads, kTopPerSm) top_logprobs_kernel(const __grid_constant__ Logprobs p) {
  __shared__ Best best;
  __shared__ float red[3][kWarps];
  __shared__ bool shared_last;
  constexpr int V = Range<T>::V;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dependency_wait();
  const Items items(p, kWarps);
  for (long long item = items.at; item < items.end; item += items.step) {
    const long long row = items.row(item);
    const int part = (int)(item - row * p.parts), token = token_of(p, row);
    if (token == 0) {
      if (part == 0 && warp == 0) write_padding(p, row);
      continue;
    }
    const float x = token > 0 ? to_float((static_cast<const T*>(p.x) + row * p.ld)[token - 1]) : 0.f;
    __syncthreads();  // the item before is done with
    const Range<T> r = range_of<T>(p, row, part);
    const Inner in(r);
    const int edge = edge_index(r, in, tid);
    const float at_edge = edge >= 0 ? to_float(r.src[edge]) : 0.f;
    Sums<T, true> sums;
    if (tid == 0) best.count = 0;  // ahead of the barriers of the first threshold
    float theta = -INFINITY;
    if (edge >= 0 && tid < 8) sums.add_one(at_edge, p.c);
    int tile = 0;
#pragma unroll 1
    for (int v = in.a; v < in.b || tile == 0; v += kTile, ++tile) {
      uint4 q[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) q[u] = v + u * kThreads + tid < in.b ? __ldcs(r.at(v) + u * kThreads + tid) : empty_row_vec<T>();
      const float most = sums.add(q, p.c);
      if (tile == 0) {
        theta = group_threshold(word_max<T>(sums.top), p.top, best);
        if (edge >= 0 && tid < 8) list_one(at_edge, edge, theta, best);
      }
      if (most > theta) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const uint32_t largest = max_word<T>(max_word<T>(q[u].x, q[u].y), max_word<T>(q[u].z, q[u].w));
          if (word_max<T>(largest) > theta) list_vector<T>(q[u], (v + u * kThreads + tid) * V - r.off, theta, best);
        }
      }
      if (tile > 0 && (tile & (tile + 1)) == 0 && v + kTile < in.b) theta = group_threshold(word_max<T>(sums.top), p.top, best);
    }
    if (edge >= 0 && tid >= 8) {
      sums.add_one(at_edge, p.c);
      list_one(at_edge, edge, theta, best);
    }
    const float3 of_warp = sums.over_warp(p.c);
    if (lane == 0) {
      red[0][warp] = of_warp.x;
      red[1][warp] = of_warp.y;
      red[2][warp] = of_warp.z;
    }
    __syncthreads();
    int count = best.count;
    if (count > kCand) {
      count = radix_list(r, p.top, best);
    } else if (count < p.top) {
      // theta of the first tile: with fewer than k above it, it is also the last one
      Range<T> first = r;
      first.v1 = min(r.v1, in.a + kTile);
      count = append_equal(first, theta, count, p.top - count, best);
    }
    select_list(count, p.top, best);
    float3 sum = make_float3(0.f, 0.f, 0.f);
    if (warp == 0) sum = join_warps<kWarps>(red, p.c);
    if (p.parts > 1) {
      const int size = record_size(p.top);
      float4* records = p.records + row * p.parts * size;
      if (warp == 0) {
        if (lane < p.top)
          __stcg(reinterpret_cast<float2*>(records + part * size + 1) + lane, make_float2(best.out_value[lane], __int_as_float(best.out_index[lane])));
        if (lane == 0) __stcg(records + part * size, make_float4(sum.x, sum.y, sum.z, 0.f));
        __threadfence();
        __syncwarp();
        if (lane == 0) shared_last = atomicInc(p.tickets + row, p.parts - 1) == p.parts - 1;
      }
      __syncthreads();
      if (!shared_last) continue;
      __threadfence();
      for (int i = tid; i < p.parts * p.top; i += kThreads) {
        // Spread (1009 is a prime, and not a product of parts and k), or threads would have elements of the same few ranks and their maxima
        // say little: 8 x 128000 f32, k = 32, 32 parts of 32 in order took 48 us for 13.
        const int of = i / p.top, at = i * 1009 % (p.parts * p.top);
        const float2 e = __ldcg(reinterpret_cast<const float2*>(records + of * size + 1) + (i - of * p.top));
        const int index = __float_as_int(e.y);
        best.value[at] = index >= 0 ? e.x : -INFINITY;
        best.index[at] = index >= 0 ? index : INT_MAX;
      }
      if (warp == 0) sum = gather_records(records, p.parts, size, p.c);
      __syncthreads();
      select_list(p.parts * p.top, p.top, best);
    }
    if (warp == 0) {
      const float log_sum = logf(sum.y);
      write_results(p, row, token, x, sum);
      if (lane < p.top) {
        const int id = best.out_index[lane];
        const bool there = id >= 0 && id != INT_MAX;
        p.top_logprobs[row * p.top + lane] = there ? scaled_apart(best.out_value[lane], sum.x, p.temperature) - log_sum : NAN;
        p.top_ids[row * p.top + lane] = there ? id + 1 : 0;
      }
    }
  }
  grid_dependency_launch();
}

// ------------------------------------------------------------------ gradients
// d = e (a + b t), e = 2^t, over a range, by W warps.  t = (x - base) c with APART, which keeps its digits whatever the magnitude of x (and
// costs a loop that HBM bounds nothing: 4096 x 65536 bf16 240.5 us for 240.4), else x c - base.
template <typename T, bool ENTROPY, bool APART, int W, int UNROLL = kUnroll>
__device__ __forceinline__ void stream_gradient(const Range<T>& r, const Inner& in, T* dst, float c, float base, float a, float b) {
  const int tid = threadIdx.x % (W * 32), edge = edge_index(r, in, tid);
  const bool aligned = ((uintptr_t)(dst - r.off) & 15) == 0;
  const Pair cc = pair(c, c), minus = pair(-base, -base), aa = pair(a, a), bb = pair(b, b);
  const float x = edge >= 0 ? to_float(r.src[edge]) : 0.f;
  each_tile<T, W, false, UNROLL>(r, in, [&](auto& q, int v) {
    constexpr int N = sizeof(q) / sizeof(uint4);
    uint4* to = reinterpret_cast<uint4*>(dst - r.off) + v + tid;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      uint32_t word[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
      for (int i = 0; i < 8 / (int)sizeof(T); ++i) {
        const Pair y = vec_pair<T>(word, i), t = APART ? mul2(add2(y, minus), cc) : fma2(y, cc, minus), e = exp2_pair(t);
        if constexpr (ENTROPY) {
          const float2 h = halves(t);
          put_pair<T>(word, i, mul2(e, fma2(bb, pair(fmaxf(h.x, kLowest), fmaxf(h.y, kLowest)), aa)));
        } else {
          put_pair<T>(word, i, mul2(e, aa));
        }
      }
      const uint4 d = make_uint4(word[0], word[1], word[2], word[3]);
      if (N > 1 || v + tid < in.b) {
        if (aligned) __stcs(to + u * W * 32, d);
        else store_edge<T>(dst, r.off, r.n, v + u * W * 32 + tid, d);
      }
    }
  });
  if (edge >= 0) {
    const float t = APART ? (x - base) * c : fmaf(x, c, -base), e = ex2_approx_ftz(t);
    dst[edge] = from_float<T>(ENTROPY ? e * fmaf(b, fmaxf(t, kLowest), a) : e * a);
  }
}
// Zeros over a range, by W warps.
template <typename T, int W>
__device__ __noinline__ void stream_zeros(const Range<T>& r, T* dst) {
  const bool aligned = ((uintptr_t)(dst - r.off) & 15) == 0;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int v = r.v0 + threadIdx.x % (W * 32); v < r.v1; v += W * 32) {
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
// Calls f(id, j, sum of the weights of this id) for the entries of this range that the calling warp, of W, has streamed, once per id: the
// lane writes over what the warp has written there.
template <int W, typename T, typename F>
__device__ __forceinline__ void patch_entries(const Range<T>& r, const Inner& in, const int* entry, const float* weight, int entries, F f) {
  __syncwarp();
  const int warp = threadIdx.x >> 5;
  for (int j = threadIdx.x & 31; j < entries; j += 32) {
    const int id = in_range(r, entry[j]);
    if (id == 0) continue;
    const int v = (id - 1 + r.off) / Range<T>::V;
    if (W > 1 && (v < in.a || v >= in.b ? 0 : (v - in.a) % kThreads >> 5) != warp) continue;
    float sum = 0.f;
    bool first = true;
    for (int i = 0; i < entries; ++i)
      if (entry[i] == id) {
        first &= i >= j;
        sum += weight[i];
      }
    if (first) f(id, j, sum);
  }
}

// ------------------------------------------------------------------ distillation, forward, and the gradient at once
// What the gradient needs to know of a row.  Maximum and sum apart, as p = 2^((x - most) c) / sum: one f32 for the logarithm of the sum of powers
// would leave p off by 2^-24 of that logarithm, and at -1e9 (a row that is masked by a number, a small temperature) nothing of the sum.
//   listed elements: d = g (whole p - q)      others: d = g outside r, r = 2^((x - rest_most) c) / rest_sum
// With a rest, r is its share of the rest's probability p_r, and outside = whole p_r - (what the list leaves over): p is 0 in f32 where the
// gradient of a small rest is not.  Else r = p, outside = 1.
// The teacher's maximum and log of its sum are apart as well, q = exp((value - largest value) / temperature - norm - norm_low); with teacher_lse
// q = exp(value / temperature - norm).
struct alignas(16) Saved {
  float most, sum;       // of the row
  float rest_most, rest_sum;
  float whole, outside;  // whole 0: the row has no gradient; -1: there is no rest, whole = outside = 1, and in `outside` lies the largest value
  float norm, norm_low;
};
static_assert(sizeof(Saved) == 32, "a row's saved values are eight f32");
struct Distill : Rows {
  const void* ids;
  int id_bits, entries;
  const void* values;
  int values_dtype;
  const float* teacher_lse;
  double per_temperature;  // 1 / temperature
  float* loss;
  Saved* saved;
};

// The teacher's side of a row, in f64: what its list leaves over is a difference from one.
struct Teacher {
  double terms, all, norm;   // sum q (log q - (z - listed_max / temperature)), sum q; norm: see Saved
  float listed_max;          // the student's largest listed logit
  union {
    float listed;            // with a rest: the sum of powers, relative to it, of the listed ids, each once
    float most;              // without: the teacher's largest value
  };
};
static_assert(sizeof(Teacher) == 2 * sizeof(float4), "a teacher takes two records");
// A warp's lists of `entries` each, in dynamic shared memory: ids (0: unused), q, the student's logits.
struct Listed {
  int* entry;
  float *q, *x;
  __device__ __forceinline__ Listed(unsigned char* store, int entries, int which) {
    entry = reinterpret_cast<int*>(store) + which * 3 * entries;
    q = reinterpret_cast<float*>(entry + entries);
    x = q + entries;
  }
};
__host__ __device__ constexpr int lists_words(int entries) { return kWarps * 3 * entries; }
enum Row { PADDING, BAD, LIVE };

// Whether a row has used entries, and ids in range only; a warp.  f(id) for each id in range.
template <typename F>
__device__ __forceinline__ Row look_at(const Distill& p, long long row, F f) {
  bool used = false, bad = false;
  for (int j = threadIdx.x & 31; j < p.entries; j += 32) {
    const long long id = load_id(p.ids, row * p.entries + j, p.id_bits);
    used |= id != 0;
    if (id < 0 || id > p.n) bad = true;
    else if (id > 0) f((int)id);
  }
  used = __any_sync(0xffffffffu, used);
  return __any_sync(0xffffffffu, bad) ? BAD : used ? LIVE : PADDING;
}
__device__ __forceinline__ void write_unused(const Distill& p, long long row, Row kind) {
  if ((threadIdx.x & 31) != 0) return;
  if (kind == BAD) atomicMax(p.status, DEV_BAD_INDEX);
  p.loss[row] = kind == BAD ? NAN : 0.f;
  p.saved[row] = {};
}
// log v, absolutely exact to 2^-24 whatever the magnitude.
__device__ __forceinline__ double log_of(float v) {
  int k;
  const float m = frexpf(v, &k);
  return fma((double)k, 0.69314718055994531, (double)logf(m));
}
// The teacher's side of a live row; a warp.  All of it is f64: a gradient q is off by the roundings of q, of g and of their product alone.
template <typename T, bool TAIL>
__device__ __noinline__ Teacher learn(const Distill& p, long long row, const Listed& t, unsigned* seen, int words) {
  const int lane = threadIdx.x & 31;
  const T* src = static_cast<const T*>(p.x) + row * p.ld;
  float most = -INFINITY, x_most = -INFINITY;
  __syncwarp();
  for (int j0 = 0; j0 < p.entries; j0 += 64) {
    int id[2];
    float v[2], x[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = j0 + 32 * i + lane;
      id[i] = j < p.entries ? (int)load_id(p.ids, row * p.entries + j, p.id_bits) : 0;
      v[i] = j < p.entries ? load_value(p.values, row * p.entries + j, p.values_dtype) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = id[i] ? to_float(src[id[i] - 1]) : -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = j0 + 32 * i + lane;
      if (j >= p.entries) break;
      t.entry[j] = id[i];
      t.q[j] = v[i];
      t.x[j] = x[i];
      x_most = fmaxf(x_most, x[i]);
      if (id[i]) most = fmaxf(most, v[i]);
    }
  }
  x_most = fmaxf(warp_max(x_most), -FLT_MAX);
  double norm, base = 0;
  if constexpr (TAIL) {
    norm = p.teacher_lse[row];
  } else {
    most = warp_max(most);
    base = most;
    double sum = 0;
    for (int j = lane; j < p.entries; j += 32)
      if (t.entry[j]) sum += exp(((double)t.q[j] - base) * p.per_temperature);
    norm = log(sum_lanes(sum));
  }
  double all = 0, terms = 0;
  for (int j = lane; j < p.entries; j += 32) {
    if (t.entry[j] == 0) continue;
    const double log_q = fma((double)t.q[j] - base, p.per_temperature, -norm);
    const double q = exp(log_q);
    all += q;
    if (q != 0) terms = fma(q, log_q - ((double)t.x[j] - (double)x_most) * p.per_temperature, terms);
    t.q[j] = (float)q;
  }
  terms = sum_lanes(terms);
  float listed = 0.f;
  if constexpr (TAIL) {
    all = sum_lanes(all);
    __syncwarp();
    // Ids that meet in a small table are looked for in the list, and all but the first of those alike marked.
    const unsigned mask = (32u << (31 - __clz(words))) - 1;
    for (int j0 = 0; j0 < p.entries; j0 += 32) {
      const int id = j0 + lane < p.entries ? t.entry[j0 + lane] : 0, own = max(id, 0);
      const bool met = id > 0 && (atomicOr(seen + ((own & mask) >> 5), 1u << (own & 31)) >> (own & 31) & 1);
      for (unsigned left = __ballot_sync(0xffffffffu, met); left; left &= left - 1) {
        const int like = __shfl_sync(0xffffffffu, id, __ffs(left) - 1);
        int first = kMaxEntries;
        for (int i = lane; i < p.entries; i += 32)
          if (abs(t.entry[i]) == like) first = min(first, i);
        first = __reduce_min_sync(0xffffffffu, first);
        for (int i = lane; i < p.entries; i += 32)
          if (i != first && t.entry[i] == like) t.entry[i] = -like;
        __syncwarp();
      }
    }
    for (int j = lane; j < p.entries; j += 32)
      if (t.entry[j] > 0) {
        listed += ex2_approx_ftz((t.x[j] - x_most) * p.c);
        seen[(t.entry[j] & mask) >> 5] = 0;
      }
    listed = warp_sum(listed);
  }
  __syncwarp();
  return {terms, TAIL ? all : 1, norm, x_most, {TAIL ? listed : most}};
}
// The maximum and the sum of powers of a row, and of what it has besides the teacher's list.  The two do not share a maximum: a student that is
// sure of what is listed leaves the rest less than f32 holds beside it.
struct Sides {
  float most, sum, rest_most, rest_sum;
};
// sum: of the row, with TAIL without what is listed.
template <bool TAIL>
__device__ __forceinline__ Sides with_listed(const Distill& p, const Teacher& t, float3 sum) {
  if constexpr (!TAIL) return {sum.x, sum.y, sum.x, sum.y};
  const float most = fmaxf(sum.x, t.listed_max);
  return {most, sum.y * ex2_approx_ftz((sum.x - most) * p.c) + t.listed * ex2_approx_ftz((t.listed_max - most) * p.c), sum.x, sum.y};
}
// What the teacher's list leaves over.
__device__ __forceinline__ double left_over(const Teacher& t) { return t.all > 1 ? 0 : 1 - t.all; }
template <bool TAIL>
__device__ __forceinline__ Saved saved_of(const Distill& p, const Teacher& t, const Sides& of) {
  const float norm = (float)t.norm;
  if constexpr (!TAIL) return {of.most, of.sum, of.most, of.sum, -1.f, t.most, norm, (float)(t.norm - (double)norm)};
  const double left = left_over(t), whole = t.all + left;
  if (of.rest_sum == 0.f) return {of.most, of.sum, of.most, of.sum, (float)whole, (float)whole, norm, 0.f};  // all else is masked, and gets 0
  const double share = exp(((double)of.rest_most - (double)of.most) * p.per_temperature) * (double)of.rest_sum / (double)of.sum;
  return {of.most, of.sum, of.rest_most, of.rest_sum, (float)whole, (float)(whole * share - left), norm, 0.f};
}
// Loss and saved values of a row; one lane.
template <bool TAIL>
__device__ __noinline__ void close_row(const Distill& p, long long row, const Teacher& t, const Sides& of) {
  const double log_total = log_of(of.sum);
  double loss = t.terms + t.all * fma((double)of.most - (double)t.listed_max, p.per_temperature, log_total);  // differences: z may be large
  if (TAIL && left_over(t) != 0)
    loss += left_over(t) * (log(left_over(t)) - fma((double)of.rest_most - (double)of.most, p.per_temperature, log_of(of.rest_sum) - log_total));
  p.loss[row] = (float)loss;
  p.saved[row] = saved_of<TAIL>(p, t, of);
}

// ------------------------------------------------------------------ backward
struct Both : Distill {
  void* dx;
  long long ld_dx;
  const float* d_loss;
};
struct Backward : Rows {
  void* dx;
  long long ld_dx;
  // log probabilities
  const void* tokens;
  int token_bits, top;
  const float *lse, *entropy, *d_logprobs, *d_entropy, *d_top;
  float lse_c, lse_c_low;  // temperature c: what lse is in units of the exponents
  const int* top_ids;
  // distillation
  const void* ids;
  int id_bits, entries;
  const void* values;
  int values_dtype;
  double per_temperature;
  const Saved* saved;
  const float* d_loss;
};

// Gradient of the log probabilities, the entropy and the alternatives of a row:
//   dx_v = 1/temperature [ sum of the gradients that meet at v - p_v (G + g_H (log p_v + H)) ],  G = the sum of all but g_H
// and of the distillation loss: see Saved.
// A CTA takes a part of a row after another; its warps share the tiles, so that 16 KB are read and written side by side (parts of a warp's
// own left HBM at 85 %), but do not wait for each other: each has the few places in its tiles that a gradient meets directly, and writes
// them behind its stream.  What a warp needs of a row the others need as well, and each loads it.
// TAIL: teacher_lse is given, and what the teacher lists is left out of the row's sum, by a bit per element, and added apart: the rest's
// probability from a difference would lose all digits where it is small.
// A part's elements but for those with a bit.
template <typename T, bool TAIL, bool KEEP>
__device__ __forceinline__ float3 sum_range(const Range<T>& r, const Inner& in, const unsigned* holes, int words, float c) {
  constexpr int V = Range<T>::V;
  const int lane = threadIdx.x & 31, edge = edge_index(r, in, lane);
  const float x = edge >= 0 ? to_float(r.src[edge]) : 0.f;
  Sums<T, false> sums;
  each_tile<T, 1, KEEP>(r, in, [&](auto& q, int v) {
    if constexpr (TAIL) {
      const unsigned hole = hole_bits<T>(holes, v - in.a);
      if (__any_sync(0xffffffffu, hole != 0)) {
#pragma unroll
        for (int u = 0; u < (int)(sizeof(q) / sizeof(uint4)); ++u) mask_holes<T>(q[u], hole >> u * V);
      }
    }
    (void)sums.add(q, c);
  });
  if (edge >= 0) {
    const int bit = (edge + r.off & V - 1) + (lane < 8 ? 0 : 16);
    if (!(TAIL && (holes[words - 1] >> bit & 1))) sums.add_one(x, c);
  }
  __syncwarp();
  return sums.over_warp(c);
}
__device__ __forceinline__ void clear_holes(unsigned* holes, int words) {
  __syncwarp();
  for (int i = threadIdx.x & 31; i < words; i += 32) holes[i] = 0;
  __syncwarp();
}
// (maximum, s) of two stretches of a row.
__device__ __forceinline__ float3 join_two(float3 a, float3 b, float c) {
  const float most = fmaxf(fmaxf(a.x, b.x), -FLT_MAX);
  return make_float3(most, fmaf(a.y, ex2_approx_ftz((a.x - most) * c), b.y * ex2_approx_ftz((b.x - most) * c)), 0.f);
}
// A warp has bits for this many elements, and takes a longer part in stretches (LONG).  Parts are that long only where rows of 300000 elements and
// more have few counters, or none.
constexpr int kStretch = 16384;
__host__ __device__ constexpr int stretch(int elem) { return kStretch * elem / 16; }  // vectors
__host__ __device__ constexpr int part_words(int per, int elem) { return hole_words(per < stretch(elem) ? per : stretch(elem), elem); }
// What a row needs, by a warp each: the sums of its parts, and (part -1) the teacher's side, which takes as long as a part of 20 KB or so: latencies
// and f64.  Each is left as a record, the teacher's in the first two; the last warp to come closes the row.  holes: zero before and after.
template <typename T, bool TAIL, bool LONG>
__device__ __forceinline__ void distill_part(const Distill& p, long long row, int part, const Listed& lists, unsigned* holes, int words) {
  const int lane = threadIdx.x & 31;
  const bool whole = p.parts == 1;  // one warp does it all
  Range<T> r = range_of<T>(p, row, max(part, 0));
  const int end = r.v1;
  if (LONG) r.v1 = min(end, r.v0 + stretch(sizeof(T)));
  auto leave_out = [&](int id) {
    if (TAIL && part >= 0 && in_range(r, id)) punch(r, Inner(r), id, holes, words);
  };
  const Row kind = look_at(p, row, leave_out);
  float4* records = p.records + row * (p.parts + 2);
  bool last = whole || part < 0, clean = false;
  if (kind != LIVE) {
    if (last) write_unused(p, row, kind);
  } else {
    __syncwarp();
    float3 sum;
    Teacher t;
    if constexpr (LONG) {
      sum = make_float3(-INFINITY, 0.f, 0.f);
      while (part >= 0) {
        sum = join_two(sum, sum_range<T, TAIL, false>(r, Inner(r), holes, words, p.c), p.c);
        if (r.v1 == end) break;
        clear_holes(holes, words);
        r.v0 = r.v1;
        r.v1 = min(end, r.v0 + stretch(sizeof(T)));
        (void)look_at(p, row, leave_out);
        __syncwarp();
      }
    } else if (part >= 0) {
      sum = sum_range<T, TAIL, false>(r, Inner(r), holes, words, p.c);
    }
    if (whole || part < 0) {
      if (TAIL && whole) clear_holes(holes, words);
      clean = whole;
      t = learn<T, TAIL>(p, row, lists, holes, words);
    }
    if (!whole) {
      unsigned order = 0;
      if (lane == 0) {
        if (part < 0) {
          __stcg(reinterpret_cast<double2*>(records), make_double2(t.terms, t.all));
          __stcg(reinterpret_cast<double2*>(records + 1), make_double2(t.norm, __hiloint2double(__float_as_int(t.listed), __float_as_int(t.listed_max))));
        } else {
          __stcg(records + 2 + part, make_float4(sum.x, sum.y, sum.z, 0.f));
        }
        __threadfence();
        order = atomicInc(p.tickets + row, p.parts);
      }
      last = __shfl_sync(0xffffffffu, order, 0) == (unsigned)p.parts;
      if (last) {
        __threadfence();
        const double2 a = __ldcg(reinterpret_cast<const double2*>(records)), b = __ldcg(reinterpret_cast<const double2*>(records + 1));
        t = {a.x, a.y, b.x, __int_as_float(__double2loint(b.y)), {__int_as_float(__double2hiint(b.y))}};
        sum = gather_records(records + 2, p.parts, 1, p.c);
      }
    }
    if (last && lane == 0) close_row<TAIL>(p, row, t, with_listed<TAIL>(p, t, sum));
  }
  if (TAIL && part >= 0 && !clean) clear_holes(holes, words);
  __syncwarp();
}

// The loss alone: rows cut among warps.
template <typename T, bool TAIL, bool LONG>
__global__ void __launch_bounds__(kThreads, kPlainPerSm) distill_kernel(const __grid_constant__ Distill p) {
  extern __shared__ __align__(16) unsigned char store[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Listed lists(store, p.entries, threadIdx.x >> 5);
  const int words = TAIL ? part_words(p.per, sizeof(T)) : 0;
  unsigned* holes = reinterpret_cast<unsigned*>(store) + lists_words(p.entries) + warp * words;
  for (int i = lane; i < words; i += 32) holes[i] = 0;
  grid_dependency_wait();
  __syncwarp();
  const int each = p.parts > 1 ? p.parts + 1 : 1;
  const Items items(p, 1, each);
  for (long long item = items.at; item < items.end; item += items.step) {
    const long long row = items.row(item);
    distill_part<T, TAIL, LONG>(p, row, (int)(item - row * each) - (each > 1), lists, holes, words);
  }
  grid_dependency_launch();
}

// A part of a row's gradient, by W warps that own each their vectors of it, and the listed elements in those.
// What the listed logits give is taken from them before the part is streamed (dx may be the logits themselves).  own_list: of the warp.
// given: the entries as learn has left them, if it has.
template <typename T, int W, bool GIVEN, typename P>
__device__ __forceinline__ void distill_gradient(const P& p, long long row, int part, const Saved& saved, const Listed& own_list,
                                                 const Listed& given) {
  int* entry = own_list.entry;
  float *weight = own_list.q, *p_all = own_list.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Range<T> r = range_of<T>(p, row, part);
  const Inner in(r);
  T* dst = static_cast<T*>(p.dx) + row * p.ld_dx;
  if (saved.whole == 0.f) {
    stream_zeros<T, W>(r, dst);
    return;
  }
  int own = 0;
  __syncwarp();
  for (int j0 = 0; j0 < p.entries; j0 += 32) {
    const int j = j0 + lane;
    const long long id = j >= p.entries ? 0 : GIVEN ? abs(given.entry[j]) : load_id(p.ids, row * p.entries + j, p.id_bits);
    if (!GIVEN && (id < 0 || id > p.n)) atomicMax(p.status, DEV_BAD_INDEX);
    bool mine = id <= p.n && in_range(r, id) != 0;
    if (W > 1 && mine) {
      const int v = (int)((id - 1 + r.off) / Range<T>::V);
      mine = (v < in.a || v >= in.b ? 0 : (v - in.a) % (W * 32) >> 5) == warp;
    }
    const unsigned all = __ballot_sync(0xffffffffu, mine);
    if (mine) {
      const int at = own + __popc(all & ((1u << lane) - 1));
      entry[at] = (int)id;
      weight[at] = __int_as_float(j);
    }
    own += __popc(all);
  }
  __syncwarp();
  const bool list_is_all = saved.whole < 0.f;
  const float whole = list_is_all ? 1.f : saved.whole, per_sum = 1.f / saved.sum;
  for (int k = lane; k < own; k += 32) {
    const int j = __float_as_int(weight[k]);
    const float of = GIVEN ? given.x[j] : to_float(r.src[entry[k] - 1]);
    p_all[k] = whole * (ex2_approx_ftz((of - saved.most) * p.c) * per_sum);
    if constexpr (GIVEN) {
      weight[k] = given.q[j];
    } else {
      const double norm = (double)saved.norm + (double)saved.norm_low, base = list_is_all ? (double)saved.outside : 0.;
      weight[k] = (float)exp(fma((double)load_value(p.values, row * p.entries + j, p.values_dtype) - base, p.per_temperature, -norm));
    }
  }
  const float g = p.d_loss[row] / p.temperature, outside = list_is_all ? 1.f : saved.outside;
  __syncwarp();
  stream_gradient<T, false, true, W>(r, in, dst, p.c, saved.rest_most, g * outside / saved.rest_sum, 0.f);
  __syncwarp();
  for (int k = lane; k < own; k += 32) {
    const int id = entry[k];
    float q = 0.f;
    bool first = true;
    for (int i = 0; i < own; ++i)
      if (entry[i] == id) {
        first &= i >= k;
        q += weight[i];
      }
    if (first) dst[id - 1] = from_float<T>(g * (p_all[k] - q));
  }
  __syncwarp();
}

// Loss and gradient at once, a row at a time by a CTA: eight warps sum an eighth each while a ninth learns the teacher's side, they meet, and
// each writes the gradient of its eighth, which comes out of L2.  The rows that are under way (four per SM) have to stay there: with five per
// SM 4096 x 65536 bf16 takes 274 us for 250, with three 254.  Two forms with more to them were slower: clusters with a warp that
// learns ahead (267), and warps that draw sums and, some rows behind, gradients from one counter (255, small batches twice as long).
template <typename T, bool TAIL>
__global__ void __launch_bounds__(kThreads + 32, kBothPerSm) distill_both_kernel(const __grid_constant__ Both p) {
  extern __shared__ __align__(16) unsigned char store[];
  __shared__ float red[2][3][kWarps];
  __shared__ Teacher teachers[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Listed lists(store, p.entries, threadIdx.x >> 5);
  const int words = TAIL ? hole_words(p.per, sizeof(T)) : 0;
  unsigned* holes = reinterpret_cast<unsigned*>(store) + lists_words(p.entries) / kWarps * (kWarps + 2) + warp * words;
  for (int i = lane; i < words; i += 32) holes[i] = 0;
  grid_dependency_wait();
  __syncwarp();
  int turn = 0;  // of two places: what a warp leaves for the others is not written over before they have all come to the next meeting
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const Range<T> r = range_of<T>(p, row, warp);
    const Inner in(r);
    const Row kind = look_at(p, row, [&](int id) {
      if (TAIL && warp < kWarps && in_range(r, id)) punch(r, in, id, holes, words);
    });
    if (kind != LIVE) {
      if (warp == kWarps) write_unused(p, row, kind);
      else stream_zeros<T, 1>(r, static_cast<T*>(p.dx) + row * p.ld_dx);
      if (TAIL) clear_holes(holes, words);
      continue;
    }
    __syncwarp();
    const Listed taught(store, p.entries, kWarps + turn);
    if (warp == kWarps) {
      const Teacher t = learn<T, TAIL>(p, row, taught, holes, words);
      if (lane == 0) teachers[turn] = t;
    } else {
      const float3 sum = sum_range<T, TAIL, true>(r, in, holes, words, p.c);
      if (lane == 0) {
        red[turn][0][warp] = sum.x;
        red[turn][1][warp] = sum.y;
        red[turn][2][warp] = 0.f;
      }
      if (TAIL) clear_holes(holes, words);
    }
    __syncthreads();
    const Teacher t = teachers[turn];
    const Sides sides = with_listed<TAIL>(p, t, join_warps<kWarps>(red[turn], p.c));
    if (warp == kWarps) {
      if (lane == 0) close_row<TAIL>(p, row, t, sides);
    } else {
      distill_gradient<T, 1, true>(p, row, warp, saved_of<TAIL>(p, t, sides), lists, taught);
    }
    turn ^= 1;
    __syncwarp();
  }
  grid_dependency_launch();
}

template <typename T>
__global__ void __launch_bounds__(kThreads, kBackwardPerSm) distill_backward_kernel(const __grid_constant__ Backward p) {
  extern __shared__ __align__(16) unsigned char store[];
  const Listed lists(store, p.entries, threadIdx.x >> 5);
  grid_dependency_wait();
  const Items items(p, kWarps);
  for (long long item = items.at; item < items.end; item += items.step) {
    const long long row = items.row(item);
    distill_gradient<T, kWarps, false>(p, row, (int)(item - row * p.parts), p.saved[row], lists, lists);
  }
  grid_dependency_launch();
}
// The ids that gradients of a row meet directly, in the range r, with those gradients and with the logits: dx may be the logits themselves.
// Returns how many, and the sum of the gradients; a warp, for itself.
struct Meeting {
  int entry[kMaxTop + 1];
  float weight[kMaxTop + 1], x[kMaxTop + 1];
  int others;  // whether a row is left for whole_rows_gradient
};
template <typename T>
__device__ __forceinline__ int meet(const Backward& p, long long row, long long token, const Range<T>& r, Meeting& m, float& all) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  auto enter = [&](int j, long long id, float w) {
    if (id < 0 || id > p.n) {
      atomicMax(p.status, DEV_BAD_INDEX);
      id = 0;
    }
    const int mine = in_range(r, id);
    m.entry[j] = mine;
    m.weight[j] = w;
    m.x[j] = mine ? to_float(r.src[mine - 1]) : 0.f;
  };
  const float g0 = p.d_logprobs ? p.d_logprobs[row] : 0.f, gt = lane < p.top ? p.d_top[row * p.top + lane] : 0.f;
  all = g0 + warp_sum(gt);
  if (lane < p.top) enter(lane, p.top_ids[row * p.top + lane], gt);
  if (lane == 0 && p.d_logprobs) enter(p.top, token, g0);
  __syncwarp();
  return p.top + (p.d_logprobs ? 1 : 0);
}

// p = e^(z - lse) is off by the rounding of lse, 2^-24 of it at most.  Up to this |lse| that is no more than 2^-17 of p (f32), or 2^-16, less
// than a tenth of a step of f16 and a hundredth of one of bf16.
template <typename T>
__device__ __forceinline__ bool lse_will_do(float lse) { return fabsf(lse) <= (sizeof(T) == 4 ? 128.f : 256.f); }
// The other rows (large logits, small temperatures, rows masked by a number): a CTA takes one as a whole, for what it writes over others may not
// read, and reads it twice, first for its maximum and sum.  Logits around 1000: 2048 x 100003 bf16 219 us (156 around 0), 512 x 50001 f32 60
// (40), 64 x 128000 bf16 38 (10).
constexpr int kWholeUnroll = 2;
template <typename T, bool ENTROPY>
__device__ __forceinline__ void whole_row_gradient(const Backward& p, long long row, long long token, Meeting& m) {
  __shared__ float red[3][kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Range<T> r = range_of<T>(p, row, 0);
  r.v1 = (r.off + r.n + Range<T>::V - 1) / Range<T>::V;
  const Inner in(r);
  T* dst = static_cast<T*>(p.dx) + row * p.ld_dx;
  float all;
  const int entries = meet(p, row, token, r, m, all), edge = edge_index(r, in, threadIdx.x);
  Sums<T, false> sums;
  each_tile<T, kWarps, true, kWholeUnroll>(r, in, [&](auto& q, int) { (void)sums.add(q, p.c); });
  if (edge >= 0) sums.add_one(to_float(r.src[edge]), p.c);
  __syncwarp();
  const float3 of_warp = sums.over_warp(p.c);
  __syncthreads();  // the row before is done with
  if (lane == 0) {
    red[0][warp] = of_warp.x;
    red[1][warp] = of_warp.y;
    red[2][warp] = 0.f;
  }
  __syncthreads();
  const float3 sum = join_warps<kWarps>(red, p.c);
  // lse says no more than these, unless it is not the row's own (a part of a vocabulary, with the lse of all)
  const float lse = p.lse[row], own = sum.x / p.temperature + logf(sum.y);
  const float per = (own == lse || fabsf(own - lse) <= 0x1p-21f * fabsf(lse) ? 1.f : expf(own - lse)) / sum.y;
  const float gh = ENTROPY ? p.d_entropy[row] : 0.f, h = ENTROPY ? p.entropy[row] : 0.f;
  const float b = -gh * kLn2 / p.temperature * per;
  const float a = -(all + gh * h) / p.temperature * per + (ENTROPY ? b * log2f(per) : 0.f);
  stream_gradient<T, ENTROPY, true, kWarps, kWholeUnroll>(r, in, dst, p.c, sum.x, a, b);
  patch_entries<kWarps>(r, in, m.entry, m.weight, entries, [&](int id, int j, float direct) {
    const float t = (m.x[j] - sum.x) * p.c, e = ex2_approx_ftz(t);
    dst[id - 1] = from_float<T>(direct / p.temperature + e * fmaf(b, fmaxf(t, kLowest), a));
  });
}
// The warps of a CTA agree on the rows by votes, whatever each has read.
// Behind the loop over the other rows, and two vectors at a time: as a call, in that loop, or four vectors at a time it slows the other rows down
// (2048 x 100003 bf16, forward and gradient 228.5 us; as a call 232).
template <typename T, bool ENTROPY>
__device__ __forceinline__ void whole_rows_gradient(const Backward& p, Meeting* lists) {
  const Items items(p, kWarps);
  for (long long item = items.at; item < items.end; item += items.step) {
    const long long row = items.row(item), token = p.tokens ? load_id(p.tokens, row, p.token_bits) : -1;
    const bool skip = item != row * p.parts || token == 0 || (p.tokens && (token < 0 || token > p.n)) || lse_will_do<T>(p.lse[row]);
    if (!__syncthreads_or(!skip)) continue;
    whole_row_gradient<T, ENTROPY>(p, row, token, lists[threadIdx.x >> 5]);
  }
}
template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(kThreads, kBackwardPerSm) logits_backward_kernel(const __grid_constant__ Backward p) {
  __shared__ Meeting lists[kWarps];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  Meeting& m = lists[threadIdx.x >> 5];
  const Items items(p, kWarps);
  if (lane == 0) m.others = 0;
  for (long long item = items.at; item < items.end; item += items.step) {
    const long long row = items.row(item);
    const Range<T> r = range_of<T>(p, row, (int)(item - row * p.parts));
    T* dst = static_cast<T*>(p.dx) + row * p.ld_dx;
    const long long token = p.tokens ? load_id(p.tokens, row, p.token_bits) : -1;
    const float lse = p.lse[row];
    const bool bad = p.tokens && (token < 0 || token > p.n);
    if (token == 0 || bad) {
      if (bad && lane == 0) atomicMax(p.status, DEV_BAD_INDEX);
      stream_zeros<T, kWarps>(r, dst);
      continue;
    }
    if (!lse_will_do<T>(lse)) {
      if (lane == 0) m.others = 1;
      continue;
    }
    const Inner in(r);
    float all;
    const int entries = meet(p, row, token, r, m, all);
    const float gh = ENTROPY ? p.d_entropy[row] : 0.f, h = ENTROPY ? p.entropy[row] : 0.f;
    // log2 p = t - lost: lse in units of c as it is, and what its f32 loses goes into a and b
    const float base = __fmul_rn(lse, p.lse_c), lost = fmaf(lse, p.lse_c, -base) + lse * p.lse_c_low, more = ex2_approx_ftz(-lost);
    const float b = -gh * kLn2 / p.temperature * more, a = -(all + gh * h) / p.temperature * more - b * lost;
    stream_gradient<T, ENTROPY, false, kWarps>(r, in, dst, p.c, base, a, b);
    patch_entries<kWarps>(r, in, m.entry, m.weight, entries, [&](int id, int j, float direct) {
      const float t = fmaf(m.x[j], p.c, -base), e = ex2_approx_ftz(t);
      dst[id - 1] = from_float<T>(direct / p.temperature + e * fmaf(b, fmaxf(t, kLowest), a));
    });
  }
  grid_dependency_launch();
  __syncwarp();
  if (__syncthreads_or(m.others)) whole_rows_gradient<T, ENTROPY>(p, lists);
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

template <typename T>
int64_t vectors(const Rows& p) {  // of a row, wherever it starts
  constexpr int V = 16 / (int)sizeof(T);
  return (p.n + V - 1) / V + 1;
}
void cut_into(Rows& p, int64_t nvec, int64_t parts) {
  p.per = (int)(((nvec + parts - 1) / parts + 31) / 32 * 32);
  p.parts = (int)parts;
}
// Rows cut among warps: into the parts for which rounds of parts take the least time.  A warp reads `alone` bytes per ns when nobody else reads
// and shares what HBM gives otherwise, a part costs `ends` besides and one more of a row 0.05 in the join (us); measured with 1 to 2220 rows of 50000 to 128000 elements.
void cut_among_warps(Rows& p, int64_t nvec, int elem, int64_t places, int64_t least, int64_t most, int more,
                     double ends) {
  const double alone = elem == 4 ? 5.1 : 3.5, all = 7600, bytes = (double)nvec * 16e-3;  // of a row, in 1000
  double best = 0;
  int64_t parts = 1;
  most = std::min({most, std::max<int64_t>(1, nvec / 128), std::max<int64_t>(1, 16 * places / std::max(1, p.rows))});  // 2 KB; 16 rounds
  least = std::min(least, most);
  for (int64_t n = least; n <= most; n = n < 64 ? n + 1 : n + n / 8) {
    const int64_t items = p.rows * (n + (n > 1 ? more : 0)), full = items / places, rest = items % places;
    auto round = [&](int64_t active) { return bytes / (double)n * (1 / alone + (double)active / all) + ends; };
    const double time = (double)full * round(places) + (rest ? round(rest) : 0) + 0.05 * (double)n;
    if (n == least || time < best) {
      best = time;
      parts = n;
    }
  }
  p.per = (int)(((nvec + parts - 1) / parts + 31) / 32 * 32);
  p.parts = (int)((nvec + p.per - 1) / p.per);
}
// Rows cut among CTAs that share nothing, in parts of whole tiles, and how many CTAs an SM gets (five, or one less): those for which rounds of
// parts, with half a tile for what begins and ends one, leave the fewest places without work.  4096 x 65536 bf16: 186 us in 7 rounds of
// four rows per SM, 201 in 6 of five; 2048 x 100003: 162 and 154.  Returns the CTAs.
int64_t cut_rows_into_parts(Rows& p, int64_t nvec, int sms) {
  const int64_t tiles = (nvec + kTile - 1) / kTile;
  double best = 0;
  int64_t per = 1, ctas = 1;
  for (int on_sm = kBackwardPerSm; on_sm >= kBackwardPerSm - 1; --on_sm) {
    const int64_t places = (int64_t)on_sm * sms;
    for (int64_t each = std::min<int64_t>(tiles, 16); each >= 1; --each) {
      const int64_t items = p.rows * ((tiles + each - 1) / each);
      const double time = (double)((items + places - 1) / places * std::min<int64_t>(on_sm, (items + sms - 1) / sms)) * ((double)each + 0.5);
      if (best == 0 || time < best) {
        best = time;
        per = each;
        ctas = std::min(items, places);
      }
    }
  }
  p.per = (int)(per * kTile);
  p.parts = (int)((nvec + p.per - 1) / p.per);
  return ctas;
}
// Parts that a row may have whose sums meet in scratch memory: as many as their records and counters have room for.
int64_t most_parts(const Rows& p, int record, int more) {
  if (p.rows > kTickets) return 1;
  return std::max<int64_t>(1, std::min<int64_t>(kMaxParts, kStreamScratchBytes / (int64_t)sizeof(float4) / p.rows / record - more));
}

// The same call for some of its rows.
template <typename T>
Logprobs rows_of(Logprobs p, int64_t first, int rows) {
  p.rows = rows;
  p.x = static_cast<const T*>(p.x) + first * p.ld;
  if (p.tokens) p.tokens = static_cast<const char*>(p.tokens) + first * (p.token_bits / 8);
  for (float** out : {&p.logprobs, &p.entropy, &p.lse})
    if (*out) *out += first;
  return p;
}
template <typename T>
Distill rows_of(Distill p, int64_t first, int rows) {
  p.rows = rows;
  p.x = static_cast<const T*>(p.x) + first * p.ld;
  p.ids = static_cast<const char*>(p.ids) + first * p.entries * (p.id_bits / 8);
  p.values = static_cast<const char*>(p.values) + first * p.entries * (p.values_dtype == CTB_F32 ? 4 : 2);
  if (p.teacher_lse) p.teacher_lse += first;
  p.loss += first;
  p.saved += first;
  return p;
}

// Launches a forward kernel whose warps cut the rows among them.  bits: dynamic shared memory for a bit per element; LONG: for parts that have more of
// them than that has room for.
template <auto KERNEL, auto LONG, typename T, typename P>
int launch_items(ctb_ctx* ctx, cudaStream_t st, P p, bool bits, bool taught, double ends, const char* who) {
  const int64_t places = (int64_t)kPlainPerSm * ctx->sm_count * kWarps, nvec = vectors<T>(p);
  if (p.rows > kTickets && nvec >= 2048 && (bits || p.rows < 8 * places)) {  // rows that there are no counters for, and too few to go whole
    const int64_t launches = (p.rows + kTickets - 1) / kTickets, each = (p.rows + launches - 1) / launches;
    for (int64_t first = 0; first < p.rows; first += each)
      if (int s = launch_items<KERNEL, LONG, T>(ctx, st, rows_of<T>(p, first, (int)std::min<int64_t>(each, p.rows - first)), bits, taught, ends, who)) return s;
    return CTB_OK;
  }
  size_t lists = 0;
  if constexpr (std::is_same<P, Distill>::value) lists = 4 * (size_t)lists_words(p.entries);
  auto go = [&] {
    const size_t smem = lists + (bits ? (size_t)kWarps * 4 * part_words(p.per, sizeof(T)) : 0);  // 41 KB at most
    int per_sm = kPlainPerSm;
    if (smem > 0) {
      per_sm = std::max(1, std::min(kPlainPerSm, (int)(kMostShared / (smem + 1024))));
    }
    const int64_t ctas = ((int64_t)p.rows * (p.parts + (taught && p.parts > 1)) + kWarps - 1) / kWarps;
    const bool stretches = bits && p.per > stretch(sizeof(T));
    launch_kernel(stretches ? LONG : KERNEL, (int)std::min<int64_t>(ctas, (int64_t)per_sm * ctx->sm_count), kThreads, smem, st, 0, p);
    CTB_CHECK_LAUNCH(who);
    return (int)CTB_OK;
  };
  cut_among_warps(p, nvec, sizeof(T), places, bits ? p.n / kStretch + 1 : 1, most_parts(p, 1, taught ? 2 : 0), taught, ends);
  if (p.parts > 1) {
    StreamScratch scratch(ctx, st);
    if (scratch.data) {
      p.records = reinterpret_cast<float4*>(scratch.data);
      p.tickets = scratch.tickets;
      return go();
    }
    cut_into(p, nvec, 1);
  }
  return go();
}

// With alternatives: parts of whole tiles, a CTA each, those for which rounds of parts take the least time.  A CTA reads 20 bytes per ns when
// nobody else reads, a part costs 3 us besides, and lists that are joined 2.5 (measured with 1 to 2220 rows of 32000 to 128000 elements).
template <typename T>
int launch_top(ctb_ctx* ctx, cudaStream_t st, Logprobs p, const char* who) {
  const int64_t nvec = vectors<T>(p), tiles = (nvec + kTile - 1) / kTile, places = (int64_t)kTopPerSm * ctx->sm_count;
  const int64_t most = std::min<int64_t>(most_parts(p, record_size(p.top), 0), kCand / p.top);
  double best = 0;
  p.per = (int)(tiles * kTile);
  p.parts = 1;
  for (int64_t n = 1; n <= std::min(most, tiles); ++n) {
    const int64_t each = (tiles + n - 1) / n, parts = (tiles + each - 1) / each, items = p.rows * parts;
    const double bytes = (double)each * kTile * 16;
    auto round = [&](int64_t active) { return std::max((double)active * bytes / 6500e3, bytes / 20e3 + 3.0); };
    const double time = (double)(items / places) * round(places) + (items % places ? round(items % places) : 0) + (parts > 1 ? 2.5 : 0);
    if (n == 1 || time < best) {
      best = time;
      p.per = (int)(each * kTile);
      p.parts = (int)parts;
    }
  }
  auto go = [&] {
    launch_kernel(top_logprobs_kernel<T>, (int)std::min<int64_t>((int64_t)p.rows * p.parts, places), kThreads, 0, st, 0, p);
    CTB_CHECK_LAUNCH(who);
    return (int)CTB_OK;
  };
  if (p.parts > 1) {
    StreamScratch scratch(ctx, st);
    if (scratch.data) {
      p.records = reinterpret_cast<float4*>(scratch.data);
      p.tickets = scratch.tickets;
      return go();
    }
    p.per = (int)(tiles * kTile);
    p.parts = 1;
  }
  return go();
}
template <typename T>
int launch_logprobs(ctb_ctx* ctx, cudaStream_t st, const Logprobs& p, const char* who) {
  return p.top ? launch_top<T>(ctx, st, p, who) : launch_items<logprobs_kernel<T>, logprobs_kernel<T>, T>(ctx, st, p, false, false, 3.0, who);
}
template <typename T>
int launch_backward(ctb_ctx* ctx, cudaStream_t st, Backward p, const char* who) {
  auto kernel = p.ids ? distill_backward_kernel<T> : p.d_entropy ? logits_backward_kernel<T, true> : logits_backward_kernel<T, false>;
  const int64_t ctas = cut_rows_into_parts(p, vectors<T>(p), ctx->sm_count);
  launch_kernel(kernel, (int)ctas, kThreads, p.ids ? 4 * (size_t)lists_words(p.entries) : 0, st, 0, p);
  CTB_CHECK_LAUNCH(who);
  return CTB_OK;
}
template <typename T>
int launch_distill(ctb_ctx* ctx, cudaStream_t st, const Distill& p, const char* who) {
  return p.teacher_lse ? launch_items<distill_kernel<T, true, false>, distill_kernel<T, true, true>, T>(ctx, st, p, true, true, 3.0, who)
                       : launch_items<distill_kernel<T, false, false>, distill_kernel<T, false, false>, T>(ctx, st, p, false, true, 3.0, who);
}
template <typename T>
size_t both_shared(const Both& p) {
  const int per = (int)((vectors<T>(p) + kWarps - 1) / kWarps + 31) / 32 * 32;
  return 4 * ((size_t)lists_words(p.entries) / kWarps * (kWarps + 2) + (p.teacher_lse ? (size_t)hole_words(per, sizeof(T)) * (kWarps + 1) : 0));
}
// Loss and gradient at once, or one after the other?  sms: above 128 KB a row takes a CTA so long that each SM wants one.  In us, one after the other and at once: 4096 x 65536 bf16 298, 250; 1500 x 50001 f32 178, 151;
// 8000 x 32000 bf16 318, 228.  Where the teacher's side takes longer than a row (20000 x 8000 bf16, with a rest: 305, 362), where the rows
// under way do not stay in L2 (1024 x 128000 f32: 281, 278), and for few long rows, one after the other.
template <typename T>
bool at_once(const Both& p, int sms) {
  const int64_t bytes = (int64_t)p.n * sizeof(T);
  return bytes >= 32 * 1024 && bytes <= 512 * 1024 && (bytes <= 128 * 1024 || p.rows >= sms) && both_shared<T>(p) <= kMostShared / kBothPerSm - 2048;
}
template <typename T>
int launch_both(ctb_ctx* ctx, cudaStream_t st, Both p, const char* who) {
  auto kernel = p.teacher_lse ? distill_both_kernel<T, true> : distill_both_kernel<T, false>;
  cut_into(p, vectors<T>(p), kWarps);
  const size_t smem = both_shared<T>(p);
  cudaError_t e = smem > 48 * 1024 ? allow_smem(kernel, kMostShared) : cudaSuccess;
  if (e != cudaSuccess) return cuda_fail(e, who);
  launch_kernel(kernel, (int)std::min<int64_t>(p.rows, (int64_t)kBothPerSm * ctx->sm_count), kThreads + 32, smem, st, 0, p);
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
  const double lse_c = (double)temperature * (double)p.c;
  p.lse_c = (float)lse_c; p.lse_c_low = (float)(lse_c - (double)p.lse_c);
  p.lse = lse; p.entropy = entropy; p.d_logprobs = d_logprobs; p.d_entropy = d_entropy; p.d_top = d_top_logprobs; p.top_ids = top_ids;
  return by_type(dtype, [&](auto t) { return launch_backward<decltype(t)>(ctx, static_cast<cudaStream_t>(stream), p, who); });
}

static int distill_forward(const char* who, ctb_ctx* ctx, void* stream, const void* logits, const void* teacher_ids, int id_bits,
                           const void* teacher_values, int values_dtype, const float* teacher_lse, float* loss, float* saved,
                           int64_t V, int64_t T, int64_t ld, int entries, float temperature, int dtype, const float* d_loss = nullptr,
                           void* d_logits = nullptr, int64_t ld_out = 0, bool* both = nullptr) {
  if (int s = check_rows(who, logits, V, T, ld, temperature, dtype)) return s;
  if (T == 0) return CTB_OK;
  if (int s = check_teacher(who, teacher_ids, id_bits, teacher_values, values_dtype, entries)) return s;
  if (teacher_lse) CTB_CHECK_PTR(who, teacher_lse);
  CTB_CHECK_PTR(who, loss);
  CTB_CHECK_PTR(who, saved);
  if ((uintptr_t)saved % 16) return fail(CTB_BAD_ALIGN, "%s: saved must be 16-byte aligned", who);
  Both p = {};
  p.x = logits; p.ld = ld; p.n = (int)V; p.rows = (int)T;
  p.c = (float)(1.4426950408889634 / (double)temperature);
  p.temperature = temperature;
  p.status = ctx->dev_status;
  p.ids = teacher_ids; p.id_bits = id_bits; p.entries = entries; p.values = teacher_values; p.values_dtype = values_dtype;
  p.teacher_lse = teacher_lse; p.per_temperature = 1 / (double)temperature; p.loss = loss; p.saved = reinterpret_cast<Saved*>(saved);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  p.d_loss = d_loss; p.dx = d_logits; p.ld_dx = ld_out;
  return by_type(dtype, [&](auto t) {
    if (both) *both = at_once<decltype(t)>(p, ctx->sm_count);
    return both && *both ? launch_both<decltype(t)>(ctx, st, p, who) : launch_distill<decltype(t)>(ctx, st, p, who);
  });
}

static int distill_backward(const char* who, ctb_ctx* ctx, void* stream, void* d_logits, const void* logits, const void* teacher_ids, int id_bits,
                            const void* teacher_values, int values_dtype, const float* saved, const float* d_loss, int64_t V, int64_t T,
                            int64_t ld_out, int64_t ld, int entries, float temperature, int dtype) {
  Backward p = {};
  p.x = logits; p.ld = ld; p.dx = d_logits; p.ld_dx = ld_out; p.n = (int)V; p.rows = (int)T;
  p.c = (float)(1.4426950408889634 / (double)temperature);
  p.temperature = temperature;
  p.status = ctx->dev_status;
  p.ids = teacher_ids; p.id_bits = id_bits; p.entries = entries; p.values = teacher_values; p.values_dtype = values_dtype;
  p.saved = reinterpret_cast<const Saved*>(saved); p.d_loss = d_loss; p.per_temperature = 1 / (double)temperature;
  return by_type(dtype, [&](auto t) { return launch_backward<decltype(t)>(ctx, static_cast<cudaStream_t>(stream), p, who); });
}

extern "C" int ctb_distill_fwd(ctb_ctx* ctx, void* stream, const void* logits, const void* teacher_ids, int id_bits,
                               const void* teacher_values, int values_dtype, const float* teacher_lse, float* loss, float* saved,
                               int64_t V, int64_t T, int64_t ld, int entries, float temperature, int dtype) {
  CTB_CHECK_CTX(ctx);
  CurrentDevice current(ctx);
  return distill_forward("ctb_distill_fwd", ctx, stream, logits, teacher_ids, id_bits, teacher_values, values_dtype, teacher_lse, loss, saved,
                         V, T, ld, entries, temperature, dtype);
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
  bool both = true;
  if (int s = distill_forward(who, ctx, stream, logits, teacher_ids, id_bits, teacher_values, values_dtype, teacher_lse, loss, saved, V, T, ld,
                              entries, temperature, dtype, d_loss, d_logits, ld_out, &both))
    return s;
  if (both) return CTB_OK;
  return distill_backward(who, ctx, stream, d_logits, logits, teacher_ids, id_bits, teacher_values, values_dtype, saved, d_loss, V, T, ld_out,
                          ld, entries, temperature, dtype);
}
