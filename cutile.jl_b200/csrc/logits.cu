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
constexpr int kMostHoles = 200 * 1024;  // bytes of shared memory, one per vector of a part
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Exponents (base 2) are held above this where they are multiplied by their power, which is 0 there: 0 * -inf would be NaN.
constexpr float kLowest = -16384.f;
// A thread's reference follows its maximum only when an element is 2^kSlack above it: powers up to 2^kSlack are harmless in f32.
constexpr float kSlack = 64.f;

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

// Vectors [v0, v1) of a row.
template <typename T>
struct Range {
  const T* src;
  int off, n, v0, v1;
};

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
      unpack_row<T>(load_row_vec(r.src, r.off, r.n, v), f);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (f[i] == value && in_row<V>(r.off, r.n, v, i)) match |= 1u << i;
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
      unpack_row<T>(load_row_vec(r.src, r.off, r.n, v), f);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint32_t key = order_key(f[i]);
        if (f[i] == f[i] && in_row<V>(r.off, r.n, v, i) && (key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1);
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
    unpack_row<T>(load_row_vec(r.src, r.off, r.n, v), f);
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

// ------------------------------------------------------------------ forward
// Arguments of the forward kernels: the logits, and what is done with a row.
struct Forward {
  const void* x;
  long long ld;
  int n, rows, parts, per;  // per: vectors of a part
  float c, temperature;     // c = log2(e) / temperature
  int* status;
  float* scratch;           // records of the parts
  unsigned* tickets;        // a counter per row
  // log probabilities
  const void* tokens;
  int token_bits, top;
  float *logprobs, *entropy, *lse, *top_logprobs;
  int* top_ids;
  // distillation
  const void* ids;
  int id_bits, entries;
  const void* values;
  int values_dtype;
  const float* teacher_lse;
  float *loss, *saved;
  // distillation with the gradient
  const float* d_loss;
  void* dx;
  long long ld_dx;
};

// Floats of a part's record: maximum, sum, entropy's sum, the best values, their indices.
__host__ __device__ constexpr int record_floats(int top) { return 4 + (2 * top + 3) / 4 * 4; }

enum Operator { LOGPROBS, DISTILL, DISTILL_GRAD };

__device__ __forceinline__ long long load_id(const void* p, long long i, int bits) {
  return bits == 64 ? static_cast<const long long*>(p)[i] : static_cast<const int*>(p)[i];
}
__device__ __forceinline__ float load_value(const void* p, long long i, int dtype) {
  if (dtype == CTB_F32) return static_cast<const float*>(p)[i];
  if (dtype == CTB_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __uint_as_float((uint32_t) static_cast<const unsigned short*>(p)[i] << 16);
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

struct Shared {
  float red[3][kWarps];
  int last;
  float grad[3];                  // what the gradient of a row needs: lse, outside, all of q
  int entry[kMaxEntries];         // ids of the teacher's entries, 0: unused
  float q[kMaxEntries];
  double log_q[kMaxEntries];
};

// The loss of a row from its maximum and sum, and what its gradient needs; one warp.  HOLES: teacher_lse is given, and sum leaves out what
// the teacher lists.  The teacher's side is in f64: what its list leaves over is a difference from one.
template <typename T, bool HOLES>
__device__ __noinline__ void finish_distill(const Forward& p, long long row, const T* src, float top_max, float sum, Shared& sh) {
  const int lane = threadIdx.x & 31;
  const double temperature = p.temperature;
  double most = -INFINITY;
  float x_most = top_max;
  for (int j = lane; j < p.entries; j += 32) {
    const int id = (int)load_id(p.ids, row * p.entries + j, p.id_bits);  // in range: rows with others have been sorted out
    const double u = (double)load_value(p.values, row * p.entries + j, p.values_dtype) / temperature;
    sh.entry[j] = id;
    sh.log_q[j] = u;
    if (id) {
      const float x = to_float(src[id - 1]);
      sh.q[j] = x;
      x_most = fmaxf(x_most, x);
      most = fmax(most, u);
    }
  }
  __syncwarp();
  double norm;
  if constexpr (HOLES) {
    norm = p.teacher_lse[row];
  } else {
    most = warp_max(most);
    double s = 0;
    for (int j = lane; j < p.entries; j += 32)
      if (sh.entry[j]) s += exp(sh.log_q[j] - most);
    norm = most + log(warp_sum(s));
  }
  float total = sum, rest = sum;
  if constexpr (HOLES) {  // the row's sum is that of the rest and, once per id, that of the entries
    x_most = ctb::warp_max(x_most);
    rest = sum * ex2_approx_ftz((top_max - x_most) * p.c);
    top_max = x_most;
    float listed = 0.f;
    for (int j = lane; j < p.entries; j += 32) {
      const int id = sh.entry[j];
      bool again = id == 0;
      for (int i = 0; i < j; ++i) again |= sh.entry[i] == id;
      if (!again) listed += ex2_approx_ftz((sh.q[j] - top_max) * p.c);
    }
    total = rest + ctb::warp_sum(listed);
  }
  const double log_total = log((double)total);
  double all = 0, terms = 0;
  for (int j = lane; j < p.entries; j += 32) {
    if (sh.entry[j] == 0) continue;
    const double log_q = sh.log_q[j] - norm, q = exp(log_q);
    const double log_p = ((double)sh.q[j] - (double)top_max) / temperature - log_total;
    if (q != 0) terms += q * (log_q - log_p);
    all += q;
    sh.q[j] = (float)q;
  }
  all = warp_sum(all);
  terms = warp_sum(terms);
  float outside = 1.f;
  if constexpr (HOLES) {
    const double left = all > 1 ? 0 : 1 - all;
    all += left;
    if (left != 0) terms += left * (log(left) - (log((double)rest) - log_total));
    outside = (float)(rest == 0.f ? all : all - left * ((double)total / (double)rest));
  } else {
    all = 1;
  }
  if (lane == 0) {
    const float lse = (float)((double)top_max / temperature + log_total);
    p.loss[row] = (float)terms;
    // (lse, outside, all, norm) with teacher_lse; else outside and all are 1, and the norm keeps 48 bits: (lse, low part, -1, norm)
    const float high = (float)norm;
    reinterpret_cast<float4*>(p.saved)[row] = HOLES ? make_float4(lse, outside, (float)all, high) : make_float4(lse, (float)(norm - (double)high), -1.f, high);
    sh.grad[0] = lse;
    sh.grad[1] = outside;
    sh.grad[2] = (float)all;
  }
}

// Gradient at the listed entries: g (all p - sum of the q of this id), once per id.  Thread j has entry j and its logit.
template <typename T>
__device__ __forceinline__ void patch_entries(T* dst, int entries, float x, float c, float lse2, float g, float all, const Shared& sh,
                                              long long lo, long long hi) {
  const int j = threadIdx.x;
  if (j >= entries) return;
  const int id = sh.entry[j];
  if (id <= lo || id > hi) return;
  float q = 0.f;
  for (int i = 0; i < entries; ++i)
    if (sh.entry[i] == id) {
      if (i < j) return;
      q += sh.q[i];
    }
  dst[id - 1] = from_float<T>(g * (all * ex2_approx_ftz(fmaf(x, c, -lse2)) - q));
}

// d = p (a + b t) with t = log2 p over vectors [v0, v1) of a row.
template <typename T, bool ENTROPY>
__device__ __noinline__ void stream_gradient(const T* src, T* dst, int off, int n, int v0, int v1, float c, float lse2, float a,
                                                float b) {
  constexpr int V = 16 / (int)sizeof(T);
  const bool aligned = ((uintptr_t)(dst - off) & 15) == 0;
  for (int base = v0 + (int)threadIdx.x; base < v1; base += kTile) {
    uint4 q[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (base + u * kThreads < v1) q[u] = load_row_vec(src, off, n, base + u * kThreads);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int v = base + u * kThreads;
      if (v >= v1) break;
      float f[V];
      unpack_row<T>(q[u], f);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float t = fmaf(f[i], c, -lse2), e = ex2_approx_ftz(t);
        f[i] = ENTROPY ? e * fmaf(b, fmaxf(t, kLowest), a) : e * a;
      }
      store_row_vec<T>(dst, off, n, v, f, aligned);
    }
  }
}
template <typename T>
__device__ __noinline__ void stream_zeros(T* dst, int off, int n, int v0, int v1) {
  constexpr int V = 16 / (int)sizeof(T);
  const bool aligned = ((uintptr_t)(dst - off) & 15) == 0;
  float f[V] = {};
  for (int v = v0 + (int)threadIdx.x; v < v1; v += kThreads) store_row_vec<T>(dst, off, n, v, f, aligned);
}

// A CTA takes (row, part) after (row, part); 256 threads with the loads of a tile in flight while the one before it is worked on, across the
// ends of rows too.  Rows are cut into parts where there are fewer rows than room for CTAs; the CTA that finishes a row's last part
// puts the parts together.
template <typename T, int OP, bool TOP, bool HOLES>
__global__ void __launch_bounds__(kThreads, 4) logits_forward_kernel(const __grid_constant__ Forward p) {
  constexpr int V = 16 / (int)sizeof(T);
  constexpr bool ENTROPY = OP == LOGPROBS;
  extern __shared__ __align__(16) unsigned char holes[];  // HOLES: per vector of the part, a bit for each element that the teacher lists
  __shared__ Shared sh;
  __shared__ typename std::conditional<TOP, Best, int>::type best_store;
  Best& best = reinterpret_cast<Best&>(best_store);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if constexpr (HOLES)
    for (int i = tid; i < (p.per + 3) / 4; i += kThreads) reinterpret_cast<unsigned*>(holes)[i] = 0;
  grid_dependency_sync();

  struct Item {
    int row, part, off, v0, v1;
    const T* src;
    long long token;
    float x_token;
  };
  const long long items = (long long)p.rows * p.parts;
  long long at = (long long)blockIdx.x - gridDim.x;
  // The next item that is not a padding row; outputs of padding rows are written on the way.
  auto advance = [&](Item& it) {
    for (;;) {
      at += gridDim.x;
      if (at >= items) return false;
      it.row = (int)(at / p.parts);
      it.part = (int)(at - (long long)it.row * p.parts);
      it.src = static_cast<const T*>(p.x) + it.row * p.ld;
      it.off = (int)(((uintptr_t)it.src & 15) / sizeof(T));
      const int nvec = (it.off + p.n + V - 1) / V;
      it.v0 = min(nvec, it.part * p.per);
      it.v1 = min(nvec, it.v0 + p.per);
      if constexpr (OP == LOGPROBS) {
        it.token = p.tokens ? load_id(p.tokens, it.row, p.token_bits) : -1;
        if (it.token != 0) {
          it.x_token = 0.f;
          if (it.token > 0 && it.token <= p.n) it.x_token = to_float(it.src[it.token - 1]);
          return true;
        }
        if (it.part == 0) {
          if (tid == 0) {
            if (p.logprobs) p.logprobs[it.row] = 0.f;
            if (p.entropy) p.entropy[it.row] = 0.f;
            if (p.lse) p.lse[it.row] = 0.f;
          }
          if (tid < p.top) {
            p.top_logprobs[(long long)it.row * p.top + tid] = 0.f;
            p.top_ids[(long long)it.row * p.top + tid] = 0;
          }
        }
      } else {
        bool used = false, bad = false;  // the same in every warp
        for (int j = lane; j < p.entries; j += 32) {
          const long long id = load_id(p.ids, (long long)it.row * p.entries + j, p.id_bits);
          used |= id != 0;
          bad |= id < 0 || id > p.n;
        }
        bad = __any_sync(0xffffffffu, bad);
        if (__any_sync(0xffffffffu, used) && !bad) return true;
        if (it.part == 0) {
          if (tid == 0) {
            if (bad) atomicMax(p.status, DEV_BAD_INDEX);
            p.loss[it.row] = bad ? NAN : 0.f;
            reinterpret_cast<float4*>(p.saved)[it.row] = make_float4(0.f, 0.f, 0.f, 0.f);
          }
          if constexpr (OP == DISTILL_GRAD) {
            T* dst = static_cast<T*>(p.dx) + it.row * p.ld_dx;
            stream_zeros<T>(dst, it.off, p.n, 0, nvec);
          }
        }
      }
    }
  };
  uint4 next[kUnroll];
  auto load = [&](const Item& it, int tile) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int v = it.v0 + tile * kTile + u * kThreads + tid;
      next[u] = v < it.v1 ? load_row_vec<T, OP == DISTILL_GRAD>(it.src, it.off, p.n, v) : empty_row_vec<T>();
    }
  };

  Item it, nit;
  bool have = advance(it);
  if (have) load(it, 0);
  while (have) {
    const int tiles = max(1, (it.v1 - it.v0 + kTile - 1) / kTile);
    bool nhave = false;
    float m = -FLT_MAX, gm = -INFINITY, theta = -INFINITY;
    float2 s2 = make_float2(0.f, 0.f), w2 = make_float2(0.f, 0.f);
    if constexpr (TOP) {
      if (tid == 0) best.count = 0;  // ahead of the barriers of the first threshold
    }
    if constexpr (HOLES) {  // the teacher's entries of this part
      if (tid < p.entries) {
        const long long id = load_id(p.ids, (long long)it.row * p.entries + tid, p.id_bits);
        const long long e = id - 1 + it.off;
        const int v = (int)(e / V) - it.v0;
        if (id > 0 && v >= 0 && v < it.v1 - it.v0)
          atomicOr(reinterpret_cast<unsigned*>(holes) + (v >> 2), 1u << ((v & 3) * 8 + (int)(e % V)));
      }
      __syncthreads();
    }
#pragma unroll 1
    for (int tile = 0; tile < tiles; ++tile) {
      uint4 cur[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) cur[u] = next[u];
      if (tile == 0) {
        nit = it;
        nhave = advance(nit);
      }
      if (tile + 1 < tiles) load(it, tile + 1);
      else if (nhave) load(nit, 0);
      float vmax[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        float f[V];
        unpack_row<T>(cur[u], f);
        if constexpr (HOLES) {
          const int v = tile * kTile + u * kThreads + tid;
          const unsigned hole = v < it.v1 - it.v0 ? holes[v] : 0u;
          if (hole)
#pragma unroll
            for (int i = 0; i < V; ++i)
              if (hole >> i & 1) f[i] = -INFINITY;
        }
        float most = f[0];
#pragma unroll
        for (int i = 1; i < V; ++i) most = fmaxf(most, f[i]);
        vmax[u] = most;
        gm = fmaxf(gm, most);
        if ((most - m) * p.c > kSlack) {
          const float d = fmaxf((m - most) * p.c, kLowest), r = ex2_approx_ftz(d);
          if constexpr (ENTROPY) {
            w2.x = r * fmaf(s2.x, d, w2.x);
            w2.y = r * fmaf(s2.y, d, w2.y);
          }
          s2.x *= r;
          s2.y *= r;
          m = most;
        }
        const float2 minus = make_float2(-m, -m), cc = make_float2(p.c, p.c);
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          float2 t = mul_pair(add_pair(make_float2(f[i], f[i + 1]), minus), cc);
          const float2 e = make_float2(ex2_approx_ftz(t.x), ex2_approx_ftz(t.y));
          s2 = add_pair(s2, e);
          if constexpr (ENTROPY) {
            t.x = fmaxf(t.x, kLowest);
            t.y = fmaxf(t.y, kLowest);
            w2 = fma_pair(e, t, w2);
          }
        }
      }
      if constexpr (TOP) {
        if (tile == 0) theta = group_threshold(gm, p.top, best);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (vmax[u] > theta) {
            float f[V];
            unpack_row<T>(cur[u], f);
            const int e0 = (it.v0 + tile * kTile + u * kThreads + tid) * V - it.off;
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
        if (tile > 0 && (tile & (tile + 1)) == 0 && tile + 1 < tiles) theta = group_threshold(gm, p.top, best);
      }
    }

    // The threads meet at the maximum of the part.
    float top_max = ctb::warp_max(gm);
    if (lane == 0) sh.red[0][warp] = top_max;
    __syncthreads();
    top_max = sh.red[0][0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) top_max = fmaxf(top_max, sh.red[0][i]);
    top_max = fmaxf(top_max, -FLT_MAX);
    {
      const float d = (m - top_max) * p.c, r = ex2_approx_ftz(d);
      const float s = s2.x + s2.y, w = r * fmaf(s, fmaxf(d, kLowest), w2.x + w2.y);
      const float a = ctb::warp_sum(s * r), b = ENTROPY ? ctb::warp_sum(w) : 0.f;
      if (lane == 0) {
        sh.red[1][warp] = a;
        sh.red[2][warp] = b;
      }
    }
    if constexpr (TOP) {
      __syncthreads();
      int n = best.count;
      const Range<T> range = {it.src, it.off, p.n, it.v0, it.v1};
      if (n > kCand) {
        n = radix_list(range, p.top, best);
      } else if (n < p.top) {
        // theta of the first tile: with fewer than k above it, it is also the last one
        const Range<T> first = {it.src, it.off, p.n, it.v0, min(it.v1, it.v0 + kTile)};
        n = append_equal(first, theta, n, p.top - n, best);
      }
      select_list(n, p.top, best);
    } else {
      __syncthreads();
    }
    float sum = 0.f, wsum = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      sum += sh.red[1][i];
      wsum += sh.red[2][i];
    }

    bool finish = true;
    if (p.parts > 1) {
      const int stride = record_floats(p.top);
      float* record = p.scratch + ((long long)it.row * p.parts + it.part) * stride;
      if (tid == 0) *reinterpret_cast<float4*>(record) = make_float4(top_max, sum, wsum, 0.f);
      if constexpr (TOP) {
        if (tid < p.top) {
          const int id = best.out_index[tid];
          record[4 + tid] = id >= 0 ? best.out_value[tid] : -INFINITY;
          reinterpret_cast<int*>(record)[4 + p.top + tid] = id;
        }
      }
      __threadfence();
      __syncthreads();
      if (tid == 0) sh.last = atomicInc(p.tickets + it.row, p.parts - 1) == (unsigned)p.parts - 1;
      __syncthreads();
      finish = sh.last;
      if (finish) {
        __threadfence();
        const float* all = p.scratch + (long long)it.row * p.parts * stride;
        const float4 mine = lane < p.parts ? __ldcg(reinterpret_cast<const float4*>(all + (long long)lane * stride))
                                           : make_float4(-FLT_MAX, 0.f, 0.f, 0.f);
        top_max = ctb::warp_max(mine.x);
        const float d = (mine.x - top_max) * p.c, r = ex2_approx_ftz(d);
        sum = ctb::warp_sum(mine.y * r);
        wsum = ctb::warp_sum(r * fmaf(mine.y, fmaxf(d, kLowest), mine.z));
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
    }

    if (finish) {
      if constexpr (OP == LOGPROBS) {
        const float log_sum = logf(sum), base = top_max / p.temperature;
        if (tid == 0) {
          if (p.lse) p.lse[it.row] = base + log_sum;
          if (p.entropy) p.entropy[it.row] = log_sum - kLn2 * (wsum / sum);
          if (p.logprobs) {
            if (it.token > p.n || it.token < 0) atomicMax(p.status, DEV_BAD_INDEX);
            p.logprobs[it.row] = it.token > p.n || it.token < 0 ? NAN : (it.x_token - top_max) / p.temperature - log_sum;
          }
        }
        if constexpr (TOP) {
          if (tid < p.top) {
            const int id = best.out_index[tid];
            p.top_logprobs[(long long)it.row * p.top + tid] = id >= 0 ? (best.out_value[tid] - top_max) / p.temperature - log_sum : NAN;
            p.top_ids[(long long)it.row * p.top + tid] = id + 1;
          }
        }
      } else if (warp == 0) {
        finish_distill<T, HOLES>(p, it.row, it.src, top_max, sum, sh);
      }
    }
    if constexpr (OP == DISTILL_GRAD) {  // one part: the row is read again, from L2
      __syncthreads();
      T* dst = static_cast<T*>(p.dx) + it.row * p.ld_dx;
      const int id = tid < p.entries ? sh.entry[tid] : 0;
      const float x = id ? to_float(it.src[id - 1]) : 0.f;
      const float lse2 = sh.grad[0] * kLog2e, g = p.d_loss[it.row] / p.temperature;
      __syncthreads();  // dst may be the logits themselves
      stream_gradient<T, false>(it.src, dst, it.off, p.n, it.v0, it.v1, p.c, lse2, g * sh.grad[1], 0.f);
      __syncthreads();
      patch_entries<T>(dst, p.entries, x, p.c, lse2, g, sh.grad[2], sh, 0, p.n);
    }
    if constexpr (HOLES) {
      __syncthreads();
      if (tid < p.entries) {
        const long long id = load_id(p.ids, (long long)it.row * p.entries + tid, p.id_bits);
        const int v = (int)((id - 1 + it.off) / V) - it.v0;
        if (id > 0 && v >= 0 && v < it.v1 - it.v0) holes[v] = 0;
      }
    }
    __syncthreads();  // what the row left in shared memory has been read
    it = nit;
    have = nhave;
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
// and of the distillation loss: g/temperature p_v outside, or g/temperature (all p_v - q_v) where the teacher lists v.
// A CTA takes part after part; the few places that a gradient meets directly are written behind the part's stream.
template <typename T, int OP>
__global__ void __launch_bounds__(kThreads, 4) logits_backward_kernel(const __grid_constant__ Backward p) {
  constexpr int V = 16 / (int)sizeof(T);
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 31;
  grid_dependency_sync();
  const long long items = (long long)p.rows * p.parts;
  for (long long at = blockIdx.x; at < items; at += gridDim.x) {
    const long long row = at / p.parts;
    const int part = (int)(at - row * p.parts);
    const T* src = static_cast<const T*>(p.x) + row * p.ld;
    T* dst = static_cast<T*>(p.dx) + row * p.ld_dx;
    const int off = (int)(((uintptr_t)src & 15) / sizeof(T)), nvec = (off + p.n + V - 1) / V;
    const int v0 = min(nvec, part * p.per), v1 = min(nvec, v0 + p.per);
    const long long lo = max(0ll, (long long)v0 * V - off), hi = (long long)v1 * V - off;  // ids (lo, hi] lie in this part
    if constexpr (OP == LOGPROBS) {
      const long long token = p.tokens ? load_id(p.tokens, row, p.token_bits) : -1;
      const bool bad = p.tokens && (token < 0 || token > p.n);
      if (token == 0 || bad) {
        if (bad && tid == 0) atomicMax(p.status, DEV_BAD_INDEX);
        stream_zeros<T>(dst, off, p.n, v0, v1);
        continue;
      }
      const float g0 = p.d_logprobs ? p.d_logprobs[row] : 0.f, gh = p.d_entropy ? p.d_entropy[row] : 0.f;
      const float h = p.d_entropy ? p.entropy[row] : 0.f, lse2 = p.lse[row] * kLog2e;
      float all = lane < p.top ? p.d_top[row * p.top + lane] : 0.f;
      all = g0 + ctb::warp_sum(all);
      // entries: the alternatives, then the token
      const int entries = p.top + (p.d_logprobs ? 1 : 0);
      __syncthreads();
      if (tid < entries) {
        long long id = tid < p.top ? p.top_ids[row * p.top + tid] : token;
        if (id < 0 || id > p.n) {
          atomicMax(p.status, DEV_BAD_INDEX);
          id = 0;
        }
        sh.entry[tid] = (int)id;
        sh.q[tid] = tid < p.top ? p.d_top[row * p.top + tid] : g0;
      }
      __syncthreads();
      const int id = tid < entries ? sh.entry[tid] : 0;
      const float x = id > lo && id <= hi ? to_float(src[id - 1]) : 0.f;
      const float a = -(all + gh * h) / p.temperature, b = -gh * kLn2 / p.temperature;
      __syncthreads();  // dst may be the logits themselves
      if (p.d_entropy) stream_gradient<T, true>(src, dst, off, p.n, v0, v1, p.c, lse2, a, b);
      else stream_gradient<T, false>(src, dst, off, p.n, v0, v1, p.c, lse2, a, 0.f);
      __syncthreads();
      if (id > lo && id <= hi) {
        float g = 0.f;
        bool again = false;
        for (int i = 0; i < entries; ++i)
          if (sh.entry[i] == id) {
            again |= i < tid;
            g += sh.q[i];
          }
        const float t = fmaf(x, p.c, -lse2);
        if (!again) dst[id - 1] = from_float<T>(g / p.temperature + ex2_approx_ftz(t) * fmaf(b, fmaxf(t, kLowest), a));
      }
    } else {
      const float4 saved = reinterpret_cast<const float4*>(p.saved)[row];
      if (saved.z == 0.f) {
        stream_zeros<T>(dst, off, p.n, v0, v1);
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
        sh.entry[tid] = (int)id;
        sh.q[tid] = (float)exp((double)load_value(p.values, row * p.entries + tid, p.values_dtype) / (double)p.temperature - norm);
      }
      __syncthreads();
      const int id = tid < p.entries ? sh.entry[tid] : 0;
      const float x = id > lo && id <= hi ? to_float(src[id - 1]) : 0.f;
      __syncthreads();  // dst may be the logits themselves
      stream_gradient<T, false>(src, dst, off, p.n, v0, v1, p.c, lse2, g * outside, 0.f);
      __syncthreads();
      patch_entries<T>(dst, p.entries, x, p.c, lse2, g, all, sh, lo, hi);
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
void cut_rows(ctb_ctx* ctx, int64_t rows, int64_t nvec, int64_t least, int most, int* parts, int* per) {
  const int64_t places = 4ll * ctx->sm_count;
  int64_t n = rows >= places ? 1 : places / rows;
  n = std::min<int64_t>(n, (nvec + kTile - 1) / kTile);
  n = std::min<int64_t>(std::max(n, least), most);
  int64_t v = (nvec + n - 1) / n;
  v = (v + 31) / 32 * 32;
  *per = (int)v;
  *parts = (int)((nvec + v - 1) / v);
}

template <typename T, int OP, bool TOP, bool HOLES>
int launch_forward(ctb_ctx* ctx, cudaStream_t st, Forward p, const char* who) {
  constexpr int V = 16 / (int)sizeof(T);
  const int64_t nvec = (p.n + V - 1) / V + 1;  // a row that starts off a vector boundary touches one more
  const int record = record_floats(p.top);
  int most = kMaxParts;
  if (p.rows > kTickets || OP == DISTILL_GRAD) most = 1;
  else most = std::max<int>(1, std::min<int64_t>(most, kStreamScratchBytes / sizeof(float) / record / p.rows));
  if (TOP) most = std::min(most, kCand / p.top);
  const int64_t least = HOLES ? (nvec + kMostHoles - 1) / kMostHoles : 1;
  cut_rows(ctx, p.rows, nvec, least, most, &p.parts, &p.per);
  size_t smem = 0;
  if (HOLES) {
    smem = ((size_t)p.per + 15) / 16 * 16;
    if (smem > kMostHoles + 64)
      return fail(CTB_UNSUPPORTED, "%s: with teacher_lse, %d rows of %d elements are too long", who, p.rows, p.n);
    cudaError_t e = allow_smem(logits_forward_kernel<T, OP, TOP, HOLES>, kMostHoles + 64);
    if (e != cudaSuccess) return cuda_fail(e, who);
  }
  auto go = [&] {
    const int64_t items = (int64_t)p.rows * p.parts;
    int per_sm = 4;
    if (HOLES) {
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, logits_forward_kernel<T, OP, TOP, HOLES>, kThreads, smem);
      per_sm = std::max(1, std::min(4, per_sm));
    }
    const int grid = (int)std::min<int64_t>(items, (int64_t)per_sm * ctx->sm_count);
    launch_kernel(logits_forward_kernel<T, OP, TOP, HOLES>, grid, kThreads, smem, st, 0, p);
  };
  if (p.parts > 1) {
    StreamScratch scratch(ctx, st);
    if (scratch.data) {
      p.scratch = scratch.data;
      p.tickets = scratch.tickets;
      go();
      CTB_CHECK_LAUNCH(who);
      return CTB_OK;
    }
    p.parts = 1;
    p.per = (int)((nvec + 31) / 32 * 32);
    if (HOLES && p.per > kMostHoles) return fail(CTB_UNSUPPORTED, "%s: no scratch for a row in parts", who);
    if (HOLES) smem = ((size_t)p.per + 15) / 16 * 16;
  }
  go();
  CTB_CHECK_LAUNCH(who);
  return CTB_OK;
}

template <int OP, bool TOP, bool HOLES>
int forward_by_type(ctb_ctx* ctx, cudaStream_t st, const Forward& p, int dtype, const char* who) {
  if (dtype == CTB_F32) return launch_forward<float, OP, TOP, HOLES>(ctx, st, p, who);
  if (dtype == CTB_F16) return launch_forward<__half, OP, TOP, HOLES>(ctx, st, p, who);
  return launch_forward<__nv_bfloat16, OP, TOP, HOLES>(ctx, st, p, who);
}

template <typename T, int OP>
int launch_backward(ctb_ctx* ctx, cudaStream_t st, Backward p, const char* who) {
  constexpr int V = 16 / (int)sizeof(T);
  const int64_t nvec = (p.n + V - 1) / V + 1;
  // parts of at most four tiles, and of one where that spreads the work over more SMs
  const int64_t tiles = p.rows * ((nvec + kTile - 1) / kTile);
  const int64_t want = tiles >= 16ll * ctx->sm_count ? 4 : 1;
  const int64_t parts = (nvec + want * kTile - 1) / (want * kTile);
  p.per = (int)(((nvec + parts - 1) / parts + 31) / 32 * 32);
  p.parts = (int)((nvec + p.per - 1) / p.per);
  const int grid = (int)std::min<int64_t>((int64_t)p.rows * p.parts, 4ll * ctx->sm_count);
  launch_kernel(logits_backward_kernel<T, OP>, grid, kThreads, 0, st, 0, p);
  CTB_CHECK_LAUNCH(who);
  return CTB_OK;
}
template <int OP>
int backward_by_type(ctb_ctx* ctx, cudaStream_t st, const Backward& p, int dtype, const char* who) {
  if (dtype == CTB_F32) return launch_backward<float, OP>(ctx, st, p, who);
  if (dtype == CTB_F16) return launch_backward<__half, OP>(ctx, st, p, who);
  return launch_backward<__nv_bfloat16, OP>(ctx, st, p, who);
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
  Forward p = {};
  p.x = logits; p.ld = ld; p.n = (int)V; p.rows = (int)T;
  p.c = (float)(1.4426950408889634 / (double)temperature);
  p.temperature = temperature;
  p.status = ctx->dev_status;
  p.tokens = tokens; p.token_bits = token_bits; p.top = top;
  p.logprobs = logprobs; p.entropy = entropy; p.lse = lse; p.top_logprobs = top_logprobs; p.top_ids = top_ids;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (top) return forward_by_type<LOGPROBS, true, false>(ctx, st, p, dtype, who);
  return forward_by_type<LOGPROBS, false, false>(ctx, st, p, dtype, who);
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
  return backward_by_type<LOGPROBS>(ctx, static_cast<cudaStream_t>(stream), p, dtype, who);
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
  Forward p = {};
  p.x = logits; p.ld = ld; p.n = (int)V; p.rows = (int)T;
  p.c = (float)(1.4426950408889634 / (double)temperature);
  p.temperature = temperature;
  p.status = ctx->dev_status;
  p.ids = teacher_ids; p.id_bits = id_bits; p.entries = entries; p.values = teacher_values; p.values_dtype = values_dtype;
  p.teacher_lse = teacher_lse; p.loss = loss; p.saved = saved;
  p.d_loss = d_loss; p.dx = d_logits; p.ld_dx = ld_out;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d_logits)
    return teacher_lse ? forward_by_type<DISTILL_GRAD, false, true>(ctx, st, p, dtype, who)
                       : forward_by_type<DISTILL_GRAD, false, false>(ctx, st, p, dtype, who);
  return teacher_lse ? forward_by_type<DISTILL, false, true>(ctx, st, p, dtype, who)
                     : forward_by_type<DISTILL, false, false>(ctx, st, p, dtype, who);
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
  return backward_by_type<DISTILL>(ctx, static_cast<cudaStream_t>(stream), p, dtype, who);
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
  const int64_t nvec = V / (16 / elem_size(dtype)) + 2;
  // One kernel where there are rows enough to give every SM its own, else the two halves, which cut rows into parts.
  if (T >= 2 * ctx->sm_count && !(teacher_lse && nvec > kMostHoles))
    return distill_forward(who, ctx, stream, logits, teacher_ids, id_bits, teacher_values, values_dtype, teacher_lse, loss, saved, d_loss,
                           d_logits, V, T, ld_out, ld, entries, temperature, dtype);
  if (int s = distill_forward(who, ctx, stream, logits, teacher_ids, id_bits, teacher_values, values_dtype, teacher_lse, loss, saved, nullptr,
                              nullptr, V, T, 0, ld, entries, temperature, dtype))
    return s;
  return distill_backward(who, ctx, stream, d_logits, logits, teacher_ids, id_bits, teacher_values, values_dtype, saved, d_loss, V, T, ld_out,
                          ld, entries, temperature, dtype);
}
