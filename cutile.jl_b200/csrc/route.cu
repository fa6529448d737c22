// Routing of tokens to experts by given logits, and its gradient, for sm_100a.
//
//   s = softmax(x) or sigmoid(x)       c = s + bias (for the choice only)
//   a group of experts scores the sum of its one or two best c; experts outside of the best groups are out
//   the k best c are chosen (ties to the lowest expert), w = scale s / max(sum of the chosen s, 1e-20), or scale s
// The bias balances the experts' load and takes no gradient.
//
// A warp takes a token, lane l experts l * EPL ... + EPL - 1, a chunk of the row that is read as 16-byte vectors.  The work is tiny (1 KB of
// logits per token of 256 experts), so latency bounds it: of the selection rounds and of the launch.  A round is one integer maximum over
// the warp (the order of f32 as that of 32-bit words) and one ballot; ties end at the lowest lane and its lowest expert.
//
// What is chosen must not hang on a rounding.  Where the order of c is that of x (no bias, and no sum of two scores per group), x itself is
// compared, and no exponential is taken but those of the chosen (and of the softmax's sum, where the weights need it).  Elsewhere c is
// computed in f32 together with a bound of its error: where two neighbours in the order lie closer than the bound and are not alike in both
// logit and bias, the warp takes the token again in f64 (one token of 300 for normal logits; that path costs 5 times the other).
#include <float.h>

#include <algorithm>

#include "ctx.h"
#include "ptx.cuh"
#include "rows.cuh"

using namespace ctb;
using namespace ctb_internal;

namespace {

constexpr int kThreads = 256;  // eight tokens: their ids fill a 32-byte sector
constexpr int kWarps = kThreads / 32;
constexpr int kMaxExperts = 512;
constexpr int kMaxTopk = 32;

struct Route {
  const void* x;
  const float* bias;
  int* ids;
  void* weights;
  int weights_dtype;
  long long ld;
  unsigned tokens;
  int experts, topk, sigmoid, groups, topk_groups, group_top, renormalize;
  float scale;
  int wide;           // rows (and bias) can be read as vectors
  int lanes_a_group;  // a power of two where the lanes' chunks make up groups, else 0
};

__device__ __forceinline__ void store_weight(void* p, long long i, int dtype, float v) {
  if (dtype == CTB_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == CTB_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ float load_weight(const void* p, long long i, int dtype) {
  if (dtype == CTB_F32) return static_cast<const float*>(p)[i];
  if (dtype == CTB_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// Words in the order of the numbers; NaN and -inf as 1, the least that exists.  In f64 that one counts as the lowest finite number.
__device__ __forceinline__ uint32_t word_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);  // -0 is 0
  return v > -INFINITY ? b ^ (0x80000000u | (uint32_t)((int)b >> 31)) : 1u;
}
__device__ __forceinline__ uint64_t word_of(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return v > -INFINITY ? b ^ (0x8000000000000000ull | (uint64_t)((int64_t)b >> 63)) : 1ull;
}
__device__ __forceinline__ float number_of(uint32_t w) {
  return w > 1 ? __uint_as_float(w ^ (w >> 31 ? 0x80000000u : 0xffffffffu)) : -INFINITY;
}
__device__ __forceinline__ double number_of(uint64_t w) {
  return w > 1 ? __longlong_as_double((long long)(w ^ (w >> 63 ? 0x8000000000000000ull : ~0ull))) : -DBL_MAX;
}
// The largest word of the warp, and the lowest lane that has it.
__device__ __forceinline__ uint32_t top_word(uint32_t w, int& who) {
  const uint32_t top = __reduce_max_sync(0xffffffffu, w);
  who = __ffs(__ballot_sync(0xffffffffu, w == top)) - 1;
  return top;
}
__device__ __forceinline__ uint64_t top_word(uint64_t w, int& who) {
  const uint32_t high = (uint32_t)(w >> 32), top = __reduce_max_sync(0xffffffffu, high);
  const uint32_t low = __reduce_max_sync(0xffffffffu, high == top ? (uint32_t)w : 0u);
  const uint64_t both = (uint64_t)top << 32 | low;
  who = __ffs(__ballot_sync(0xffffffffu, w == both)) - 1;
  return both;
}
// e^v to a relative 2^-22 where it is a normal f32: expf of v's leading bits, and the rest's first order.
__device__ __forceinline__ float exp_of(double v) {
  const float high = (float)v, e = expf(high);
  return fmaf(e, (float)(v - (double)high), e);
}
// A lane's chunk of a row: EPL elements from `at` on, -inf from `end` on.  wide: chunks are vectors, and end a multiple of EPL.
template <int BYTES>
struct alignas(BYTES < 16 ? BYTES : 16) Chunk {
  uint32_t w[(BYTES + 3) / 4];
};
template <typename T, int EPL>
__device__ __forceinline__ void load_chunk(const T* src, int at, int end, bool wide, float (&x)[EPL]) {
  constexpr int kBytes = EPL * sizeof(T);
  if constexpr (kBytes >= 4) {
    if (wide) {
      Chunk<kBytes> c = {};
      if (at < end) c = *reinterpret_cast<const Chunk<kBytes>*>(src + at);
#pragma unroll
      for (int i = 0; i < EPL; ++i) x[i] = at < end ? to_float(reinterpret_cast<const T*>(c.w)[i]) : -INFINITY;
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) x[i] = at + i < end ? to_float(src[at + i]) : -INFINITY;
}
template <typename T, int EPL>
__device__ __forceinline__ void store_chunk(T* dst, int at, int end, bool wide, const float (&x)[EPL]) {
  constexpr int kBytes = EPL * sizeof(T);
  if constexpr (kBytes >= 4) {
    if (wide) {
      Chunk<kBytes> c;
#pragma unroll
      for (int i = 0; i < EPL; ++i) reinterpret_cast<T*>(c.w)[i] = from_float<T>(x[i]);
      if (at < end) *reinterpret_cast<Chunk<kBytes>*>(dst + at) = c;
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (at + i < end) dst[at + i] = from_float<T>(x[i]);
}

// A token; a warp.  scratch: a word per expert of its own, where lanes' chunks do not make up groups.  True: nothing has been written, the
// order is in doubt (never with EXACT).
template <typename T, int EPL, bool EXACT>
__device__ __forceinline__ bool route_token(const Route& p, unsigned t, void* scratch) {
  using Word = typename std::conditional<EXACT, uint64_t, uint32_t>::type;
  using Number = typename std::conditional<EXACT, double, float>::type;
  const int lane = threadIdx.x & 31, first = lane * EPL;
  const bool grouped = p.topk_groups < p.groups;
  const bool by_logit = !EXACT && !p.bias && !(grouped && p.group_top == 2);
  float x[EPL], most = -INFINITY;
  bool odd = false;
  load_chunk<T, EPL>(static_cast<const T*>(p.x) + (long long)t * p.ld, first, p.experts, p.wide, x);
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    most = fmaxf(most, x[i]);
    odd |= !(x[i] < INFINITY);
  }
  most = number_of(__reduce_max_sync(0xffffffffu, word_of(most)));
  if (!EXACT && (__any_sync(0xffffffffu, odd) || most == -INFINITY)) return true;
  // 1. words of c, 0 for what does not exist.  Errors of f32 scores, with the bounds of __expf (2 + 1.2 |v| steps) and __fdividef (2 steps):
  // a sigmoid is off by s (1 - s) (2 + 1.2 |x|) 2^-23 + 2^-24 + 2^-22 < 2^-21, a softmax by 2^-17 of its largest score.
  Word word[EPL];
  double sum = 1;
  float error = 0.f;  // of a score, at most
  if (!p.sigmoid && !(by_logit && p.renormalize)) {
    sum = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      if constexpr (EXACT) {
        if (first + i < p.experts) sum += exp((double)x[i] - (double)most);
      } else {
        const float d = x[i] - most, e = expf(d), back = d + most;  // d and what it lost: x - most = d + ((x - back) - (most - (back - d)))
        sum += (double)(x[i] > -INFINITY ? fmaf(e, (x[i] - back) - (most - (back - d)), e) : 0.f);
      }
    }
    sum = sum_lanes(sum);
  }
  if (by_logit) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) word[i] = word_of((Number)x[i]);
  } else {
    const float rate = 1.f / (float)sum;
    error = p.sigmoid ? 0x1p-21f : 0x1p-17f * rate;
    float bias[EPL];
    if (p.bias) load_chunk<float, EPL>(p.bias, first, p.experts, p.wide, bias);
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      Number s;
      if constexpr (EXACT) s = p.sigmoid ? 1 / (1 + exp(-(double)x[i])) : exp((double)x[i] - (double)most) / sum;
      else s = p.sigmoid ? __fdividef(1.f, 1.f + __expf(-x[i])) : __expf(x[i] - most) * rate;
      word[i] = word_of(p.bias ? s + (Number)bias[i] : s);
    }
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (first + i >= p.experts) word[i] = 0;
  // 2. groups
  if (grouped) {
    const int size = p.experts / p.groups;
    Word a = 0, b = 0;  // the lane's group's best two
    if (p.lanes_a_group) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        b = max(b, min(a, word[i]));
        a = max(a, word[i]);
      }
      for (int o = 1; o < p.lanes_a_group; o <<= 1) {
        const Word oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
        b = max(max(b, ob), min(a, oa));
        a = max(a, oa);
      }
      a = __shfl_sync(0xffffffffu, a, lane * p.lanes_a_group);
      b = __shfl_sync(0xffffffffu, b, lane * p.lanes_a_group);
    } else {
      Word* v = static_cast<Word*>(scratch);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (first + i < p.experts) v[first + i] = word[i];
      __syncwarp();
      if (lane < p.groups)
        for (int i = 0; i < size; ++i) {
          const Word w = v[lane * size + i];
          b = max(b, min(a, w));
          a = max(a, w);
        }
      __syncwarp();
    }
    const Number score = p.group_top == 2 ? number_of(a) + number_of(b) : number_of(a);  // lane g: of group g
    float slack = 0.f;
    if (!EXACT && !by_logit)
      slack = p.group_top == 2 ? 2 * error + (fabsf((float)number_of(a)) + fabsf((float)number_of(b))) * 0x1p-22f
                               : error + fabsf((float)number_of(a)) * 0x1p-22f;
    int rank = 0;
    unsigned close = 0;
    for (int g = 0; g < p.groups; ++g) {
      const Number o = __shfl_sync(0xffffffffu, score, g);
      rank += o > score || (o == score && g < lane);
      if constexpr (!EXACT) {
        const float s = __shfl_sync(0xffffffffu, slack, g);
        if (!by_logit && !(fabsf(o - score) > s + slack)) close |= 1u << g;
      }
    }
    const bool in = lane < p.groups && rank < p.topk_groups;
    const unsigned kept = __ballot_sync(0xffffffffu, in);
    if (!EXACT && __any_sync(0xffffffffu, in && (close & ~kept) != 0)) return true;  // close groups, one kept and the other out
    if (p.lanes_a_group) {
      if (!(kept >> (lane / p.lanes_a_group) & 1)) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) word[i] = 0;
      }
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (first + i < p.experts && !(kept >> ((first + i) / size) & 1)) word[i] = 0;
    }
  }
  const bool sure = !EXACT && !p.bias;  // the order is that of the logits
  if (sure && !by_logit) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) word[i] = word[i] ? word_of((Number)x[i]) : 0;
  }
  // 3. the choices, and where their order can be in doubt the two after them
  Word my_word = 0;  // lane j: word and expert of the j-th choice
  int my_id = 0;
  const bool mine = lane < p.topk;
  const int rounds = sure || EXACT ? p.topk : min(p.topk + 2, 32);
  if (!EXACT && sizeof(T) == 2 && sure) {
    // 16-bit logits take 19 bits as f32, and leave room for the expert: no two words are alike
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (word[i]) word[i] = (max((uint32_t)word[i], 512u) & ~511u) | (uint32_t)(511 - first - i);
    for (int j = 0; j < rounds; ++j) {
      uint32_t best = 0;
#pragma unroll
      for (int i = 0; i < EPL; ++i) best = max(best, (uint32_t)word[i]);
      best = __reduce_max_sync(0xffffffffu, best);
      if (lane == j) my_word = best;
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (word[i] == best) word[i] = 0;
    }
    my_id = mine ? 511 - (int)(my_word & 511) : 0;
  } else {
    for (int j = 0; j < rounds; ++j) {
      Word best = 0;
#pragma unroll
      for (int i = 0; i < EPL; ++i) best = max(best, word[i]);
      int who, at = 0;
      const Word top = top_word(best, who);
#pragma unroll
      for (int i = EPL - 1; i >= 0; --i)
        if (word[i] == top) at = i;
      const int id = __shfl_sync(0xffffffffu, first + at, who);
      if (lane == j) {
        my_word = top;
        my_id = id;
      }
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (id == first + i) word[i] = 0;
    }
  }
  float my_x = 0.f;
  if (lane < rounds && (mine || my_word)) my_x = to_float(static_cast<const T*>(p.x)[(long long)t * p.ld + my_id]);
  if constexpr (!EXACT) {
    // far from where scores of different logits may be alike
    if (__any_sync(0xffffffffu, mine && (p.sigmoid ? !(my_x >= -80.f && my_x <= 16.f) : !(my_x - most >= -80.f)))) return true;
    if (!sure) {
      const bool there = lane < rounds && my_word > 1;
      const float my_bias = there ? p.bias[my_id] : 0.f, c = there ? number_of(my_word) : -INFINITY;
      float next = __shfl_down_sync(0xffffffffu, c, 1);
      const float next_x = __shfl_down_sync(0xffffffffu, my_x, 1);
      const float next_bias = __shfl_down_sync(0xffffffffu, my_bias, 1);
      if (p.topk == 32) {  // no lane holds what comes after the last choice
        Word best = 0;
#pragma unroll
        for (int i = 0; i < EPL; ++i) best = max(best, word[i]);
        int who;
        best = top_word(best, who);
        if (lane == 31) next = best > 1 ? number_of(best) : -INFINITY;
      }
      auto close = [&](float below) { return there && below > -INFINITY && !(c - below > 2 * error + (fabsf(c) + fabsf(below)) * 0x1p-22f); };
      // Alike in both, two choices are in order.  What comes after the last one is not: behind it there may be one that is only close.
      const bool doubt = mine && close(next) && (lane == p.topk - 1 || !(my_x == next_x && my_bias == next_bias));
      if (__any_sync(0xffffffffu, doubt)) {
        // The choices and the one after them in f64, where the next one cannot be among the best either.
        const float second = __shfl_sync(0xffffffffu, c, (p.topk + 1) & 31);
        if (!p.sigmoid || p.topk > 30 || __any_sync(0xffffffffu, lane == p.topk - 1 && close(second)) ||
            __any_sync(0xffffffffu, lane <= p.topk && !(there && fabsf(c) < INFINITY && my_x >= -80.f)))
          return true;
        const double exact = 1 / (1 + exp(-(double)my_x)) + (double)my_bias;
        int rank = 0;
        for (int j = 0; j <= p.topk; ++j) {
          const double o = __shfl_sync(0xffffffffu, exact, j);
          const int id = __shfl_sync(0xffffffffu, my_id, j);
          rank += o > exact || (o == exact && id < my_id);
        }
        int from = 0;
        for (int j = 0; j <= p.topk; ++j) {
          const int r = __shfl_sync(0xffffffffu, rank, j);
          if (r == lane) from = j;
        }
        my_id = __shfl_sync(0xffffffffu, my_id, from);
        my_x = __shfl_sync(0xffffffffu, my_x, from);
        if (__any_sync(0xffffffffu, mine && my_x > 16.f)) return true;
      }
    }
  }
  // 4. weights, from accurate scores of the chosen
  double s = 0;
  if (mine) {
    const double v = p.sigmoid ? -(double)my_x : (double)my_x - (double)most, e = EXACT ? exp(v) : (double)exp_of(v);
    s = p.sigmoid ? 1 / (1 + e) : e / sum;
  }
  double scale = p.scale;
  if (p.renormalize) {
    const double chosen = sum_lanes(s);
    scale /= chosen < 1e-20 ? 1e-20 : chosen;
  }
  if (mine) {
    const long long at = (long long)lane * p.tokens + t;
    p.ids[at] = my_id + 1;
    store_weight(p.weights, at, p.weights_dtype, (float)(s * scale));
  }
  return false;
}
template <typename T, int EPL>
__device__ __noinline__ void route_exactly(const Route& p, unsigned t, void* scratch) {
  route_token<T, EPL, true>(p, t, scratch);
}

template <typename T, int EPL>
__global__ void __launch_bounds__(kThreads, EPL <= 4 ? 6 : EPL <= 8 ? 5 : 2) route_kernel(const __grid_constant__ Route p) {
  extern __shared__ double scratch[];  // with groups that are not lanes' chunks
  const int warp = threadIdx.x >> 5;
  grid_dependency_wait();
  for (unsigned t = blockIdx.x * kWarps + warp; t < p.tokens; t += gridDim.x * kWarps) {  // 2^31 and a round more at most
    if (route_token<T, EPL, false>(p, t, scratch + warp * p.experts)) route_exactly<T, EPL>(p, t, scratch + warp * p.experts);
    __syncwarp();
  }
  grid_dependency_launch();
}

struct RouteBackward {
  const void* x;
  void* dx;
  const void* ids;
  int id_bits;
  const void* d_weights;
  int weights_dtype;
  long long ld, ld_dx;
  unsigned tokens;
  int experts, topk, sigmoid, renormalize;
  float scale;
  int* status;
  int wide;
};

// With dw_j the gradient of the j-th weight (0 for the other experts), e a token's powers (softmax) or scores, S the sum of all powers, R that of
// the chosen e, C that of dw_j e_j, and s' = s (1 - s) of a sigmoid:
//   softmax: dx_v = scale / S e_v (dw_v - C / S)      renormalised: dx_v = scale / R e_v (dw_v - C / R) for the chosen, else 0
//   sigmoid: dx_v = scale s'_v dw_v                   renormalised: dx_v = scale / R s'_v (dw_v - C / R)
// (a chosen sum below 1e-20 is a constant, and the gradient that without renormalisation).  s' comes from e^-|x| without a difference.  The
// brackets are the sum of e_w (dw_v - dw_w), of which little is left where one expert has nearly all of it or the gradients are alike:
//   - renormalised, dw is taken relative to that of the largest chosen e: f32 is then off by (2 topk + 1) 2^-23 of the sum of sizes;
//   - else f32 is off by 17 * 2^-23 of it while an eighth of S is not chosen, and beyond S and C are f64 (f64 for all tokens: 16384 x 128 bf16
//     with its gradient 18.5 us for 17.4, for what conversions take).
template <typename T, int EPL>
__global__ void __launch_bounds__(kThreads) route_backward_kernel(const RouteBackward p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = lane * EPL;
  grid_dependency_wait();
  for (unsigned t = blockIdx.x * kWarps + warp; t < p.tokens; t += gridDim.x * kWarps) {
    const T* src = static_cast<const T*>(p.x) + (long long)t * p.ld;
    T* dst = static_cast<T*>(p.dx) + (long long)t * p.ld_dx;
    float s[EPL], most = -INFINITY;  // logits, then what they give to d
    load_chunk<T, EPL>(src, first, p.experts, p.wide, s);
    int id = 0;
    float dw = 0.f;
    if (lane < p.topk) {
      const long long at = (long long)lane * p.tokens + t;
      dw = load_weight(p.d_weights, at, p.weights_dtype);
      const long long e = p.id_bits == 64 ? static_cast<const long long*>(p.ids)[at] : static_cast<const int*>(p.ids)[at];
      if (e < 0 || e > p.experts) atomicMax(p.status, DEV_BAD_INDEX);
      else id = (int)e;
      if (!id) dw = 0.f;
    }
    float xj = 0.f;  // logit of this lane's choice, from the lane that holds it
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const float x = __shfl_sync(0xffffffffu, s[i], max(id - 1, 0) / EPL);
      if (max(id - 1, 0) % EPL == i) xj = x;
      most = fmaxf(most, s[i]);
    }
    float ej, all = 1.f;  // e of this lane's choice; S
    if (p.sigmoid) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const float e = expf(-fabsf(s[i])), inverse = 1.f / (1.f + e);
        s[i] = e * inverse * inverse;
      }
      const float e = expf(-fabsf(xj));
      ej = (xj < 0.f ? e : 1.f) / (1.f + e);
    } else {
      most = number_of(__reduce_max_sync(0xffffffffu, word_of(most)));
      all = 0.f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        s[i] = expf(s[i] - most);
        if (first + i < p.experts) all += s[i];
      }
      all = warp_sum(all);
      ej = expf(xj - most);
    }
    if (!id) ej = 0.f;
    float factor = p.scale, mean = 0.f, all_low = 0.f, mean_low = 0.f;  // mean: C
    bool apart = !p.sigmoid, exact = false;  // apart: from dw S - C, once what meets at an expert is added up
    if (p.renormalize) {
      const uint32_t bits = __float_as_uint(ej), top = __reduce_max_sync(0xffffffffu, bits);
      const float of = __shfl_sync(0xffffffffu, dw, __ffs(__ballot_sync(0xffffffffu, bits == top)) - 1);
      const float chosen = warp_sum(ej);
      mean = warp_sum((id ? dw - of : 0.f) * ej);
      if (chosen < 1e-20f * all) {
        factor *= 1e20f;
        mean = fmaf(of, chosen, mean);
      } else {
        apart = false;
        const float per = 1.f / chosen;
        dw = id ? fmaf(dw - of, chosen, -mean) * per : 0.f;
        factor *= per;
      }
    } else if (!p.sigmoid) {
      const unsigned chosen = __reduce_add_sync(0xffffffffu, (unsigned)(ej * 0x1p24f));  // near enough
      exact = (float)chosen > 0.875f * 0x1p24f * all;
      if (!exact) {
        mean = warp_sum(dw * ej);
      } else {
        double a = 0;
#pragma unroll
        for (int i = 0; i < EPL; ++i)
          if (first + i < p.experts) a += (double)s[i];
        a = sum_lanes(a);
        const double b = sum_lanes((double)dw * (double)ej);
        all = (float)a;
        all_low = (float)(a - (double)all);
        mean = (float)b;
        mean_low = (float)(b - (double)mean);
      }
    }
    float d[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) d[i] = 0.f;
    for (int j = 0; j < p.topk; ++j) {
      const int e = __shfl_sync(0xffffffffu, id, j) - 1;
      const float v = __shfl_sync(0xffffffffu, dw, j);
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (e == first + i) d[i] += v;
    }
    if (apart) {
      const float per = 1.f / all;
#pragma unroll
      for (int i = 0; i < EPL; ++i) d[i] = fmaf(d[i], all, -mean) + (exact ? fmaf(d[i], all_low, -mean_low) : 0.f);
      factor *= per * per;
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) d[i] *= factor * s[i];
    store_chunk<T, EPL>(dst, first, p.experts, p.wide, d);
  }
  grid_dependency_launch();
}

int check_route(const char* who, const void* logits, int64_t T, int64_t E, int64_t ld, int topk, int score, float scale, int dtype,
                int weights_dtype) {
  if (dtype != CTB_F32 && dtype != CTB_F16 && dtype != CTB_BF16) return fail(CTB_BAD_ARG, "%s: dtype must be CTB_F32, CTB_F16 or CTB_BF16", who);
  if (weights_dtype != CTB_F32 && weights_dtype != CTB_F16 && weights_dtype != CTB_BF16)
    return fail(CTB_BAD_ARG, "%s: the weights' type must be CTB_F32, CTB_F16 or CTB_BF16", who);
  if (T < 0 || E <= 0 || T > INT32_MAX) return fail(CTB_BAD_ARG, "%s: bad shape E=%lld T=%lld", who, (long long)E, (long long)T);
  if (E > kMaxExperts) return fail(CTB_UNSUPPORTED, "%s: at most %d experts are implemented, got %lld", who, kMaxExperts, (long long)E);
  if (ld < E) return fail(CTB_BAD_ARG, "%s: leading dimension smaller than E", who);
  if (topk < 1 || topk > E) return fail(CTB_BAD_ARG, "%s: topk must lie between 1 and the number of experts", who);
  if (topk > kMaxTopk) return fail(CTB_UNSUPPORTED, "%s: at most %d experts per token are implemented", who, kMaxTopk);
  if (score != CTB_SCORE_SOFTMAX && score != CTB_SCORE_SIGMOID) return fail(CTB_BAD_ARG, "%s: unknown score function %d", who, score);
  if (!(fabsf(scale) <= FLT_MAX)) return fail(CTB_BAD_ARG, "%s: scale must be finite", who);
  if (T == 0) return CTB_OK;
  if (!is_device_ptr(logits)) return fail(CTB_BAD_ARG, "%s: logits is not a device pointer", who);
  if ((uintptr_t)logits % (dtype == CTB_F32 ? 4 : 2)) return fail(CTB_BAD_ALIGN, "%s: logits must be aligned to their element size", who);
  return CTB_OK;
}

template <typename F>
void by_experts(int E, F f) {
  if (E <= 32) f(std::integral_constant<int, 1>());
  else if (E <= 64) f(std::integral_constant<int, 2>());
  else if (E <= 128) f(std::integral_constant<int, 4>());
  else if (E <= 256) f(std::integral_constant<int, 8>());
  else f(std::integral_constant<int, 16>());
}

// Whether chunks of `epl` elements of rows at p are vectors.
bool wide_rows(const void* p, long long ld, int experts, int epl, int elem) {
  const int bytes = std::min(16, epl * elem);
  return experts % epl == 0 && (uintptr_t)p % bytes == 0 && ld * elem % bytes == 0;
}
template <typename T>
int launch_route(ctb_ctx* ctx, cudaStream_t st, Route p) {
  const int grid = (int)std::min<int64_t>((p.tokens + kWarps - 1) / kWarps, 16ll * ctx->sm_count);
  by_experts(p.experts, [&](auto epl) {
    constexpr int kEach = decltype(epl)::value;
    const int size = p.experts / p.groups, lanes = size % kEach == 0 ? size / kEach : 0;
    p.lanes_a_group = (lanes & (lanes - 1)) == 0 ? lanes : 0;
    const size_t smem = p.topk_groups < p.groups && !p.lanes_a_group ? (size_t)kWarps * p.experts * sizeof(double) : 0;
    p.wide = wide_rows(p.x, p.ld, p.experts, kEach, sizeof(T)) && wide_rows(p.bias, 0, p.experts, kEach, sizeof(float));
    launch_kernel(route_kernel<T, kEach>, grid, kThreads, smem, st, 0, p);
  });
  CTB_CHECK_LAUNCH("ctb_moe_route launch");
  return CTB_OK;
}
template <typename T>
int launch_route_backward(ctb_ctx* ctx, cudaStream_t st, RouteBackward p) {
  const int grid = (int)std::min<int64_t>((p.tokens + kWarps - 1) / kWarps, 16ll * ctx->sm_count);
  by_experts(p.experts, [&](auto epl) {
    constexpr int kEach = decltype(epl)::value;
    p.wide = wide_rows(p.x, p.ld, p.experts, kEach, sizeof(T)) && wide_rows(p.dx, p.ld_dx, p.experts, kEach, sizeof(T));
    launch_kernel(route_backward_kernel<T, kEach>, grid, kThreads, 0, st, 0, p);
  });
  CTB_CHECK_LAUNCH("ctb_moe_route_bwd launch");
  return CTB_OK;
}

}  // namespace

extern "C" int ctb_moe_route(ctb_ctx* ctx, void* stream, const void* logits, const float* bias, int32_t* topk_ids, void* topk_weights,
                             int weights_dtype, int64_t T, int64_t E, int64_t ld, int topk, int score, int groups, int topk_groups,
                             int group_top, int renormalize, float scale, int dtype) {
  const char* who = "ctb_moe_route";
  CTB_CHECK_CTX(ctx);
  CurrentDevice current(ctx);
  if (int s = check_route(who, logits, T, E, ld, topk, score, scale, dtype, weights_dtype)) return s;
  if (groups < 1 || E % groups != 0) return fail(CTB_BAD_ARG, "%s: %lld experts cannot be cut into %d groups", who, (long long)E, groups);
  if (groups > 32) return fail(CTB_UNSUPPORTED, "%s: at most 32 groups are implemented", who);
  if (topk_groups < 1 || topk_groups > groups) return fail(CTB_BAD_ARG, "%s: topk_groups must lie between 1 and groups", who);
  if (topk > topk_groups * (E / groups))
    return fail(CTB_BAD_ARG, "%s: %d groups of %lld experts hold fewer than topk=%d", who, topk_groups, (long long)(E / groups), topk);
  if (group_top != 1 && group_top != 2) return fail(CTB_BAD_ARG, "%s: group_top must be 1 or 2", who);
  if (group_top == 2 && groups > topk_groups && E / groups < 2) return fail(CTB_BAD_ARG, "%s: group_top = 2 needs groups of two experts or more", who);
  if (T == 0) return CTB_OK;
  if (bias) CTB_CHECK_DEV(bias);
  CTB_CHECK_DEV(topk_ids);
  CTB_CHECK_DEV(topk_weights);
  const Route p = {logits, bias, topk_ids, topk_weights, weights_dtype, ld, (unsigned)T, (int)E, topk, score == CTB_SCORE_SIGMOID, groups, topk_groups,
                   group_top, renormalize != 0, scale, 0, 0};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == CTB_F32) return launch_route<float>(ctx, st, p);
  if (dtype == CTB_F16) return launch_route<__half>(ctx, st, p);
  return launch_route<__nv_bfloat16>(ctx, st, p);
}

extern "C" int ctb_moe_route_bwd(ctb_ctx* ctx, void* stream, void* d_logits, const void* logits, const void* topk_ids, int ids_bits,
                                 const void* d_weights, int weights_dtype, int64_t T, int64_t E, int64_t ld_out, int64_t ld, int topk,
                                 int score, int renormalize, float scale, int dtype) {
  const char* who = "ctb_moe_route_bwd";
  CTB_CHECK_CTX(ctx);
  CurrentDevice current(ctx);
  if (int s = check_route(who, logits, T, E, ld, topk, score, scale, dtype, weights_dtype)) return s;
  if (ids_bits != 32 && ids_bits != 64) return fail(CTB_BAD_ARG, "%s: ids must be 32- or 64-bit integers", who);
  if (ld_out < E) return fail(CTB_BAD_ARG, "%s: leading dimension of d_logits smaller than E", who);
  if (T == 0) return CTB_OK;
  CTB_CHECK_DEV(d_logits);
  CTB_CHECK_DEV(topk_ids);
  CTB_CHECK_DEV(d_weights);
  if ((uintptr_t)d_logits % (dtype == CTB_F32 ? 4 : 2)) return fail(CTB_BAD_ALIGN, "%s: d_logits must be aligned to their element size", who);
  if (int s = check_in_place(who, logits, ld, d_logits, ld_out, E, T, dtype == CTB_F32 ? 4 : 2)) return s;
  const RouteBackward p = {logits, d_logits, topk_ids, ids_bits, d_weights, weights_dtype, ld, ld_out, (unsigned)T, (int)E, topk,
                           score == CTB_SCORE_SIGMOID, renormalize != 0, scale, ctx->dev_status, 0};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == CTB_F32) return launch_route_backward<float>(ctx, st, p);
  if (dtype == CTB_F16) return launch_route_backward<__half>(ctx, st, p);
  return launch_route_backward<__nv_bfloat16>(ctx, st, p);
}
