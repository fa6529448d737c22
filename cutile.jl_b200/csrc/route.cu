// Routing of tokens to experts by given logits, and its gradient, for sm_100a.
//
//   s = softmax(x) or sigmoid(x)       c = s + bias (for the choice only)
//   a group of experts scores the sum of its one or two best c; experts outside of the best groups are out
//   the k best c are chosen (ties to the lowest expert), w = scale s / max(sum of the chosen s, 1e-20), or scale s
// The bias balances the experts' load and takes no gradient.
//
// A warp takes a token.  The work is tiny (1 KB of logits per token of 256 experts), so latency bounds it: of the selection rounds and
// of the launch.  What is chosen must not hang on a rounding: c is compared in f64.
#include <float.h>

#include <algorithm>

#include "ctx.h"
#include "ptx.cuh"
#include "rows.cuh"

using namespace ctb;
using namespace ctb_internal;

namespace {

constexpr int kThreads = 128;
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
  int tokens, experts, topk, sigmoid, groups, topk_groups, group_top, renormalize;
  float scale;
};

__device__ __forceinline__ double sum_lanes(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

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

// Lane l holds experts l, l + 32, ...
template <typename T, int EPL>
__global__ void __launch_bounds__(kThreads) route_kernel(const Route p) {
  extern __shared__ double values[];  // with groups: c of the warp's token
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_dependency_sync();
  for (int t = blockIdx.x * kWarps + warp; t < p.tokens; t += gridDim.x * kWarps) {
    const T* src = static_cast<const T*>(p.x) + t * p.ld;
    double s[EPL], c[EPL];
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane + 32 * i;
      const float x = e < p.experts ? to_float(src[e]) : -INFINITY;
      most = fmaxf(most, x);
      s[i] = x;
    }
    if (p.sigmoid) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) s[i] = 1 / (1 + exp(-s[i]));
    } else {
      most = warp_max(most);
      double sum = 0;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        s[i] = exp(s[i] - (double)most);
        if (lane + 32 * i < p.experts) sum += s[i];
      }
      sum = sum_lanes(sum);
#pragma unroll
      for (int i = 0; i < EPL; ++i) s[i] /= sum;
    }
    unsigned out = 0;  // bit i: the expert does not exist, is in a group that is out, or has been chosen
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane + 32 * i;
      c[i] = s[i];
      if (e >= p.experts) {
        out |= 1u << i;
      } else {
        if (p.bias) c[i] += (double)p.bias[e];
        if (!(c[i] > -DBL_MAX)) c[i] = -DBL_MAX;  // NaN and -inf come last, but before what is out
      }
    }
    if (p.topk_groups < p.groups) {
      double* v = values + warp * p.experts;
      const int size = p.experts / p.groups;
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (lane + 32 * i < p.experts) v[lane + 32 * i] = c[i];
      __syncwarp();
      double score = -INFINITY;
      if (lane < p.groups) {
        double a = -INFINITY, b = -INFINITY;
        for (int i = 0; i < size; ++i) {
          const double x = v[lane * size + i];
          b = fmax(b, fmin(a, x));
          a = fmax(a, x);
        }
        score = p.group_top == 2 ? a + b : a;
      }
      int rank = 0;
      for (int g = 0; g < p.groups; ++g) {
        const double o = __shfl_sync(0xffffffffu, score, g);
        rank += o > score || (o == score && g < lane);
      }
      const unsigned kept = __ballot_sync(0xffffffffu, lane < p.groups && rank < p.topk_groups);
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (lane + 32 * i < p.experts && !(kept >> ((lane + 32 * i) / size) & 1)) out |= 1u << i;
      __syncwarp();
    }
    double mine = 0;  // lane j: score and expert of the j-th choice
    int my_id = 0;
    for (int j = 0; j < p.topk; ++j) {
      double best = -INFINITY, best_s = 0;
      int id = 0x7fffffff;
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (!(out >> i & 1) && c[i] > best) {  // ascending experts: the first of equal ones stays
          best = c[i];
          best_s = s[i];
          id = lane + 32 * i;
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const double ob = __shfl_xor_sync(0xffffffffu, best, o), os = __shfl_xor_sync(0xffffffffu, best_s, o);
        const int oi = __shfl_xor_sync(0xffffffffu, id, o);
        if (ob > best || (ob == best && oi < id)) {
          best = ob;
          best_s = os;
          id = oi;
        }
      }
      if (lane == j) {
        mine = best_s;
        my_id = id;
      }
      if ((id & 31) == lane) out |= 1u << (id >> 5);
    }
    double scale = p.scale;
    if (p.renormalize) {
      const double sum = sum_lanes(lane < p.topk ? mine : 0.0);
      scale /= sum < 1e-20 ? 1e-20 : sum;
    }
    if (lane < p.topk) {
      const long long at = (long long)lane * p.tokens + t;
      p.ids[at] = my_id + 1;
      store_weight(p.weights, at, p.weights_dtype, (float)(mine * scale));
    }
  }
}

struct RouteBackward {
  const void* x;
  void* dx;
  const void* ids;
  int id_bits;
  const void* d_weights;
  int weights_dtype;
  long long ld, ld_dx;
  int tokens, experts, topk, sigmoid, renormalize;
  float scale;
  int* status;
};

// With u_j the gradient that reaches s_j of the j-th choice (0 for the others):
//   sigmoid: dx_e = u_e s_e (1 - s_e)        softmax: dx_e = s_e (u_e - sum_j u_j s_j), a sum that is 0 for renormalised weights
template <typename T, int EPL>
__global__ void __launch_bounds__(kThreads) route_backward_kernel(const RouteBackward p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_dependency_sync();
  for (int t = blockIdx.x * kWarps + warp; t < p.tokens; t += gridDim.x * kWarps) {
    const T* src = static_cast<const T*>(p.x) + t * p.ld;
    T* dst = static_cast<T*>(p.dx) + t * p.ld_dx;
    int id = 0;
    float dw = 0.f, xj = 0.f;
    if (lane < p.topk) {
      const long long at = (long long)lane * p.tokens + t;
      const long long e = p.id_bits == 64 ? static_cast<const long long*>(p.ids)[at] : static_cast<const int*>(p.ids)[at];
      if (e < 0 || e > p.experts) atomicMax(p.status, DEV_BAD_INDEX);
      else id = (int)e;
      if (id) {
        dw = load_weight(p.d_weights, at, p.weights_dtype);
        xj = to_float(src[id - 1]);
      }
    }
    float s[EPL], most = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      s[i] = lane + 32 * i < p.experts ? to_float(src[lane + 32 * i]) : -INFINITY;
      most = fmaxf(most, s[i]);
    }
    float sj;  // score of this lane's choice
    if (p.sigmoid) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) s[i] = 1.f / (1.f + expf(-s[i]));
      sj = 1.f / (1.f + expf(-xj));
    } else {
      most = warp_max(most);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        s[i] = expf(s[i] - most);
        if (lane + 32 * i < p.experts) sum += s[i];
      }
      sum = warp_sum(sum);
#pragma unroll
      for (int i = 0; i < EPL; ++i) s[i] /= sum;
      sj = expf(xj - most) / sum;
    }
    if (!id) sj = 0.f;
    float u = p.scale * dw;
    if (p.renormalize) {
      const float sum = warp_sum(sj), total = fmaxf(sum, 1e-20f);
      const float mean = sum < 1e-20f ? 0.f : warp_sum(dw * sj) / total;  // below, the total is a constant
      u = p.scale * (dw - mean) / total;
    }
    if (!id) u = 0.f;
    const float common = p.sigmoid || p.renormalize ? 0.f : warp_sum(u * sj);
    float d[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) d[i] = -common;
    for (int j = 0; j < p.topk; ++j) {
      const int e = __shfl_sync(0xffffffffu, id, j) - 1;
      const float v = __shfl_sync(0xffffffffu, u, j);
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (e == lane + 32 * i) d[i] += v;
    }
    __syncwarp();  // dst may be the logits themselves: the choices' logits have been read
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (lane + 32 * i < p.experts) dst[lane + 32 * i] = from_float<T>(d[i] * s[i] * (p.sigmoid ? 1.f - s[i] : 1.f));
  }
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

template <typename T, typename F>
void by_experts(int E, F f) {
  if (E <= 32) f(std::integral_constant<int, 1>());
  else if (E <= 64) f(std::integral_constant<int, 2>());
  else if (E <= 128) f(std::integral_constant<int, 4>());
  else if (E <= 256) f(std::integral_constant<int, 8>());
  else f(std::integral_constant<int, 16>());
}

template <typename T>
int launch_route(ctb_ctx* ctx, cudaStream_t st, const Route& p) {
  const int grid = (int)std::min<int64_t>((p.tokens + kWarps - 1) / kWarps, 16ll * ctx->sm_count);
  const size_t smem = p.topk_groups < p.groups ? (size_t)kWarps * p.experts * sizeof(double) : 0;
  by_experts<T>(p.experts, [&](auto epl) { launch_kernel(route_kernel<T, decltype(epl)::value>, grid, kThreads, smem, st, 0, p); });
  CTB_CHECK_LAUNCH("ctb_moe_route launch");
  return CTB_OK;
}
template <typename T>
int launch_route_backward(ctb_ctx* ctx, cudaStream_t st, const RouteBackward& p) {
  const int grid = (int)std::min<int64_t>((p.tokens + kWarps - 1) / kWarps, 16ll * ctx->sm_count);
  by_experts<T>(p.experts, [&](auto epl) { launch_kernel(route_backward_kernel<T, decltype(epl)::value>, grid, kThreads, 0, st, 0, p); });
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
  const Route p = {logits, bias, topk_ids, topk_weights, weights_dtype, ld, (int)T, (int)E, topk, score == CTB_SCORE_SIGMOID, groups, topk_groups,
                   group_top, renormalize != 0, scale};
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
  const RouteBackward p = {logits, d_logits, topk_ids, ids_bits, d_weights, weights_dtype, ld, ld_out, (int)T, (int)E, topk,
                           score == CTB_SCORE_SIGMOID, renormalize != 0, scale, ctx->dev_status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == CTB_F32) return launch_route_backward<float>(ctx, st, p);
  if (dtype == CTB_F16) return launch_route_backward<__half>(ctx, st, p);
  return launch_route_backward<__nv_bfloat16>(ctx, st, p);
}
