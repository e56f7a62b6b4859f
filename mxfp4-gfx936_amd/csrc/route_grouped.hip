// Expert router with groups: softmax or sigmoid scores, a balance bias that
// acts on the choice only, the best groups first, top-k among their experts,
// weights renormalised and scaled.  No counterpart in the reference, whose
// tests route by softmax -> top-k (test:242-244; route.hip).
//
//   s_i = softmax(l)_i or 1 / (1 + exp(-l_i))
//   v_i = s_i + bias_i, or without a bias l_i, whose order is the score's
//   group value = max v, or the sum of the two largest s (+ bias)
//   weight = s_i, 0 where v_i = -inf; / sum over the chosen; * scale
//
// One wave per token row; lane l holds experts l, l + 64, ...  The choice is
// a comparison of sums of exponentials, and any rounding of them can turn
// it, so scores and values are FP64: a 64-bit FMA costs this GPU's vector
// units what a 32-bit one does, and the row's weights round to FP32 once.
// The group values are taken from the row's values in LDS, P lanes a group;
// a group is kept if fewer than topk_groups are better (by value, then by
// lower id), which needs no sort.  Then top_k rounds of an argmax over the
// wave, ties to the lower expert id.
#include <climits>
#include <math.h>

#include "common.h"

namespace mx {
namespace {

struct RouteArgs {
  const void* logits;
  const float* bias;  // [ne] or nullptr
  float* w_out;
  void* id_out;
  int64_t m, ld;
  int ne, top_k, groups, keep, x_dtype, ids64;
  int sigmoid, top2, renorm;
  float scale;
  int gsize;          // experts per group
  uint32_t gmagic;    // ceil(2^20 / gsize): e / gsize for e < 1024
  int glanes_log2;    // lanes that read a group's values together
};

constexpr double kNone = -INFINITY;

__device__ __forceinline__ double shfl_xor_f64(double v, int mask) {
  const int lo = __shfl_xor(__double2loint(v), mask), hi = __shfl_xor(__double2hiint(v), mask);
  return __hiloint2double(hi, lo);
}
__device__ __forceinline__ double lane_f64(double v, int lane) {  // uniform lane
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane),
                          __builtin_amdgcn_readlane(__double2loint(v), lane));
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += shfl_xor_f64(v, d);
  return v;
}
__device__ __forceinline__ double wave_max(double v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = fmax(v, shfl_xor_f64(v, d));
  return v;
}

// A logit; NaN counts as -inf (an expert out of service)
__device__ __forceinline__ double load_logit(const RouteArgs& a, int64_t row, int e) {
  const int64_t i = row * a.ld + e;
  float v;
  if (a.x_dtype == MXFP4_DT_F32) v = static_cast<const float*>(a.logits)[i];
  else if (a.x_dtype == MXFP4_DT_BF16) v = (float)static_cast<const __bf16*>(a.logits)[i];
  else v = (float)static_cast<const _Float16*>(a.logits)[i];
  return v != v ? kNone : (double)v;
}

// exp(l - top) with exp(inf - inf) = 1: logits of +inf share the softmax
__device__ __forceinline__ double softmax_term(double l, double top) {
  return l == kNone ? 0.0 : (l == top ? 1.0 : exp(l - top));
}
__device__ __forceinline__ double sigmoid(double l) { return 1.0 / (1.0 + exp(-l)); }

template <int J>
__global__ __launch_bounds__(256) void route_grouped(RouteArgs a) {
  __shared__ double vals[4][64 * J];
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  if (row >= a.m) return;  // whole waves; no barriers

  double l[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int e = lane + 64 * j;
    l[j] = e < a.ne ? load_logit(a, row, e) : kNone;
  }
  // softmax: the row's largest logit and the sum of the terms
  const bool all_scores = a.bias || a.top2;
  double top = kNone, total = 0.0;
  if (!a.sigmoid) {
#pragma unroll
    for (int j = 0; j < J; ++j) top = fmax(top, l[j]);
    top = wave_max(top);
    if (all_scores || !a.renorm) {
#pragma unroll
      for (int j = 0; j < J; ++j) total += softmax_term(l[j], top);
      total = wave_sum(total);
    }
  }
  auto score = [&](double x) {
    if (a.sigmoid) return sigmoid(x);
    return total > 0.0 ? softmax_term(x, top) / total : 0.0;
  };

  double v[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int e = lane + 64 * j;
    v[j] = l[j];
    double g = v[j];  // what the group values are made of
    if (all_scores && e < a.ne) {
      g = score(l[j]);
      if (a.bias) {
        const float b = a.bias[e];
        g = b < INFINITY ? g + (double)b : kNone;  // NaN and +inf: out of service
        v[j] = g;
      }
    }
    if (a.groups > 1 && e < a.ne) vals[wave][e] = g;
  }

  uint32_t out = 0;  // bit j: expert lane + 64 j is not a candidate (any more)
  if (a.groups > 1) {
    // one wave writes and reads its own row of LDS, in order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int P = 1 << a.glanes_log2;
    const int g = lane >> a.glanes_log2, p = lane & (P - 1);
    double t1 = kNone, t2 = kNone;
    if (g < a.groups) {
      for (int i = p; i < a.gsize; i += P) {
        const double x = vals[wave][g * a.gsize + i];
        t2 = fmax(t2, fmin(t1, x));
        t1 = fmax(t1, x);
      }
    }
    for (int d = 1; d < P; d <<= 1) {
      const double o1 = shfl_xor_f64(t1, d), o2 = shfl_xor_f64(t2, d);
      t2 = fmax(fmin(t1, o1), fmax(t2, o2));
      t1 = fmax(t1, o1);
    }
    const double gv = a.top2 ? t1 + t2 : t1;
    int rank = 0;
    for (int h = 0; h < a.groups; ++h) {
      const double o = lane_f64(gv, h << a.glanes_log2);
      rank += (o > gv || (o == gv && h < g)) ? 1 : 0;
    }
    const uint64_t kept = __ballot(g < a.groups && p == 0 && rank < a.keep);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const uint32_t e = lane + 64 * j;
      const int ge = (int)((e * a.gmagic) >> 20);
      if (!((kept >> ((ge << a.glanes_log2) & 63)) & 1u)) out |= 1u << j;
    }
  }

  double mine = kNone;  // slot `lane` (lanes < top_k): value and expert
  int mine_id = 0;
  for (int r = 0; r < a.top_k; ++r) {
    double best = kNone;
    int bi = INT_MAX;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int e = lane + 64 * j;
      if (e < a.ne && !((out >> j) & 1u) && (bi == INT_MAX || v[j] > best)) {
        best = v[j];
        bi = e;
      }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double ov = shfl_xor_f64(best, d);
      const int oi = __shfl_xor(bi, d);
      if (oi != INT_MAX && (bi == INT_MAX || ov > best || (ov == best && oi < bi))) {
        best = ov;
        bi = oi;
      }
    }
    if (lane == r) {
      mine = best;
      mine_id = bi;
    }
    if ((bi & 63) == lane) out |= 1u << (bi >> 6);
  }

  // weights of the chosen, one per lane; a renormalised softmax needs only
  // their own largest logit
  const bool on = lane < a.top_k;
  const bool live = on && mine != kNone;
  const double x = live ? load_logit(a, row, mine_id) : kNone;
  double s = 0.0;
  if (a.renorm) {
    if (a.sigmoid) {
      s = live ? sigmoid(x) : 0.0;
    } else {
      const double t = wave_max(x);
      s = softmax_term(x, t);
    }
    const double sum = wave_sum(s);
    s = sum > 0.0 ? s / sum : 0.0;
  } else if (live) {
    s = score(x);
  }
  if (on) {
    const int64_t o = row * a.top_k + lane;
    a.w_out[o] = (float)(s * (double)a.scale);
    if (a.ids64) static_cast<int64_t*>(a.id_out)[o] = mine_id;
    else static_cast<int32_t*>(a.id_out)[o] = mine_id;
  }
}

}  // namespace
}  // namespace mx

extern "C" int mxfp4_moe_route_grouped(const void* logits, int x_dtype, int64_t m, int num_experts,
                                       int64_t row_stride, const float* bias, int scoring,
                                       int num_groups, int topk_groups, int group_score, int top_k,
                                       int renormalize, float scale, float* topk_weights,
                                       void* topk_ids, int ids_dtype, void* stream) {
  using namespace mx;
  if (x_dtype != MXFP4_DT_F32 && x_dtype != MXFP4_DT_BF16 && x_dtype != MXFP4_DT_F16) {
    set_error("grouped router: unsupported logits dtype %d", x_dtype);
    return MXFP4_ERR_TYPE;
  }
  if (ids_dtype != MXFP4_DT_I32 && ids_dtype != MXFP4_DT_I64) {
    set_error("grouped router: topk_ids must be int32 or int64 (dtype code %d)", ids_dtype);
    return MXFP4_ERR_TYPE;
  }
  if ((scoring != MXFP4_SCORE_SOFTMAX && scoring != MXFP4_SCORE_SIGMOID) ||
      (group_score != MXFP4_GROUP_MAX && group_score != MXFP4_GROUP_TOP2)) {
    set_error("grouped router: unknown scoring %d or group score %d", scoring, group_score);
    return MXFP4_ERR_VALUE;
  }
  if (m < 0 || num_experts < 1 || num_experts > 1024 || row_stride < num_experts) {
    set_error("grouped router: invalid sizes (m %lld, experts %d, row stride %lld)", (long long)m,
              num_experts, (long long)row_stride);
    return MXFP4_ERR_VALUE;
  }
  if (num_groups < 1 || num_groups > 64 || num_experts % num_groups != 0 || topk_groups < 1 ||
      topk_groups > num_groups) {
    set_error("grouped router: %d of %d groups of %d experts", topk_groups, num_groups, num_experts);
    return MXFP4_ERR_VALUE;
  }
  const int gsize = num_experts / num_groups;
  if (group_score == MXFP4_GROUP_TOP2 && num_groups > 1 && gsize < 2) {
    set_error("grouped router: the two best of a group need groups of two experts");
    return MXFP4_ERR_VALUE;
  }
  if (top_k < 1 || top_k > 64 || top_k > topk_groups * gsize) {
    set_error("grouped router: unsupported top_k %d for %d groups of %d experts", top_k,
              topk_groups, gsize);
    return MXFP4_ERR_VALUE;
  }
  if (!(scale > -INFINITY && scale < INFINITY)) {
    set_error("grouped router: scale must be finite");
    return MXFP4_ERR_VALUE;
  }
  if ((m + 3) / 4 > 0x7FFFFF) {  // 2^31 threads a launch
    set_error("grouped router: too many rows (%lld)", (long long)m);
    return MXFP4_ERR_VALUE;
  }
  if (m == 0) return MXFP4_OK;
  RouteArgs a{};
  a.logits = logits;
  a.bias = bias;
  a.w_out = topk_weights;
  a.id_out = topk_ids;
  a.m = m;
  a.ld = row_stride;
  a.ne = num_experts;
  a.top_k = top_k;
  // all groups kept: no choice among them
  a.groups = topk_groups == num_groups ? 1 : num_groups;
  a.keep = topk_groups;
  a.x_dtype = x_dtype;
  a.ids64 = ids_dtype == MXFP4_DT_I64;
  a.sigmoid = scoring == MXFP4_SCORE_SIGMOID;
  a.top2 = a.groups > 1 && group_score == MXFP4_GROUP_TOP2;
  a.renorm = renormalize != 0;
  a.scale = scale;
  a.gsize = num_experts / a.groups;
  a.gmagic = ((1u << 20) + a.gsize - 1) / a.gsize;
  a.glanes_log2 = 0;
  while ((a.groups << (a.glanes_log2 + 1)) <= 64) ++a.glanes_log2;
  const unsigned grid = (unsigned)((m + 3) / 4);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int j = (num_experts + 63) / 64;
  if (j <= 1) route_grouped<1><<<grid, 256, 0, st>>>(a);
  else if (j <= 2) route_grouped<2><<<grid, 256, 0, st>>>(a);
  else if (j <= 4) route_grouped<4><<<grid, 256, 0, st>>>(a);
  else if (j <= 8) route_grouped<8><<<grid, 256, 0, st>>>(a);
  else route_grouped<16><<<grid, 256, 0, st>>>(a);
  return launch_status("grouped router launch");
}
