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
// The choice is a comparison of sums of exponentials, and any rounding of them
// can turn it, so scores and values are FP64: a 64-bit FMA costs this GPU's
// vector units what a 32-bit one does, and the row's weights round to FP32 once.
// A group is kept if fewer than topk_groups are better (by value, then by lower
// id), which needs no sort.
//
// Bound by a wave's own chain more than by instructions or memory (9.2 MB at
// 8192 x 256 are 1.8 us).  Counters at 8192 x 256 with a bias, 13.1 us: 2048
// waves, two a SIMD, all there from start to end; a wave issues 1880 vector
// instructions for its four rows, which keeps a SIMD's vector unit at work half
// of the time, and waits for half of its own; the instruction cache has 1% of
// its fetches missing.
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
  int glanes_log2;    // lanes that hold (16 a row) or read (64) a group's values together
  int per;            // 16 lanes a row: consecutive experts of a lane
  int esize, vec;     // bytes of a logit; `per` logits are aligned 16-byte pieces
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

// A logit; NaN counts as -inf: score 0, and without a bias out of service (with
// one its value is the bias, which alone takes experts out of the choice)
__device__ __forceinline__ double load_logit(const RouteArgs& a, int64_t row, int e) {
  const int64_t i = row * a.ld + e;
  float v;
  if (a.x_dtype == MXFP4_DT_F32) v = static_cast<const float*>(a.logits)[i];
  else if (a.x_dtype == MXFP4_DT_BF16) v = (float)static_cast<const __bf16*>(a.logits)[i];
  else v = (float)static_cast<const _Float16*>(a.logits)[i];
  return v != v ? kNone : (double)v;
}

// `per` consecutive logits of a row from expert e0 on, in 16-byte pieces where
// they are aligned; -inf past the last expert
template <int J>
__device__ __forceinline__ void load_row(const RouteArgs& a, int64_t row, int e0, int per,
                                         double (&l)[J]) {
  const char* p = static_cast<const char*>(a.logits) + (row * a.ld + e0) * a.esize;
  if (a.vec) {  // all of them are experts
    float f[J];
    if (a.x_dtype == MXFP4_DT_F32) {
#pragma unroll
      for (int j = 0; j < J; j += 4) {
        if (j >= per) continue;
        const f32x4 t = *reinterpret_cast<const f32x4*>(p + j * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[j + i] = t[i];
      }
    } else if constexpr (J >= 8) {
#pragma unroll
      for (int j = 0; j < J; j += 8) {
        if (j >= per) continue;
        const u16x8 t = *reinterpret_cast<const u16x8*>(p + j * 2);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint16_t b = t[i];
          f[j + i] = a.x_dtype == MXFP4_DT_BF16 ? (float)__builtin_bit_cast(__bf16, b)
                                                : (float)__builtin_bit_cast(_Float16, b);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < J; ++j) l[j] = j >= per || f[j] != f[j] ? kNone : (double)f[j];
  } else {
#pragma unroll
    for (int j = 0; j < J; ++j)
      l[j] = j < per && e0 + j < a.ne ? load_logit(a, row, e0 + j) : kNone;
  }
}

__device__ __forceinline__ void store_slot(const RouteArgs& a, int64_t row, int slot, double s,
                                           int id) {
  const int64_t o = row * a.top_k + slot;
  a.w_out[o] = (float)(s * (double)a.scale);
  if (a.ids64) static_cast<int64_t*>(a.id_out)[o] = id;
  else static_cast<int32_t*>(a.id_out)[o] = id;
}

// exp(x) for x <= 0: 2^n e^r, n = x / ln 2 rounded, |r| <= ln 2 / 2 (ln 2 in two
// parts), e^r by its Taylor series to r^13 (the next term is under 2^-57 of the
// sum).  Fewer instructions than the general function.
__device__ __forceinline__ double exp_neg(double x) {
  x = __builtin_fmax(x, -1100.0);  // 0 from about -745 on; also for -inf
  const double n = __builtin_rint(x * 1.4426950408889634);
  double r = fma(n, -0.6931471805599453, x);
  r = fma(n, -2.3190468138462996e-17, r);
  double p = 1.0 / 6227020800.0;
  p = fma(p, r, 1.0 / 479001600.0);
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return ldexp(p, (int)n);
}
// 1 / d for d in [1, 2]: the hardware's estimate and two Newton steps
__device__ __forceinline__ double recip12(double d) {
  double y = __builtin_amdgcn_rcp(d);
  y = fma(fma(-d, y, 1.0), y, y);
  return fma(fma(-d, y, 1.0), y, y);
}

// exp(l - top) with exp(inf - inf) = 1: logits of +inf share the softmax
__device__ __forceinline__ double softmax_term(double l, double top) {
  const double t = exp_neg(l - top);
  return l == kNone ? 0.0 : (l == top ? 1.0 : t);
}
// 1 / (1 + e^-l) from e^-|l|, which neither overflows nor loses the small side
__device__ __forceinline__ double sigmoid(double l) {
  const double e = exp_neg(-__builtin_fabs(l));
  return (l >= 0.0 ? 1.0 : e) * recip12(1.0 + e);
}

// ------------------------------------------------------------ top_k searches
// One wave a row; lane l holds experts l, l + 64, ...; the group values are read
// from the row's values in LDS, some lanes a group.  Then top_k rounds of an
// argmax over the wave, ties to the lower id.  For top_k beyond 8 and groups
// that are not whole lanes: 8192 rows, E = 256, top-8 of 4 of 8 groups 26 us
// (route_top8 13).
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
  if (on) store_slot(a, row, lane, s, mine_id);
}

// ------------------------------------------------------------------- top-8
// L lanes a row (16: four rows a wave); lane l holds experts l * per .. + per - 1,
// so that a group is L / groups lanes.  The choice is one sort instead of top_k
// searches: the keys are the values with the expert's id in their low 10 bits
// (so that the larger double is the larger value, then the lower id, and no
// index moves beside it), each lane sorts its own, and butterfly steps over the
// lanes merge their best eight: max(a[i], b[7 - i]) of two sorted lists are the
// best eight of both, a bitonic list, sorted by three more rounds.
//
// Without a bias the value is a logit and the 10 bits are free (24 of 53 are
// used).  With one they are the value's lowest: where two keys that meet at the
// chosen ones are equal above them, the row is chosen again by comparing whole
// values.
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140;  // DPP

template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  const int lo = __builtin_amdgcn_mov_dpp(__double2loint(v), CTRL, 0xF, 0xF, true);
  const int hi = __builtin_amdgcn_mov_dpp(__double2hiint(v), CTRL, 0xF, 0xF, true);
  return __hiloint2double(hi, lo);
}
// The two sides of lanes l ^ 16 (W = 16) or l ^ 32, as both see them: the even
// rows' (the lower half's) value and the odd rows'
template <int W>
__device__ __forceinline__ void sides(double v, double& even, double& odd) {
  const uint32_t lo = (uint32_t)__double2loint(v), hi = (uint32_t)__double2hiint(v);
  if constexpr (W == 16) {
    const auto x = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
    const auto y = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    even = __hiloint2double((int)y[0], (int)x[0]);
    odd = __hiloint2double((int)y[1], (int)x[1]);
  } else {
    const auto x = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
    const auto y = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
    even = __hiloint2double((int)y[0], (int)x[0]);
    odd = __hiloint2double((int)y[1], (int)x[1]);
  }
}
// f over the L lanes of a row, in every lane: partners' values are equal within
// the 2, 4, 8 lanes reduced before, so mirrors do for xor 4 and 8
template <int L, typename F>
__device__ __forceinline__ double row_all(double v, F f) {
  v = f(v, dpp64<kXor1>(v));
  v = f(v, dpp64<kXor2>(v));
  v = f(v, dpp64<kHalfMirror>(v));
  v = f(v, dpp64<kMirror>(v));
  if constexpr (L == 64) {
    double a, b;
    sides<16>(v, a, b);
    v = f(a, b);
    sides<32>(v, a, b);
    v = f(a, b);
  }
  return v;
}
__device__ __forceinline__ double larger(double a, double b) { return __builtin_fmax(a, b); }
__device__ __forceinline__ double smaller(double a, double b) { return __builtin_fmin(a, b); }

// Keys below every value: experts out of service, experts of other groups
constexpr uint32_t kDeadHi = 0xFFE00000u, kOutHi = 0xFFEF0000u;

__device__ __forceinline__ double make_key(double v, int e) {
  const uint64_t b = __double_as_longlong(v + 0.0);  // -0 is 0
  uint32_t hi = (uint32_t)(b >> 32);
  const uint32_t lo = (uint32_t)b & ~1023u;
  if (hi == 0x7FF00000u) hi = 0x7FE00000u;  // inf: no NaN by its low bits
  if (hi == 0xFFF00000u) hi = kDeadHi;
  return __hiloint2double((int)hi, (int)(lo | (uint32_t)((int)hi < 0 ? e : 1023 - e)));
}
__device__ __forceinline__ int key_id(double k) {
  const int b = __double2loint(k) & 1023;
  return __double2hiint(k) < 0 ? b : 1023 - b;
}
// equal but for the ids
__device__ __forceinline__ bool same_value(double a, double b) {
  return __double2hiint(a) == __double2hiint(b) &&
         ((uint32_t)(__double2loint(a) ^ __double2loint(b)) & ~1023u) == 0;
}

__device__ __forceinline__ void exchange(double& a, double& b) {  // a >= b after
  const double x = larger(a, b);
  b = smaller(a, b);
  a = x;
}
__device__ __forceinline__ void sort8(double (&v)[8]) {
  constexpr int net[19][2] = {{0, 1}, {2, 3}, {4, 5}, {6, 7}, {0, 2}, {1, 3}, {4, 6},
                              {5, 7}, {1, 2}, {5, 6}, {0, 4}, {3, 7}, {1, 5}, {2, 6},
                              {1, 4}, {3, 6}, {2, 4}, {3, 5}, {3, 4}};
#pragma unroll
  for (int i = 0; i < 19; ++i) exchange(v[net[i][0]], v[net[i][1]]);
}
__device__ __forceinline__ void merge8(double (&a)[8], const double (&b)[8]) {  // best 8 of both
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = larger(a[i], b[7 - i]);
#pragma unroll
  for (int d = 4; d; d >>= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (!(i & d)) exchange(a[i], a[i + d]);
}
template <int CTRL>
__device__ __forceinline__ void merge_lanes(double (&a)[8]) {
  double b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = dpp64<CTRL>(a[i]);
  merge8(a, b);
}

template <int W>
__device__ __forceinline__ void merge_sides(double (&a)[8]) {
  double b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sides<W>(a[i], a[i], b[i]);
  merge8(a, b);
}

__device__ __forceinline__ void best_two(double& t1, double& t2, double o1, double o2) {
  t2 = larger(smaller(t1, o1), larger(t2, o2));
  t1 = larger(t1, o1);
}
template <int CTRL>
__device__ __forceinline__ void best_two(double& t1, double& t2) {
  best_two(t1, t2, dpp64<CTRL>(t1), dpp64<CTRL>(t2));
}
__device__ __forceinline__ void better_of(double& best, int& bi, double ov, int oi) {
  if (oi != INT_MAX && (bi == INT_MAX || ov > best || (ov == best && oi < bi))) {
    best = ov;
    bi = oi;
  }
}

template <int L, int J>
__global__ __launch_bounds__(256) void route_top8(RouteArgs a) {
  static_assert(L == 16 || L == 64, "16 or 64 lanes a row");
  const int lane = threadIdx.x & (L - 1);  // within the row
  const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (row >= a.m) return;  // whole rows of lanes; no barriers
  const int per = a.per, e0 = lane * per;

  double l[J];
  load_row<J>(a, row, e0, per, l);
  const bool all_scores = a.bias || a.top2;
  double top = kNone, total = 0.0;
  if (!a.sigmoid) {
#pragma unroll
    for (int j = 0; j < J; ++j) top = larger(top, l[j]);
    top = row_all<L>(top, larger);
    if (all_scores || !a.renorm) {
#pragma unroll
      for (int j = 0; j < J; ++j) total += softmax_term(l[j], top);
      total = row_all<L>(total, [](double x, double y) { return x + y; });
    }
  }
  const double inv = total > 0.0 ? 1.0 / total : 0.0;
  auto mine = [&](int j) { return j < per && e0 + j < a.ne; };

  double v[J];
  double t1 = kNone, t2 = kNone;  // the two largest that a group value is made of
  if (all_scores) {
    // of experts past the last one too: no branch in the row
    if (a.sigmoid) {
#pragma unroll
      for (int j = 0; j < J; ++j) v[j] = sigmoid(l[j]);
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j) v[j] = softmax_term(l[j], top) * inv;
    }
    if (a.bias) {
      float b[J];
#pragma unroll
      for (int j = 0; j < J; ++j) b[j] = a.bias[mine(j) ? e0 + j : 0];
#pragma unroll
      for (int j = 0; j < J; ++j)  // NaN and +inf: out of service
        v[j] = b[j] < INFINITY ? v[j] + (double)b[j] : kNone;
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const double x = mine(j) ? v[j] : kNone;
      t2 = larger(t2, smaller(t1, x));
      t1 = larger(t1, x);
    }
  }
  if (!a.bias) {
#pragma unroll
    for (int j = 0; j < J; ++j) v[j] = l[j];
    if (!a.top2) {
#pragma unroll
      for (int j = 0; j < J; ++j) t1 = larger(t1, l[j]);
    }
  }
  bool kept = true;
  if (a.groups > 1) {
    const int p = a.glanes_log2;  // log2 of a group's lanes
    if (p >= 1) best_two<kXor1>(t1, t2);
    if (p >= 2) best_two<kXor2>(t1, t2);
    if (p >= 3) best_two<kHalfMirror>(t1, t2);
    if (L == 64 && p >= 4) best_two<kMirror>(t1, t2);
    if (L == 64 && p >= 5) {
      double a1, b1, a2, b2;
      sides<16>(t1, a1, b1);
      sides<16>(t2, a2, b2);
      t1 = a1, t2 = a2;
      best_two(t1, t2, b1, b2);
    }
    const double gv = a.top2 ? t1 + t2 : t1;
    const int first = (lane >> p) << p;  // of this lane's group
    int rank = 0;
    auto meet = [&](double o, int h) {  // the group whose first lane is h
      rank += (o > gv || (o == gv && h < first)) ? 1 : 0;
    };
    if constexpr (L == 64) {
      for (int h = 0; h < 64; h += 1 << p) meet(lane_f64(gv, h), h);
    } else {
      static_for<0, 16>([&](auto hc) {  // broadcast within the row
        constexpr int h = decltype(hc)::value;
        if ((h & ((1 << p) - 1)) == 0) meet(dpp64<0x150 + h>(gv), h);
      });
    }
    kept = rank < a.keep;
  }

  double key[J];
#pragma unroll
  for (int j = 0; j < J; ++j)
    key[j] = mine(j) && kept ? make_key(v[j], e0 + j) : __hiloint2double((int)kOutHi, e0 + j);
  double best[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) best[i] = i < J ? key[i] : __hiloint2double((int)kOutHi, 1023);
  if constexpr (J == 4) {  // the other four are the least already
    exchange(best[0], best[1]);
    exchange(best[2], best[3]);
    exchange(best[0], best[2]);
    exchange(best[1], best[3]);
    exchange(best[1], best[2]);
  } else {
    sort8(best);
  }
  if constexpr (J > 8) {
    double more[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) more[i] = key[8 + i];
    sort8(more);
    merge8(best, more);
  }
  merge_lanes<kXor1>(best);
  merge_lanes<kXor2>(best);
  merge_lanes<kHalfMirror>(best);
  merge_lanes<kMirror>(best);
  if constexpr (L == 64) {
    merge_sides<16>(best);
    merge_sides<32>(best);
  }

  double slot = best[0], last = best[0];  // this lane's, and the last one chosen
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    if (lane == i) slot = best[i];
    if (a.top_k > i) last = best[i];
  }
  int id = key_id(slot);
  bool live = (uint32_t)__double2hiint(slot) != kDeadHi;
  if (a.bias) {
    bool unsure = false;
#pragma unroll
    for (int i = 1; i < 8; ++i) unsure |= i < a.top_k && same_value(best[i - 1], best[i]);
#pragma unroll
    for (int j = 0; j < J; ++j) unsure |= key[j] < last && same_value(key[j], last);
    if (__ballot(unsure)) {  // in any of the wave's rows
      uint32_t out = 0;
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (!mine(j) || !kept) out |= 1u << j;
      for (int r = 0; r < a.top_k; ++r) {
        double bv = kNone;
        int bi = INT_MAX;
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (!((out >> j) & 1u) && (bi == INT_MAX || v[j] > bv)) {
            bv = v[j];
            bi = e0 + j;
          }
#pragma unroll
        for (int d = 1; d < L; d <<= 1) better_of(bv, bi, shfl_xor_f64(bv, d), __shfl_xor(bi, d));
        if (lane == r) {
          id = bi;
          live = bv != kNone;
        }
        if (bi >= e0 && bi < e0 + per) out |= 1u << (bi - e0);
      }
    }
  }

  const bool on = lane < a.top_k;
  live = live && on;
  const double x = live ? load_logit(a, row, id) : kNone;
  double s = 0.0;
  if (a.renorm) {
    if (a.sigmoid) s = live ? sigmoid(x) : 0.0;
    else s = softmax_term(x, row_all<L>(x, larger));
    const double sum = row_all<L>(s, [](double p, double q) { return p + q; });
    s = sum > 0.0 ? s / sum : 0.0;
  } else if (live) {
    s = a.sigmoid ? sigmoid(x) : softmax_term(x, top) * inv;
  }
  if (on) store_slot(a, row, lane, s, id);
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
    set_error("grouped router: %d of %d groups of %d experts", topk_groups, num_groups,
              num_experts);
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
  hipStream_t st = static_cast<hipStream_t>(stream);
  // Lists of eight, groups of whole lanes; anything else takes the searches.  16
  // lanes a row do the least work (E = 256 with a bias: 8192 rows 13.6 us, a
  // wave a row 17.9; softmax alone 6.4, 13.6; E = 128 softmax 5.6, 13.2).  A wave
  // a row is the quicker while a lane would hold more than 8 experts and the rows
  // do not fill the GPU: at E = 256 with a bias up to 3100 rows (1 row 4.7 us, 16
  // lanes 8.0; 2048 rows 6.8, 10.6; 3000 9.0, 10.6; 3600 11.0, 10.1), softmax
  // alone up to 1500 (1024 rows 5.1, 6.3; 1536 6.1, 6.1; 2500 7.2, 6.1).  2048
  // lies between the two.  With fewer experts both take the same.
  auto whole = [&](int lanes) {
    return a.groups == 1 || (num_experts % lanes == 0 && lanes % a.groups == 0);
  };
  int lanes = 0;
  if (top_k <= 8) {
    const bool can16 = num_experts <= 256 && whole(16);
    if (can16 && (num_experts <= 128 || m > 2048)) lanes = 16;
    else if (whole(64)) lanes = 64;
    else if (can16) lanes = 16;
  }
  auto group_lanes = [&](int of) {
    int log2 = 0;
    while ((a.groups << (log2 + 1)) <= of) ++log2;
    return log2;
  };
  if (lanes) {
    a.glanes_log2 = group_lanes(lanes);
    a.per = (num_experts + lanes - 1) / lanes;
    a.esize = x_dtype == MXFP4_DT_F32 ? 4 : 2;
    a.vec = num_experts % lanes == 0 && a.per * a.esize % 16 == 0 &&
            ((reinterpret_cast<uintptr_t>(logits) | (uintptr_t)(row_stride * a.esize)) & 15) == 0;
    const unsigned grid = (unsigned)((m * lanes + 255) / 256);
    if (lanes == 16) {
      if (a.per <= 4) route_top8<16, 4><<<grid, 256, 0, st>>>(a);
      else if (a.per <= 8) route_top8<16, 8><<<grid, 256, 0, st>>>(a);
      else route_top8<16, 16><<<grid, 256, 0, st>>>(a);
    } else {
      if (a.per <= 4) route_top8<64, 4><<<grid, 256, 0, st>>>(a);
      else if (a.per <= 8) route_top8<64, 8><<<grid, 256, 0, st>>>(a);
      else route_top8<64, 16><<<grid, 256, 0, st>>>(a);
    }
    return launch_status("grouped router launch");
  }
  a.glanes_log2 = group_lanes(64);
  const unsigned grid = (unsigned)((m + 3) / 4);
  const int j = (num_experts + 63) / 64;
  if (j <= 1) route_grouped<1><<<grid, 256, 0, st>>>(a);
  else if (j <= 2) route_grouped<2><<<grid, 256, 0, st>>>(a);
  else if (j <= 4) route_grouped<4><<<grid, 256, 0, st>>>(a);
  else if (j <= 8) route_grouped<8><<<grid, 256, 0, st>>>(a);
  else route_grouped<16><<<grid, 256, 0, st>>>(a);
  return launch_status("grouped router launch");
}
