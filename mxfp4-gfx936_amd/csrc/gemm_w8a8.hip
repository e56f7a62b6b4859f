// W8A8 GEMM: int8 activations with a scale per token times int8 weights with
// a scale per output channel.  No counterpart in the reference.
//
//   out[i, j] = round(float(sum_k a[i, k] w[j, k]) * sa[i] * sw[j] + bias[j])
//
// The sum is exact: products of two bytes added in int32 by the integer
// MFMA (v_mfma_i32_16x16x64_i8), which K <= 131071 cannot overflow (2^14 per
// product), so tiles, waves and splits of K may add in any order and give
// the same bits.  FP32 from there (one rounding of the sum, two products,
// one addition), one rounding to the output type.
//
// Operands of the MFMA: lane l supplies 16 consecutive K bytes of row l % 16
// (K = (l / 16) * 16 ..); the weights are its A operand and the activations
// its B operand, so lane l receives columns (l / 16) * 4 .. + 3 of row l % 16
// and writes them side by side.
#include "common.h"

namespace mx {
namespace {

struct W8Args {
  const uint8_t* a;
  const float* a_scale;
  const uint8_t* w;
  const float* w_scale;
  const void* bias;  // [n] of the output type or nullptr
  void* out;
  int64_t m, n;
  int k;
};

__device__ __forceinline__ i32x4 mfma_i8(i32x4 a, i32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// Four output values of row `row`, columns col .. col + 3 (col % 4 == 0)
template <typename TO>
__device__ __forceinline__ void finish4(const W8Args& g, int64_t row, int64_t col, i32x4 acc,
                                        bool vec) {
  if (row >= g.m || col >= g.n) return;
  const float sa = g.a_scale[row];
  TO* const o = static_cast<TO*>(g.out) + row * g.n + col;
  TO r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v = 0.f;
    if (col + i < g.n) {
      v = (float)acc[i] * sa * g.w_scale[col + i];
      if (g.bias) v += to_f32(static_cast<const TO*>(g.bias)[col + i]);
    }
    r[i] = from_f32<TO>(v);
  }
  if (vec && col + 4 <= g.n) {
    typedef TO T4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<T4*>(o) = T4{r[0], r[1], r[2], r[3]};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + i < g.n) o[i] = r[i];
  }
}

// One workgroup of 4 waves computes 64 rows x 64 columns, 64 bytes of K at a
// time through LDS.
template <typename TO>
__global__ __launch_bounds__(256) void w8a8_tile(W8Args g, int nbn) {
  constexpr int LD = 80;  // bytes of an LDS row: 64 and a pad against bank conflicts
  __shared__ __attribute__((aligned(16))) uint8_t As[64 * LD];
  __shared__ __attribute__((aligned(16))) uint8_t Ws[64 * LD];
  const int tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6;
  const int c16 = lane & 15, grp = lane >> 4;
  const int64_t row0 = (int64_t)(blockIdx.x / nbn) * 64;
  const int64_t col0 = (int64_t)(blockIdx.x % nbn) * 64;
  const int r = tid >> 2, ch = (tid & 3) * 16;
  const bool a_ok = row0 + r < g.m, w_ok = col0 + r < g.n;
  const uint8_t* ap = g.a + (a_ok ? row0 + r : 0) * g.k + ch;
  const uint8_t* wp = g.w + (w_ok ? col0 + r : 0) * g.k + ch;
  i32x4 acc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = i32x4{0, 0, 0, 0};
  for (int k0 = 0; k0 < g.k; k0 += 64) {
    const bool in = k0 + ch < g.k;
    const i32x4 zero = {0, 0, 0, 0};
    const i32x4 av = a_ok && in ? *reinterpret_cast<const i32x4*>(ap + k0) : zero;
    const i32x4 wv = w_ok && in ? *reinterpret_cast<const i32x4*>(wp + k0) : zero;
    __syncthreads();
    *reinterpret_cast<i32x4*>(As + r * LD + ch) = av;
    *reinterpret_cast<i32x4*>(Ws + r * LD + ch) = wv;
    __syncthreads();
    const i32x4 b = *reinterpret_cast<const i32x4*>(As + (wave * 16 + c16) * LD + grp * 16);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      acc[i] = mfma_i8(*reinterpret_cast<const i32x4*>(Ws + (i * 16 + c16) * LD + grp * 16), b,
                       acc[i]);
  }
  const bool vec = g.n % 4 == 0 && !(reinterpret_cast<uintptr_t>(g.out) & 15);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    finish4<TO>(g, row0 + wave * 16 + c16, col0 + i * 16 + grp * 4, acc[i], vec);
}

template <typename TO>
int launch_typed(const W8Args& g, hipStream_t st) {
  const int64_t nbm = (g.m + 63) / 64, nbn = (g.n + 63) / 64;
  if (nbm * nbn > 0x7FFFFF) {  // 2^31 threads a launch
    set_error("w8a8: too many tiles (%lld x %lld)", (long long)nbm, (long long)nbn);
    return MXFP4_ERR_VALUE;
  }
  w8a8_tile<TO><<<(unsigned)(nbm * nbn), 256, 0, st>>>(g, (int)nbn);
  return launch_status("w8a8 launch");
}

}  // namespace
}  // namespace mx

extern "C" int mxfp4_linear_w8a8(const int8_t* a, const float* a_scales, int64_t m, int64_t k,
                                 const int8_t* w, const float* w_scales, int64_t n,
                                 const void* bias, void* out, int out_dtype, void* stream) {
  using namespace mx;
  if (out_dtype != MXFP4_DT_BF16 && out_dtype != MXFP4_DT_F16 && out_dtype != MXFP4_DT_F32) {
    set_error("w8a8: unsupported output dtype %d", out_dtype);
    return MXFP4_ERR_TYPE;
  }
  if (m < 0 || n < 0 || k < 32 || k % 32 != 0 || k > MXFP4_W8A8_MAX_K) {
    set_error("w8a8: K must be divisible by 32 and at most %d, got %lld (m %lld, n %lld)",
              MXFP4_W8A8_MAX_K, (long long)k, (long long)m, (long long)n);
    return MXFP4_ERR_VALUE;
  }
  if (m > 0x7FFFFFFF || n > 0x7FFFFFFF) {
    set_error("w8a8: too many rows or columns (m %lld, n %lld)", (long long)m, (long long)n);
    return MXFP4_ERR_VALUE;
  }
  if (((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(w)) & 15) != 0) {
    set_error("w8a8: operands must be 16-byte aligned");
    return MXFP4_ERR_VALUE;
  }
  if (m == 0 || n == 0) return MXFP4_OK;
  W8Args g{};
  g.a = reinterpret_cast<const uint8_t*>(a);
  g.a_scale = a_scales;
  g.w = reinterpret_cast<const uint8_t*>(w);
  g.w_scale = w_scales;
  g.bias = bias;
  g.out = out;
  g.m = m;
  g.n = n;
  g.k = (int)k;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (out_dtype) {
    case MXFP4_DT_BF16: return launch_typed<__bf16>(g, st);
    case MXFP4_DT_F16: return launch_typed<_Float16>(g, st);
    default: return launch_typed<float>(g, st);
  }
}
