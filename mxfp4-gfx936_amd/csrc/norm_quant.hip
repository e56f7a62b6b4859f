// RMS norm with the residual's addition and an 8-bit output with scales, and
// the int8 quantizer by rows, which is its last step alone.  No counterpart
// in the reference.
//
//   h = x + residual (FP32)            residual_out = h rounded to x's type
//   y = h * w * rsqrt(mean(h^2) + eps)          normed = y rounded likewise
//   int8: s = max(max|y| / 127, 2^-126), q = y / s to the nearest (even) integer
//   MX FP8 (blocks of 32): E = floor(log2 max|y|) - emax, q = y * 2^-E rounded
//         to e4m3 (emax 8) / e5m2 (15), saturating; scale byte E + 127
//
// HBM bound: x, the residual and the weights are read once, every output is
// written once.  A workgroup holds a row in registers from its load to its
// last store, so one reduction over the row is enough: h * w does not need
// the mean, and max|y| = max|h * w| * rsqrt(..) is reduced together with the
// sum of squares.  That sum is FP64 (no square of an FP32 value leaves its
// range, and the order of the sum does not show); everything per element is
// FP32.  The quotient y / s is the correctly rounded one: q0 = y * r with r =
// 1 / s, then Markstein's step q0 + (y - q0 * s) * r, two FMAs instead of a
// division.
//
// bf16, residual, int8 out, cold inputs: 8192 x 4096 46.1 us (235 MB, 5.1 TB/s,
// what a large copy reaches), 8192 x 2048 23.8, 2048 x 16384 48.2; the quantizer
// alone at 8192 x 4096 19.4 us (5.2 TB/s).  One row of 2048 2.6 us.  Rows off 16
// bytes go element by element and far from that: 8192 x 4097 297 us, the
// quantizer 71; 2048 x 2049 43 and 14 (2048 x 2048 8.4 and 4.6).
//
// A non-finite row (int8) has scale NaN, a non-finite block (MX) scale byte
// 255, with zeros for its values: it stays what it is for the product.
#include "common.h"

namespace mx {
namespace {

enum { KIND_QUANT = 0, KIND_NORM = 1, KIND_NORM_MX = 2 };

struct NormArgs {
  const void* x;
  const void* residual;  // or nullptr
  const void* weight;
  void* q;
  void* scales;
  void* residual_out;  // or nullptr (no residual)
  void* normed;        // or nullptr
  int64_t rows, ldx, ldr;
  int k, w_f32, e5m2;
  float eps;
};

__device__ __forceinline__ float pow2f(int e) {  // 2^e, e in [-127, 127]
  return e >= -126 ? __uint_as_float((uint32_t)(e + 127) << 23) : __uint_as_float(0x00400000u);
}
__device__ __forceinline__ int floor_log2_bits(uint32_t b) {  // of a finite float's bits, > 0
  const int ex = (int)(b >> 23);
  return ex ? ex - 127 : (31 - __builtin_clz(b)) - 149;
}
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// V consecutive elements as FP32 (V = 8: 16-byte aligned)
template <typename T, int V>
__device__ __forceinline__ void load_elems(const T* p, float (&o)[V]) {
  if constexpr (V == 1) {
    o[0] = (float)*p;
  } else if constexpr (sizeof(T) == 4) {
    const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[i] = a[i];
      o[4 + i] = b[i];
    }
  } else {
    typedef T T8 __attribute__((ext_vector_type(8)));
    const T8 a = *reinterpret_cast<const T8*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (float)a[i];
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_elems(T* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    *p = from_f32<T>(v[0]);
  } else if constexpr (sizeof(T) == 4) {
    reinterpret_cast<f32x4*>(p)[0] = f32x4{v[0], v[1], v[2], v[3]};
    reinterpret_cast<f32x4*>(p)[1] = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    typedef T T8 __attribute__((ext_vector_type(8)));
    T8 a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = from_f32<T>(v[i]);
    *reinterpret_cast<T8*>(p) = a;
  }
}

__device__ __forceinline__ int quant_i8(float y, float s, float r) {
  float q = y * r;
  q = fmaf(fmaf(-q, s, y), r, q);
  return (int)rintf(fminf(fmaxf(q, -127.f), 127.f));
}

// V values of a lane to FP8 (two or one byte at a time), saturating
__device__ __forceinline__ uint32_t fp8_pair(float a, float b, bool e5m2) {
  return e5m2 ? (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false)
              : (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
}

// NT threads a row, C chunks of V elements a thread: V = 8 takes rows in
// 16-byte pieces, V = 1 rows of any length, stride and alignment.  C = 0: a
// row too long for registers, read a second time for its last step.  A
// workgroup takes rows blockIdx.x, + gridDim.x, ...  Every element is written
// by the thread that read it, after it did: residual_out may be an input.
template <typename T, int KIND, int V, int NT, int C>
__global__ __launch_bounds__(NT) void norm_quant(NormArgs a) {
  constexpr int NW = NT / 64;
  constexpr bool NORM = KIND != KIND_QUANT;
  __shared__ double red_ss[2][NW];
  __shared__ uint32_t red_max[2][NW];
  const int tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6;
  const int k = a.k;
  int par = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, par ^= 1) {
    const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
    const T* rr = static_cast<const T*>(a.residual) + (a.residual ? row * a.ldr : 0);
    double ss = 0.0;
    uint32_t amax = 0;

    auto load = [&](int at, float (&v)[V]) {  // v = h
      load_elems<T, V>(xr + at, v);
      if (NORM && a.residual) {
        float r[V];
        load_elems<T, V>(rr + at, r);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] += r[i];
      }
    };
    auto weigh = [&](int at, float (&v)[V]) {  // v = h * w
      if constexpr (NORM) {
        float w[V];
        if (a.w_f32) load_elems<float, V>(static_cast<const float*>(a.weight) + at, w);
        else load_elems<T, V>(static_cast<const T*>(a.weight) + at, w);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] *= w[i];
      }
    };
    auto store_sum = [&](int at, const float (&v)[V]) {
      if (NORM && a.residual_out)
        store_elems<T, V>(static_cast<T*>(a.residual_out) + row * k + at, v);
    };
    auto squares = [&](const float (&v)[V]) {
      if constexpr (NORM) {
#pragma unroll
        for (int i = 0; i < V; ++i) ss = fma((double)v[i], (double)v[i], ss);
      }
    };
    auto largest = [&](const float (&v)[V]) {
      // magnitude bits order as the floats, NaN above infinity
#pragma unroll
      for (int i = 0; i < V; ++i) amax = umax(amax, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    };

    float v[C ? C : 1][V];
    if constexpr (C > 0) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int at = (tid + c * NT) * V;
#pragma unroll
        for (int i = 0; i < V; ++i) v[c][i] = 0.f;
        if (at < k) load(at, v[c]);
      }
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int at = (tid + c * NT) * V;
        if (at >= k) continue;
        store_sum(at, v[c]);
        squares(v[c]);
        weigh(at, v[c]);
        largest(v[c]);
      }
    } else {
      for (int at = tid * V; at < k; at += NT * V) {
        load(at, v[0]);
        squares(v[0]);
        weigh(at, v[0]);
        largest(v[0]);
      }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      if constexpr (NORM) {
        const int lo = __shfl_xor(__double2loint(ss), d), hi = __shfl_xor(__double2hiint(ss), d);
        ss += __hiloint2double(hi, lo);
      }
      if constexpr (KIND != KIND_NORM_MX) amax = umax(amax, (uint32_t)__shfl_xor((int)amax, d));
    }
    if constexpr (NW > 1) {
      // two sets of slots: the next row's writes do not meet this row's reads
      if (lane == 0) {
        red_ss[par][wave] = ss;
        red_max[par][wave] = amax;
      }
      __syncthreads();
      ss = red_ss[par][0];
      amax = red_max[par][0];
#pragma unroll
      for (int i = 1; i < NW; ++i) {
        ss += red_ss[par][i];
        amax = umax(amax, red_max[par][i]);
      }
    }

    float rs = 1.f;  // y = v * rs
    if constexpr (NORM) rs = (float)(1.0 / sqrt(ss / (double)k + (double)a.eps));
    // int8: the largest |v| * rs is the largest |y|, rounded as it was
    const float top = __uint_as_float(amax) * rs;
    const bool bad = !(top < INFINITY);
    const float s = fmaxf(top / 127.f, 1.17549435e-38f);
    const float r = 1.f / s;
    if (KIND != KIND_NORM_MX && tid == 0) static_cast<float*>(a.scales)[row] = bad ? NAN : s;

    auto emit = [&](int at, float (&y)[V]) {
      if constexpr (NORM) {
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] *= rs;
        if (a.normed) store_elems<T, V>(static_cast<T*>(a.normed) + row * k + at, y);
      }
      uint8_t* q = static_cast<uint8_t*>(a.q) + row * k + at;
      if constexpr (KIND != KIND_NORM_MX) {
        if constexpr (V == 1) {
          *q = bad ? 0 : (uint8_t)quant_i8(y[0], s, r);
        } else {
          uint32_t p[2] = {0, 0};
          if (!bad) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              p[i >> 2] |= ((uint32_t)quant_i8(y[i], s, r) & 0xFFu) << ((i & 3) * 8);
          }
          *reinterpret_cast<i32x2*>(q) = i32x2{(int)p[0], (int)p[1]};
        }
      } else {
        // the 32 / V lanes of a block come here together: k % 32 == 0
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) m = umax(m, __float_as_uint(y[i]) & 0x7FFFFFFFu);
#pragma unroll
        for (int d = 1; d < 32 / V; d <<= 1) m = umax(m, (uint32_t)__shfl_xor((int)m, d));
        int e = m ? floor_log2_bits(m) - (a.e5m2 ? 15 : 8) : -127;
        e = e < -127 ? -127 : e;
        const bool nan = m >= 0x7F800000u;
        const float inv = pow2f(-e);
        const float most = a.e5m2 ? 57344.f : 448.f;
        float z[V];
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = nan ? 0.f : fminf(fmaxf(y[i] * inv, -most), most);
        if ((at & 31) == 0)
          static_cast<uint8_t*>(a.scales)[row * (k >> 5) + (at >> 5)] =
              nan ? 255 : (uint8_t)(e + 127);
        if constexpr (V == 1) {
          *q = (uint8_t)fp8_pair(z[0], 0.f, a.e5m2);
        } else {
          uint32_t p[2];
#pragma unroll
          for (int i = 0; i < 2; ++i)
            p[i] = (fp8_pair(z[4 * i], z[4 * i + 1], a.e5m2) & 0xFFFFu) |
                   (fp8_pair(z[4 * i + 2], z[4 * i + 3], a.e5m2) << 16);
          *reinterpret_cast<i32x2*>(q) = i32x2{(int)p[0], (int)p[1]};
        }
      }
    };
    if constexpr (C > 0) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int at = (tid + c * NT) * V;
        if (at < k) emit(at, v[c]);
      }
    } else {
      for (int at = tid * V; at < k; at += NT * V) {
        load(at, v[0]);
        store_sum(at, v[0]);
        weigh(at, v[0]);
        emit(at, v[0]);
      }
    }
  }
}

// More workgroups than the GPU holds at any of the sizes; the rows beyond them
// are taken in turn.
constexpr int64_t kMaxGrid = 16384;

template <typename T, int KIND, int V, int NT, int C>
void launch_shape(const NormArgs& a, hipStream_t st) {
  const unsigned grid = (unsigned)(a.rows < kMaxGrid ? a.rows : kMaxGrid);
  norm_quant<T, KIND, V, NT, C><<<grid, NT, 0, st>>>(a);
}

template <typename T, int KIND>
void launch_rows(const NormArgs& a, bool vec, hipStream_t st) {
  constexpr bool HALF = sizeof(T) == 2;
  if (!vec) {
    if (a.k <= 2048) launch_shape<T, KIND, 1, 256, 8>(a, st);
    else if (a.k <= 16384) launch_shape<T, KIND, 1, 1024, 16>(a, st);
    else launch_shape<T, KIND, 1, 1024, 0>(a, st);
    return;
  }
  // Threads and pieces by the row's length.  Fewer threads with more of the row
  // each where both fit: 2048 x 16384 bf16 512 x 4 48.2 us, 1024 x 2 57.0; 16384 x
  // 1024 128 threads 24.8, 256 half of them idle 30.2; 8192 x 2048 128 x 2 23.8, 256
  // x 1 24.5, but in FP32 (twice the bytes a piece) 37.9 and 35.0; 4096 x 8192
  // FP32 512 x 2 83.8, 256 x 4 89.6.  Rows that do not fill the GPU are a matter of
  // latency, and more threads the quicker.  K = 2048, 256 x 1 and 128 x 2: 1 row 2.6
  // us, 3.2; 130 3.6, 4.3; 512 4.4, 5.2; 1000 5.4, 5.8; 2048 7.7, 8.4; 4096 14.8,
  // 13.2.  K = 4096, 512 x 1 and 256 x 2: 130 rows 4.0, 4.6; 512 5.5, 5.8; 1000 8.0,
  // 8.3; 1200 9.5, 9.0; 4096 25.0, 23.6; in FP32 512 rows 6.6, 7.3; 4096 34.2, 37.5.
  // 512 rows, two a CU, lie below every crossing.
  const bool few = a.rows <= 512;
  if (a.k <= 512) launch_shape<T, KIND, 8, 64, 1>(a, st);
  else if (a.k <= 1024) launch_shape<T, KIND, 8, 128, 1>(a, st);
  else if (a.k <= 2048 && HALF && !few) launch_shape<T, KIND, 8, 128, 2>(a, st);
  else if (a.k <= 2048) launch_shape<T, KIND, 8, 256, 1>(a, st);
  else if (a.k <= 4096 && few) launch_shape<T, KIND, 8, 512, 1>(a, st);
  else if (a.k <= 4096) launch_shape<T, KIND, 8, 256, 2>(a, st);
  else if (a.k <= 8192) launch_shape<T, KIND, 8, 512, 2>(a, st);
  else if (a.k <= 16384) launch_shape<T, KIND, 8, 512, 4>(a, st);
  else launch_shape<T, KIND, 8, 1024, 0>(a, st);
}

template <int KIND>
int launch_kind(const NormArgs& a, int x_dtype, hipStream_t st) {
  const int es = x_dtype == MXFP4_DT_F32 ? 4 : 2;
  auto odd = [](const void* p, int64_t stride_bytes) {
    return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)stride_bytes) & 15) != 0;
  };
  // 8 elements at a time need 16-byte aligned rows everywhere (q: 8 bytes)
  bool vec = a.k % 8 == 0 && !odd(a.x, a.ldx * es) && !(reinterpret_cast<uintptr_t>(a.q) & 7);
  if (a.residual) vec = vec && !odd(a.residual, a.ldr * es) && !odd(a.residual_out, a.k * es);
  if (a.normed) vec = vec && !odd(a.normed, a.k * es);
  if (a.weight) vec = vec && !odd(a.weight, 0);
  switch (x_dtype) {
    case MXFP4_DT_BF16: launch_rows<__bf16, KIND>(a, vec, st); break;
    case MXFP4_DT_F16: launch_rows<_Float16, KIND>(a, vec, st); break;
    default: launch_rows<float, KIND>(a, vec, st); break;
  }
  return launch_status("8-bit row quantizer launch");
}

int check_rows(const char* what, int x_dtype, int64_t rows, int64_t k, int64_t stride) {
  if (x_dtype != MXFP4_DT_BF16 && x_dtype != MXFP4_DT_F16 && x_dtype != MXFP4_DT_F32) {
    set_error("%s: unsupported input dtype %d", what, x_dtype);
    return MXFP4_ERR_TYPE;
  }
  if (rows < 0 || k < 1 || k > MXFP4_NORM_MAX_K || stride < k) {
    set_error("%s: invalid sizes (rows %lld, K %lld of 1 to %d, row stride %lld)", what,
              (long long)rows, (long long)k, MXFP4_NORM_MAX_K, (long long)stride);
    return MXFP4_ERR_VALUE;
  }
  return MXFP4_OK;
}

}  // namespace
}  // namespace mx

extern "C" int mxfp4_quant_int8(const void* x, int x_dtype, int64_t rows, int64_t k,
                                int64_t x_row_stride, int8_t* q, float* scales, void* stream) {
  using namespace mx;
  const int rc = check_rows("int8 quantizer", x_dtype, rows, k, x_row_stride);
  if (rc != MXFP4_OK || rows == 0) return rc;
  NormArgs a{};
  a.x = x;
  a.ldx = x_row_stride;
  a.q = q;
  a.scales = scales;
  a.rows = rows;
  a.k = (int)k;
  return launch_kind<KIND_QUANT>(a, x_dtype, static_cast<hipStream_t>(stream));
}

extern "C" int mxfp4_rms_norm_quant(const void* x, int x_dtype, int64_t rows, int64_t k,
                                    int64_t x_row_stride, const void* residual,
                                    int64_t residual_row_stride, const void* weight,
                                    int weight_dtype, float eps, int q_dtype, void* q,
                                    void* scales, void* residual_out, void* normed, void* stream) {
  using namespace mx;
  const int rc = check_rows("RMS norm", x_dtype, rows, k, x_row_stride);
  if (rc != MXFP4_OK) return rc;
  if (weight_dtype != x_dtype && weight_dtype != MXFP4_DT_F32) {
    set_error("RMS norm: the weight is of x's dtype or FP32, got dtype %d", weight_dtype);
    return MXFP4_ERR_TYPE;
  }
  if (q_dtype != MXFP4_DT_I8 && q_dtype != MXFP4_DT_F8E4M3 && q_dtype != MXFP4_DT_F8E5M2) {
    set_error("RMS norm: unsupported output dtype %d", q_dtype);
    return MXFP4_ERR_TYPE;
  }
  if (q_dtype != MXFP4_DT_I8 && k % 32 != 0) {
    set_error("RMS norm: MX blocks need K divisible by 32, got %lld", (long long)k);
    return MXFP4_ERR_VALUE;
  }
  if ((residual != nullptr) != (residual_out != nullptr) ||
      (residual != nullptr && residual_row_stride < k)) {
    set_error("RMS norm: residual and residual_out go together, rows of at least K");
    return MXFP4_ERR_VALUE;
  }
  // in place a row must lie where it is read: another stride would write rows
  // that other workgroups still read
  if (residual_out != nullptr && rows > 1 &&
      ((residual_out == residual && residual_row_stride != k) ||
       (residual_out == x && x_row_stride != k))) {
    set_error("RMS norm: residual_out in place needs rows of stride K");
    return MXFP4_ERR_VALUE;
  }
  if (!(eps > 0.f && eps < INFINITY)) {
    set_error("RMS norm: eps must be positive and finite");
    return MXFP4_ERR_VALUE;
  }
  if (rows == 0) return MXFP4_OK;
  NormArgs a{};
  a.x = x;
  a.ldx = x_row_stride;
  a.residual = residual;
  a.ldr = residual_row_stride;
  a.weight = weight;
  a.q = q;
  a.scales = scales;
  a.residual_out = residual_out;
  a.normed = normed;
  a.rows = rows;
  a.k = (int)k;
  a.w_f32 = weight_dtype == MXFP4_DT_F32;
  a.e5m2 = q_dtype == MXFP4_DT_F8E5M2;
  a.eps = eps;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (q_dtype == MXFP4_DT_I8) return launch_kind<KIND_NORM>(a, x_dtype, st);
  return launch_kind<KIND_NORM_MX>(a, x_dtype, st);
}
