// Quantizers to FP8 (e4m3) with an FP32 scale for each 128 values: the inputs of
// the block-scaled FP8 products.  No counterpart in the reference.
//
//   rows:    s = max(max|x| / 448, 2^-126) over 128 values along a row
//   SiLU-mul rows: the same of h = g / (1 + exp(-g)) * u, x = [g | u]
//   blocks:  s over 128 rows x 128 columns (weights)
//   q = x / s rounded to the nearest e4m3 (ties to even)
//
// 16-bit values x often lie next to the middle between two e4m3 steps, where the
// FP32 quotient's own rounding would decide: its last bit is set where the
// division leaves a remainder (rounding to odd), so that the second rounding is
// the exact quotient's.  Below s = 2^-90, where a remainder may lie below every FP32
// number, x and s are taken times 2^64.  That takes a dozen operations a value; x * (1 / s),
// off by two FP32 steps at most, gives the same e4m3 value unless it lies within four of a
// middle or among e4m3's subnormals, and only a wave that has such a value does the division.
// max|x| <= 448 s (1 + 2^-23): no value saturates.  A group with a value that is
// not finite has s = NaN and q = 0.
#include "gemm.h"

namespace mx {
namespace {

constexpr uint32_t kInf = 0x7F800000u;

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// x / s, last bit set where it is not exact; r = 1 / s
__device__ __forceinline__ float quotient(float x, float s, float r) {
  float q = x * r;
  q = fmaf(fmaf(-q, s, x), r, q);
  const float rem = fmaf(-q, s, x);
  const uint32_t b = __float_as_uint(q);
  // to the odd one of q and its neighbour on the remainder's side
  const uint32_t odd = (b - ((__float_as_uint(rem) ^ b) >> 31)) | 1u;
  return rem == 0.f ? q : __uint_as_float(odd);
}

template <int V>
__device__ __forceinline__ void quotients(const float (&x)[V], float s, float r, float (&q)[V]) {
  if (__any(s < 0x1p-90f)) {  // a branch: the factors in every wave cost 2 to 4%
    const float up = s < 0x1p-90f ? 0x1p64f : 1.f;
#pragma unroll
    for (int i = 0; i < V; ++i) q[i] = quotient(x[i] * up, s * up, r * (1.f / up));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) q[i] = quotient(x[i], s, r);
  }
}

__device__ __forceinline__ float scale_of(uint32_t amax) {
  return amax < kInf ? fmaxf(__uint_as_float(amax) / 448.f, 0x1p-126f)
                     : __uint_as_float(0x7FC00000u);
}

// SiLU(g) * u.  exp2 and the reciprocal to an ulp or two; -g / ln 2 rounded once, so
// that the result's relative error is about |g| * 2^-24: FP8 keeps 2^-4.  Below -80 the
// sum is taken times 2^-32, whose reciprocal is then still a normal number (1 / (1 + e)
// itself would be flushed to 0 from -87.3 on); 0 from about -110 on.
__device__ __forceinline__ float silu_mul(float g, float u) {
  const bool low = g < -80.f;
  const float one = low ? 0x1p-32f : 1.f;
  const float e = __builtin_amdgcn_exp2f(fmaf(g, -1.44269504088896f, low ? -32.f : 0.f));
  return g * __builtin_amdgcn_rcpf(one + e) * u * one;
}

// 16 bytes (fp32: twice) as 8 values
template <typename T, int NL>
__device__ __forceinline__ void values_of(const i32x4 (&raw)[NL], float (&o)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __uint_as_float((uint32_t)raw[i / 4][i % 4]);
  } else {
    typedef T T8 __attribute__((ext_vector_type(8)));
    const T8 a = __builtin_bit_cast(T8, raw[0]);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (float)a[i];
  }
}

__device__ __forceinline__ void store_fp8(uint8_t* p, const float (&v)[8], float s, bool finite) {
  const float r = 1.f / s;
  float q[8];
  uint32_t middle = ~0u, small = ~0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    q[i] = v[i] * r;
    const uint32_t b = __float_as_uint(q[i]);
    // the 20 bits below e4m3's, from four steps below the middle on
    const uint32_t m = (b + 0x80004u) << 12, a = (b << 1) - 1u;
    middle = middle < m ? middle : m;
    small = small < a ? small : a;  // magnitudes but 0, doubled
  }
  if (__any(middle < 8u << 12 || small < 0x3C800000u << 1))  // 2^-6
    quotients<8>(v, s, r, q);
  int w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i], q[4 * i + 1], 0, false);
    w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i + 2], q[4 * i + 3], t, true);
  }
  *reinterpret_cast<i32x2*>(p) = finite ? i32x2{w[0], w[1]} : i32x2{0, 0};
}

__device__ __forceinline__ uint8_t fp8_of(float q, bool finite) {
  return finite ? (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(q, 0.f, 0, false) : 0;
}

struct RowArgs {
  const void* x;
  int64_t rows, k, ldx;
  uint8_t* q;
  float* scales;
  int64_t ss_row, ss_block;  // strides of the scales, in values
};

// A workgroup takes R rows x 4 groups: with V = 8 a wave has one row's 512 columns at a
// time (16 lanes a group), with V = 1 (rows off 16 bytes) one group (64 lanes, two
// values each).  The scales go through LDS, so that those of consecutive rows, which lie
// side by side where the blocks are outermost, are stored together: 64 bytes with R =
// 16.  HBM bound then (8192 x 4096 bf16 24.8 us, 4.1 TB/s; 4096 x 4096 fp32 15.2, 5.5; with
// a wait at each row's load 1.20 times the time; R = 8 1.04; a row's parts far apart in
// time, so that all read the same few of the memory's channels, 1.13).  Grids that do not
// fill the GPU take R = 4, a row a wave, for the shorter chain: 200 x 768 SiLU-mul 4.8 ->
// 3.3 us, 1 x 2048 3.4 -> 2.8.  Where K ends inside the 512 columns of a part (768: half of
// the second), the lanes past it load what they do not use: 4072 x 768 SiLU-mul 7.4 us, 2.4
// times its bytes.
template <typename T, int V, bool SILU, int R>
__global__ __launch_bounds__(256) void quant_rows(RowArgs a) {
  __shared__ float sc[4][R];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t blocks = (a.k + 127) >> 7;
  const uint32_t parts = (uint32_t)((a.k + 511) >> 9);  // workgroups a row; gridDim: of whole rows
  const int64_t b0 = (int64_t)(blockIdx.x % parts) * 4;
  const uint32_t step = gridDim.x / parts;
  for (int64_t row0 = (int64_t)(blockIdx.x / parts) * R; row0 < a.rows;
       row0 += (int64_t)step * R) {
    if constexpr (V == 8) {
      const int64_t col = b0 * 128 + lane * 8;
      const bool in = col < a.k;
      // every load before the first value is used; past the end the last row's again, and
      // past K the row's first 16 bytes, which count as zeros
      constexpr int NL = sizeof(T) == 4 ? 2 : 1, G = SILU ? 2 : 1;
      i32x4 raw[R / 4][G][NL];
#pragma unroll
      for (int i = 0; i < R / 4; ++i) {
        const int64_t row = row0 + i * 4 + wave;
        const T* p = static_cast<const T*>(a.x) + (row < a.rows ? row : a.rows - 1) * a.ldx;
#pragma unroll
        for (int h = 0; h < G; ++h)
#pragma unroll
          for (int l = 0; l < NL; ++l)
            raw[i][h][l] = reinterpret_cast<const i32x4*>(p + h * a.k + (in ? col : 0))[l];
      }
#pragma unroll
      for (int i = 0; i < R / 4; ++i) {
        const int64_t row = row0 + i * 4 + wave;
        float v[8], u[8];
        values_of<T>(raw[i][0], v);
        if constexpr (SILU) {
          values_of<T>(raw[i][1], u);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = silu_mul(v[j], u[j]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = in ? v[j] : 0.f;
        uint32_t amax = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = umax(amax, __float_as_uint(v[j]) & 0x7FFFFFFFu);
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) amax = umax(amax, __shfl_xor((int)amax, off));
        const float s = scale_of(amax);
        if (in && row < a.rows) store_fp8(a.q + row * a.k + col, v, s, amax < kInf);
        if ((lane & 15) == 0) sc[lane >> 4][i * 4 + wave] = s;
      }
    } else {
#pragma unroll 2
      for (int i = 0; i < R; ++i) {  // this wave's group of row i
        const int64_t row = row0 + i;
        float v[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int64_t col = (b0 + wave) * 128 + j * 64 + lane;
          if (col < a.k && row < a.rows) {
            const T* p = static_cast<const T*>(a.x) + row * a.ldx + col;
            v[j] = (float)*p;
            if constexpr (SILU) v[j] = silu_mul(v[j], (float)p[a.k]);
          }
        }
        uint32_t amax = umax(__float_as_uint(v[0]) & 0x7FFFFFFFu,
                             __float_as_uint(v[1]) & 0x7FFFFFFFu);
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) amax = umax(amax, __shfl_xor((int)amax, off));
        const float s = scale_of(amax);
        float q[2];
        quotients<2>(v, s, 1.f / s, q);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int64_t col = (b0 + wave) * 128 + j * 64 + lane;
          if (col < a.k && row < a.rows) a.q[row * a.k + col] = fp8_of(q[j], amax < kInf);
        }
        if (lane == 0) sc[wave][i] = s;
      }
    }
    __syncthreads();
    if (tid < 4 * R) {
      const int64_t b = b0 + tid / R, row = row0 + tid % R;
      if (b < blocks && row < a.rows)
        a.scales[row * a.ss_row + b * a.ss_block] = sc[tid / R][tid % R];
    }
    __syncthreads();
  }
}

// A workgroup a block of 128 x 128; thread: 8 (or, V = 1, strided single) columns of
// rows tid / 16 + 16 i.  HBM bound from a round of the CUs on: 8192 x 4096 bf16 25 us, 4.0
// TB/s; an expert's 1536 x 2048 fp32, 192 workgroups, 7.3.
template <typename T, int V>
__global__ __launch_bounds__(256) void quant_blocks(const T* __restrict__ x, int64_t rows,
                                                    int64_t k, int64_t ldx,
                                                    uint8_t* __restrict__ q,
                                                    float* __restrict__ scales) {
  __shared__ uint32_t part[4];
  const int tid = threadIdx.x;
  const int64_t kb = (k + 127) >> 7;
  const int64_t bi = blockIdx.x / kb, bj = blockIdx.x % kb;
  float v[64];
  auto col_of = [&](int j) {
    return bj * 128 + (V == 8 ? (tid & 15) * 8 + j : (tid & 15) + 16 * j);
  };
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = bi * 128 + (tid >> 4) + 16 * i;
    float t[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (row < rows) {
      if constexpr (V == 8) {
        if (col_of(0) < k) {
          constexpr int NL = sizeof(T) == 4 ? 2 : 1;
          i32x4 raw[NL];
#pragma unroll
          for (int l = 0; l < NL; ++l)
            raw[l] = reinterpret_cast<const i32x4*>(x + row * ldx + col_of(0))[l];
          values_of<T>(raw, t);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col_of(j) < k) t[j] = (float)x[row * ldx + col_of(j)];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[i * 8 + j] = t[j];
      amax = umax(amax, __float_as_uint(t[j]) & 0x7FFFFFFFu);
    }
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) amax = umax(amax, __shfl_xor((int)amax, off));
  if ((tid & 63) == 0) part[tid >> 6] = amax;
  __syncthreads();
  amax = umax(umax(part[0], part[1]), umax(part[2], part[3]));
  const float s = scale_of(amax);
  if (tid == 0) scales[blockIdx.x] = s;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = bi * 128 + (tid >> 4) + 16 * i;
    if (row >= rows) continue;
    float t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = v[i * 8 + j];
    if constexpr (V == 8) {
      if (col_of(0) < k) store_fp8(q + row * k + col_of(0), t, s, amax < kInf);
    } else {
      float z[8];
      quotients<8>(t, s, 1.f / s, z);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col_of(j) < k) q[row * k + col_of(j)] = fp8_of(z[j], amax < kInf);
    }
  }
}

template <typename T, int R>
void launch_rows(const RowArgs& a, bool silu, bool vec, hipStream_t st) {
  const int64_t nx = (a.rows + R - 1) / R, ny = (a.k + 511) / 512;
  const int64_t most = 0x7FFFFF / ny;  // 2^31 threads a launch
  const unsigned grid = (unsigned)((nx < most ? nx : most) * ny);
  if (silu) {
    if (vec) quant_rows<T, 8, true, R><<<grid, 256, 0, st>>>(a);
    else quant_rows<T, 1, true, R><<<grid, 256, 0, st>>>(a);
  } else {
    if (vec) quant_rows<T, 8, false, R><<<grid, 256, 0, st>>>(a);
    else quant_rows<T, 1, false, R><<<grid, 256, 0, st>>>(a);
  }
}

template <typename T>
void launch_rows(const RowArgs& a, bool silu, bool vec, hipStream_t st) {
  // 16 rows a workgroup fill the GPU from two a CU on
  const bool few = (a.rows + 15) / 16 * ((a.k + 511) / 512) < 2 * device_cus();
  if (few) launch_rows<T, 4>(a, silu, vec, st);
  else launch_rows<T, 16>(a, silu, vec, st);
}

}  // namespace
}  // namespace mx

extern "C" int mxfp4_quant_fp8_rows(const void* x, int x_dtype, int64_t rows, int64_t k,
                                    int64_t x_row_stride, int silu_mul, uint8_t* q, float* scales,
                                    int64_t scale_row_stride, int64_t scale_block_stride,
                                    void* stream) {
  using namespace mx;
  if (x_dtype != MXFP4_DT_BF16 && x_dtype != MXFP4_DT_F16 && x_dtype != MXFP4_DT_F32) {
    set_error("fp8 quantizer: unsupported input dtype %d", x_dtype);
    return MXFP4_ERR_TYPE;
  }
  const int64_t width = silu_mul ? 2 * k : k;
  if (rows < 0 || k < 1 || k > MXFP4_FP8_MAX_K || x_row_stride < width ||
      scale_row_stride < 1 || scale_block_stride < 1) {
    set_error("fp8 quantizer: rows of 1 to %d values, got %lld (stride %lld, rows %lld)",
              MXFP4_FP8_MAX_K, (long long)k, (long long)x_row_stride, (long long)rows);
    return MXFP4_ERR_VALUE;
  }
  if (rows == 0) return MXFP4_OK;
  const RowArgs a{x, rows, k, x_row_stride, q, scales, scale_row_stride, scale_block_stride};
  const int64_t b = x_dtype == MXFP4_DT_F32 ? 4 : 2;
  const uintptr_t low = reinterpret_cast<uintptr_t>(x) | (uintptr_t)(x_row_stride * b);
  const bool vec = k % 8 == 0 && (low & 15) == 0 && (reinterpret_cast<uintptr_t>(q) & 7) == 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (x_dtype) {
    case MXFP4_DT_BF16: launch_rows<__bf16>(a, silu_mul != 0, vec, st); break;
    case MXFP4_DT_F16: launch_rows<_Float16>(a, silu_mul != 0, vec, st); break;
    default: launch_rows<float>(a, silu_mul != 0, vec, st); break;
  }
  return launch_status("fp8 quantizer launch");
}

extern "C" int mxfp4_quant_fp8_blocks(const void* x, int x_dtype, int64_t rows, int64_t k,
                                      int64_t x_row_stride, uint8_t* q, float* scales,
                                      void* stream) {
  using namespace mx;
  if (x_dtype != MXFP4_DT_BF16 && x_dtype != MXFP4_DT_F16 && x_dtype != MXFP4_DT_F32) {
    set_error("fp8 quantizer: unsupported input dtype %d", x_dtype);
    return MXFP4_ERR_TYPE;
  }
  const int64_t blocks = rows < 0 || k < 1 ? 0 : ((rows + 127) / 128) * ((k + 127) / 128);
  if (rows < 0 || k < 1 || k > MXFP4_FP8_MAX_K || x_row_stride < k || blocks > 0x7FFFFF) {
    set_error("fp8 quantizer: %lld rows of %lld values (stride %lld)", (long long)rows,
              (long long)k, (long long)x_row_stride);
    return MXFP4_ERR_VALUE;
  }
  if (rows == 0) return MXFP4_OK;
  const int64_t b = x_dtype == MXFP4_DT_F32 ? 4 : 2;
  const uintptr_t low = reinterpret_cast<uintptr_t>(x) | (uintptr_t)(x_row_stride * b);
  const bool vec = k % 8 == 0 && (low & 15) == 0 && (reinterpret_cast<uintptr_t>(q) & 7) == 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto go = [&](auto type) {
    typedef decltype(type) T;
    if (vec)
      quant_blocks<T, 8><<<(unsigned)blocks, 256, 0, st>>>(static_cast<const T*>(x), rows, k,
                                                           x_row_stride, q, scales);
    else
      quant_blocks<T, 1><<<(unsigned)blocks, 256, 0, st>>>(static_cast<const T*>(x), rows, k,
                                                           x_row_stride, q, scales);
  };
  switch (x_dtype) {
    case MXFP4_DT_BF16: go(__bf16{}); break;
    case MXFP4_DT_F16: go(_Float16{}); break;
    default: go(float{}); break;
  }
  return launch_status("fp8 quantizer launch");
}
