// W8A8 GEMM: int8 activations with a scale per token times int8 weights with
// a scale per output channel.  No counterpart in the reference.
//
//   out[i, j] = round(float(sum_k a[i, k] w[j, k]) * sa[i] * sw[j] + bias[j])
//
// The sum is exact: products of two bytes added in int32 by the integer
// MFMA (v_mfma_i32_16x16x64_i8), which K <= 131071 cannot overflow (2^14 per
// product), so tiles, waves and splits of K may add in any order and give
// the same bits.  FP32 from there (the sum rounded, times sa, times sw, or by
// one FMA with the bias), one rounding to the output type.
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

// One output value, the same bits in every kernel: the FMA is spelled out
__device__ __forceinline__ float scaled(int acc, float sa, float sw) {
  return (float)acc * sa * sw;
}
__device__ __forceinline__ float scaled(int acc, float sa, float sw, float bias) {
  return fmaf((float)acc * sa, sw, bias);
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
      const float sw = g.w_scale[col + i];
      v = g.bias ? scaled(acc[i], sa, sw, to_f32(static_cast<const TO*>(g.bias)[col + i]))
                 : scaled(acc[i], sa, sw);
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

// ---------------------------------------------------------------- large grids
// 256 x 256 tiles, 2 x 2 waves of 128 x 128 (one per SIMD, 16 32x32 blocks,
// 256 accumulator registers), K in 128-byte stages moved global -> LDS by
// 16-byte-per-lane loads, two stages in LDS.  What bounds such a tile is LDS:
// per 128 bytes of K the waves read (128 + 128) rows each, 128 KB, and the
// loads write 64 KB, 1536 cycles at 128 bytes a cycle, beside 2048 cycles of
// MFMA; 2 x 4 waves of 128 x 64 would read 192 KB, as long as the MFMAs take.
// With one wave a SIMD nothing else hides a wait, so a half stage's fragments
// are read while the half before it is multiplied.
//
// A row's stage is its whole 128-byte line; chunk c of row r sits in slot c ^
// ((r / 2) % 8), which the lane that fills a slot undoes, so that the 16 lanes
// of a read cover all 64 banks.  The 32x32x32 MFMA takes 16 K bytes of row l %
// 32 from lane l (K = (l / 32) * 16 ..).
typedef int i32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ void tile_of_dense(int nbm, int nbn, int idx, int nwg, int& bm,
                                              int& bn) {
  // workgroup i runs on XCD i % 8: each XCD gets a contiguous range of tiles,
  // walked in groups of 4 row blocks, its operands L2 resident
  const int x = idx % 8, i = idx / 8;
  const int per = nwg / 8, rem = nwg % 8;
  const int pid = x * per + (x < rem ? x : rem) + i;
  constexpr int GROUP = 4;
  const int first = (pid / (GROUP * nbn)) * GROUP;
  const int gsize = (nbm - first) < GROUP ? (nbm - first) : GROUP;
  // scalars for the buffer resources: the divisions run on vector registers
  bm = __builtin_amdgcn_readfirstlane(first + (pid % (GROUP * nbn)) % gsize);
  bn = __builtin_amdgcn_readfirstlane((pid % (GROUP * nbn)) / gsize);
}

template <typename TO>
__global__ __launch_bounds__(256, 1) void w8a8_pf(W8Args g, int nbm, int nbn) {
  constexpr int ROWS = 256, STAGE = 2 * ROWS * 128;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * STAGE];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  int bm, bn;
  tile_of_dense(nbm, nbn, blockIdx.x, gridDim.x, bm, bn);
  const int64_t row0 = (int64_t)bm * ROWS, col0 = (int64_t)bn * ROWS;
  const int rows = (int)(g.m - row0 < ROWS ? g.m - row0 : ROWS);
  const int cols = (int)(g.n - col0 < ROWS ? g.n - col0 : ROWS);
  const i32x4 rA = make_rsrc(g.a + row0 * g.k, (uint32_t)rows * g.k);
  const i32x4 rW = make_rsrc(g.w + col0 * g.k, (uint32_t)cols * g.k);

  // wave-load j of this wave: rows j * 32 + wave * 8 + lane / 8
  uint32_t a_off[8], w_off[8];
  const int lrow = wave * 8 + (lane >> 3);
  const int chunk = ((lane & 7) ^ ((lrow >> 1) & 7)) * 16;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int r = j * 32 + lrow;
    a_off[j] = r < rows ? (uint32_t)r * g.k + chunk : kOOB;
    w_off[j] = r < cols ? (uint32_t)r * g.k + chunk : kOOB;
  }
  const int nk = (g.k + 127) >> 7;
  // load j of stage kt: 1 KB of A, 1 KB of W
  auto issue1 = [&](int kt, int j) {
    uint8_t* base = smem + (kt & 1) * STAGE;
    const bool in = chunk < g.k - kt * 128;  // the last stage may be a part
    llvm_amdgcn_raw_buffer_load_lds(rA, lds_ptr(base + (j * 4 + wave) * 1024), 16,
                                    (int)(in ? a_off[j] : kOOB), kt * 128, 0, 0);
    llvm_amdgcn_raw_buffer_load_lds(rW, lds_ptr(base + ROWS * 128 + (j * 4 + wave) * 1024), 16,
                                    (int)(in ? w_off[j] : kOOB), kt * 128, 0, 0);
  };
  auto issue = [&](int kt) {
#pragma unroll
    for (int j = 0; j < 8; ++j) issue1(kt, j);
  };

  i32x16 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

  const int c32 = lane & 31, half = lane >> 5, swz = (lane >> 1) & 7;
  const int a_rd = (wm * 128 + c32) * 128;
  const int w_rd = ROWS * 128 + (wn * 128 + c32) * 128;
  struct Frags {
    i32x4 a[4][2], w[4][2];
  };
  // block i's fragments of half stage `phase`, K 32 t of it
  auto read1 = [&](Frags& f, int kt, int phase, int t, int i) {
    const uint8_t* base = smem + (kt & 1) * STAGE;
    const int slot = (((phase * 2 + t) * 2 + half) ^ swz) * 16;
    f.w[i][t] = *reinterpret_cast<const i32x4*>(base + w_rd + slot + i * 4096);
    f.a[i][t] = *reinterpret_cast<const i32x4*>(base + a_rd + slot + i * 4096);
  };
  auto read = [&](Frags& f, int kt, int phase) {
#pragma unroll
    for (int i = 0; i < 8; ++i) read1(f, kt, phase, i >> 2, i & 3);
  };
  auto multiply = [&](const Frags& f) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[j][t], f.a[i][t], acc[i][j], 0, 0, 0);
  };
  Frags f0, f1;
  issue(0);
  asm volatile("" ::: "memory");
  if (nk > 1) {
    issue(1);
    wait_vmcnt<16>();
  } else {
    wait_vmcnt<0>();
  }
  barrier_only();
  read(f0, 0, 0);
  int kt = 0;
  for (; kt + 2 < nk; ++kt) {
    read(f1, kt, 1);
    multiply(f0);
#pragma unroll
    for (int i = 0; i < 16; ++i) {  // a fragment read, then two MFMAs
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
    }
    // the next stage has landed, and this one is read by all: its place is free
    wait_vmcnt<0>();
    wait_lgkm0();
    barrier_only();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      issue1(kt + 2, i);
      read1(f0, kt + 1, 0, i >> 2, i & 3);
    }
    multiply(f1);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
  }
  for (; kt < nk; ++kt) {
    read(f1, kt, 1);
    multiply(f0);
    if (kt + 1 < nk) {
      wait_vmcnt<0>();
      wait_lgkm0();
      barrier_only();
      read(f0, kt + 1, 0);
    }
    multiply(f1);
  }

  // lane: row l % 32 of its blocks, columns q * 8 + half * 4 .. + 3 (q = 0 .. 3)
  const bool vec = g.n % (16 / (int)sizeof(TO)) == 0 && !(reinterpret_cast<uintptr_t>(g.out) & 15);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float sw[16], bias[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int64_t col = col0 + wn * 128 + j * 32 + (e >> 2) * 8 + half * 4 + (e & 3);
      const bool in = col < g.n;
      sw[e] = in ? g.w_scale[col] : 0.f;
      bias[e] = in && g.bias ? to_f32(static_cast<const TO*>(g.bias)[col]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = row0 + wm * 128 + i * 32 + c32;
      const bool row_in = row < g.m;
      const float sa = row_in ? g.a_scale[row] : 0.f;
      TO* const crow = static_cast<TO*>(g.out) + (row_in ? row : 0) * g.n;
      const int64_t cb = col0 + wn * 128 + j * 32;
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e)
        v[e] = g.bias ? scaled(acc[i][j][e], sa, sw[e], bias[e]) : scaled(acc[i][j][e], sa, sw[e]);
      if constexpr (sizeof(TO) == 4) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int64_t col = cb + q * 8 + half * 4;
          if (!row_in) continue;
          if (vec && col + 4 <= g.n) {
            *reinterpret_cast<f32x4*>(crow + col) =
                f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
          } else {
            for (int e = 0; e < 4; ++e)
              if (col + e < g.n) crow[col + e] = v[4 * q + e];
          }
        }
      } else {
        // the lane halves trade: the lower one gets columns q * 8 .. + 7 of q =
        // 2p, the upper one of q = 2p + 1
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          uint32_t lo[2], hi[2];
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            auto pack = [&](int e) {
              return (uint32_t)__builtin_bit_cast(uint16_t, from_f32<TO>(v[e])) |
                     ((uint32_t)__builtin_bit_cast(uint16_t, from_f32<TO>(v[e + 1])) << 16);
            };
            const auto sw2 = __builtin_amdgcn_permlane32_swap(pack(p * 8 + 2 * w),
                                                             pack(p * 8 + 4 + 2 * w), false, false);
            lo[w] = sw2[0];
            hi[w] = sw2[1];
          }
          const int64_t col = cb + (2 * p + half) * 8;
          if (!row_in) continue;
          const uint32_t o[4] = {lo[0], lo[1], hi[0], hi[1]};
          if (vec && col + 8 <= g.n) {
            *reinterpret_cast<i32x4*>(crow + col) =
                i32x4{(int)o[0], (int)o[1], (int)o[2], (int)o[3]};
          } else {
            for (int e = 0; e < 8; ++e)
              if (col + e < g.n)
                crow[col + e] = __builtin_bit_cast(TO, (uint16_t)(o[e >> 1] >> (16 * (e & 1))));
          }
        }
      }
    }
  }
}

template <typename TO>
int launch_typed(const W8Args& g, hipStream_t st) {
  const int64_t nbm = (g.m + 63) / 64, nbn = (g.n + 63) / 64;
  if (nbm * nbn > 0x7FFFFF) {  // 2^31 threads a launch
    set_error("w8a8: too many tiles (%lld x %lld)", (long long)nbm, (long long)nbn);
    return MXFP4_ERR_VALUE;
  }
  const int64_t bm = (g.m + 255) / 256, bn = (g.n + 255) / 256;
  if (bm * bn >= 160) {
    w8a8_pf<TO><<<(unsigned)(bm * bn), 256, 0, st>>>(g, (int)bm, (int)bn);
    return launch_status("w8a8 launch");
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
