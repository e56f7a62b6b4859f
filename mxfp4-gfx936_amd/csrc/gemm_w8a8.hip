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
#include <cstdlib>

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

extern "C" __device__ uint16_t llvm_amdgcn_raw_buffer_load_i16(i32x4 rsrc, uint32_t voffset,
                                                               int soffset, int aux)
    __asm("llvm.amdgcn.raw.buffer.load.i16");

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

// One bias value by its index in the range; 0 past it
template <typename TO>
__device__ __forceinline__ float load_bias(i32x4 rsrc, int i) {
  if constexpr (sizeof(TO) == 4) {
    return __uint_as_float(buf_load4(rsrc, (uint32_t)i * 4));
  } else {
    return to_f32(__builtin_bit_cast(
        TO, (uint16_t)llvm_amdgcn_raw_buffer_load_i16(rsrc, (uint32_t)i * 2, 0, 0)));
  }
}

template <int FM, int FN>
struct PfShape {
  static constexpr int BM = 64 * FM, BN = 64 * FN;
  static constexpr int A_BYTES = BM * 128, W_BYTES = BN * 128;  // of a stage
  // a third A stage where LDS holds it
  static constexpr int NA = 3 * A_BYTES + 2 * W_BYTES <= 163840 ? 3 : 2;
  static constexpr int LDS = NA * A_BYTES + 2 * W_BYTES;
  static constexpr int NM = FM * FN;  // MFMAs of a phase
};

template <typename TO, int FM, int FN>
__global__ __launch_bounds__(256, 1) void w8a8_pf(W8Args g, int nbm, int nbn) {
  typedef PfShape<FM, FN> S;
  constexpr int BM = S::BM, BN = S::BN, LA = 2 * FM, LW = 2 * FN;  // loads of a wave and stage
  constexpr int HELD = S::NM >= 8 ? 4 : 1;  // MFMAs kept for after the barrier
  __shared__ __attribute__((aligned(1024))) uint8_t smem[S::LDS];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  int bm, bn;
  tile_of_dense(nbm, nbn, blockIdx.x, gridDim.x, bm, bn);
  const int64_t row0 = (int64_t)bm * BM, col0 = (int64_t)bn * BN;
  const int rows = (int)(g.m - row0 < BM ? g.m - row0 : BM);
  const int cols = (int)(g.n - col0 < BN ? g.n - col0 : BN);
  const i32x4 rA = make_rsrc(g.a + row0 * g.k, (uint32_t)rows * g.k);
  const i32x4 rW = make_rsrc(g.w + col0 * g.k, (uint32_t)cols * g.k);

  // wave-load j of this wave: rows j * 32 + wave * 8 + lane / 8
  uint32_t a_off[LA], w_off[LW];
  const int lrow = wave * 8 + (lane >> 3);
  const int chunk = ((lane & 7) ^ ((lrow >> 1) & 7)) * 16;
#pragma unroll
  for (int j = 0; j < LA; ++j) {
    const int r = j * 32 + lrow;
    a_off[j] = r < rows ? (uint32_t)r * g.k + chunk : kOOB;
  }
#pragma unroll
  for (int j = 0; j < LW; ++j) {
    const int r = j * 32 + lrow;
    w_off[j] = r < cols ? (uint32_t)r * g.k + chunk : kOOB;
  }
  const int nk = (g.k + 127) >> 7;
  // 1 KB of stage kt; the last stage may be a part
  auto load_a = [&](int kt, int slot, int j) {
    llvm_amdgcn_raw_buffer_load_lds(rA, lds_ptr(smem + slot * S::A_BYTES + (j * 4 + wave) * 1024),
                                    16, (int)(chunk < g.k - kt * 128 ? a_off[j] : kOOB), kt * 128,
                                    0, 0);
  };
  auto load_w = [&](int kt, int j) {
    llvm_amdgcn_raw_buffer_load_lds(
        rW, lds_ptr(smem + S::NA * S::A_BYTES + (kt & 1) * S::W_BYTES + (j * 4 + wave) * 1024), 16,
        (int)(chunk < g.k - kt * 128 ? w_off[j] : kOOB), kt * 128, 0, 0);
  };

  i32x16 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

  const int c32 = lane & 31, half = lane >> 5, swz = (lane >> 1) & 7;
  const int a_rd = (wm * FM * 32 + c32) * 128;
  const int w_rd = S::NA * S::A_BYTES + (wn * FN * 32 + c32) * 128;
  i32x4 fa[2][FM], fw[2][FN];  // fragments of the even and the odd phases
  // fragment i of phase p (K p * 32 .. + 32): first the weights', then A's
  auto read = [&](auto pc, int kt, int slot, auto ic) {
    constexpr int p = decltype(pc)::value, i = decltype(ic)::value;
    const int at = ((p * 2 + half) ^ swz) * 16;
    if constexpr (i < FN)
      fw[p & 1][i] = *reinterpret_cast<const i32x4*>(smem + (kt & 1) * S::W_BYTES + w_rd + at +
                                                     i * 4096);
    else
      fa[p & 1][i - FN] = *reinterpret_cast<const i32x4*>(smem + slot * S::A_BYTES + a_rd + at +
                                                          (i - FN) * 4096);
  };
  auto multiply = [&](auto pc, auto from, auto to) {
    constexpr int p = decltype(pc)::value;
    static_for<decltype(from)::value, decltype(to)::value>([&](auto mc) {
      constexpr int i = decltype(mc)::value / FN, j = decltype(mc)::value % FN;
      acc[i][j] =
          __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[p & 1][j], fa[p & 1][i], acc[i][j], 0, 0, 0);
    });
  };
  // The order of a phase: NR reads and NL loads, one of each in turn, spread
  // over the first three quarters of NM MFMAs
  auto order = [&](auto nr, auto nl, auto nm) {
    constexpr int NR = decltype(nr)::value, NL = decltype(nl)::value, M = decltype(nm)::value;
    constexpr int N = NR > NL ? NR : NL, SPAN = M * 3 / 4;
    static_for<0, N>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      constexpr int mf = SPAN * (i + 1) / N - SPAN * i / N;
      if constexpr (i < NL) __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
      if constexpr (i < NR) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      if constexpr (mf > 0) __builtin_amdgcn_sched_group_barrier(0x008, mf, 0);
    });
    __builtin_amdgcn_sched_group_barrier(0x008, M - SPAN, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
#define C_(v) std::integral_constant<int, (v)>{}
  constexpr int NR = FM + FN, NM = S::NM;

  int s0 = 0, s1 = 1, s2 = S::NA == 3 ? 2 : 0;  // A's slots of stages kt, kt + 1, kt + 2
  // One stage; MORE: how many follow it (2: at least two)
  auto stage = [&](int kt, auto more) {
    constexpr int MORE = decltype(more)::value;
    constexpr bool early = MORE == 2 && S::NA == 3;
    static_for<0, 3>([&](auto pc) {
      constexpr int p = decltype(pc)::value;
      constexpr int first = p == 0 ? 0 : LA / 2, nl = early && p < 2 ? LA / 2 : 0;
      static_for<0, (NR > nl ? NR : nl)>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if constexpr (i < nl) load_a(kt + 2, s2, first + i);
        if constexpr (i < NR) read(C_(p + 1), kt, s0, ic);
      });
      multiply(pc, C_(0), C_(p == 2 ? NM - HELD : NM));
      order(C_(NR), C_(nl), C_(p == 2 ? NM - HELD : NM));
    });
    if constexpr (MORE > 0) {
      // the next stage has landed, and this one is read by all: its place is free
      wait_vmcnt<early ? LA : 0>();
      wait_lgkm0();
      barrier_only();
      __builtin_amdgcn_sched_barrier(0);
      multiply(C_(2), C_(NM - HELD), C_(NM));
      constexpr int nl = MORE == 2 ? LW + (S::NA == 3 ? 0 : LA) : 0;
      static_for<0, (NR > nl ? NR : nl)>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if constexpr (i < nl) {
          if constexpr (i < LW) load_w(kt + 2, i);
          else load_a(kt + 2, s2, i - LW);
        }
        if constexpr (i < NR) read(C_(0), kt + 1, s1, ic);
      });
      multiply(C_(3), C_(0), C_(NM));
      order(C_(NR), C_(nl), C_(NM + HELD));
      const int t = s0;
      s0 = s1;
      s1 = s2;
      s2 = S::NA == 3 ? t : s0;
    } else {
      multiply(C_(2), C_(NM - HELD), C_(NM));
      multiply(C_(3), C_(0), C_(NM));
    }
  };

  static_for<0, LA>([&](auto j) { load_a(0, 0, decltype(j)::value); });
  static_for<0, LW>([&](auto j) { load_w(0, decltype(j)::value); });
  asm volatile("" ::: "memory");
  if (nk > 1) {
    static_for<0, LA>([&](auto j) { load_a(1, 1, decltype(j)::value); });
    static_for<0, LW>([&](auto j) { load_w(1, decltype(j)::value); });
    wait_vmcnt<LA + LW>();
  } else {
    wait_vmcnt<0>();
  }
  barrier_only();
  static_for<0, NR>([&](auto i) { read(C_(0), 0, 0, i); });
  int kt = 0;
  for (; kt + 2 < nk; ++kt) stage(kt, C_(2));
  if (kt + 1 < nk) {
    stage(kt, C_(1));
    ++kt;
  }
  stage(kt, C_(0));
#undef C_

  // lane: row l % 32 of its blocks, columns q * 8 + half * 4 .. + 3 (q = 0 ..
  // 3).  Scales and bias by range-checked loads, without a branch; a tile
  // inside the output stores without one too.
  const i32x4 rSW = make_rsrc(g.w_scale + col0, (uint32_t)cols * 4);
  const i32x4 rSA = make_rsrc(g.a_scale + row0, (uint32_t)rows * 4);
  const i32x4 rB = make_rsrc(static_cast<const TO*>(g.bias) + (g.bias ? col0 : 0),
                             g.bias ? (uint32_t)(cols * sizeof(TO)) : 0u);
  const bool vec = g.n % (16 / (int)sizeof(TO)) == 0 && !(reinterpret_cast<uintptr_t>(g.out) & 15);
  const bool full = vec && rows == BM && cols == BN;
  float sa[FM];
#pragma unroll
  for (int i = 0; i < FM; ++i)
    sa[i] = __uint_as_float(buf_load4(rSA, ((wm * FM + i) * 32 + c32) * 4));
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    const int cb = (wn * FN + j) * 32;  // the block's columns
    float sw[16], bias[16];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const i32x4 v = buf_load16(rSW, (cb + q * 8 + half * 4) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sw[4 * q + e] = __int_as_float(v[e]);
        if (g.bias) bias[4 * q + e] = load_bias<TO>(rB, cb + q * 8 + half * 4 + e);
      }
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int r = (wm * FM + i) * 32 + c32;
      TO* const crow = static_cast<TO*>(g.out) + (row0 + r) * g.n + col0;
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e)
        v[e] = g.bias ? scaled(acc[i][j][e], sa[i], sw[e], bias[e])
                      : scaled(acc[i][j][e], sa[i], sw[e]);
      if constexpr (sizeof(TO) == 4) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = cb + q * 8 + half * 4;
          if (full || (vec && r < rows && c + 4 <= cols)) {
            *reinterpret_cast<f32x4*>(crow + c) =
                f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
          } else if (r < rows) {
            for (int e = 0; e < 4; ++e)
              if (c + e < cols) crow[c + e] = v[4 * q + e];
          }
        }
      } else {
        // the lane halves trade: the lower one gets columns q * 8 .. + 7 of q =
        // 2p, the upper one of q = 2p + 1
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          uint32_t o[4];
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            auto pack = [&](int e) {
              return (uint32_t)__builtin_bit_cast(uint16_t, from_f32<TO>(v[e])) |
                     ((uint32_t)__builtin_bit_cast(uint16_t, from_f32<TO>(v[e + 1])) << 16);
            };
            const auto t = __builtin_amdgcn_permlane32_swap(pack(p * 8 + 2 * w),
                                                            pack(p * 8 + 4 + 2 * w), false, false);
            o[w] = t[0];
            o[2 + w] = t[1];
          }
          const int c = cb + (2 * p + half) * 8;
          if (full || (vec && r < rows && c + 8 <= cols)) {
            *reinterpret_cast<i32x4*>(crow + c) =
                i32x4{(int)o[0], (int)o[1], (int)o[2], (int)o[3]};
          } else if (r < rows) {
            for (int e = 0; e < 8; ++e)
              if (c + e < cols)
                crow[c + e] = __builtin_bit_cast(TO, (uint16_t)(o[e >> 1] >> (16 * (e & 1))));
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
  static const char* force = getenv("W8CFG");
  auto pf = [&](auto fm, auto fn) {
    constexpr int FM = decltype(fm)::value, FN = decltype(fn)::value;
    typedef PfShape<FM, FN> S;
    const int64_t bm = (g.m + S::BM - 1) / S::BM, bn = (g.n + S::BN - 1) / S::BN;
    w8a8_pf<TO, FM, FN><<<(unsigned)(bm * bn), 256, 0, st>>>(g, (int)bm, (int)bn);
    return launch_status("w8a8 launch");
  };
#define C_(v) std::integral_constant<int, (v)>{}
  int cfg = force ? atoi(force) : (((g.m + 255) / 256) * ((g.n + 255) / 256) >= 160 ? 44 : 0);
  switch (cfg) {
    case 44: return pf(C_(4), C_(4));
    case 45: return pf(C_(4), C_(5));
    case 43: return pf(C_(4), C_(3));
    case 33: return pf(C_(3), C_(3));
    case 42: return pf(C_(4), C_(2));
    case 24: return pf(C_(2), C_(4));
    case 22: return pf(C_(2), C_(2));
    default: break;
  }
#undef C_
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
