// W8A8 GEMM: int8 activations with a scale per token times int8 weights with
// a scale per output channel.  No counterpart in the reference.
//
//   out[i, j] = round(float(sum_k a[i, k] w[j, k]) * sa[i] * sw[j] + bias[j])
//
// The sum is exact: products of two bytes added in int32 by the integer MFMAs,
// which K <= 131071 cannot overflow (2^14 per product), so tiles, waves and
// splits of K may add in any order and give the same bits.  FP32 from there (the
// sum rounded, times sa, then one FMA with sw and the bias), one rounding to the
// output type.
//
// Operands of the 16x16x64 MFMA: lane l supplies 16 consecutive K bytes of row l %
// 16 (K = (l / 16) * 16 ..); of the 32x32x32 one, of row l % 32 (K = (l / 32) * 16
// ..).  The weights are the A operand and the activations the B operand, so a
// lane receives consecutive columns of one row.
#include "gemm.h"

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

// One output value, the same bits in every kernel.  Without a bias it is -0.0:
// then the FMA is the product, to its sign.
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
      v = scaled(acc[i], sa, g.w_scale[col + i],
                 g.bias ? to_f32(static_cast<const TO*>(g.bias)[col + i]) : -0.f);
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

// ---------------------------------------------------------------- large grids
// Tiles of 64 FM x 64 FN, 2 x 2 waves of FM x FN blocks of 32 x 32; at the largest,
// 256 x 256, one wave a SIMD with 256 accumulator registers.  K moves global ->
// LDS in 128-byte stages by 16-byte-per-lane loads.
//
// What bounds such a tile is LDS and then power.  Per 128 bytes of K the four
// waves of 128 x 128 read 128 KB and the loads write 64 KB, 1536 cycles at 128
// bytes a cycle, beside 2048 cycles of MFMA; 2 x 4 waves of 128 x 64 would read
// 192 KB, as long as the MFMAs take.  With one wave a SIMD nothing else hides a
// wait, so the fragments of 32 bytes of K (a phase) are read while those before
// them are multiplied, and loads and reads are dealt out among the MFMAs.  The
// barrier of a stage comes before its last phase, some MFMAs kept back for the
// waves that wait at it.  LDS holds three stages of A, whose loads run two
// stages ahead, and two of W.
//
// Counters at 8192^3 (random bytes, 437 us, 2.5 POP/s): MFMAs busy 75% of the
// cycles, no LDS conflicts, 128 bytes an L2 request; the clock falls to 1.6 GHz.
// 8192 x 4096 x 4096: 119 us, of zeros 91.  Kept from the sums to the output: no
// branch (loads of scales by column under a condition cost 6 us a tile).
//
// KG > 1: groups of four waves take every KG-th stage of the same tile, for grids
// that would leave a SIMD one wave of small tiles (1021 x 4096 x 2048, 128 x 64:
// 16.4 us with one group, 14.0 with two).
//
// A row's stage is its whole 128-byte line; chunk c of row r sits in slot c ^
// ((r / 2) % 8), which the lane that fills a slot undoes, so that the 16 lanes
// of a read cover all 64 banks.
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

template <int FM, int FN, int KG>
struct PfShape {
  static constexpr int BM = 64 * FM, BN = 64 * FN;
  static constexpr int A_BYTES = BM * 128, W_BYTES = BN * 128;  // of a stage
  static constexpr int W_AT = 3 * A_BYTES;  // A's three stages first
  static constexpr int LDS = W_AT + 2 * W_BYTES;
  static_assert(KG * LDS <= 163840, "the stages fit a CU's LDS");
  static constexpr int NM = FM * FN;  // MFMAs of a phase
};

// ROW16: the output's rows are 16-byte aligned.  (Two kernels: with both ways
// to store in one, the sums of either are moved out of the accumulators first.)
template <typename TO, int FM, int FN, int KG, bool ROW16>
__global__ __launch_bounds__(256 * KG, 1) void w8a8_pf(W8Args g, int nbm, int nbn) {
  typedef PfShape<FM, FN, KG> S;
  constexpr int BM = S::BM, BN = S::BN, LA = 2 * FM, LW = 2 * FN;  // loads of a wave and stage
  constexpr int HELD = S::NM >= 8 ? 4 : 1;  // MFMAs kept for after the barrier
  __shared__ __attribute__((aligned(1024))) uint8_t lds[KG * S::LDS];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int group = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 8);
  const int wave = __builtin_amdgcn_readfirstlane((tid >> 6) & 3);
  const int wm = wave >> 1, wn = wave & 1;
  uint8_t* const smem = lds + group * S::LDS;
  int bm, bn;
  tile_of_dense(nbm, nbn, blockIdx.x, gridDim.x, bm, bn);
  const int64_t row0 = (int64_t)bm * BM, col0 = (int64_t)bn * BN;
  const int rows = (int)(g.m - row0 < BM ? g.m - row0 : BM);
  const int cols = (int)(g.n - col0 < BN ? g.n - col0 : BN);
  const i32x4 rA = make_rsrc(g.a + row0 * g.k, (uint32_t)rows * g.k);
  const i32x4 rW = make_rsrc(g.w + col0 * g.k, (uint32_t)cols * g.k);

  const int c32 = lane & 31, half = lane >> 5;
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
  // group q takes stages q, q + KG, ..; all the same number: past K are zeros
  const int nk = (g.k + 128 * KG - 1) / (128 * KG);
  auto k0 = [&](int kt) { return (kt * KG + group) * 128; };
  // 1 KB of stage kt; the last stage may be a part
  auto load_a = [&](int kt, int slot, int j) {
    llvm_amdgcn_raw_buffer_load_lds(rA, lds_ptr(smem + slot * S::A_BYTES + (j * 4 + wave) * 1024),
                                    16, (int)(chunk < g.k - k0(kt) ? a_off[j] : kOOB), k0(kt), 0,
                                    0);
  };
  auto load_w = [&](int kt, int j) {
    llvm_amdgcn_raw_buffer_load_lds(
        rW, lds_ptr(smem + S::W_AT + (kt & 1) * S::W_BYTES + (j * 4 + wave) * 1024), 16,
        (int)(chunk < g.k - k0(kt) ? w_off[j] : kOOB), k0(kt), 0, 0);
  };

  // The scales of the lane's row and columns (row l % 32 of its blocks, columns
  // q * 8 + half * 4 .. + 3, q = 0 .. 3), range-checked, on their way while K
  // is multiplied
  const i32x4 rSW = make_rsrc(g.w_scale + col0, (uint32_t)cols * 4);
  const i32x4 rSA = make_rsrc(g.a_scale + row0, (uint32_t)rows * 4);
  f32x4 sw[FN][4];
  float sa[FM];
#pragma unroll
  for (int i = 0; i < FM; ++i)
    sa[i] = __uint_as_float(buf_load4(rSA, ((wm * FM + i) * 32 + c32) * 4));
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      sw[j][q] = __builtin_bit_cast(
          f32x4, buf_load16(rSW, ((wn * FN + j) * 32 + q * 8 + half * 4) * 4));

  i32x16 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

  const int swz = (lane >> 1) & 7;
  const int a_rd = (wm * FM * 32 + c32) * 128;
  const int w_rd = S::W_AT + (wn * FN * 32 + c32) * 128;
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

  int s0 = 0, s1 = 1, s2 = 2;  // A's slots of stages kt, kt + 1, kt + 2
  // One stage; MORE: how many follow it (2: at least two)
  auto stage = [&](int kt, auto more) {
    constexpr int MORE = decltype(more)::value;
    static_for<0, 3>([&](auto pc) {
      constexpr int p = decltype(pc)::value;
      constexpr int first = p == 0 ? 0 : LA / 2, nl = MORE == 2 && p < 2 ? LA / 2 : 0;
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
      wait_vmcnt<MORE == 2 ? LA : 0>();  // all but A of the stage after it
      wait_lgkm0();
      barrier_only();
      __builtin_amdgcn_sched_barrier(0);
      multiply(C_(2), C_(NM - HELD), C_(NM));
      constexpr int nl = MORE == 2 ? LW : 0;
      static_for<0, (NR > nl ? NR : nl)>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if constexpr (i < nl) load_w(kt + 2, i);
        if constexpr (i < NR) read(C_(0), kt + 1, s1, ic);
      });
      multiply(C_(3), C_(0), C_(NM));
      order(C_(NR), C_(nl), C_(NM + HELD));
      const int t = s0;
      s0 = s1;
      s1 = s2;
      s2 = t;
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

  if constexpr (KG > 1) {  // the first group adds the others' sums
    wait_lgkm0();  // the sums take the fragments' place: every wave has read its last
    barrier_only();
    i32x4* const sums = reinterpret_cast<i32x4*>(lds);
    auto at = [&](int q, int i, int j, int e) {
      return ((((q - 1) * 4 + wave) * S::NM + i * FN + j) * 4 + e) * 64 + lane;
    };
    if (group > 0) {
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sums[at(group, i, j, e)] = i32x4{acc[i][j][4 * e], acc[i][j][4 * e + 1],
                                             acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]};
    }
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int q = 1; q < KG; ++q)
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const i32x4 v = sums[at(q, i, j, e)];
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[i][j][4 * e + x] += v[x];
          }
  }

  const i32x4 rB = make_rsrc(static_cast<const TO*>(g.bias) + (g.bias ? col0 : 0),
                             g.bias ? (uint32_t)(cols * sizeof(TO)) : 0u);
  auto bias_of = [&](int j, float (&b)[16]) {
#pragma unroll
    for (int e = 0; e < 16; ++e) b[e] = -0.f;
    if (g.bias) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        b[e] = load_bias<TO>(rB, (wn * FN + j) * 32 + (e >> 2) * 8 + half * 4 + (e & 3));
    }
  };
  TO* const tile = static_cast<TO*>(g.out) + row0 * g.n + col0;
  if constexpr (ROW16) {
    // from the registers, 16 bytes a lane
    const bool full = rows == BM && cols == BN;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int cb = (wn * FN + j) * 32;  // the block's columns
      float bias[16];
      bias_of(j, bias);
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int r = (wm * FM + i) * 32 + c32;
        TO* const crow = tile + (int64_t)r * g.n;
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e)
          v[e] = scaled(acc[i][j][e], sa[i], sw[j][e >> 2][e & 3], bias[e]);
        if constexpr (sizeof(TO) == 4) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int c = cb + q * 8 + half * 4;
            if (full || (r < rows && c < cols))
              *reinterpret_cast<f32x4*>(crow + c) =
                  f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
          }
        } else {
          // the lane halves trade: the lower one gets columns q * 8 .. + 7 of q
          // = 2p, the upper one of q = 2p + 1
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            uint32_t o[4];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              auto pack = [&](int e) {
                return (uint32_t)__builtin_bit_cast(uint16_t, from_f32<TO>(v[e])) |
                       ((uint32_t)__builtin_bit_cast(uint16_t, from_f32<TO>(v[e + 1])) << 16);
              };
              const auto t = __builtin_amdgcn_permlane32_swap(
                  pack(p * 8 + 2 * w), pack(p * 8 + 4 + 2 * w), false, false);
              o[w] = t[0];
              o[2 + w] = t[1];
            }
            const int c = cb + (2 * p + half) * 8;
            if (full || (r < rows && c < cols))
              *reinterpret_cast<i32x4*>(crow + c) =
                  i32x4{(int)o[0], (int)o[1], (int)o[2], (int)o[3]};
          }
        }
      }
    }
  } else {
    // through LDS, 32 rows of the wave's columns at a time, so that the lanes of a
    // store write side by side: a dword each, for 2-byte types the pairs that lie
    // on 4 bytes (7281 x 512 x 9865: 227 us with 2-byte stores, 108)
    constexpr int WC = FN * 32, RS = WC + 16 / (int)sizeof(TO);
    static_assert(4 * 32 * RS * sizeof(TO) <= KG * S::LDS, "the waves' rows fit LDS");
    TO* const mine = reinterpret_cast<TO*>(lds) + wave * 32 * RS;
    const int wcols = cols - wn * WC;  // columns of this wave inside the output
    __syncthreads();                   // every wave is done with what LDS holds
#pragma unroll
    for (int i = 0; i < FM; ++i) {
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        float bias[16];
        bias_of(j, bias);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          typedef TO T4 __attribute__((ext_vector_type(4)));
          T4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = scaled(acc[i][j][4 * q + e], sa[i], sw[j][q][e], bias[4 * q + e]);
            v[e] = from_f32<TO>(x);
          }
          *reinterpret_cast<T4*>(mine + c32 * RS + j * 32 + q * 8 + half * 4) = v;
        }
      }
      // this wave's own rows: written, then read, in order
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      const int r0 = (wm * FM + i) * 32;
      if constexpr (sizeof(TO) == 4) {
#pragma unroll 4
        for (int t = 0; t < WC / 2; ++t) {
          const int r = (t * 64 + lane) / WC, c = (t * 64 + lane) % WC;
          if (r0 + r < rows && c < wcols)
            tile[(int64_t)(r0 + r) * g.n + wn * WC + c] = mine[r * RS + c];
        }
      } else {
        constexpr int LPR = WC / 2;  // lanes a row
#pragma unroll 4
        for (int t = 0; t < LPR / 2; ++t) {
          const int r = (t * 64 + lane) / LPR, l = lane % LPR;
          if (r0 + r >= rows) continue;
          TO* const o = tile + (int64_t)(r0 + r) * g.n + wn * WC;
          const int odd = (int)(reinterpret_cast<uintptr_t>(o) >> 1) & 1;
          const int c = 2 * l + odd;
          const TO x = mine[r * RS + c], y = mine[r * RS + c + 1];
          if (c + 1 < wcols && c + 1 < WC) {
            *reinterpret_cast<uint32_t*>(o + c) =
                (uint32_t)__builtin_bit_cast(uint16_t, x) |
                ((uint32_t)__builtin_bit_cast(uint16_t, y) << 16);
          } else if (c < wcols) {
            o[c] = x;
          }
          if (odd && l == 0 && wcols > 0) o[0] = mine[r * RS];  // before the first pair
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
}

// ---------------------------------------------------------------- small grids
// Tiles of FM x FN blocks of 16 x 16, a workgroup of W waves each; wave w takes
// the 128-byte pieces w, w + W, ... of K and multiplies the whole tile, so the
// waves meet only where their sums are added.  A piece goes through LDS all
// the same, in a place of the wave's own and without a barrier: 8 lanes then
// load a row's whole line.  As MFMA fragments straight into registers (16 rows x
// 64 bytes a load, two requests for a line) a CU received 14 bytes a cycle
// instead of 30 and more: 48 x 4096 x 2048 8.3 us, this 4.5.  D pieces of a wave
// are in flight.
template <typename TO, int FM, int FN, int W, int D>
__global__ __launch_bounds__(64 * W) void w8a8_kl(W8Args g, int nbm, int nbn) {
  constexpr int BM = FM * 16, BN = FN * 16, NB = FM * FN;
  constexpr int NL = (BM + BN) / 8, LA = BM / 8;  // loads of a piece; of A
  constexpr int PIECE = (BM + BN) * 128;
  static_assert(NB * 1024 <= D * PIECE, "the sums take the place of the pieces");
  __shared__ __attribute__((aligned(1024))) uint8_t smem[W * D * PIECE];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, grp = lane >> 4;
  int bm, bn;
  tile_of_dense(nbm, nbn, blockIdx.x, gridDim.x, bm, bn);
  const int64_t row0 = (int64_t)bm * BM, col0 = (int64_t)bn * BN;
  const int rows = (int)(g.m - row0 < BM ? g.m - row0 : BM);
  const int cols = (int)(g.n - col0 < BN ? g.n - col0 : BN);
  const i32x4 rA = make_rsrc(g.a + row0 * g.k, (uint32_t)rows * g.k);
  const i32x4 rW = make_rsrc(g.w + col0 * g.k, (uint32_t)cols * g.k);
  // load i: rows i * 8 + lane / 8 of A, then of W; slot lane % 8 of a row holds
  // its chunk (lane % 8) ^ ((row / 2) % 8)
  uint32_t off[NL];
  int chunk[2];  // of even and odd i: a row's (row / 2) % 8 repeats every 16 rows
#pragma unroll
  for (int i = 0; i < 2; ++i) chunk[i] = ((lane & 7) ^ (i * 4 + (lane >> 4))) * 16;
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int r = (i < LA ? i : i - LA) * 8 + (lane >> 3);
    off[i] = r < (i < LA ? rows : cols) ? (uint32_t)r * g.k + chunk[i & 1] : kOOB;
  }
  uint8_t* const mine = smem + wave * (D * PIECE);
  auto load = [&](int d, int piece) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const bool in = chunk[i & 1] < g.k - piece * 128;  // past the end: zeros
      llvm_amdgcn_raw_buffer_load_lds(i < LA ? rA : rW, lds_ptr(mine + d * PIECE + i * 1024), 16,
                                      (int)(in ? off[i] : kOOB), piece * 128, 0, 0);
    }
  };
  i32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = i32x4{0, 0, 0, 0};

  const int np = (g.k + 127) >> 7;  // pieces of K
#pragma unroll
  for (int d = 0; d < D; ++d) {
    load(d, wave + d * W);
    asm volatile("" ::: "memory");
  }
  const int rd = c16 * 128, swz = c16 >> 1;
  int d = 0;
  for (int p = wave; p < np; p += W) {
    wait_vmcnt<(D - 1) * NL>();
    const uint8_t* base = mine + d * PIECE + rd;
    i32x4 fa[FM][2], fw[FN][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = ((h * 4 + grp) ^ swz) * 16;
#pragma unroll
      for (int i = 0; i < FM; ++i)
        fa[i][h] = *reinterpret_cast<const i32x4*>(base + at + i * 2048);
#pragma unroll
      for (int j = 0; j < FN; ++j)
        fw[j][h] = *reinterpret_cast<const i32x4*>(base + at + BM * 128 + j * 2048);
    }
    wait_lgkm0();  // read: its place is free
    load(d, p + D * W);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma_i8(fw[j][h], fa[i][h], acc[i][j]);
    d = d + 1 == D ? 0 : d + 1;
  }
  wait_vmcnt<0>();
  i32x4* const sums = reinterpret_cast<i32x4*>(mine);
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) sums[(i * FN + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  const bool vec = g.n % 4 == 0 && !(reinterpret_cast<uintptr_t>(g.out) & 15);
  for (int u = tid; u < NB * 64; u += 64 * W) {
    const int b = u >> 6, l = u & 63;
    i32x4 s = reinterpret_cast<const i32x4*>(smem)[u];
#pragma unroll
    for (int w = 1; w < W; ++w) s += reinterpret_cast<const i32x4*>(smem + w * (D * PIECE))[u];
    finish4<TO>(g, row0 + (b / FN) * 16 + (l & 15), col0 + (b % FN) * 16 + (l >> 4) * 4, s, vec);
  }
}

// ------------------------------------------------------------------ dispatch
// The kernels' tiles, and what they cost by the rounds that a grid takes: us =
// start + rounds * (tile + stages * stage) + tiles / CUs * stages * load, rounds =
// tiles / CUs rounded up; the last term is what the work takes more with every
// CU at it (power, memory).  Least squares over 140 sizes (M 1 .. 8192, K 512 ..
// 14000, N 256 .. 12000, bf16 out): the kernel that this puts first took 1.01 times
// the fastest of the eight's time on average, 1.23 times at worst (large products
// 1.001 and 1.02).  It ranks them and does not predict: of 65 sizes and tiles half
// came within 9% of it, 37 x 14016 x 8960 took 45 us instead of 25.5, 506 x 12128 x
// 6656 68 instead of 56.  It knows neither the bytes that every block of rows reads
// again, nor that a CU holds two or more workgroups of the smaller tiles, nor
// wider outputs; and it has no cost of odd rows for 128 x 64 tiles (7281 x 512 x
// 9865: 223 us, by the rule 124).  Any single tile is 1.5 to 10 times slower
// somewhere: the largest one alone multiplies at the full rate (8192 x 4096 x
// 4096 119 us, 128 x 128 tiles 137), the smaller ones fill the GPU (1021 x 4096 x
// 2048: 128 x 64 with two groups 14.0 us, 256 x 256 47), and with few rows the
// waves that split K read the weights fastest (1 x 2048 x 5120 4.2 us, 128 x 128
// 8.9).  Rows off 16 bytes cost the large tiles most: 7281 x 512 x 9865 128 x 128
// 108 us, 256 x 256 154.
struct Config {
  int bm, bn, kstage, threads;  // kstage: bytes of K of a stage
  float start, tile, stage, load;  // us
  float odd;                    // us of a round more for rows off 16 bytes
};
enum { PF44, PF42, PF22, PF21, PF11, KL22, KL12, KL11, CONFIGS };
constexpr Config kConfigs[CONFIGS] = {
    {256, 256, 128, 256, 0.26f, 7.82f, 0.937f, 0.659f, 17.f},   // PF44
    {256, 128, 128, 256, 0.0f, 4.78f, 0.602f, 0.303f, 10.4f},   // PF42
    {128, 128, 128, 256, 2.11f, 1.14f, 0.441f, 0.135f, 2.6f},   // PF22
    {128, 64, 256, 512, 1.27f, 2.12f, 0.444f, 0.258f, 0.f},     // PF21, two groups
    {64, 64, 256, 512, 2.9f, 0.39f, 0.329f, 0.137f, 0.8f},      // PF11, two groups
    {32, 32, 1024, 512, 3.74f, 0.1f, 0.425f, 0.42f, 0.f},       // KL22, 8 waves
    {16, 32, 512, 256, 3.92f, 0.0f, 0.161f, 0.152f, 0.f},       // KL12, 4 waves
    {16, 16, 1024, 512, 3.34f, 0.49f, 0.204f, 0.179f, 0.f},     // KL11, 8 waves
};

// The config of a size, -1 if no grid can hold it (2^31 threads a launch); row16:
// the output's rows are 16-byte aligned
int choose(int64_t m, int64_t k, int64_t n, bool row16, int64_t cus) {
  int best = -1;
  double least = 0.0;
  for (int c = 0; c < CONFIGS; ++c) {
    const Config& f = kConfigs[c];
    const int64_t nbm = (m + f.bm - 1) / f.bm, nbn = (n + f.bn - 1) / f.bn;
    if (nbm > 0x7FFFFFFF / f.threads / nbn) continue;
    const int64_t rounds = (nbm * nbn + cus - 1) / cus, stages = (k + f.kstage - 1) / f.kstage;
    const double tile = f.tile + (double)stages * f.stage + (row16 ? 0.f : f.odd);
    const double us = f.start + (double)rounds * tile +
                      (double)(nbm * nbn) / (double)cus * (double)stages * f.load;
    if (best < 0 || us < least) {
      best = c;
      least = us;
    }
  }
  return best;
}

template <typename TO>
int launch_typed(const W8Args& g, hipStream_t st) {
  const int cus = device_cus();
  const bool row16 =
      g.n % (16 / (int)sizeof(TO)) == 0 && !(reinterpret_cast<uintptr_t>(g.out) & 15);
  const int cfg = choose(g.m, g.k, g.n, row16, cus > 0 ? cus : 256);
  if (cfg < 0) {
    set_error("w8a8: too many rows or columns (m %lld, n %lld)", (long long)g.m, (long long)g.n);
    return MXFP4_ERR_VALUE;
  }
  const int nbm = (int)((g.m + kConfigs[cfg].bm - 1) / kConfigs[cfg].bm);
  const int nbn = (int)((g.n + kConfigs[cfg].bn - 1) / kConfigs[cfg].bn);
  const unsigned grid = (unsigned)nbm * (unsigned)nbn;
  auto pf = [&](auto fm, auto fn, auto kg) {
    constexpr int FM = decltype(fm)::value, FN = decltype(fn)::value, KG = decltype(kg)::value;
    if (row16) w8a8_pf<TO, FM, FN, KG, true><<<grid, 256 * KG, 0, st>>>(g, nbm, nbn);
    else w8a8_pf<TO, FM, FN, KG, false><<<grid, 256 * KG, 0, st>>>(g, nbm, nbn);
  };
#define C_(v) std::integral_constant<int, (v)>{}
  switch (cfg) {
    case PF44: pf(C_(4), C_(4), C_(1)); break;
    case PF42: pf(C_(4), C_(2), C_(1)); break;
    case PF22: pf(C_(2), C_(2), C_(1)); break;
    case PF21: pf(C_(2), C_(1), C_(2)); break;
    case PF11: pf(C_(1), C_(1), C_(2)); break;
    case KL22: w8a8_kl<TO, 2, 2, 8, 1><<<grid, 512, 0, st>>>(g, nbm, nbn); break;
    case KL12: w8a8_kl<TO, 1, 2, 4, 2><<<grid, 256, 0, st>>>(g, nbm, nbn); break;
    default: w8a8_kl<TO, 1, 1, 8, 2><<<grid, 512, 0, st>>>(g, nbm, nbn); break;
  }
#undef C_
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

// Test hook: the tile that a size runs with, rows * 65536 + columns; 0 if none
extern "C" int mxfp4_test_w8a8_tile(int64_t m, int64_t k, int64_t n, int row16, int64_t cus) {
  const int c = mx::choose(m, k, n, row16 != 0, cus);
  return c < 0 ? 0 : mx::kConfigs[c].bm * 65536 + mx::kConfigs[c].bn;
}
