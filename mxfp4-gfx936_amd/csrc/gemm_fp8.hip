// FP8 (e4m3) GEMM with a scale for each 128 values of K: activations a row each,
// weights a block of 128 rows x 128.  Dense, and by expert on rows that are sorted
// by expert.  No counterpart in the reference.
//
//   out[i, j] = sum_b sa[i, b] * sw[j / 128, b] * (sum_{k in block b} a[i, k] w[j, k]) (+ bias[j])
//
// One 16x16x128 f8f6f4 MFMA is one block's inner sum, from a zero accumulator; FP32
// FMAs then add it, times sa * sw, to the running sums: 4 of them beside the MFMA's
// 32 cycles.  The MFMA adds the products in groups of 8 consecutive K, whose bits
// below about 2^-13 of the group's largest product are dropped (the 16x16x32 FP8
// MFMA drops the same ones); on values quantized per 128 that is 1.4e-5 of the
// result (2-norm), half a step of bf16 being 2e-3.  Everything after it is FP32,
// with one rounding to the output type.
//
// Operands: lane l supplies row l % 16; which 32 of a row's 128 bytes it takes does not
// matter as long as both operands agree: here chunks l / 16 and l / 16 + 4 of 16 bytes.
// The weights are the A operand and the activations the B operand, so a lane
// receives columns (l / 16) * 4 .. + 3 of row l % 16: one row's scale a lane and
// block of rows, one weight scale for the whole wave.
#include <cmath>

#include "gemm.h"

namespace mx {
namespace {

struct F8Args {
  const uint8_t* a;
  const float* sa;
  int64_t sa_row, sa_block;  // strides of the activations' scales, in values
  const uint8_t* w;
  const float* sw;
  const void* bias;  // [n] of the output type or nullptr (dense)
  void* out;
  int64_t m;  // rows of the output
  int64_t n;
  int k, kb;  // kb: blocks of K
  // by expert: rows offsets[e] .. offsets[e + 1] are expert e's, zeros from
  // offsets[experts] on; routes (or nullptr): row p reads activation routes[p] / top_k
  const int32_t* offsets;
  const int32_t* routes;
  int64_t a_rows;
  int top_k, experts;
  int row16;  // the output's rows are 16-byte aligned
};

__device__ __forceinline__ f32x4 mfma_f8(i32x4 a0, i32x4 a1, i32x4 b0, i32x4 b1) {
  const i32x8 a = {a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]};
  const i32x8 b = {b0[0], b0[1], b0[2], b0[3], b1[0], b1[1], b1[2], b1[3]};
  // formats 0 (e4m3), scale bytes 127 (1.0)
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0,
                                                          127, 0, 127);
}

// ------------------------------------------------------------- tile -> work
struct Tile {
  int64_t row0;  // first output row
  int rows;      // rows of the tile
  int bn;        // column tile
  int expert;    // -1: rows of zeros
};

__device__ __forceinline__ void dense_tile(int nbm, int nbn, int idx, int nwg, int& bm, int& bn) {
  // workgroup i runs on XCD i % 8: each XCD gets a contiguous range of tiles,
  // walked in groups of 4 row blocks, its operands L2 resident
  const int x = idx % 8, i = idx / 8;
  const int per = nwg / 8, rem = nwg % 8;
  const int pid = x * per + (x < rem ? x : rem) + i;
  constexpr int GROUP = 4;
  const int first = (pid / (GROUP * nbn)) * GROUP;
  const int gsize = (nbm - first) < GROUP ? (nbm - first) : GROUP;
  bm = __builtin_amdgcn_readfirstlane(first + (pid % (GROUP * nbn)) % gsize);
  bn = __builtin_amdgcn_readfirstlane((pid % (GROUP * nbn)) / gsize);
}

// Inclusive sum over the lanes so far, by DPP: within 16 lanes, then over them
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);   // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);   // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);   // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return v;
}

// Row blocks of BM rows, each expert's (and the rows behind the last one's) starting at
// its own first row; the live ones are split into 8 contiguous ranges, one an
// XCD, each walked with all column tiles of a row block before the next: an
// expert's weights go into few L2s.  Every wave finds its tile for itself, 256 experts
// at a time: one wait for the offsets, which are read again only if there are more.
// False: no work left.
template <int BM>
__device__ __forceinline__ bool expert_tile(const F8Args& g, int nbn, Tile& t) {
  constexpr int Q = 4;
  const int lane = threadIdx.x & 63;
  const int rows = (int)g.m, groups = g.experts + 1;
  int from[Q], count[Q];
  // of groups e0 + 64 q + lane; inside the rows whatever the offsets hold
  auto read = [&](int e0) {
    int next[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int e = e0 + q * 64 + lane;
      from[q] = g.offsets[e < groups ? e : 0];
      next[q] = g.offsets[e + 1 < groups ? e + 1 : 0];
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int e = e0 + q * 64 + lane;
      auto inside = [&](int v) { return v < 0 ? 0 : v < rows ? v : rows; };
      from[q] = inside(from[q]);
      count[q] = e < groups ? (e + 1 < groups ? inside(next[q]) : rows) - from[q] : 0;
      count[q] = count[q] > 0 ? count[q] : 0;
    }
  };
  auto blocks = [&](int q) { return (count[q] + BM - 1) / BM; };
  int live = 0;
  for (int e0 = 0; e0 < groups; e0 += Q * 64) {
    read(e0);
#pragma unroll
    for (int q = 0; q < Q; ++q) live += blocks(q);
  }
  live = __builtin_amdgcn_readlane(wave_scan(live), 63);
  const int x = blockIdx.x % 8, i = blockIdx.x / 8;
  const int lo = (int)((int64_t)live * x / 8), hi = (int)((int64_t)live * (x + 1) / 8);
  const int b = lo + i / nbn;
  t.bn = __builtin_amdgcn_readfirstlane(i % nbn);
  if (b >= hi) return false;
  int base = 0;
  for (int e0 = 0; e0 < groups; e0 += Q * 64) {
    if (groups > Q * 64) read(e0);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int c = blocks(q);
      const int end = base + wave_scan(c);
      const uint64_t past = __ballot(end > b);
      if (past) {
        const int l = __builtin_ctzll(past);
        const int e = e0 + q * 64 + l;
        const int first = __builtin_amdgcn_readlane(end, l) - __builtin_amdgcn_readlane(c, l);
        const int at = (b - first) * BM;
        const int left = __builtin_amdgcn_readlane(count[q], l) - at;
        t.row0 = __builtin_amdgcn_readlane(from[q], l) + at;
        t.rows = left < BM ? left : BM;
        t.expert = e < g.experts ? e : -1;
        return true;
      }
      base = __builtin_amdgcn_readlane(end, 63);
    }
  }
  return false;
}

template <int BM, bool GROUPED>
__device__ __forceinline__ bool find_tile(const F8Args& g, int nbm, int nbn, Tile& t) {
  if constexpr (GROUPED) {
    return expert_tile<BM>(g, nbn, t);
  } else {
    int bm;
    dense_tile(nbm, nbn, blockIdx.x, gridDim.x, bm, t.bn);
    t.row0 = (int64_t)bm * BM;
    t.rows = (int)(g.m - t.row0 < BM ? g.m - t.row0 : BM);
    t.expert = 0;
    return true;
  }
}

// The activation row that row r of the tile reads, counted from the base that
// a_base gives; -1: none (a row past the tile or a route outside the activations)
template <bool GROUPED>
__device__ __forceinline__ int64_t a_row(const F8Args& g, const Tile& t, int r) {
  if (r >= t.rows) return -1;
  if constexpr (GROUPED) {
    if (g.routes) {
      const int32_t route = g.routes[t.row0 + r];
      if (route < 0) return -1;
      const int64_t row = route / g.top_k;
      return row < g.a_rows ? row : -1;
    }
  }
  return r;
}
template <bool GROUPED>
__device__ __forceinline__ int64_t a_base(const F8Args& g, const Tile& t) {
  return GROUPED && g.routes ? 0 : t.row0;
}

template <typename TO>
__device__ __forceinline__ void zero_rows(const F8Args& g, const Tile& t, int64_t col0, int cols,
                                          int threads) {
  TO* const o = static_cast<TO*>(g.out) + t.row0 * g.n + col0;
  for (int u = threadIdx.x; u < t.rows * cols; u += threads)
    o[(int64_t)(u / cols) * g.n + u % cols] = from_f32<TO>(0.f);
}

// Four output values of row `row`, columns col .. col + 3
template <typename TO>
__device__ __forceinline__ void finish4(const F8Args& g, int64_t row, int64_t col, f32x4 v,
                                        bool vec) {
  TO* const o = static_cast<TO*>(g.out) + row * g.n + col;
  TO r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float b = 0.f;
    if (g.bias && col + i < g.n) b = to_f32(static_cast<const TO*>(g.bias)[col + i]);
    r[i] = from_f32<TO>(g.bias ? v[i] + b : v[i]);
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
// Tiles of WM x WN waves, each FM x FN blocks of 16 x 16; ST stages of 128 bytes of K in
// LDS, of which ST - 1 are on their way while one is multiplied.  A row's stage is
// its whole 128-byte line; chunk c of row r sits in slot c ^ ((r / 2) % 8), which the
// lane that fills a slot undoes, so that the 16 lanes of a read cover all 64 banks.
// The rows' scales of a stage go to LDS as well, in the order in which a lane reads
// its FM of them at once; a wave's weight scales of 64 stages are a lane's value
// each, read by the stage's number.
//
// What bounds it.  256 x 256 in 8 waves: LDS and power; a stage's 192 KB of fragment
// reads and 64 KB of writes take as many cycles as its MFMAs, 2048 (8192 x 4096 x 4096
// 122 us, 2.26 PFLOP/s: MFMAs 62% of the time at 2.0 GHz, and 7 us a tile for its first
// load and its stores).  Smaller tiles: the loads from L2, about 28 bytes a cycle and CU,
// and rows that begin off 128 bytes (K no multiple of it), whose pieces are two lines
// each (1021 x 4016 x 2050 26.4 us, 1024 x 4096 x 2048 15.9).  By expert with few rows
// each: the weights' stream (16 x 8 routes, 66 of 128 experts hit, 5.2 TB/s, 509 x 8 4.1),
// else both: 4096 x 8 routes, 2048 -> 1536, 185 us, MFMAs 37%, CUs idle 17% at the end.
// Measured and slower: weights from memory to registers (256 x 256: 300 us against 122);
// 4 to 6 stages (nothing gained on small tiles); the next stage's fragments in a second
// set of registers (4096^3 80 -> 72 us, other sizes the same or slower); a stage's lines
// fetched into L2 two stages ahead (by expert 176 -> 185 us, dense 128 -> 136); row
// blocks skipped in a wave that has some rows (spills; whole waves are skipped).
template <int FM, int FN, int WM, int WN, int ST, int KG>
struct PfShape {
  static constexpr int NW = WM * WN, BM = WM * FM * 16, BN = WN * FN * 16;
  static constexpr int A_BYTES = BM * 128, W_BYTES = BN * 128;
  static constexpr int SROWS = BM < 64 ? 64 : BM;  // rows that the scales' loads cover
  static constexpr int STAGE = A_BYTES + W_BYTES + SROWS * 4;
  static constexpr int LA = A_BYTES / 1024 / NW, LW = W_BYTES / 1024 / NW;  // loads of a wave
  static constexpr int LOADS = LA + LW + 1;
  static_assert(A_BYTES % (1024 * NW) == 0 && W_BYTES % (1024 * NW) == 0, "even shares");
  static_assert(SROWS % 64 == 0 && SROWS / 64 <= NW, "a wave one load of scales");
  static_assert(128 % (FN * 16) == 0, "one weight scale a wave");
  static_assert(ST >= 2 && KG * ST * STAGE <= 163840, "the stages fit a CU's LDS");
  static_assert((KG - 1) * NW * FM * FN * 1024 <= KG * ST * STAGE, "the groups' sums fit");
  // a row of a wave's columns in LDS on its way out
  template <typename TO>
  static constexpr int out_row() { return FN * 16 + 16 / (int)sizeof(TO); }
};

template <typename TO, int FM, int FN, int WM, int WN, int ST, int KG, int MINW, bool GROUPED>
__global__ __launch_bounds__(64 * WM * WN * KG, MINW) void f8_pf(F8Args g, int nbm, int nbn) {
  typedef PfShape<FM, FN, WM, WN, ST, KG> S;
  constexpr int BM = S::BM, BN = S::BN, NW = S::NW;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[KG * ST * S::STAGE];
  Tile t;
  if (!find_tile<BM, GROUPED>(g, nbm, nbn, t)) return;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave_of_all = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = KG == 1 ? 0 : wave_of_all / NW;
  const int wave = KG == 1 ? wave_of_all : wave_of_all % NW;
  uint8_t* const lds = smem + group * (ST * S::STAGE);
  const int wm = wave / WN, wn = wave % WN;
  const int c16 = lane & 15, grp = lane >> 4;
  const int64_t col0 = (int64_t)t.bn * BN;
  const int cols = (int)(g.n - col0 < BN ? g.n - col0 : BN);
  if (GROUPED && t.expert < 0) {
    zero_rows<TO>(g, t, col0, cols, 64 * NW * KG);
    return;
  }
  const int64_t ab = a_base<GROUPED>(g, t);
  const int64_t a_rows = GROUPED && g.routes ? g.a_rows : t.rows;
  const i32x4 rA = make_rsrc(g.a + ab * g.k, (uint32_t)(a_rows * g.k));
  const int64_t we = GROUPED ? t.expert : 0;
  const i32x4 rW = make_rsrc(g.w + (we * g.n + col0) * g.k, (uint32_t)cols * g.k);
  const int64_t scales_end = (a_rows - 1) * g.sa_row + (g.kb - 1) * g.sa_block + 1;
  const i32x4 rSA = make_rsrc(g.sa + ab * g.sa_row, (uint32_t)(scales_end * 4));
  // this wave's weight scales, one a stage
  const int64_t nblocks = (g.n + 127) >> 7;
  const int64_t cblk = (col0 + wn * FN * 16) >> 7;
  const float* const sw = g.sw + (we * nblocks + (cblk < nblocks ? cblk : nblocks - 1)) * g.kb;
  const i32x4 rSW = make_rsrc(sw, (uint32_t)g.kb * 4);

  uint32_t a_off[S::LA], w_off[S::LW];
  const int lrow = wave * 8 + (lane >> 3);
  const int chunk = ((lane & 7) ^ ((lrow >> 1) & 7)) * 16;
#pragma unroll
  for (int j = 0; j < S::LA; ++j) {
    const int64_t r = a_row<GROUPED>(g, t, j * NW * 8 + lrow);
    a_off[j] = r >= 0 ? (uint32_t)(r * g.k) + chunk : kOOB;
  }
#pragma unroll
  for (int j = 0; j < S::LW; ++j) {
    const int r = j * NW * 8 + lrow;
    w_off[j] = r < cols ? (uint32_t)r * g.k + chunk : kOOB;
  }
  // slot s of the scales: row (s / (FM 16)) FM 16 + (s % FM) 16 + s / FM % 16
  const int sl = wave % (S::SROWS / 64) * 64 + lane;
  const int64_t srow =
      a_row<GROUPED>(g, t, sl / (FM * 16) * (FM * 16) + sl % FM * 16 + sl / FM % 16);
  const uint32_t s_off = srow >= 0 ? (uint32_t)(srow * g.sa_row * 4) : kOOB;

  // Group q takes the whole blocks q, q + KG, .. of K, all the same number of stages; one
  // past the last loads the last again, and counts nothing: its scales are taken as 0.
  const int nfull = g.k >> 7;
  const int nk = (nfull + KG - 1) / KG;
  auto block_of = [&](int kt) {
    const int b = kt * KG + group;
    return b < nfull ? b : nfull - 1;
  };
  // load l of block b; in: whether the lane's 16 bytes lie inside K
  auto load = [&](int b, bool in, uint8_t* st, auto lc) {
    constexpr int l = decltype(lc)::value;
    if constexpr (l < S::LA) {
      llvm_amdgcn_raw_buffer_load_lds(rA, lds_ptr(st + (l * NW + wave) * 1024), 16,
                                      (int)(in ? a_off[l] : kOOB), b * 128, 0, 0);
    } else if constexpr (l < S::LA + S::LW) {
      constexpr int j = l - S::LA;
      llvm_amdgcn_raw_buffer_load_lds(rW, lds_ptr(st + S::A_BYTES + (j * NW + wave) * 1024), 16,
                                      (int)(in ? w_off[j] : kOOB), b * 128, 0, 0);
    } else {
      llvm_amdgcn_raw_buffer_load_lds(
          rSA, lds_ptr(st + S::A_BYTES + S::W_BYTES + wave % (S::SROWS / 64) * 256), 4, (int)s_off,
          (int)(b * g.sa_block * 4), 0, 0);
    }
  };
  auto load_all = [&](int b, bool in, int slot) {
    static_for<0, S::LOADS>([&](auto l) { load(b, in, lds + slot * S::STAGE, l); });
    asm volatile("" ::: "memory");
  };

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // by expert a tile may be mostly empty: whether the wave has any rows
  const bool rows_here = !GROUPED || __builtin_amdgcn_readfirstlane(t.rows - wm * FM * 16) > 0;
  const int swz = c16 >> 1;
  const int lo = (grp ^ swz) * 16, hi = ((grp + 4) ^ swz) * 16;
  const int a_at = (wm * FM * 16 + c16) * 128, w_at = S::A_BYTES + (wn * FN * 16 + c16) * 128;
  const int s_at = S::A_BYTES + S::W_BYTES + (wm * 16 + c16) * FM * 4;
  // A stage's fragments, A's two at a time, and row scales
  constexpr int LAG = 2, NM = FM * FN;
  i32x4 w0[FN], w1[FN], a0[2], a1[2];
  float f[FM];
#define C_(v) std::integral_constant<int, (v)>{}
  auto read_a = [&](const uint8_t* st, auto ic) {
    constexpr int i = decltype(ic)::value;
    a0[i & 1] = *reinterpret_cast<const i32x4*>(st + a_at + i * 2048 + lo);
    a1[i & 1] = *reinterpret_cast<const i32x4*>(st + a_at + i * 2048 + hi);
  };
  auto read = [&](const uint8_t* st) {
    static_for<0, FN>([&](auto jc) {
      constexpr int j = decltype(jc)::value;
      w0[j] = *reinterpret_cast<const i32x4*>(st + w_at + j * 2048 + lo);
      w1[j] = *reinterpret_cast<const i32x4*>(st + w_at + j * 2048 + hi);
      if constexpr (j == 0) read_a(st, C_(0));
    });
#pragma unroll
    for (int i = 0; i < FM; ++i) f[i] = reinterpret_cast<const float*>(st + s_at)[i];
  };
  // The MFMAs of a stage; MFMA u's sums are added after MFMA u + LAG has begun, and
  // `between` (loads) is dealt out behind the first ones
  auto multiply = [&](const uint8_t* st, bool counts, float sb, auto&& between) {
    f32x4 z[LAG + 1];
    static_for<0, NM + LAG>([&](auto uc) {
      constexpr int u = decltype(uc)::value;
      if constexpr (u < NM) {
        constexpr int i = u / FN, j = u % FN;
        if constexpr (j == 0 && i + 1 < FM) read_a(st, C_(i + 1));
        z[u % (LAG + 1)] = mfma_f8(w0[j], w1[j], a0[i & 1], a1[i & 1]);
        __builtin_amdgcn_sched_barrier(0);
        between(uc);
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (u >= LAG) {
        constexpr int i = (u - LAG) / FN, j = (u - LAG) % FN;
        if constexpr (j == 0) f[i] = KG == 1 || counts ? f[i] * sb : 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[i][j][e] = fmaf(z[(u - LAG) % (LAG + 1)][e], f[i], acc[i][j][e]);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };

  if (nfull > 0) {
    // The pipeline: ST - 1 stages are on their way or in LDS before stage kt is multiplied
    constexpr int PER = (2 * S::LOADS + NM - 1) / NM;
    constexpr int SEG = 64 / ST * ST;  // weight scales are a lane's each
    auto weight_scales = [&](int kt) {
      const int b = (kt + lane) * KG + group;
      return __uint_as_float(buf_load4(rSW, b < nfull ? (uint32_t)b * 4 : kOOB));
    };
    float sbv = weight_scales(0);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int q = 0; q < ST - 1; ++q) load_all(block_of(q), true, q);
    for (int base = 0; base < nk; base += SEG) {
      if (base > 0) sbv = weight_scales(base);
      const int n = nk - base < SEG ? nk - base : SEG;
      for (int q = 0; q < n;) {
        static_for<0, ST>([&](auto sc) {
          constexpr int slot = decltype(sc)::value;
          if (q < n) {
            wait_vmcnt<(ST - 2) * S::LOADS>();  // stage kt has landed
            wait_lgkm0();                       // this wave has read the one before
            barrier_only();
            const int b = block_of(base + q + ST - 1);
            if (rows_here) {
              read(lds + slot * S::STAGE);
              __builtin_amdgcn_sched_barrier(0);
              const float sb = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sbv), q));
              const bool counts = (base + q) * KG + group < nfull;
              multiply(lds + slot * S::STAGE, counts, sb, [&](auto mc) {
                constexpr int m = decltype(mc)::value;
                static_for<m * PER, (m + 1) * PER>([&](auto l) {
                  if constexpr (decltype(l)::value < S::LOADS)
                    load(b, true, lds + (slot + ST - 1) % ST * S::STAGE, l);
                });
              });
            } else {
              load_all(b, true, (slot + ST - 1) % ST);
            }
            ++q;
          }
        });
      }
    }
  }
  if (g.k & 127) {
    // the last block is a part, zeros past K: the first group's, on its own
    wait_vmcnt<0>();
    wait_lgkm0();
    barrier_only();
    load_all(nfull, chunk < g.k - nfull * 128, 0);
    const float sb = __uint_as_float(buf_load4(rSW, (uint32_t)nfull * 4));
    wait_vmcnt<0>();
    barrier_only();
    read(lds);
    __builtin_amdgcn_sched_barrier(0);
    multiply(lds, group == 0, sb, [](auto) {});
  }
#undef C_
  // the loads past K have landed as well, and this wave has read its last stage
  wait_vmcnt<0>();
  wait_lgkm0();
  if constexpr (KG > 1) {  // the first group adds the others' sums
    barrier_only();
    f32x4* const sums = reinterpret_cast<f32x4*>(smem);
    auto at = [&](int q, int i, int j) {
      return (((q - 1) * NW + wave) * FM * FN + i * FN + j) * 64 + lane;
    };
    if (group > 0) {
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) sums[at(group, i, j)] = acc[i][j];
    }
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int q = 1; q < KG; ++q)
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] += sums[at(q, i, j)];
  }

  const int cb = wn * FN * 16;  // the wave's columns
  const int wcols = cols - cb;  // those inside the output (may be none)
  TO* const tile = static_cast<TO*>(g.out) + t.row0 * g.n + col0 + cb;
  const TO* const bias = g.bias ? static_cast<const TO*>(g.bias) + col0 + cb : nullptr;
  if constexpr (sizeof(TO) == 2 && FN % 2 == 0) {
    if (g.row16) {
      // 16 bytes a lane: odd and even 16 lanes trade, so that a lane has 8 columns of block
      // j (even 16 lanes) or j + 1 (odd) and 64 bytes of a row lie together
      const int cl = (grp & 1) * 16 + (grp >> 1) * 8;  // the lane's columns within 32
#pragma unroll
      for (int j = 0; j < FN; j += 2) {
        const int c = j * 16 + cl;
        float b[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) b[e] = bias && c < wcols ? to_f32(bias[c + e]) : 0.f;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          const int r = (wm * FM + i) * 16 + c16;
          float v[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[i][j][e]),
                                                            __float_as_uint(acc[i][j + 1][e]),
                                                            false, false);
            v[e] = __uint_as_float(x[0]);
            v[4 + e] = __uint_as_float(x[1]);
          }
          uint32_t o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = bias ? v[2 * e] + b[2 * e] : v[2 * e];
            const float q = bias ? v[2 * e + 1] + b[2 * e + 1] : v[2 * e + 1];
            o[e] = (uint32_t)__builtin_bit_cast(uint16_t, from_f32<TO>(p)) |
                   ((uint32_t)__builtin_bit_cast(uint16_t, from_f32<TO>(q)) << 16);
          }
          if (r < t.rows && c < wcols)
            *reinterpret_cast<i32x4*>(tile + (int64_t)r * g.n + c) =
                i32x4{(int)o[0], (int)o[1], (int)o[2], (int)o[3]};
        }
      }
      return;
    }
  } else {
    if (g.row16) {
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int r = (wm * FM + i) * 16 + c16;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const int c = j * 16 + grp * 4;
          if (r < t.rows && c < wcols) finish4<TO>(g, t.row0 + r, col0 + cb + c, acc[i][j], true);
        }
      }
      return;
    }
  }
  // Rows off 16 bytes: through LDS, 16 rows of the wave's columns at a time, so that the
  // lanes of a store write side by side: a dword each, for 2-byte types the pairs that
  // lie on 4 bytes
  constexpr int WC = FN * 16, RS = S::template out_row<TO>();
  static_assert(NW * 16 * RS * sizeof(TO) <= KG * ST * S::STAGE, "the waves' rows fit LDS");
  TO* const mine = reinterpret_cast<TO*>(smem) + wave * 16 * RS;
  wait_lgkm0();
  barrier_only();  // every wave has read its last stage, and the sums
#pragma unroll
  for (int i = 0; i < FM; ++i) {
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      typedef TO T4 __attribute__((ext_vector_type(4)));
      T4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = j * 16 + grp * 4 + e;
        const float b = bias && c < wcols ? to_f32(bias[c]) : 0.f;
        v[e] = from_f32<TO>(bias ? acc[i][j][e] + b : acc[i][j][e]);
      }
      *reinterpret_cast<T4*>(mine + c16 * RS + j * 16 + grp * 4) = v;
    }
    // this wave's own rows: written, then read, in order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int r0 = (wm * FM + i) * 16;
    if constexpr (sizeof(TO) == 4) {
#pragma unroll 4
      for (int u = 0; u < WC / 4; ++u) {
        const int r = (u * 64 + lane) / WC, c = (u * 64 + lane) % WC;
        if (r0 + r < t.rows && c < wcols) tile[(int64_t)(r0 + r) * g.n + c] = mine[r * RS + c];
      }
    } else {
      constexpr int LPR = WC / 2;  // lanes a row
#pragma unroll 4
      for (int u = 0; u < LPR / 4; ++u) {
        const int r = (u * 64 + lane) / LPR, l = lane % LPR;
        if (r0 + r >= t.rows) continue;
        TO* const o = tile + (int64_t)(r0 + r) * g.n;
        const int odd = (int)(reinterpret_cast<uintptr_t>(o) >> 1) & 1;
        const int c = 2 * l + odd;
        if (c + 1 < wcols && c + 1 < WC) {
          *reinterpret_cast<uint32_t*>(o + c) =
              (uint32_t)__builtin_bit_cast(uint16_t, mine[r * RS + c]) |
              ((uint32_t)__builtin_bit_cast(uint16_t, mine[r * RS + c + 1]) << 16);
        } else if (c < wcols && c < WC) {
          o[c] = mine[r * RS + c];
        }
        if (odd && l == 0 && wcols > 0) o[0] = mine[r * RS];  // before the first pair
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// ---------------------------------------------------------------- small grids
// Tiles of FM x FN blocks of 16 x 16, a workgroup of W waves each; wave w takes the
// blocks w, w + W, ... of K and multiplies the whole tile, so the waves meet only
// where their sums are added (in wave order).  A block goes through LDS in a place of
// the wave's own and without a barrier: 8 lanes then load a row's whole line.  D blocks
// of a wave are in flight.  Bound by the chain of one launch (1 x 2048 x 5120 4.5 us, 2.3
// TB/s; the pipelined 64 x 32 tile 6.5) and then by the weights' stream (48 x 4096 x
// 2048 6.8 us with 16 x 32 tiles, 6.9 with the 32 x 32 that run; 64 x 32 pipelined 8.4);
// from about 128 rows on the pipelined tiles share the weights among more rows (130 x 2048
// x 5120: 12.5 us here, 8.0 there).
template <typename TO, int FM, int FN, int W, int D, bool GROUPED>
__global__ __launch_bounds__(64 * W) void f8_kl(F8Args g, int nbm, int nbn) {
  constexpr int BM = FM * 16, BN = FN * 16, NB = FM * FN;
  constexpr int NL = (BM + BN) / 8, LA = BM / 8;  // loads of a block; of A
  constexpr int PIECE = (BM + BN) * 128;
  static_assert(NB * 1024 <= D * PIECE, "the sums take the place of the pieces");
  static_assert(128 % BN == 0, "one weight scale a tile");
  __shared__ __attribute__((aligned(1024))) uint8_t smem[W * D * PIECE];
  Tile t;
  if (!find_tile<BM, GROUPED>(g, nbm, nbn, t)) return;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, grp = lane >> 4;
  const int64_t col0 = (int64_t)t.bn * BN;
  const int cols = (int)(g.n - col0 < BN ? g.n - col0 : BN);
  if (GROUPED && t.expert < 0) {
    zero_rows<TO>(g, t, col0, cols, 64 * W);
    return;
  }
  const int64_t ab = a_base<GROUPED>(g, t);
  const int64_t a_rows = GROUPED && g.routes ? g.a_rows : t.rows;
  const i32x4 rA = make_rsrc(g.a + ab * g.k, (uint32_t)(a_rows * g.k));
  const int64_t we = GROUPED ? t.expert : 0;
  const i32x4 rW = make_rsrc(g.w + (we * g.n + col0) * g.k, (uint32_t)cols * g.k);
  const int64_t scales_end = (a_rows - 1) * g.sa_row + (g.kb - 1) * g.sa_block + 1;
  const i32x4 rSA = make_rsrc(g.sa + ab * g.sa_row, (uint32_t)(scales_end * 4));
  const i32x4 rSW = make_rsrc(g.sw + (we * ((g.n + 127) >> 7) + (col0 >> 7)) * g.kb,
                              (uint32_t)g.kb * 4);
  // load i: rows i * 8 + lane / 8 of A, then of W; slot lane % 8 of a row holds its
  // chunk (lane % 8) ^ ((row / 2) % 8)
  uint32_t off[NL], s_off[FM];
  int chunk[2];  // of even and odd i: a row's (row / 2) % 8 repeats every 16 rows
#pragma unroll
  for (int i = 0; i < 2; ++i) chunk[i] = ((lane & 7) ^ (i * 4 + (lane >> 4))) * 16;
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    if (i < LA) {
      const int64_t r = a_row<GROUPED>(g, t, i * 8 + (lane >> 3));
      off[i] = r >= 0 ? (uint32_t)(r * g.k) + chunk[i & 1] : kOOB;
    } else {
      const int r = (i - LA) * 8 + (lane >> 3);
      off[i] = r < cols ? (uint32_t)r * g.k + chunk[i & 1] : kOOB;
    }
  }
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int64_t r = a_row<GROUPED>(g, t, i * 16 + c16);
    s_off[i] = r >= 0 ? (uint32_t)(r * g.sa_row * 4) : kOOB;
  }
  uint8_t* const mine = smem + wave * (D * PIECE);
  auto load = [&](int d, int piece) {
    auto one = [&](int i, uint32_t voff, int at) {
      llvm_amdgcn_raw_buffer_load_lds(i < LA ? rA : rW, lds_ptr(mine + d * PIECE + i * 1024), 16,
                                      (int)voff, at, 0, 0);
    };
    if (piece * 128 + 128 <= g.k) {
#pragma unroll
      for (int i = 0; i < NL; ++i) one(i, off[i], piece * 128);
    } else {  // a part of a block, or none: zeros past K
      const int at = piece < g.kb ? piece * 128 : 0;
#pragma unroll
      for (int i = 0; i < NL; ++i)
        one(i, chunk[i & 1] < g.k - piece * 128 ? off[i] : kOOB, at);
    }
  };
  // scales of block `piece`; past the last its row scales again, and a weight scale of 0
  auto scales = [&](int piece, float (&sa)[FM], float& sw) {
    const int b = piece < g.kb ? piece : g.kb - 1;
#pragma unroll
    for (int i = 0; i < FM; ++i)
      sa[i] = __uint_as_float((uint32_t)llvm_amdgcn_raw_buffer_load_i32(
          rSA, s_off[i], (int)(b * g.sa_block * 4), 0));
    sw = __uint_as_float(buf_load4(rSW, piece < g.kb ? (uint32_t)piece * 4 : kOOB));
  };
  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  float sa[D][FM], sw[D];
#pragma unroll
  for (int d = 0; d < D; ++d) {
    scales(wave + d * W, sa[d], sw[d]);
    load(d, wave + d * W);
    asm volatile("" ::: "memory");
  }
  const int rd = c16 * 128, swz = c16 >> 1;
  for (int p0 = wave; p0 < g.kb; p0 += D * W) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int p = p0 + d * W;
      if (p < g.kb) {
        // all but the loads to LDS of the D - 1 blocks after this one (those of the
        // scales the compiler may have moved: they do not count)
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
        float f[FM];
#pragma unroll
        for (int i = 0; i < FM; ++i) f[i] = sa[d][i] * sw[d];
        wait_lgkm0();  // read: its place is free
        scales(p + D * W, sa[d], sw[d]);
        load(d, p + D * W);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) {
            const f32x4 z = mfma_f8(fw[j][0], fw[j][1], fa[i][0], fa[i][1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(z[e], f[i], acc[i][j][e]);
          }
      }
    }
  }
  wait_vmcnt<0>();
  f32x4* const sums = reinterpret_cast<f32x4*>(mine);
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) sums[(i * FN + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  const bool vec = g.n % 4 == 0 && !(reinterpret_cast<uintptr_t>(g.out) & 15);
  for (int u = tid; u < NB * 64; u += 64 * W) {
    const int b = u >> 6, l = u & 63;
    f32x4 s = reinterpret_cast<const f32x4*>(smem)[u];
#pragma unroll
    for (int w = 1; w < W; ++w) s += reinterpret_cast<const f32x4*>(smem + w * (D * PIECE))[u];
    const int r = (b / FN) * 16 + (l & 15);
    const int64_t col = col0 + (b % FN) * 16 + (l >> 4) * 4;
    if (r < t.rows && col < g.n) finish4<TO>(g, t.row0 + r, col, s, vec);
  }
}

// ------------------------------------------------------------------ dispatch
// The kernels' tiles, and what they cost:
//   us = start + rounds * (tile + stages * stage) + shifts * stages * shift
//        + tiles / CUs * (stages * (load + part) + odd) + MB of the experts' weights * weights
// rounds = tiles / CUs and shifts = tiles / (CUs * resident workgroups), each rounded up
// (by expert, where the tiles are only estimated, not).  part: K ends inside a block, so
// that rows begin off 128 bytes and a row's piece is two lines; odd: output rows off 16
// bytes.  Non-negative least squares of the relative error over 218 dense and 75 grouped
// sizes, every kernel timed at each.  It ranks them, no more: the chosen one takes 1.7%
// longer than the best on average over the fitted dense sizes (at worst 1.55 times: 19 x
// 512 x 2304), 1.0% over 256 others of 1 to 128 rows (1.22 times); 2.0% over the fitted
// grouped ones, 4.6% over 75 others (1.26 times: 955 x 8 routes over 128, 5760 -> 512).
// Dense sizes of 129 to 8192 rows that were not fitted, 86 of them: 2.0% (1.20 times).  One
// error is regular: at up to 128 rows, K of at most 2048 and a grid of 16 x 32 tiles that the
// CUs take at once KL32 is chosen where KL16X32 is 9 to 12% faster.
// What a wrong one costs (us, graphs of calls with three sets of inputs in turn): 1 x 2048 x
// 5120 KL16X32 4.5, PF64 6.7, PF256 25; 48 x 2048 x 2048 KL32 5.1, KL16X32 4.6, PF64 6.7;
// 130 x 2048 x 5120 PF64G 8.0, KL32 12.5, PF128 15.5; 1021 x 4016 x 2050 PF64D 26.4, PF128X64
// 30.7; 4096 x 2048 x 5120 PF128 53, PF128W 53, PF256 59, PF64 76; 8192 x 4096 x 4096 PF256
// 126, PF128 143.  By expert: 16 x 8 routes over 128, 2048 -> 1536, GR32X256 44, GR64 49,
// GR256 59, GR16 97; 509 x 8, 768 -> 2048, GR64X128R 53, GR64X128 54, GR256 66; 4096 x 8,
// 2048 -> 1536, GR256 187, GR128 190, GR64 251.
struct Config {
  int bm, bn, kstage, threads, resident;  // kstage: K of a stage
  float start, tile, shift, stage, load, odd, part, weights;  // us
};
// W: 8 waves; D: two stages of the three of PF64; G, 64X32: two and four groups of waves
enum { PF256, PF128, PF128W, PF128X64, PF64, PF64D, PF64G, PF64X32, KL32, KL16X32, KL16, DENSE };
constexpr Config kDense[DENSE] = {
    {256, 256, 128, 512, 1, 0.924f, 6.876f, 1.235f, 0.f, 0.473f, 22.992f, 0.453f, 0.f},
    {128, 128, 128, 256, 2, 2.813f, 1.729f, 0.625f, 0.f, 0.185f, 5.204f, 0.243f, 0.f},
    {128, 128, 128, 512, 2, 1.94f, 2.031f, 0.565f, 0.f, 0.232f, 2.71f, 0.279f, 0.f},
    {128, 64, 128, 256, 2, 3.005f, 1.313f, 0.105f, 0.206f, 0.032f, 2.162f, 0.142f, 0.f},
    {64, 64, 128, 256, 3, 3.167f, 0.693f, 0.124f, 0.118f, 0.026f, 0.657f, 0.087f, 0.f},
    {64, 64, 128, 256, 4, 2.789f, 0.567f, 0.404f, 0.f, 0.092f, 0.544f, 0.055f, 0.f},
    {64, 64, 256, 512, 1, 2.056f, 2.425f, 0.369f, 0.f, 0.019f, 1.737f, 0.261f, 0.f},
    {64, 32, 512, 512, 1, 2.083f, 2.711f, 0.508f, 0.f, 0.019f, 1.575f, 0.299f, 0.f},
    {32, 32, 1024, 512, 2, 2.891f, 0.675f, 0.329f, 0.31f, 0.31f, 0.141f, 0.046f, 0.f},
    {16, 32, 512, 256, 3, 2.889f, 0.451f, 0.355f, 0.01f, 0.172f, 0.048f, 0.012f, 0.f},
    {16, 16, 1024, 512, 2, 2.854f, 0.594f, 0.106f, 0.265f, 0.081f, 0.009f, 0.056f, 0.f},
};
// R: one row of waves
enum { GR256, GR128, GR64X128, GR64X128R, GR64, GR32X256, GR16X32, GR16, GROUPS };
constexpr Config kGrouped[GROUPS] = {
    {256, 256, 128, 512, 1, 0.f, 7.851f, 0.f, 1.19f, 0.618f, 0.f, 0.f, 0.082f},
    {128, 128, 128, 256, 2, 3.063f, 2.703f, 0.f, 0.592f, 0.155f, 0.f, 0.f, 0.01f},
    {64, 128, 128, 256, 2, 3.284f, 2.018f, 0.f, 0.312f, 0.133f, 0.f, 0.f, 0.036f},
    {64, 128, 128, 256, 3, 3.655f, 0.826f, 0.f, 0.551f, 0.f, 0.f, 0.f, 0.034f},
    {64, 64, 128, 256, 3, 3.773f, 1.06f, 0.f, 0.27f, 0.035f, 0.f, 0.f, 0.002f},
    {32, 256, 128, 256, 2, 2.68f, 1.737f, 0.f, 0.697f, 0.f, 0.f, 0.f, 0.072f},
    {16, 32, 512, 256, 3, 4.616f, 0.596f, 0.f, 0.44f, 0.163f, 0.f, 0.f, 0.f},
    {16, 16, 1024, 512, 2, 4.278f, 1.777f, 0.f, 0.f, 0.372f, 0.f, 0.f, 0.047f},
};

// Row blocks that a grid must hold: by expert, each group of rows may end with a part of
// one, and the eight XCDs get the same number.
int64_t row_blocks(int64_t m, int bm, int experts) {
  if (experts == 0) return (m + bm - 1) / bm;
  const int64_t groups = experts + 1;
  return (m / bm + (m < groups ? m : groups) + 7) / 8 * 8;
}

// The config of a size, -1 if no grid can hold it (2^31 threads a launch).  experts: 0
// for the dense product.  By expert the rows of each are not known on the host: as many
// experts as evenly spread routes would meet are taken to share them evenly, half a
// block of rows lost in each that has more than half a one.
int choose(int64_t m, int64_t k, int64_t n, int experts, bool row16, int64_t cus) {
  const Config* const configs = experts ? kGrouped : kDense;
  const int count = experts ? (int)GROUPS : (int)DENSE;
  double active = 0.0, mb = 0.0;
  if (experts) {
    active = experts * (1.0 - pow(1.0 - 1.0 / experts, (double)m));
    mb = active * (double)n * (double)k * 1e-6;
  }
  int best = -1;
  double least = 0.0;
  for (int c = 0; c < count; ++c) {
    const Config& f = configs[c];
    const int64_t nbn = (n + f.bn - 1) / f.bn;
    if (row_blocks(m, f.bm, experts) > 0x7FFFFFFF / f.threads / nbn) continue;
    double tiles, rounds, shifts = 0.0;
    if (experts) {
      const double rows = (double)m / active;
      tiles = (rows < 0.5 * f.bm ? 1.0 : rows / f.bm + 0.5) * active;
      tiles = (tiles > 1.0 ? tiles : 1.0) * (double)nbn;
      rounds = tiles > (double)cus ? tiles / (double)cus : 1.0;
    } else {
      const int64_t all = (m + f.bm - 1) / f.bm * nbn;
      tiles = (double)all;
      rounds = (double)((all + cus - 1) / cus);
      shifts = (double)((all + cus * f.resident - 1) / (cus * f.resident));
    }
    const double stages = (double)((k + f.kstage - 1) / f.kstage);
    const double share = tiles / (double)cus;
    const double load = f.load + (k % 128 ? f.part : 0.f);
    const double us = f.start + rounds * (f.tile + stages * f.stage) + shifts * stages * f.shift +
                      share * (stages * load + (row16 ? 0.f : f.odd)) + mb * f.weights;
    if (best < 0 || us < least) {
      best = c;
      least = us;
    }
  }
  return best;
}

template <typename TO, bool GROUPED>
int launch_typed(F8Args g, hipStream_t st) {
  const int cus = device_cus();
  g.row16 = g.n % (16 / (int)sizeof(TO)) == 0 && !(reinterpret_cast<uintptr_t>(g.out) & 15);
  const int cfg = choose(g.m, g.k, g.n, g.experts, g.row16, cus > 0 ? cus : 256);
  if (cfg < 0) {
    set_error("fp8 linear: too many rows or columns (m %lld, n %lld)", (long long)g.m,
              (long long)g.n);
    return MXFP4_ERR_VALUE;
  }
  const Config& f = GROUPED ? kGrouped[cfg] : kDense[cfg];
  const int bm = (int)row_blocks(g.m, f.bm, g.experts), bn = (int)((g.n + f.bn - 1) / f.bn);
  const unsigned grid = (unsigned)bm * (unsigned)bn;
  const int nt = f.threads;
  if constexpr (GROUPED) {
    switch (cfg) {
      case GR256: f8_pf<TO, 8, 4, 2, 4, 2, 1, 2, true><<<grid, nt, 0, st>>>(g, bm, bn); break;
      case GR128: f8_pf<TO, 4, 4, 2, 2, 2, 1, 2, true><<<grid, nt, 0, st>>>(g, bm, bn); break;
      case GR64X128: f8_pf<TO, 2, 4, 2, 2, 3, 1, 2, true><<<grid, nt, 0, st>>>(g, bm, bn); break;
      case GR64X128R: f8_pf<TO, 4, 2, 1, 4, 2, 1, 2, true><<<grid, nt, 0, st>>>(g, bm, bn); break;
      case GR64: f8_pf<TO, 2, 2, 2, 2, 3, 1, 2, true><<<grid, nt, 0, st>>>(g, bm, bn); break;
      case GR32X256: f8_pf<TO, 2, 4, 1, 4, 2, 1, 2, true><<<grid, nt, 0, st>>>(g, bm, bn); break;
      case GR16X32: f8_kl<TO, 1, 2, 4, 2, true><<<grid, nt, 0, st>>>(g, bm, bn); break;
      default: f8_kl<TO, 1, 1, 8, 2, true><<<grid, nt, 0, st>>>(g, bm, bn); break;
    }
  } else {
    switch (cfg) {
      case PF256: f8_pf<TO, 8, 4, 2, 4, 2, 1, 2, false><<<grid, nt, 0, st>>>(g, bm, bn); break;
      case PF128: f8_pf<TO, 4, 4, 2, 2, 2, 1, 2, false><<<grid, nt, 0, st>>>(g, bm, bn); break;
      case PF128W: f8_pf<TO, 4, 2, 2, 4, 2, 1, 2, false><<<grid, nt, 0, st>>>(g, bm, bn); break;
      case PF128X64: f8_pf<TO, 4, 2, 2, 2, 3, 1, 2, false><<<grid, nt, 0, st>>>(g, bm, bn); break;
      case PF64: f8_pf<TO, 2, 2, 2, 2, 3, 1, 2, false><<<grid, nt, 0, st>>>(g, bm, bn); break;
      case PF64D: f8_pf<TO, 2, 2, 2, 2, 2, 1, 2, false><<<grid, nt, 0, st>>>(g, bm, bn); break;
      case PF64G: f8_pf<TO, 2, 2, 2, 2, 3, 2, 2, false><<<grid, nt, 0, st>>>(g, bm, bn); break;
      case PF64X32: f8_pf<TO, 2, 2, 2, 1, 3, 4, 2, false><<<grid, nt, 0, st>>>(g, bm, bn); break;
      case KL32: f8_kl<TO, 2, 2, 8, 1, false><<<grid, nt, 0, st>>>(g, bm, bn); break;
      case KL16X32: f8_kl<TO, 1, 2, 4, 2, false><<<grid, nt, 0, st>>>(g, bm, bn); break;
      default: f8_kl<TO, 1, 1, 8, 2, false><<<grid, nt, 0, st>>>(g, bm, bn); break;
    }
  }
  return launch_status("fp8 linear launch");
}

template <bool GROUPED>
int launch(const F8Args& g, int out_dtype, hipStream_t st) {
  switch (out_dtype) {
    case MXFP4_DT_BF16: return launch_typed<__bf16, GROUPED>(g, st);
    case MXFP4_DT_F16: return launch_typed<_Float16, GROUPED>(g, st);
    default: return launch_typed<float, GROUPED>(g, st);
  }
}

int check(const F8Args& g, int64_t k, int out_dtype) {
  if (out_dtype != MXFP4_DT_BF16 && out_dtype != MXFP4_DT_F16 && out_dtype != MXFP4_DT_F32) {
    set_error("fp8 linear: unsupported output dtype %d", out_dtype);
    return MXFP4_ERR_TYPE;
  }
  if (g.m < 0 || g.n < 0 || g.a_rows < 0 || k < 16 || k % 16 != 0 || k > MXFP4_FP8_MAX_K) {
    set_error("fp8 linear: K must be divisible by 16 and at most %d, got %lld (m %lld, n %lld)",
              MXFP4_FP8_MAX_K, (long long)k, (long long)g.m, (long long)g.n);
    return MXFP4_ERR_VALUE;
  }
  if (g.m > 0x7FFFFFFF || g.n > 0x7FFFFFFF) {
    set_error("fp8 linear: too many rows or columns (m %lld, n %lld)", (long long)g.m,
              (long long)g.n);
    return MXFP4_ERR_VALUE;
  }
  if (((reinterpret_cast<uintptr_t>(g.a) | reinterpret_cast<uintptr_t>(g.w)) & 15) != 0) {
    set_error("fp8 linear: operands must be 16-byte aligned");
    return MXFP4_ERR_VALUE;
  }
  // the scales are addressed through 32 bits, all of them: 2^29 values
  const int64_t most = 0x1FFFFFFF;
  if (g.sa_row < 1 || g.sa_block < 1 || g.sa_row > most || g.sa_block > most / g.kb ||
      (g.a_rows > 0 && g.a_rows - 1 > (most - (g.kb - 1) * g.sa_block - 1) / g.sa_row)) {
    set_error("fp8 linear: activation scales of %lld rows, strides %lld and %lld",
              (long long)g.a_rows, (long long)g.sa_row, (long long)g.sa_block);
    return MXFP4_ERR_VALUE;
  }
  return MXFP4_OK;
}

}  // namespace
}  // namespace mx

extern "C" int mxfp4_linear_fp8(const uint8_t* a, const float* a_scales,
                                int64_t a_scale_row_stride, int64_t a_scale_block_stride,
                                int64_t m, int64_t k, const uint8_t* w, const float* w_scales,
                                int64_t n, const void* bias, void* out, int out_dtype,
                                void* stream) {
  using namespace mx;
  F8Args g{};
  g.a = a;
  g.sa = a_scales;
  g.sa_row = a_scale_row_stride;
  g.sa_block = a_scale_block_stride;
  g.w = w;
  g.sw = w_scales;
  g.bias = bias;
  g.out = out;
  g.m = g.a_rows = m;
  g.n = n;
  g.k = (int)k;
  g.kb = (int)((k + 127) >> 7);
  const int rc = check(g, k, out_dtype);
  if (rc) return rc;
  if (m == 0 || n == 0) return MXFP4_OK;
  return launch<false>(g, out_dtype, static_cast<hipStream_t>(stream));
}

extern "C" int mxfp4_grouped_linear_fp8(const uint8_t* a, const float* a_scales,
                                        int64_t a_scale_row_stride, int64_t a_scale_block_stride,
                                        int64_t a_rows, int64_t k, const uint8_t* w,
                                        const float* w_scales, int num_experts, int64_t n,
                                        const int32_t* offsets, const int32_t* routes, int top_k,
                                        int64_t rows, void* out, int out_dtype, void* stream) {
  using namespace mx;
  F8Args g{};
  g.a = a;
  g.sa = a_scales;
  g.sa_row = a_scale_row_stride;
  g.sa_block = a_scale_block_stride;
  g.w = w;
  g.sw = w_scales;
  g.out = out;
  g.m = rows;
  g.n = n;
  g.k = (int)k;
  g.kb = (int)((k + 127) >> 7);
  g.offsets = offsets;
  g.routes = routes;
  g.a_rows = a_rows;
  g.top_k = top_k;
  g.experts = num_experts;
  const int rc = check(g, k, out_dtype);
  if (rc) return rc;
  if (num_experts < 1 || num_experts > 1024 || top_k < 1 || (!routes && a_rows != rows)) {
    set_error("fp8 linear: %d experts, top_k %d, %lld activation rows of %lld", num_experts, top_k,
              (long long)a_rows, (long long)rows);
    return MXFP4_ERR_VALUE;
  }
  // gathered activations are addressed through 32 bits, all of them
  if (routes && a_rows > 0x7FFFFFFF / k) {
    set_error("fp8 linear: %lld gathered activation rows of %lld bytes reach 2 GiB",
              (long long)a_rows, (long long)k);
    return MXFP4_ERR_VALUE;
  }
  if (rows == 0 || n == 0) return MXFP4_OK;
  if (a_rows == 0) {
    set_error("fp8 linear: no activation rows for %lld routes", (long long)rows);
    return MXFP4_ERR_VALUE;
  }
  return launch<true>(g, out_dtype, static_cast<hipStream_t>(stream));
}

// Test hook: the number of the kernel that a size runs with (experts: 0 for the dense
// product), -1 if none; how many there are if m is 0
extern "C" int mxfp4_test_fp8_kernel(int64_t m, int64_t k, int64_t n, int experts, int row16,
                                     int64_t cus) {
  if (m == 0) return experts ? (int)mx::GROUPS : (int)mx::DENSE;
  return mx::choose(m, k, n, experts, row16 != 0, cus);
}
