// Tokens sorted by expert and back.  No counterpart in the reference.
//
// Route r = t * top_k + s is slot s of token t; its expert is its id where that is
// in [0, E), else it is dropped.  The order is a counting sort into E + 1 buckets,
// the last one the dropped routes':
//   offsets[x]  = routes of experts below x (offsets[E]: all that are not dropped)
//   position[r] = offsets[expert] + routes before r of the same expert; -1: dropped
//   routes      = its inverse, -1 from offsets[E] on
//
// The moves go by token, not by sorted row, so that a token's row is read once
// and written to its top_k places (or gathered from them), whatever top_k is:
//   sort     rows[position[t, s]] = x[t], zeros from offsets[E] on
//   combine  out[t] = sum_s w[t, s] * y[position[t, s]]          (FP32, slot order)
//   its gradient  dy[position[t, s]] = w[t, s] * g[t], dw[t, s] = <g[t], y[position[t, s]]>
// and the gradient of sort is combine without weights.  Every output row has one
// writer and every sum a fixed order: no atomics, the same bits on every call.
#include "common.h"

namespace mx {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kMaxBuckets = kMaxExperts + 1;

template <typename TI>
__device__ __forceinline__ int bucket_of(TI id, int experts) {
  const int64_t e = (int64_t)id;
  return e >= 0 && e < experts ? (int)e : experts;
}

// Lanes of the wave in the same bucket as this one; `in`: the lane has a route.
__device__ __forceinline__ uint64_t same_bucket(int b, bool in, int bits) {
  uint64_t same = __ballot(in);
  for (int i = 0; i < bits; ++i) {
    const bool one = (b >> i) & 1;
    const uint64_t has = __ballot(one);
    same &= one ? has : ~has;
  }
  return same;
}

__device__ __forceinline__ int lanes_before(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

__device__ __forceinline__ int wave_scan(int v) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int u = __shfl_up(v, off);
    if (lane >= off) v += u;
  }
  return v;
}

struct SortOut {
  int32_t* offsets;
  int32_t* routes;
  int32_t* position;
};

__device__ __forceinline__ void put_route(const SortOut& o, int64_t r, int p, bool dropped) {
  o.routes[p] = dropped ? -1 : (int32_t)r;
  o.position[r] = dropped ? -1 : p;
}

// From per-bucket counts to places.  `pre`, `tot`: routes of a thread's EPT buckets
// before this chunk and in all; wpos[wave][bucket] holds the waves' counts of the
// chunk and receives their first places.  Writes offsets if `first`.
template <int NT, int EPT>
__device__ __forceinline__ void place_of(const int (&pre)[EPT], const int (&tot)[EPT], int nb,
                                         int* wpos, int* part, bool first, int32_t* offsets) {
  constexpr int W = NT / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int local = 0;
#pragma unroll
  for (int j = 0; j < EPT; ++j) local += tot[j];
  int sum = wave_scan(local);
  if (lane == 63) part[wave] = sum;
  __syncthreads();
  for (int w = 0; w < wave; ++w) sum += part[w];
  int start = sum - local;
#pragma unroll
  for (int j = 0; j < EPT; ++j) {
    const int x = tid * EPT + j;
    if (x < nb) {
      if (first) offsets[x] = start;
      int p = start + pre[j];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int c = wpos[w * nb + x];
        wpos[w * nb + x] = p;
        p += c;
      }
    }
    start += tot[j];
  }
  __syncthreads();
}

// The whole order in one launch, up to kOneLaunch routes: workgroup c places the 512
// routes of chunk c and counts all others itself (earlier ones in the low half of a
// word, later ones in the high half, kOneCopies copies against lanes that meet
// in one bucket), so that no workgroup waits for another.  Bound by the launch and one
// chain: 1024 routes over 128 experts 4.3 us (two launches 7.1), 16384 7.6 (8.7), 32768
// 10.9 (9.4).
constexpr int kOneChunk = 512;
constexpr int64_t kOneLaunch = 16384;
constexpr int kOneCopies = 4;

template <typename TI, bool ONE>
__global__ __launch_bounds__(kOneChunk) void sort_one(const TI* __restrict__ ids, int64_t n,
                                                      int experts, int bits, SortOut o) {
  constexpr int NT = kOneChunk, W = NT / 64;
  constexpr int EPT = (kMaxBuckets + NT - 1) / NT;
  constexpr int B = 8;  // id loads of a thread in flight
  __shared__ int wpos[W * kMaxBuckets];
  __shared__ uint32_t cnt[ONE ? 1 : kOneCopies * kMaxBuckets];
  __shared__ int part[W];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int nb = experts + 1;
  const int c = (int)blockIdx.x;
  const int64_t mine = (int64_t)c * NT + tid;
  const bool in = mine < n;
  const int b = in ? bucket_of(ids[mine], experts) : 0;
  for (int i = tid; i < W * nb; i += NT) wpos[i] = 0;
  if constexpr (!ONE) {
    uint32_t* const my = cnt + (lane % kOneCopies) * nb;
    for (int i = tid; i < kOneCopies * nb; i += NT) cnt[i] = 0;
    __syncthreads();
    for (int64_t i0 = 0; i0 < n; i0 += B * NT) {
      TI v[B];
#pragma unroll
      for (int q = 0; q < B; ++q) v[q] = i0 + q * NT + tid < n ? ids[i0 + q * NT + tid] : (TI)0;
#pragma unroll
      for (int q = 0; q < B; ++q) {
        const int cc = (int)(i0 / NT) + q;
        if (cc != c && i0 + q * NT + tid < n)
          atomicAdd(&my[bucket_of(v[q], experts)], cc < c ? 1u : 1u << 16);
      }
    }
  } else {
    __syncthreads();
  }
  const uint64_t same = same_bucket(b, in, bits);
  const int rank = lanes_before(same);
  if (in && rank == 0) wpos[wave * nb + b] = __popcll(same);
  __syncthreads();
  int pre[EPT], tot[EPT];
#pragma unroll
  for (int j = 0; j < EPT; ++j) {
    const int x = tid * EPT + j;
    pre[j] = tot[j] = 0;
    if (x < nb) {
      uint32_t others = 0;
#pragma unroll
      for (int q = 0; q < (ONE ? 0 : kOneCopies); ++q) others += cnt[q * nb + x];
      pre[j] = (int)(others & 0xFFFF);
      tot[j] = pre[j] + (int)(others >> 16);
#pragma unroll
      for (int w = 0; w < W; ++w) tot[j] += wpos[w * nb + x];
    }
  }
  place_of<NT, EPT>(pre, tot, nb, wpos, part, c == 0, o.offsets);
  if (in) put_route(o, mine, wpos[wave * nb + b] + rank, b == experts);
}

// More routes: counts by chunk, then (beyond kScanChunks chunks one workgroup turns
// them into first places, else each workgroup sums them itself) the places.  131072
// routes over 8, 128, 1024 experts 10.9, 12.5, 21.9 us (with the scan 12.8, 14.9, 22.1),
// 2^20 34.8, 45.9, 99.5 (43.0, 51.8, 98.6); the sums grow with the square of the
// routes, the scan (one workgroup: 2^23 routes over 128 experts 351) does not.  A launch
// and one chain of four sub-chunks bound the smallest of these: 32768 routes are 16
// workgroups, 2.8 + 7.2 us.
constexpr int kChunk = 2048;
constexpr int kScanChunks = 512;

template <typename TI>
__global__ __launch_bounds__(512) void sort_count(const TI* __restrict__ ids, int64_t n,
                                                  int experts, int32_t* __restrict__ counts) {
  __shared__ int hist[kMaxBuckets];
  const int nb = experts + 1;
  for (int x = threadIdx.x; x < nb; x += 512) hist[x] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kChunk;
#pragma unroll
  for (int i = 0; i < kChunk / 512; ++i) {
    const int64_t r = base + i * 512 + threadIdx.x;
    if (r < n) atomicAdd(&hist[bucket_of(ids[r], experts)], 1);
  }
  __syncthreads();
  for (int x = threadIdx.x; x < nb; x += 512) counts[(int64_t)blockIdx.x * nb + x] = hist[x];
}

// counts[chunk][bucket] -> routes of the bucket in earlier chunks, and offsets
__global__ __launch_bounds__(1024) void sort_scan(int32_t* __restrict__ counts, int64_t chunks,
                                                  int nb, int32_t* __restrict__ offsets) {
  __shared__ int total[kMaxBuckets];
  __shared__ int part[16];
  const int tid = threadIdx.x;
  for (int x = tid; x < nb; x += 1024) {
    int sum = 0;
    for (int64_t c0 = 0; c0 < chunks; c0 += 8) {
      int v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = c0 + q < chunks ? counts[(c0 + q) * nb + x] : 0;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        if (c0 + q < chunks) counts[(c0 + q) * nb + x] = sum;
        sum += v[q];
      }
    }
    total[x] = sum;
  }
  __syncthreads();
  // two buckets a thread
  const int a = 2 * tid < nb ? total[2 * tid] : 0, b = 2 * tid + 1 < nb ? total[2 * tid + 1] : 0;
  int sum = wave_scan(a + b);
  if ((tid & 63) == 63) part[tid >> 6] = sum;
  __syncthreads();
  for (int w = 0; w < tid >> 6; ++w) sum += part[w];
  if (2 * tid < nb) offsets[2 * tid] = sum - a - b;
  if (2 * tid + 1 < nb) offsets[2 * tid + 1] = sum - b;
}

template <typename TI, bool SCANNED>
__global__ __launch_bounds__(512) void sort_place(const TI* __restrict__ ids, int64_t n,
                                                  int experts, int bits,
                                                  const int32_t* __restrict__ counts, int chunks,
                                                  SortOut o) {
  constexpr int NT = 512, W = NT / 64, RPT = kChunk / NT;
  constexpr int EPT = (kMaxBuckets + NT - 1) / NT;
  __shared__ int wpos[W * kMaxBuckets];
  __shared__ int s_pre[SCANNED ? 1 : kMaxBuckets], s_tot[SCANNED ? 1 : kMaxBuckets];
  __shared__ int part[W];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int nb = experts + 1;
  const int64_t c = blockIdx.x;
  const int64_t base = c * kChunk + wave * (RPT * 64) + lane;
  int b[RPT], rank[RPT];
  bool in[RPT];
#pragma unroll
  for (int j = 0; j < RPT; ++j) {
    in[j] = base + j * 64 < n;
    b[j] = in[j] ? bucket_of(ids[base + j * 64], experts) : 0;
  }
  for (int i = tid; i < W * nb; i += NT) wpos[i] = 0;
  if constexpr (!SCANNED) {
    for (int x = tid; x < nb; x += NT) {
      int pre = 0, tot = 0;
      for (int q0 = 0; q0 < chunks; q0 += 8) {
        int v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = q0 + q < chunks ? counts[(q0 + q) * nb + x] : 0;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          tot += v[q];
          if (q0 + q < c) pre += v[q];
        }
      }
      s_pre[x] = pre;
      s_tot[x] = tot;
    }
  }
  __syncthreads();
  // the wave's own part of wpos: its sub-chunks in order, no barrier between them
#pragma unroll
  for (int j = 0; j < RPT; ++j) {
    const uint64_t same = same_bucket(b[j], in[j], bits);
    const int before = lanes_before(same);
    rank[j] = 0;
    if (in[j]) rank[j] = wpos[wave * nb + b[j]] + before;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in[j] && before == 0) wpos[wave * nb + b[j]] += __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  __syncthreads();
  if constexpr (SCANNED) {
    for (int x = tid; x < nb; x += NT) {
      int p = o.offsets[x] + counts[c * nb + x];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int v = wpos[w * nb + x];
        wpos[w * nb + x] = p;
        p += v;
      }
    }
    __syncthreads();
  } else {
    int pre[EPT], tot[EPT];
#pragma unroll
    for (int j = 0; j < EPT; ++j) {
      const int x = tid * EPT + j;
      pre[j] = x < nb ? s_pre[x] : 0;
      tot[j] = x < nb ? s_tot[x] : 0;
    }
    place_of<NT, EPT>(pre, tot, nb, wpos, part, c == 0, o.offsets);
  }
#pragma unroll
  for (int j = 0; j < RPT; ++j)
    if (in[j])
      put_route(o, base + j * 64, wpos[wave * nb + b[j]] + rank[j], b[j] == experts);
}

template <typename TI>
int launch_sort(const TI* ids, int64_t n, int experts, const SortOut& o, int32_t* counts,
                hipStream_t st) {
  int bits = 0;
  while ((experts >> bits) != 0) ++bits;
  if (n <= kOneChunk) {
    sort_one<TI, true><<<1, kOneChunk, 0, st>>>(ids, n, experts, bits, o);
  } else if (n <= kOneLaunch) {
    const int grid = (int)((n + kOneChunk - 1) / kOneChunk);
    sort_one<TI, false><<<grid, kOneChunk, 0, st>>>(ids, n, experts, bits, o);
  } else {
    const int chunks = (int)((n + kChunk - 1) / kChunk);
    sort_count<TI><<<chunks, 512, 0, st>>>(ids, n, experts, counts);
    if (chunks <= kScanChunks) {
      sort_place<TI, false><<<chunks, 512, 0, st>>>(ids, n, experts, bits, counts, chunks, o);
    } else {
      sort_scan<<<1, 1024, 0, st>>>(counts, chunks, experts + 1, o.offsets);
      sort_place<TI, true><<<chunks, 512, 0, st>>>(ids, n, experts, bits, counts, chunks, o);
    }
  }
  return launch_status("sort routes launch");
}

// ------------------------------------------------------------------- moves

// A vector of V elements of T and its FP32 values
template <typename T, int V>
struct Vec {
  typedef T type __attribute__((ext_vector_type(V)));
};
template <typename T>
struct Vec<T, 1> {
  typedef T type;
};
template <typename T, int V>
__device__ __forceinline__ float at(const typename Vec<T, V>::type& v, int i) {
  if constexpr (V == 1) return (float)v;
  else return (float)v[i];
}
template <typename T, int V>
__device__ __forceinline__ typename Vec<T, V>::type rounded(const float (&f)[V]) {
  if constexpr (V == 1) {
    return from_f32<T>(f[0]);
  } else {
    typename Vec<T, V>::type o;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = from_f32<T>(f[i]);
    return o;
  }
}

// A token's places and weights, a lane's each (top_k <= 64): one load, and then scalars
// by their slot's number; a place outside the rows counts as none.  at() and weight() read
// other lanes: every lane has to be active where they are called.
struct Slots {
  int p;
  float w;
  __device__ __forceinline__ Slots(const int32_t* position, const float* weights, int64_t t,
                                   int top_k, int64_t rows) {
    const int lane = threadIdx.x & 63;
    const int64_t r = t * top_k + (lane < top_k ? lane : 0);
    const int raw = position[r];
    w = weights ? weights[r] : 1.f;
    p = lane < top_k && raw >= 0 && raw < rows ? raw : -1;
  }
  // -1 past the last slot too
  __device__ __forceinline__ int at(int s) const { return __builtin_amdgcn_readlane(p, s); }
  __device__ __forceinline__ float weight(int s) const {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), s));
  }
};

// HBM bound, near or above a large copy's 5.1 TB/s: 4096 x 8 routes of 2048 bf16 sort 26 us
// (151 MB), combine 29 alone and 34 to 44 behind the sort, its gradients 48 (286 MB).  A
// token's places in one load instead of one for each slot: combine 46 -> 43 us there.
// Rows off 16 bytes go by elements (units of 4, 2 or 1 bytes in the sort): 509 x 4 routes
// of 1407 fp32 7.6, 6.2 and 13.4 us.
constexpr int kSlots = 8;  // rows of a thread in flight

// x's rows, units of U (1, 2, 4 or 16 bytes), to their places; token blockIdx.x, ..,
// units blockIdx.y * 256 + thread.  The rows behind the last expert's, `units` of
// zeros, are dealt out over the tokens.
template <typename U>
__global__ __launch_bounds__(256) void sort_rows(const U* __restrict__ x, int64_t m, int64_t units,
                                                 int64_t ldx, const int32_t* __restrict__ position,
                                                 const int32_t* __restrict__ live, int top_k,
                                                 U* __restrict__ rows) {
  const int64_t n = m * top_k;
  const int64_t first_dead = *live;
  for (int64_t t = blockIdx.x; t < m; t += gridDim.x) {
    const Slots slots(position, nullptr, t, top_k, n);
    for (int64_t u0 = (int64_t)blockIdx.y * 256; u0 < units; u0 += (int64_t)gridDim.y * 256) {
      const int64_t u = u0 + threadIdx.x;
      const bool in = u < units;
      const U v = x[t * ldx + (in ? u : u0)];
      for (int s = 0; s < top_k; ++s) {
        const int p = slots.at(s);
        if (in && p >= 0) rows[p * units + u] = v;
      }
      for (int64_t p = t; p < n; p += m)
        if (in && p >= first_dead) rows[p * units + u] = U{};
    }
  }
}

template <typename T, int V>
__global__ __launch_bounds__(256) void combine_rows(const T* __restrict__ y, int64_t rows,
                                                    int64_t h, int64_t ldy,
                                                    const int32_t* __restrict__ position,
                                                    int64_t m, int top_k,
                                                    const float* __restrict__ weights,
                                                    T* __restrict__ out) {
  typedef typename Vec<T, V>::type TV;
  const int64_t units = h / V;
  for (int64_t t = blockIdx.x; t < m; t += gridDim.x) {
    const Slots slots(position, weights, t, top_k, rows);
    for (int64_t u0 = (int64_t)blockIdx.y * 256; u0 < units; u0 += (int64_t)gridDim.y * 256) {
      const int64_t u = u0 + threadIdx.x;
      const bool in = u < units;
      const T* const yu = y + (in ? u : u0) * V;
      float acc[V];
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = 0.f;
      for (int s0 = 0; s0 < top_k; s0 += kSlots) {
        // all loads before the first addition; a slot without a row reads the first one
        TV v[kSlots];
        if (rows > 0) {
#pragma unroll
          for (int s = 0; s < kSlots; ++s) {
            const int p = slots.at(s0 + s);
            v[s] = *reinterpret_cast<const TV*>(yu + (p < 0 ? 0 : p) * ldy);
          }
        }
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
          if (slots.at(s0 + s) >= 0) {
            const float w = slots.weight(s0 + s);
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = fmaf(w, at<T, V>(v[s], i), acc[i]);
          }
        }
      }
      if (in) *reinterpret_cast<TV*>(out + t * h + u * V) = rounded<T, V>(acc);
    }
  }
}

// dy and dw (either may be null) of a token's slots, in one pass over y.  dw's sum:
// each thread its units in order, then the waves by a tree.
template <typename T, int V>
__global__ __launch_bounds__(256) void combine_grad(const T* __restrict__ g, int64_t m, int64_t h,
                                                    int64_t ldg, const T* __restrict__ y,
                                                    int64_t ldy,
                                                    const int32_t* __restrict__ position,
                                                    const int32_t* __restrict__ live, int top_k,
                                                    const float* __restrict__ weights,
                                                    T* __restrict__ dy, float* __restrict__ dw) {
  typedef typename Vec<T, V>::type TV;
  __shared__ float part[kSlots][4];
  const int64_t units = h / V;
  const int64_t n = m * top_k;
  const int64_t first_dead = *live;
  const int tid = threadIdx.x;
  for (int64_t t = blockIdx.x; t < m; t += gridDim.x) {
    const Slots slots(position, weights, t, top_k, n);
    for (int s0 = 0; s0 < top_k; s0 += kSlots) {
      int p[kSlots];
      float w[kSlots], dot[kSlots];
#pragma unroll
      for (int s = 0; s < kSlots; ++s) {
        p[s] = slots.at(s0 + s);
        w[s] = slots.weight(s0 + s);
        dot[s] = 0.f;
      }
      for (int64_t u0 = 0; u0 < units; u0 += 256) {
        const int64_t u = u0 + tid;
        if (u >= units) continue;
        const TV gv = *reinterpret_cast<const TV*>(g + t * ldg + u * V);
        TV v[kSlots];
        if (dw) {
#pragma unroll
          for (int s = 0; s < kSlots; ++s)
            v[s] = *reinterpret_cast<const TV*>(y + (p[s] < 0 ? 0 : p[s]) * ldy + u * V);
        }
        float f[V];
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = at<T, V>(gv, i);
        if (dw) {
#pragma unroll
          for (int s = 0; s < kSlots; ++s)
            if (p[s] >= 0) {
#pragma unroll
              for (int i = 0; i < V; ++i) dot[s] = fmaf(f[i], at<T, V>(v[s], i), dot[s]);
            }
        }
        if (dy) {
#pragma unroll
          for (int s = 0; s < kSlots; ++s)
            if (p[s] >= 0) {
              float o[V];
#pragma unroll
              for (int i = 0; i < V; ++i) o[i] = w[s] * f[i];
              *reinterpret_cast<TV*>(dy + p[s] * h + u * V) = rounded<T, V>(o);
            }
        }
      }
      if (dw) {
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
#pragma unroll
          for (int off = 32; off; off >>= 1) dot[s] += __shfl_xor(dot[s], off);
          if ((tid & 63) == 0) part[s][tid >> 6] = dot[s];
        }
        __syncthreads();
        if (tid < kSlots && s0 + tid < top_k)
          dw[t * top_k + s0 + tid] =
              (part[tid][0] + part[tid][1]) + (part[tid][2] + part[tid][3]);
        __syncthreads();
      }
    }
    if (dy) {
      for (int64_t p = t; p < n; p += m) {
        if (p < first_dead) continue;
        float zero[V];
#pragma unroll
        for (int i = 0; i < V; ++i) zero[i] = 0.f;
        for (int64_t u = tid; u < units; u += 256)
          *reinterpret_cast<TV*>(dy + p * h + u * V) = rounded<T, V>(zero);
      }
    }
  }
}

// Workgroups by token and by 256 units of a row
dim3 token_grid(int64_t m, int64_t units) {
  const int64_t x = m < 0x7FFFFF ? m : 0x7FFFFF;  // 2^31 threads a launch
  int64_t y = (units + 255) / 256;
  if (y > 65535) y = 65535;
  if (x * y > 0x7FFFFF) y = 0x7FFFFF / x;
  return dim3((unsigned)x, (unsigned)(y > 0 ? y : 1));
}

int elem_bytes(int dtype) {
  switch (dtype) {
    case MXFP4_DT_F32: case MXFP4_DT_I32: return 4;
    case MXFP4_DT_BF16: case MXFP4_DT_F16: return 2;
    case MXFP4_DT_I64: return 8;
    default: return 1;
  }
}

int check_rows(const char* what, int64_t m, int64_t h, int top_k) {
  if (m < 0 || h < 1 || top_k < 1 || top_k > 64 || m > 0x3FFFFFFF / top_k) {
    set_error("%s: unsupported sizes (tokens %lld, row %lld, top_k %d)", what, (long long)m,
              (long long)h, top_k);
    return MXFP4_ERR_VALUE;
  }
  return MXFP4_OK;
}

// T and whether 16-byte vectors fit -> f(T{}, integral_constant<int, V>{})
template <typename F>
void by_type(int dtype, bool vec, F&& f) {
#define C_(v) std::integral_constant<int, (v)>{}
  switch (dtype) {
    case MXFP4_DT_BF16: vec ? f(__bf16{}, C_(8)) : f(__bf16{}, C_(1)); break;
    case MXFP4_DT_F16: vec ? f(_Float16{}, C_(8)) : f(_Float16{}, C_(1)); break;
    default: vec ? f(float{}, C_(4)) : f(float{}, C_(1)); break;
  }
#undef C_
}

bool float_dtype(int d) {
  return d == MXFP4_DT_F32 || d == MXFP4_DT_BF16 || d == MXFP4_DT_F16;
}

}  // namespace
}  // namespace mx

extern "C" int mxfp4_sort_routes_workspace_size(int64_t n, int num_experts, int64_t* bytes) {
  using namespace mx;
  if (n < 0 || n > 0x3FFFFFFF || num_experts < 1 || num_experts > kMaxExperts) {
    set_error("sort routes: unsupported sizes (routes %lld, experts %d)", (long long)n,
              num_experts);
    return MXFP4_ERR_VALUE;
  }
  *bytes = n <= kOneLaunch ? 0 : (n + kChunk - 1) / kChunk * (num_experts + 1) * 4;
  return MXFP4_OK;
}

extern "C" int mxfp4_sort_routes(const void* topk_ids, int ids_dtype, int64_t n, int num_experts,
                                 int32_t* offsets, int32_t* routes, int32_t* position,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace mx;
  if (ids_dtype != MXFP4_DT_I32 && ids_dtype != MXFP4_DT_I64) {
    set_error("topk_ids must be int32 or int64");
    return MXFP4_ERR_TYPE;
  }
  int64_t need = 0;
  const int rc = mxfp4_sort_routes_workspace_size(n, num_experts, &need);
  if (rc) return rc;
  if (workspace_bytes < need || (need && (reinterpret_cast<uintptr_t>(workspace) & 3))) {
    set_error("sort routes: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
              (long long)need);
    return MXFP4_ERR_VALUE;
  }
  const SortOut o{offsets, routes, position};
  hipStream_t st = static_cast<hipStream_t>(stream);
  int32_t* const counts = static_cast<int32_t*>(workspace);
  if (ids_dtype == MXFP4_DT_I32)
    return launch_sort(static_cast<const int32_t*>(topk_ids), n, num_experts, o, counts, st);
  return launch_sort(static_cast<const int64_t*>(topk_ids), n, num_experts, o, counts, st);
}

extern "C" int mxfp4_sort_tokens(const void* x, int dtype, int64_t m, int64_t h,
                                 int64_t x_row_stride, const int32_t* position,
                                 const int32_t* offsets, int num_experts, int top_k, void* rows,
                                 void* stream) {
  using namespace mx;
  if (dtype < MXFP4_DT_F32 || dtype > MXFP4_DT_I8) {
    set_error("sort tokens: unsupported dtype %d", dtype);
    return MXFP4_ERR_TYPE;
  }
  const int rc = check_rows("sort tokens", m, h, top_k);
  if (rc) return rc;
  if (x_row_stride < h || num_experts < 1 || num_experts > kMaxExperts) {
    set_error("sort tokens: row stride %lld of rows of %lld, experts %d", (long long)x_row_stride,
              (long long)h, num_experts);
    return MXFP4_ERR_VALUE;
  }
  if (m == 0) return MXFP4_OK;
  const int64_t b = elem_bytes(dtype), row = h * b, ld = x_row_stride * b;
  const uint64_t low = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(rows) |
                       (uint64_t)row | (uint64_t)ld;
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto go = [&](auto unit) {
    typedef decltype(unit) U;
    const int64_t s = (int64_t)sizeof(U);
    sort_rows<U><<<token_grid(m, row / s), 256, 0, st>>>(
        static_cast<const U*>(x), m, row / s, ld / s, position, offsets + num_experts, top_k,
        static_cast<U*>(rows));
  };
  if (low % 16 == 0) go(i32x4{});
  else if (low % 4 == 0) go(uint32_t{});
  else if (low % 2 == 0) go(uint16_t{});
  else go(uint8_t{});
  return launch_status("sort tokens launch");
}

extern "C" int mxfp4_combine_tokens(const void* y, int dtype, int64_t rows, int64_t h,
                                    int64_t y_row_stride, const int32_t* position, int64_t m,
                                    int top_k, const float* weights, void* out, void* stream) {
  using namespace mx;
  if (!float_dtype(dtype)) {
    set_error("combine tokens: unsupported dtype %d", dtype);
    return MXFP4_ERR_TYPE;
  }
  const int rc = check_rows("combine tokens", m, h, top_k);
  if (rc) return rc;
  if (y_row_stride < h || rows < 0) {
    set_error("combine tokens: row stride %lld of rows of %lld", (long long)y_row_stride,
              (long long)h);
    return MXFP4_ERR_VALUE;
  }
  if (m == 0) return MXFP4_OK;
  const int64_t b = elem_bytes(dtype);
  const bool vec = ((reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(out) |
                     (uintptr_t)(h * b) | (uintptr_t)(y_row_stride * b)) & 15) == 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  by_type(dtype, vec, [&](auto type, auto v) {
    typedef decltype(type) T;
    constexpr int V = decltype(v)::value;
    combine_rows<T, V><<<token_grid(m, h / V), 256, 0, st>>>(
        static_cast<const T*>(y), rows, h, y_row_stride, position, m, top_k, weights,
        static_cast<T*>(out));
  });
  return launch_status("combine tokens launch");
}

extern "C" int mxfp4_combine_tokens_grad(const void* g, int dtype, int64_t m, int64_t h,
                                         int64_t g_row_stride, const void* y, int64_t y_row_stride,
                                         const int32_t* position, const int32_t* offsets,
                                         int num_experts, int top_k, const float* weights,
                                         void* dy, float* dweights, void* stream) {
  using namespace mx;
  if (!float_dtype(dtype)) {
    set_error("combine tokens gradient: unsupported dtype %d", dtype);
    return MXFP4_ERR_TYPE;
  }
  const int rc = check_rows("combine tokens gradient", m, h, top_k);
  if (rc) return rc;
  if (g_row_stride < h || (dweights && y_row_stride < h) || num_experts < 1 ||
      num_experts > kMaxExperts) {
    set_error("combine tokens gradient: row strides %lld, %lld of rows of %lld, experts %d",
              (long long)g_row_stride, (long long)y_row_stride, (long long)h, num_experts);
    return MXFP4_ERR_VALUE;
  }
  if (m == 0 || (dy == nullptr && dweights == nullptr)) return MXFP4_OK;
  const int64_t b = elem_bytes(dtype);
  uintptr_t low = reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(dy) |
                  (uintptr_t)(h * b) | (uintptr_t)(g_row_stride * b);
  if (dweights) low |= reinterpret_cast<uintptr_t>(y) | (uintptr_t)(y_row_stride * b);
  hipStream_t st = static_cast<hipStream_t>(stream);
  by_type(dtype, low % 16 == 0, [&](auto type, auto v) {
    typedef decltype(type) T;
    constexpr int V = decltype(v)::value;
    combine_grad<T, V><<<token_grid(m, 1), 256, 0, st>>>(
        static_cast<const T*>(g), m, h, g_row_stride, static_cast<const T*>(y), y_row_stride,
        position, offsets + num_experts, top_k, weights, static_cast<T*>(dy), dweights);
  });
  return launch_status("combine tokens gradient launch");
}
