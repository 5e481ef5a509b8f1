// Sampling (mpc_sample): one token per row of logits by temperature, top-k, top-p and min-p from one
// uniform number. It stands beside softmax, sort and argmax of the op set; the reference has no
// sampler.
//
// All three filters keep a prefix of the tokens ranked by (logit descending, index ascending), so the kept
// set is "every token above a threshold logit, and the first r tokens equal to it", and no row is sorted:
//   1. the largest logit;
//   2. a histogram of counts over 4096 bins of T / 128 below it finds the bin where the ranks reach top_k, or
//      estimates the one where the weights reach top_p of their total;
//   3. the tokens of that bin and the bins above it (at most 2048; else the bin alone) are gathered and sorted,
//      and the border is found among them exactly, with the exact weight of what lies above. A bin of more
//      than 2048 tokens is cut again, by the bits of its logits; an estimate that was off moves on.
//   4. Where the gathered tokens are the whole kept set (any usual top_k, a narrow top_p) the draw is among them.
//      Else every warp sums the kept weights of its stretch of the row, and the one that the draw falls into
//      walks its stretch.
// Rows are read again by each step, from L1 or L2; HBM is read once.
//
// Weights w = exp((l - max) / T) in f64 are held as integers of 2^-shift (shift = 62 - log2 of the row's length, at
// most 51), so that sums are exact whatever their order: the same row always gives the same token, and
// the borders of top-p and of the drawn interval move by less than 1e-11 of the total.
//
// A cluster of 1 to 8 CTAs takes a row, as many as keep the SMs busy: a few rows are bound by latency, many by the
// f64 exponentials of the rows without top_k (about 12 double operations a token) and by the passes over L2.
#include <cooperative_groups.h>

#include "kv_cache.cuh"
#include "mpc_internal.h"

namespace cg = cooperative_groups;

namespace mpc {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaxCluster = 8;
constexpr int kBins = 4096, kPer = kBins / kThreads, kList = 2048;
constexpr float kBinsPerNat = 128.0f;

struct SampleParams {
  const void *logits;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t *top_k;
  int32_t *token, *kept;
  float *prob;
  long long stride;
  int vocab, d_top_k, shift;
  float d_temperature, d_top_p, d_min_p;
};

// Keys of the logits' order; NaN and -inf share the lowest, 0 (they are never kept).
__device__ __forceinline__ uint32_t key_of(float f) {
  const uint32_t b = __float_as_uint(f == 0.0f ? 0.0f : f);  // -0 ties with 0
  return !(f > -INFINITY) ? 0u : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

typedef unsigned long long u64;

struct Sums {  // one warp's stretch: kept weight and tokens above the threshold, tokens equal to it
  u64 w;
  unsigned n, ties;
};
struct Verdict {  // what the gathered tokens say
  u64 total;
  uint32_t key;
  unsigned ties;
  int again;
};
struct Shared {
  double table[32];  // 2^(i / 32)
  unsigned hist[kBins];  // later the merged list
  unsigned cum[kBins];   // tokens in bins 0..b, of the whole row
  u64 list[kList];
  u64 scratch[kWarps], s_above, s_in, total;
  Sums sums[kWarps], all[kWarps * kMaxCluster];
  float fscratch[kWarps];
  unsigned n_list, key_min, key_max;
  int b0, b1;
  Verdict verdict;
};

// Vectors of 16 bytes, aligned, over one row: vector v holds elements v * VE - mis ..+VE-1.
template <int DT>
struct Reader {
  static constexpr int VE = DT == MPC_F32 ? 4 : 8;
  using T = typename std::conditional<DT == MPC_F32, float, uint16_t>::type;
  const T *x;
  int V, mis, vectors;
  __device__ void set(const void *base, long long at, int n) {
    x = static_cast<const T *>(base) + at;
    V = n;
    mis = (int)(((uintptr_t)x & 15) / sizeof(T));
    vectors = (V + mis + VE - 1) / VE;
  }
  __device__ float one(int i) const {
    if constexpr (DT == MPC_F32) return __ldg(x + i);
    else if constexpr (DT == MPC_BF16) return __uint_as_float((uint32_t)__ldg(x + i) << 16);
    else return __half2float(__ushort_as_half(__ldg(x + i)));
  }
  __device__ int index(int v) const { return v * VE - mis; }
  __device__ void load(int v, float (&f)[VE]) const {
    const int i0 = index(v);
    if (i0 >= 0 && i0 + VE <= V) {
      const uint4 r = __ldg(reinterpret_cast<const uint4 *>(x + i0));
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (DT == MPC_F32) {
          f[k] = __uint_as_float(w[k]);
        } else {
          const float2 p = DT == MPC_BF16 ? bf16x2_to_f32(w[k]) : f16x2_to_f32(w[k]);
          f[2 * k] = p.x, f[2 * k + 1] = p.y;
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < VE; ++k) f[k] = i0 + k >= 0 && i0 + k < V ? one(i0 + k) : -INFINITY;
    }
  }
  // The largest of a thread's elements of vectors v0 + lane, + 32, ..; -inf where there is none.
  __device__ __forceinline__ float largest(int v0, int v1) const {
    float best = -INFINITY;
    if constexpr (DT == MPC_F32) {
      each(v0, v1, [&](float f, int) { best = fmaxf(best, f); });
    } else {
      // Pairs by the packed maximum of the type (a NaN gives the other number).
      uint32_t m = DT == MPC_BF16 ? 0xff80ff80u : 0xfc00fc00u;
      for (int v = v0 + (threadIdx.x & 31); v < v1; v += 32) {
        const int i0 = index(v);
        if (i0 >= 0 && i0 + VE <= V) {
          const uint4 r = __ldg(reinterpret_cast<const uint4 *>(x + i0));
          m = max2(m, max2(max2(r.x, r.y), max2(r.z, r.w)));
        } else {
          for (int k = 0; k < VE; ++k)
            if (i0 + k >= 0 && i0 + k < V) best = fmaxf(best, one(i0 + k));
        }
      }
      const float2 p = DT == MPC_BF16 ? bf16x2_to_f32(m) : f16x2_to_f32(m);
      best = fmaxf(best, fmaxf(p.x, p.y));
    }
    return best;
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (DT == MPC_BF16) asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  // fn(logit, index) over vectors v0 + lane, + 32, ..; elements outside the row come as -inf.
  template <typename Fn>
  __device__ __forceinline__ void each(int v0, int v1, Fn fn) const {
    constexpr int U = 16 / VE;  // 64 bytes (f32) or 32 in flight
    for (int v = v0 + (threadIdx.x & 31); v < v1; v += 32 * U) {
      float f[U][VE];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (v + 32 * u < v1) load(v + 32 * u, f[u]);
        else
#pragma unroll
          for (int k = 0; k < VE; ++k) f[u][k] = -INFINITY;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < VE; ++k) fn(f[u][k], index(v + 32 * u) + k);
    }
  }
};

// w = 2^(y), y = (l - top) log2(e) / T, as 2^n * 2^(i / 32) * 2^r with |r| <= 1/64: the second from a table, the
// last by its series to r^5 (the next term is below 3e-15).
struct Weights {
  double c, unit;  // log2(e) / T; 2^-shift
  float top;
  int shift;
  const double *table;
  __device__ __forceinline__ void parts(float f, double &s, double &p) const {
    constexpr double L = 0.69314718055994530942;
    double y = f == top ? 0.0 : ((double)f - (double)top) * c;
    y = fmax(y, -1000.0);  // also for NaN: logits below an infinite one
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the rounded integer
    const double t = fma(y, 32.0, magic);
    const int k = __double2loint(t);
    const double r = fma(t - magic, -1.0 / 32, y);
    p = fma(r, L * L * L * L * L / 120, L * L * L * L / 24);
    p = fma(p, r, L * L * L / 6);
    p = fma(p, r, L * L / 2);
    p = fma(p, r, L);
    p = fma(p, r, 1.0);
    const double e = table[k & 31];
    s = __hiloint2double(__double2hiint(e) + ((k >> 5) + shift) * (1 << 20), __double2loint(e));
  }
  __device__ __forceinline__ double weight(float f) const {
    double s, p;
    parts(f, s, p);
    return s * p * unit;
  }
  // The nearest whole number of units: below 2^52, so it appears in the low bits next to 2^52.
  __device__ __forceinline__ u64 whole(float f) const {
    double s, p;
    parts(f, s, p);
    return (u64)__double_as_longlong(fma(s, p, 4503599627370496.0)) - 0x4330000000000000ull;
  }
};

template <typename T>
__device__ __forceinline__ T warp_incl(T v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const T o = __shfl_up_sync(0xffffffffu, v, m);
    if (lane >= m) v += o;
  }
  return v;
}
// Inclusive prefix over the block's threads; *all: the sum.
template <typename T>
__device__ __forceinline__ T block_incl(T v, T *sm, T *all) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  v = warp_incl(v);
  __syncthreads();
  if (lane == 31) sm[w] = v;
  __syncthreads();
  T before = 0, sum = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < w) before += sm[i];
    sum += sm[i];
  }
  *all = sum;
  return v + before;
}

// Sorts n2 (a power of two) numbers in shared memory, descending or ascending.
__device__ void sort(u64 *a, int n2, bool descending) {
  for (int k = 2; k <= n2; k <<= 1)
    for (int j = k >> 1; j; j >>= 1) {
      __syncthreads();
      for (int q = threadIdx.x; q < n2 / 2; q += kThreads) {
        const int i = (q & ~(j - 1)) << 1 | (q & (j - 1)), l = i + j;
        const u64 x = a[i], y = a[l];
        if ((x < y) == (((i & k) == 0) == descending)) a[i] = y, a[l] = x;
      }
    }
  __syncthreads();
}

// The histogram's bins: by value below the largest logit (the last bin is not used: what lies deeper is not
// counted), or by the keys of an interval.
struct Bins {
  float top, scale;  // by value: bins of T / 128
  uint32_t lo, hi;   // by key: the interval; lo 0: by value
  int shift;
  // 2^23 + the distance below top in bins: its bits are the bin's number, and NaN and infinities compare as deep.
  __device__ __forceinline__ float place(float f) const { return fmaf(top - f, scale, 8388608.0f); }
  static __device__ __forceinline__ int bin(float place) { return __float_as_int(place) - 0x4b000000; }
  __device__ __forceinline__ int of_key(uint32_t key) const { return (int)((hi - key) >> shift); }
  // The weight of a bin's middle, for estimates.
  __device__ __forceinline__ float middle(int b, float per_nat) const {
    if (!lo) return __expf(-(float)b / kBinsPerNat);
    const uint32_t k = hi - min(hi - lo, ((uint32_t)b << shift) + ((1u << shift) >> 1));
    const float x = (top - logit_of(k)) * per_nat;
    return x > 0.0f ? __expf(-x) : 1.0f;
  }
  __device__ __forceinline__ void whole_row(uint32_t top_key) {
    lo = 1, hi = top_key, shift = 0;
    while (((hi - lo) >> shift) >= kBins) ++shift;
  }
};

template <int DT>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared &sm = *reinterpret_cast<Shared *>(raw);
  const auto cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int row = blockIdx.x / C, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Reader<DT> rd;
  rd.set(p.logits, row * p.stride, p.vocab);
  const int per_cta = (rd.vectors + C - 1) / C, per_warp = (per_cta + kWarps - 1) / kWarps;
  const int c1 = min(rd.vectors, (rank + 1) * per_cta);
  const int v0 = min(c1, rank * per_cta + warp * per_warp), v1 = min(c1, v0 + per_warp);
  const float t = p.temperature ? p.temperature[row] : p.d_temperature;
  const float top_p = p.top_p ? p.top_p[row] : p.d_top_p;
  const float min_p = p.min_p ? p.min_p[row] : p.d_min_p;
  const int top_k = p.top_k ? p.top_k[row] : p.d_top_k;
  if (threadIdx.x < 32) sm.table[threadIdx.x] = exp2(threadIdx.x / 32.0);

  // 1. The largest logit.
  uint32_t top_key = key_of(rd.largest(v0, v1));
  top_key = __reduce_max_sync(0xffffffffu, top_key);
  if (threadIdx.x == 0) sm.key_max = 0, sm.key_min = 0xffffffffu;
  __syncthreads();
  if (lane == 0) atomicMax(&sm.key_max, top_key);
  cl.sync();
  for (int i = 0; i < C; ++i) top_key = max(top_key, *cl.map_shared_rank(&sm.key_max, i));
  if (top_key == 0 || !(t > 0.0f)) {
    const float top = top_key ? logit_of(top_key) : 0.0f;
    unsigned at = 0xffffffffu;  // its lowest index
    if (top_key) rd.each(v0, v1, [&](float f, int i) {
      if (f == top) at = min(at, (unsigned)i);
    });
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) atomicMin(&sm.key_min, at);
    cl.sync();
    if (rank == 0 && threadIdx.x == 0) {
      for (int i = 0; i < C; ++i) at = min(at, *cl.map_shared_rank(&sm.key_min, i));
      p.token[row] = (int)at;  // none: -1
      if (p.prob) p.prob[row] = top_key ? 1.0f : 0.0f;
      if (p.kept) p.kept[row] = top_key ? 1 : 0;
    }
    cl.sync();  // nobody reads a CTA that has gone
    return;
  }
  Weights wt;
  wt.top = logit_of(top_key);
  wt.c = 1.4426950408889634074 / (double)t;
  wt.shift = p.shift;
  wt.unit = ldexp(1.0, -p.shift);
  wt.table = sm.table;
  const float u = fminf(fmaxf(p.u[row], 0.0f), 1.0f);
  auto draw_of = [&](u64 total) {
    const u64 d = (u64)__double2ll_rd((double)u * (double)total);
    return d < total ? d : total - 1;
  };
  auto passes = [&](uint32_t key, double w) { return key == top_key || !(w < (double)min_p); };

  // 2., 3. The threshold: keys above `key` are kept, and the first `ties` tokens of that key.
  uint32_t key = 0;
  unsigned ties = 0;
  bool by_k = top_k > 0 && top_k < p.vocab;
  const bool by_p = top_p < 1.0f;
  if (by_k || by_p) {
    Bins bins;
    bins.top = wt.top, bins.scale = kBinsPerNat / t, bins.lo = bins.hi = 0, bins.shift = 0;
    const bool by_value = fabsf(wt.top) < INFINITY && bins.scale > 0.0f && bins.scale < INFINITY;
    if (!by_value) bins.whole_row(top_key);
    bool counting = by_k;
    unsigned n_above = 0;           // tokens above the interval
    u64 base = 0, span = 0;         // weight above it, in it (by weight)
    u64 total = 0, want = 0;        // by weight: ranks before which less than `want` lies are kept
    bool known = false;             // total is
    auto want_of = [&](u64 sum) {
      const double lim = top_p > 0.0f ? (double)top_p * (double)sum : 0.0;
      const u64 w = (u64)__double2ll_ru(lim);
      return w < 1 ? 1 : w > sum ? sum : w;
    };
    for (bool found = false; !found;) {
      // The histogram of the interval.
      for (int i = threadIdx.x; i < kBins; i += kThreads) sm.hist[i] = 0;
      __syncthreads();
      u64 w = 0, sum;
      const bool weigh = !counting && !known;
      constexpr float kDeep = 8388608.0f + (kBins - 1);
      if (bins.lo) {
        rd.each(v0, v1, [&](float f, int) {
          const uint32_t k = key_of(f);
          if (k == 0) return;
          if (weigh) w += wt.whole(f);
          if (k >= bins.lo && k <= bins.hi) atomicAdd(&sm.hist[bins.of_key(k)], 1u);
        });
      } else if (weigh) {
        rd.each(v0, v1, [&](float f, int) {
          if (!(f > -INFINITY)) return;
          w += wt.whole(f);
          const float at = bins.place(f);
          if (at < kDeep) atomicAdd(&sm.hist[Bins::bin(at)], 1u);
        });
      } else {
        rd.each(v0, v1, [&](float f, int) {
          const float at = bins.place(f);
          if (at < kDeep) atomicAdd(&sm.hist[Bins::bin(at)], 1u);
        });
      }
      if (weigh) {
        block_incl(w, sm.scratch, &sum);
        if (threadIdx.x == 0) sm.total = sum;
      }
      cl.sync();
      unsigned cnt[kPer] = {};
      for (int i = 0; i < C; ++i) {
        const uint4 *h = reinterpret_cast<const uint4 *>(cl.map_shared_rank(sm.hist, i) + threadIdx.x * kPer);
#pragma unroll
        for (int j = 0; j < kPer / 4; ++j) {
          const uint4 x = h[j];
          cnt[4 * j] += x.x, cnt[4 * j + 1] += x.y, cnt[4 * j + 2] += x.z, cnt[4 * j + 3] += x.w;
        }
        if (weigh) total += *cl.map_shared_rank(&sm.total, i);
      }
      if (weigh) known = true, want = want_of(total), span = total;
      unsigned mine = 0, tokens;
#pragma unroll
      for (int j = 0; j < kPer; ++j) mine += cnt[j];
      unsigned before = block_incl(mine, reinterpret_cast<unsigned *>(sm.scratch), &tokens) - mine;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const unsigned incl = before + cnt[j];
        sm.cum[threadIdx.x * kPer + j] = incl;
        if (counting && n_above + before < (unsigned)top_k && n_above + incl >= (unsigned)top_k) sm.b1 = threadIdx.x * kPer + j;
        before = incl;
      }
      __syncthreads();
      if (counting && n_above + tokens < (unsigned)top_k) {
        cl.sync();
        if (!bins.lo) {  // top_k reaches below the counted bins
          bins.whole_row(top_key);
          continue;
        }
        by_k = counting = false;  // fewer tokens than top_k
        bins.lo = by_value ? 0 : bins.lo;
        if (!by_p) break;
        continue;
      }
      auto pop = [&](int a, int b) { return sm.cum[b] - (a ? sm.cum[a - 1] : 0u); };
      // The bin where the estimated weights reach `goal`, within [lo, hi], into sm.b1.
      auto by_weight = [&](float goal, int lo, int hi) {
        float e[kPer], part = 0.0f, all;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const int b = threadIdx.x * kPer + j;
          e[j] = (float)pop(b, b) * bins.middle(b, 1.0f / t);
          part += e[j];
        }
        float upto = block_incl(part, sm.fscratch, &all) - part;
        if (threadIdx.x == 0) sm.b1 = hi;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          upto += e[j];
          if (upto >= goal) atomicMin(&sm.b1, threadIdx.x * kPer + j);
        }
        __syncthreads();
        const int b = max(sm.b1, lo);
        __syncthreads();
        return b;
      };
      auto estimate = [&](int upto) {  // of the weights of bins 0..upto
        float part = 0.0f, all;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const int b = threadIdx.x * kPer + j;
          if (b <= upto) part += (float)pop(b, b) * bins.middle(b, 1.0f / t);
        }
        block_incl(part, sm.fscratch, &all);
        return all;
      };
      int bx;
      if (counting) bx = sm.b1;
      else bx = by_weight(span ? estimate(kBins - 1) * (float)((double)(want - base) / (double)span) : (float)((double)(want - base) * wt.unit), 0, kBins - 1);
      for (;;) {
        // The window [b0, b1]: all down to the border where the list holds that, else the bins next to it.
        int b1 = counting ? bx : min(bx + 1, kBins - 1);
        int b0 = pop(0, b1) <= kList ? 0 : counting ? bx : max(bx - 1, 0);
        if (pop(b0, b1) > kList) b0 = b1 = bx;
        const bool gather = pop(b0, b1) <= kList;
        const bool need = !counting || by_p;
        __syncthreads();
        if (threadIdx.x == 0) sm.n_list = 0, sm.key_min = 0xffffffffu, sm.key_max = 0;
        __syncthreads();
        u64 above = 0, in = 0;
        auto take = [&](float f, int i, uint32_t k, int b) {
          if (b < b0) {
            if (need) above += wt.whole(f);
          } else {
            if (!counting) in += wt.whole(f);
            if (gather) sm.list[atomicAdd(&sm.n_list, 1u)] = (u64)k << 32 | (0xffffffffu - (unsigned)i);
            else atomicMin(&sm.key_min, k), atomicMax(&sm.key_max, k);
          }
        };
        if (bins.lo) {
          rd.each(v0, v1, [&](float f, int i) {
            const uint32_t k = key_of(f);
            if (k < bins.lo) return;
            const int b = k > bins.hi ? -1 : bins.of_key(k);
            if (b <= b1) take(f, i, k, b);
          });
        } else {
          const float limit = 8388608.0f + (float)b1;
          rd.each(v0, v1, [&](float f, int i) {
            const float at = bins.place(f);
            if (at <= limit) take(f, i, key_of(f), Bins::bin(at));
          });
        }
        block_incl(above, sm.scratch, &sum);
        if (threadIdx.x == 0) sm.s_above = sum;
        block_incl(in, sm.scratch, &sum);
        if (threadIdx.x == 0) sm.s_in = sum;
        cl.sync();
        above = in = 0;
        uint32_t kmin = 0xffffffffu, kmax = 0;
        for (int i = 0; i < C; ++i) {
          above += *cl.map_shared_rank(&sm.s_above, i);
          in += *cl.map_shared_rank(&sm.s_in, i);
          kmin = min(kmin, *cl.map_shared_rank(&sm.key_min, i));
          kmax = max(kmax, *cl.map_shared_rank(&sm.key_max, i));
        }
        if (!counting && want <= above) {  // the border lies further up
          const float e = estimate(b0 - 1);
          bx = min(b0 - 1, by_weight((float)(e * ((double)(want - base) / (double)(above - base))), 0, b0 - 1));
          cl.sync();
          continue;
        }
        if (!counting && !bins.lo && b1 >= kBins - 2 && want > above + in) {  // below the counted bins
          bins.whole_row(top_key);
          n_above = 0, base = span = 0;
          cl.sync();
          break;
        }
        if (!counting && want > above + in) {  // further down
          const float e = estimate(b1);
          bx = by_weight((float)(e * ((double)(want - base) / (double)(above + in - base))), b1 + 1, kBins - 1);
          cl.sync();
          continue;
        }
        const unsigned over = n_above + (b0 ? sm.cum[b0 - 1] : 0u);  // tokens above the window
        if (!gather && kmin < kmax) {  // cut the window again by its keys
          bins.lo = kmin, bins.hi = kmax, bins.shift = 0;
          while (((kmax - kmin) >> bins.shift) >= kBins) ++bins.shift;
          n_above = over, base = above, span = counting ? 0 : in;
          cl.sync();
          break;
        }
        if (!gather) {  // more equal logits than the list holds
          const u64 each = wt.whole(logit_of(kmin));
          key = kmin;
          found = true;
          if (counting) {
            ties = (unsigned)top_k - over;
            if (by_p) {
              total = above + ties * each, want = want_of(total);
              if (want <= above) found = false;
            }
          } else {
            ties = pop(b0, b1);
          }
          if (found && by_p && each) ties = (unsigned)min((u64)ties, (want - above + each - 1) / each);
          if (!found) {  // top-p's border lies above top-k's: find it by weight, from the whole row
            counting = false, known = true, base = span = 0, n_above = 0;
            if (by_value) bins.lo = 0;
            else bins.whole_row(top_key);
          }
          cl.sync();
          break;
        }
        // The first CTA sorts the gathered tokens and finds the border among them.
        if (rank == 0) {
          u64 *const all = reinterpret_cast<u64 *>(sm.hist);
          int n = 0;
          for (int i = 0; i < C; ++i) {
            const int m = (int)*cl.map_shared_rank(&sm.n_list, i);
            const u64 *from = cl.map_shared_rank(sm.list, i);
            for (int j = threadIdx.x; j < m; j += kThreads) all[n + j] = from[j];
            n += m;
          }
          int n2 = 32;
          while (n2 < n) n2 <<= 1;
          for (int j = n + threadIdx.x; j < n2; j += kThreads) all[j] = 0;
          sort(all, n2, true);
          const int lim = counting ? min(n, (int)((unsigned)top_k - over)) : n;
          // Thread i weighs ranks 4i ..+3.
          u64 q[kList / kThreads], part = 0;
          const int r0 = threadIdx.x * (kList / kThreads);
#pragma unroll
          for (int j = 0; j < kList / kThreads; ++j) {
            q[j] = r0 + j < lim && by_p ? wt.whole(logit_of((uint32_t)(all[r0 + j] >> 32))) : 0;
            part += q[j];
          }
          u64 upto = block_incl(part, sm.scratch, &sum) - part;
          u64 goal = want;
          bool again = false;
          if (counting && by_p) {
            total = above + sum, goal = want_of(total);
            again = goal <= above;
          }
          unsigned kept = 0;
          upto += above;
#pragma unroll
          for (int j = 0; j < kList / kThreads; ++j) {
            kept += r0 + j < lim && (!by_p || upto < goal);
            upto += q[j];
          }
          unsigned n_kept;
          block_incl(kept, reinterpret_cast<unsigned *>(sm.scratch), &n_kept);
          if (over == 0) {
            // 4. The kept set is among the gathered tokens: min-p, then the draw in the order of the indices.
            kept = 0;
            for (unsigned j = threadIdx.x; j < n_kept; j += kThreads) {
              const uint32_t k = (uint32_t)(all[j] >> 32);
              kept += passes(k, wt.weight(logit_of(k)));
            }
            block_incl(kept, reinterpret_cast<unsigned *>(sm.scratch), &n_kept);
            n2 = 32;
            while (n2 < (int)n_kept) n2 <<= 1;
            for (int j = threadIdx.x; j < n2; j += kThreads) {
              const u64 x = all[j];
              all[j] = j < (int)n_kept ? (u64)(0xffffffffu - (uint32_t)x) << 32 | x >> 32 : ~0ull;
            }
            sort(all, n2, false);
            part = 0;
#pragma unroll
            for (int j = 0; j < kList / kThreads; ++j) {
              q[j] = r0 + j < (int)n_kept ? wt.whole(logit_of((uint32_t)all[r0 + j])) : 0;
              part += q[j];
            }
            upto = block_incl(part, sm.scratch, &sum) - part;
            const u64 d = draw_of(sum);
#pragma unroll
            for (int j = 0; j < kList / kThreads; ++j) {
              if (upto <= d && d < upto + q[j]) {
                const u64 x = all[r0 + j];
                p.token[row] = (int32_t)(x >> 32);
                if (p.prob) p.prob[row] = (float)(wt.weight(logit_of((uint32_t)x)) / ((double)sum * wt.unit));
              }
              upto += q[j];
            }
            if (threadIdx.x == 0 && p.kept) p.kept[row] = (int32_t)n_kept;
          } else if (threadIdx.x == 0) {
            Verdict v;
            v.total = total, v.again = again, v.key = 0, v.ties = 0;
            if (!again) {
              v.key = (uint32_t)(all[n_kept - 1] >> 32);
              for (int j = (int)n_kept - 1; j >= 0 && (uint32_t)(all[j] >> 32) == v.key; --j) ++v.ties;
            }
            sm.verdict = v;
          }
        }
        cl.sync();
        if (over == 0) return;  // the first CTA has drawn
        const Verdict v = *cl.map_shared_rank(&sm.verdict, 0);
        cl.sync();
        if (v.again) {
          counting = false, known = true, base = span = 0, n_above = 0;
          if (by_value) bins.lo = 0;
          else bins.whole_row(top_key);
          total = v.total, want = want_of(total);
        } else {
          key = v.key, ties = v.ties, found = true;
        }
        break;
      }
    }
  }

  // 4. Every warp's kept weight, and the one that the draw falls into.
  float far = -INFINITY;  // below it w < min_p for sure
  if (min_p > 0.0f) {
    const float x = wt.top + t * logf(min_p) - (0.01f * t + 1e-6f * fabsf(wt.top));
    if (x == x) far = fminf(x, wt.top);
  }
  const float at_key = key ? logit_of(key) : __int_as_float(0x7fffffff);  // none: NaN
  const float low = fmaxf(fmaxf(key ? at_key : -INFINITY, far), -3.402823466e38f);  // tokens below are not kept
  {
    Sums s{0, 0, 0};
    rd.each(v0, v1, [&](float f, int) {
      if (!(f >= low)) return;
      if (f == at_key) {
        ++s.ties;
        return;
      }
      double a, b;
      wt.parts(f, a, b);
      if (min_p > 0.0f && f != wt.top && a * b * wt.unit < (double)min_p) return;
      s.w += (u64)__double_as_longlong(fma(a, b, 4503599627370496.0)) - 0x4330000000000000ull;
      ++s.n;
    });
#pragma unroll
    for (int m = 16; m; m >>= 1) {
      s.w += __shfl_xor_sync(0xffffffffu, s.w, m);
      s.n += __shfl_xor_sync(0xffffffffu, s.n, m);
      s.ties += __shfl_xor_sync(0xffffffffu, s.ties, m);
    }
    if (lane == 0) sm.sums[warp] = s;
  }
  cl.sync();
  for (int i = threadIdx.x; i < C * kWarps; i += kThreads) sm.all[i] = cl.map_shared_rank(sm.sums, i / kWarps)[i % kWarps];
  __syncthreads();
  const u64 tie_w = key ? wt.whole(logit_of(key)) : 0;
  if (key && !passes(key, wt.weight(logit_of(key)))) ties = 0;
  // Each warp walks the stretches up to its own, lane by lane of 32.
  u64 total = 0, before = 0, mine = 0;
  unsigned kept = 0, tie_before = 0, tie_at = 0;
  const int self = rank * kWarps + warp;
  for (int i0 = 0; i0 < C * kWarps; i0 += 32) {
    Sums s{0, 0, 0};
    if (i0 + lane < C * kWarps) s = sm.all[i0 + lane];
    const unsigned tie_incl = tie_at + warp_incl(s.ties), tie_excl = tie_incl - s.ties;
    const unsigned take = min(ties, tie_incl) - min(ties, tie_excl);
    const u64 w = s.w + take * tie_w, incl = total + warp_incl(w);
    const unsigned n = warp_incl(s.n + take);
    if (i0 <= self && self < i0 + 32) {
      mine = __shfl_sync(0xffffffffu, w, self - i0);
      before = __shfl_sync(0xffffffffu, incl, self - i0) - mine;
      tie_before = __shfl_sync(0xffffffffu, tie_excl, self - i0);
    }
    total = __shfl_sync(0xffffffffu, incl, 31);
    kept += __shfl_sync(0xffffffffu, n, 31);
    tie_at = __shfl_sync(0xffffffffu, tie_incl, 31);
  }
  if (rank == 0 && threadIdx.x == 0 && p.kept) p.kept[row] = (int32_t)kept;
  const u64 d = draw_of(total);
  if (before <= d && d < before + mine) {
    constexpr int VE = Reader<DT>::VE;
    u64 at = before;
    unsigned tie = tie_before;
    for (int v = v0; v < v1; v += 32) {
      float f[VE];
#pragma unroll
      for (int k = 0; k < VE; ++k) f[k] = -INFINITY;
      if (v + lane < v1) rd.load(v + lane, f);
      unsigned eq = 0;
#pragma unroll
      for (int k = 0; k < VE; ++k) eq += f[k] == at_key;
      const unsigned eq_incl = warp_incl(eq);
      unsigned my_tie = tie + eq_incl - eq;
      u64 q[VE], part = 0;
#pragma unroll
      for (int k = 0; k < VE; ++k) {
        q[k] = 0;
        if (!(f[k] >= low)) continue;
        if (f[k] == at_key) {
          if (my_tie++ < ties) q[k] = tie_w;
        } else if (!(min_p > 0.0f) || f[k] == wt.top || !(wt.weight(f[k]) < (double)min_p)) {
          q[k] = wt.whole(f[k]);
        }
        part += q[k];
      }
      const u64 incl = at + warp_incl(part);
      u64 upto = incl - part;
      if (upto <= d && d < incl) {
#pragma unroll
        for (int k = 0; k < VE; ++k) {
          if (upto <= d && d < upto + q[k]) {
            p.token[row] = rd.index(v + lane) + k;
            if (p.prob) p.prob[row] = (float)(wt.weight(f[k]) / ((double)total * wt.unit));
          }
          upto += q[k];
        }
      }
      at = __shfl_sync(0xffffffffu, incl, 31);
      if (at > d) break;
      tie += __shfl_sync(0xffffffffu, eq_incl, 31);
    }
  }
  cl.sync();
}

template <int DT>
int launch_sample(mpc_device *dev, const SampleParams &p, int rows, cudaStream_t st) {
  static bool configured[64] = {};
  const int ord = dev->ordinal & 63;
  if (!configured[ord]) {
    MPC_CUDA(dev, cudaFuncSetAttribute(sample_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared)));
    configured[ord] = true;
  }
  // CTAs per row: up to two for every SM, of at least 2048 tokens.
  int c = 1;
  while (c < kMaxCluster && (long long)rows * c < 2ll * dev->prop.multiProcessorCount && p.vocab >= 2 * c * 2048) c *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)rows * c), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = sizeof(Shared), cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)c, at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  MPC_CUDA(dev, cudaLaunchKernelEx(&cfg, sample_kernel<DT>, p));
  dev->launches++;
  return MPC_OK;
}

}  // namespace
}  // namespace mpc

using namespace mpc;

extern "C" int mpc_sample(mpc_device *dev, const mpc_sample_desc *d, const void *logits, const float *u,
                          const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                          int32_t *token, float *prob, int32_t *kept, mpc_stream s) {
  int rc = enter(dev);
  if (rc) return rc;
  if (!d) return fail(MPC_ERR_INVALID, "mpc_sample: null descriptor");
  if (d->dtype < MPC_F32 || d->dtype > MPC_BF16) return fail(MPC_ERR_INVALID, "mpc_sample: logits of dtype %d", d->dtype);
  if (d->rows < 0 || d->vocab < 0 || d->row_stride < 0)
    return fail(MPC_ERR_INVALID, "mpc_sample: negative extent or stride");
  if (d->rows > INT32_MAX || d->vocab > (1 << 30))
    return fail(MPC_ERR_UNSUPPORTED, "mpc_sample: more than 2^31 - 1 rows or 2^30 tokens");
  if (d->rows == 0) return MPC_OK;
  if (d->vocab == 0) return fail(MPC_ERR_INVALID, "mpc_sample: rows of no tokens");
  if (!logits || !u || !token) return fail(MPC_ERR_INVALID, "mpc_sample: null pointer");
  SampleParams p{};
  p.logits = logits, p.u = u, p.temperature = temperature, p.top_p = top_p, p.min_p = min_p, p.top_k = top_k;
  p.token = token, p.kept = kept, p.prob = prob, p.stride = d->row_stride, p.vocab = (int)d->vocab;
  p.d_top_k = d->top_k, p.d_temperature = d->temperature, p.d_top_p = d->top_p, p.d_min_p = d->min_p;
  int log2v = 0;
  while ((int64_t(1) << log2v) < d->vocab) ++log2v;
  p.shift = log2v < 11 ? 51 : 62 - log2v;  // V weights of at most 2^shift stay below 2^63, each below 2^52
  cudaStream_t st = stream_of(dev, s);
  const int rows = (int)d->rows;
  if (d->dtype == MPC_F32) return launch_sample<MPC_F32>(dev, p, rows, st);
  if (d->dtype == MPC_BF16) return launch_sample<MPC_BF16>(dev, p, rows, st);
  return launch_sample<MPC_F16>(dev, p, rows, st);
}
