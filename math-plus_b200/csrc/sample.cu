// Sampling (mpc_sample): one token per row of logits by temperature, top-k, top-p and min-p from one
// uniform number. It stands beside softmax, sort and argmax of the op set; the reference has no
// sampler.
//
// All three filters keep a prefix of the tokens ranked by (logit descending, index ascending), so the kept
// set is "every token above a threshold logit, and the first r tokens equal to it", and no row is sorted:
//   1. the largest logit;
//   2. a bound below the border: for a small top_k, the least over the CTAs of their (top_k / CTAs)-th largest of the
//      256 threads' maxima, since top_k tokens reach it for sure. Else a histogram of counts over 8192 bins of
//      T / 256 below the largest gives the bin where the ranks reach top_k or, with the weights' exact total, an
//      estimate of the one where the weights reach top_p of it;
//   3. the tokens between the bound (or the bin, by weight the next one too) and what lies surely above are gathered
//      (at most 256), the exact weight of those above is summed, and the border is found among the gathered, each
//      compared with every other. An estimate that was off moves; a bin of more tokens is cut again, by the bits
//      of its logits.
//   4. Where the gathered tokens are the whole kept set (a small top_k, a narrow top_p) the draw is among them.
//      Else every warp has the kept weight of its stretch of the row, and the block with the one that the draw falls
//      into goes through that stretch again, a piece per thread.
// Rows are read again by each step, from L1 or L2; HBM is read once.
//
// Weights w = exp((l - max) / T) in f64 are held as integers of 2^-shift (shift = 62 - log2 of the row's length, at
// most 51), so that sums are exact whatever their order: the same row always gives the same token. The roundings of V
// weights move the borders of top-p and of the drawn interval by at most V 2^-(shift + 1) of the largest weight, at
// worst (a tail of weights just under half a unit): 2^-31 at 2^16 tokens, 2^-23, two steps of u next to 1, at 2^20.
// Rows of more tokens are refused.
//
// A cluster of 1 to 8 CTAs takes a row. A few rows are bound by latency (cluster barriers and remote reads), many by the
// passes over the row and their f64 exponentials (10 double operations each, at 33.5 M tokens a fifth of the time without
// filters by the published rate; the rest is latency at 16 warps an SM). Measured (GPU time of a replayed call): 4 rows of
// 50257 bf16 with mixed settings 14.7 us (alike: greedy 6, top_k 50 15, top_p 0.9 26, top_k 1000 with top_p and min_p 45);
// 256 rows of 131071 f32 with mixed settings 173 us (greedy 57, top_k 50 102, no filter 104, top_p 0.9 265); 134 MB at
// 6.55 TB/s are 20.5 us.
#include <cooperative_groups.h>

#include "kv_cache.cuh"
#include "mpc_internal.h"
#include "sm100.cuh"

namespace cg = cooperative_groups;

namespace mpc {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kMaxCluster = 8;
// kSmallK: top_k up to which the threads' maxima give the bound. Measured (by them / by the histogram) at top_k 1, 50, 100,
// 192: 4 rows of 50257 bf16 12.2 / 13.9, 15.3 / 16.6, 17.7 / 17.7, 27.8 / 21.0 us; 256 of 131071 f32 87 / 113,
// 102 / 130, 115 / 142, 167 / 159 us.
constexpr int kBins = 8192, kList = kThreads, kSmallK = 192;
constexpr float kBinsPerNat = 256.0f;

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
struct Share {  // one CTA's part of step 2: over its share of the bins, tokens and estimated weights; the weights' exact
  u64 total;    // total over its stretch
  unsigned n;
  float e;
};
struct Border {  // a bin, the tokens above it and in it, the estimated weight above it
  int bin;       // -1: none
  unsigned over, pop;
  float e;
};
struct Gathered {  // one CTA's part of step 3
  u64 above, in;  // weight above the window; in it, where it is too much to be gathered
  unsigned n, key_min, key_max;
};
struct Verdict {  // what the gathered tokens say
  u64 total;
  uint32_t key;
  unsigned ties;
  int next;  // 0: the border is found; 1: it lies further up, 2: down; 3: top-p's lies above top-k's
};
struct Shared {
  double table[32];  // 2^(i / 32 + shift)
  u64 list[kList];  // the gathered tokens of this CTA's stretch
  u64 all[kList];   // of the row (the first CTA)
  u64 q[kThreads];
  unsigned counts[kBins];
  u64 scratch[kWarps];
  Share share;
  // Of each warp's and each CTA's share of the bins: where the border is reached; the last bin with tokens.
  Border reached_in[kWarps], last_in[kWarps], reached[kMaxCluster], last[kMaxCluster];
  unsigned warp_n[kWarps];
  float warp_e[kWarps];
  Gathered gathered;
  Verdict verdict;
  Sums sums[kWarps], every[kWarps * kMaxCluster];
  union {
    float largest[kThreads];
    float queue[kWarps][544];  // a batch of 512 and 31 that wait
  };
  unsigned waiting[kWarps];
  unsigned key_max, key_min, key_kth;
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
  // fn(16 logits, v) over vectors v0 + lane, + 32, ..: logit k is element element(v, k). All lanes of a warp go
  // through as many batches; elements outside the row or the stretch come as -inf.
  static constexpr int U = 16 / VE;
  __device__ __forceinline__ int element(int v, int k) const { return index(v + 32 * (k / VE)) + k % VE; }
  template <typename Fn>
  __device__ __forceinline__ void batches(int v0, int v1, Fn fn) const {
    const int lane = threadIdx.x & 31;
    for (int w = v0; w < v1; w += 32 * U) {
      const int v = w + lane;
      float f[U][VE];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (v + 32 * u < v1) load(v + 32 * u, f[u]);
        else
#pragma unroll
          for (int k = 0; k < VE; ++k) f[u][k] = -INFINITY;
      }
      fn(reinterpret_cast<const float(&)[16]>(f), v);
    }
  }
  template <typename Fn>
  __device__ __forceinline__ void each(int v0, int v1, Fn fn) const {  // fn(logit, index)
    batches(v0, v1, [&](const float(&f)[16], int v) {
#pragma unroll
      for (int k = 0; k < 16; ++k) fn(f[k], element(v, k));
    });
  }
};

// w = 2^(y), y = (l - top) log2(e) / T, as 2^n * 2^(i / 32) * 2^r with |r| <= 1/64: the second from a table, the
// last by its series to r^4 (the next term is below 1.3e-12 and changes sign with r).
constexpr u64 kMagicBits = 0x4330000000000000ull;  // 2^52: the nearest whole number of a sum with it is in its low bits
struct Weights {
  double c, unit;  // log2(e) / T; 2^-shift
  float top, floor;
  bool plain;  // logits below `floor` weigh nothing, and clamping to it is safe
  const double *table;
  __device__ __forceinline__ void of(double y, double &s, double &p) const {
    constexpr double L = 0.69314718055994530942;
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the rounded integer
    const double t = fma(y, 32.0, magic);
    const int k = __double2loint(t);
    const double r = fma(t - magic, -1.0 / 32, y);
    p = fma(r, L * L * L * L / 24, L * L * L / 6);
    p = fma(p, r, L * L / 2);
    p = fma(p, r, L);
    p = fma(p, r, 1.0);
    const double e = table[k & 31];
    s = __hiloint2double(__double2hiint(e) + ((k & ~31) << 15), __double2loint(e));
  }
  __device__ __forceinline__ void parts(float f, double &s, double &p) const {
    const double y = f == top ? 0.0 : ((double)f - (double)top) * c;
    of(fmax(y, -900.0), s, p);  // fmax also for NaN: logits below an infinite one
  }
  __device__ __forceinline__ double weight(float f) const {
    double s, p;
    parts(f, s, p);
    return s * p * unit;
  }
  // The nearest whole number of units: below 2^52.
  __device__ __forceinline__ u64 whole(float f) const {
    double s, p;
    parts(f, s, p);
    return (u64)__double_as_longlong(fma(s, p, 4503599627370496.0)) - kMagicBits;
  }
  // The same, for any f (0 for NaN and -inf), where `plain`.
  __device__ __forceinline__ void parts_any(float f, double &s, double &p) const {
    of(((double)fmaxf(f, floor) - (double)top) * c, s, p);
  }
  __device__ __forceinline__ u64 whole_any(float f) const {
    double s, p;
    parts_any(f, s, p);
    return (u64)__double_as_longlong(fma(s, p, 4503599627370496.0)) - kMagicBits;
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

// counts[bin] + 1 where `at` is below `end`, without a branch; counts0 is the shared address less the bits of 2^23.
__device__ __forceinline__ void count_if(uint32_t counts0, float at, float end) {
  asm volatile("{\n .reg .pred p;\n setp.lt.f32 p, %1, %2;\n @p red.shared.add.u32 [%0], 1;\n}\n" ::"r"(
                   counts0 + 4 * (uint32_t)__float_as_int(at)),
               "f"(at), "f"(end));
}

// The histogram's bins: by value below the largest logit (the last bin is not used: what lies deeper is not
// counted), or by the keys of an interval.
struct Bins {
  float top, scale;  // by value: bins of T / 256
  uint32_t lo, hi;   // by key: the interval; lo 0: by value
  int shift;
  // 2^23 + the distance below top in bins: its bits are the bin's number, and NaN and infinities compare as deep.
  __device__ __forceinline__ float place(float f) const { return fmaf(top - f, scale, 8388608.0f); }
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

template <int DT, int C>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared &sm = *reinterpret_cast<Shared *>(raw);
  const auto cl = cg::this_cluster();
  const int rank = (int)cl.block_rank();
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
  if (threadIdx.x < 32) sm.table[threadIdx.x] = ldexp(exp2(threadIdx.x / 32.0), p.shift);

  Weights wt;
  wt.c = 1.4426950408889634074 / (double)t;
  wt.unit = ldexp(1.0, -p.shift);
  wt.table = sm.table;

  // 1. The largest logit.
  const float largest = rd.largest(v0, v1);
  uint32_t top_key = key_of(largest);
  bool by_k = top_k > 0 && top_k < p.vocab;
  bool quick = by_k && top_k <= kSmallK;
  if (quick) sm.largest[threadIdx.x] = largest;
  top_key = __reduce_max_sync(0xffffffffu, top_key);
  if (threadIdx.x == 0) sm.key_max = sm.key_kth = 0, sm.key_min = 0xffffffffu;
  __syncthreads();
  if (lane == 0) atomicMax(&sm.key_max, top_key);
  if (quick) {  // the thread whose maximum has rank ceil(top_k / C) - 1 of the CTA's
    int above = 0;
#pragma unroll 8
    for (int i = 0; i < kThreads; ++i) above += sm.largest[i] > largest || (sm.largest[i] == largest && i < (int)threadIdx.x);
    if (above == (top_k + C - 1) / C - 1) sm.key_kth = key_of(largest);
  }
  cl.sync();
  // Lane i reads CTA i: one remote latency.
  top_key = __reduce_max_sync(0xffffffffu, lane < C ? *cl.map_shared_rank(&sm.key_max, lane) : 0u);
  const uint32_t bound = __reduce_min_sync(0xffffffffu, lane < C ? *cl.map_shared_rank(&sm.key_kth, lane) : 0xffffffffu);
  if (top_key == 0 || !(t > 0.0f) || min_p > 1.0f) {  // nothing to draw among: with min_p above 1 the first rank is left
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
  wt.top = logit_of(top_key);
  wt.floor = wt.top - 46.0f * t;  // 2^-66
  wt.plain = wt.top - wt.floor >= 40.0f * t && wt.floor >= -3.402823466e38f;  // not where t is lost next to top
  const float u = fminf(fmaxf(p.u[row], 0.0f), 1.0f);
  auto draw_of = [&](u64 total) {
    const u64 d = (u64)__double2ll_rd((double)u * (double)total);
    return d < total ? d : total - 1;
  };
  // Whether a kept token passes min_p.
  auto passes = [&](float f) { return !(min_p > 0.0f) || f == wt.top || !(wt.weight(f) < (double)min_p); };
  float far = -INFINITY, sure = -INFINITY;  // below `far` w < min_p, from `sure` on not, f32's rounding allowed for
  if (min_p > 0.0f) {
    const float x = wt.top + t * logf(min_p), slack = 0.01f * t + 1e-6f * fabsf(wt.top);
    sure = wt.top;
    if (x - slack == x - slack) far = fminf(x - slack, wt.top), sure = fminf(x + slack, wt.top);
  }
  bool summed = false;  // the warps' sums are those of the tokens above the window, whose own are in the lists
  u64 add_up = 0;
  Sums s{0, 0, 0};

  // 2., 3. The threshold: keys above `key` are kept, and the first `ties` tokens of that key.
  uint32_t key = 0;
  unsigned ties = 0;
  const bool by_p = top_p < 1.0f;
  if (by_k || by_p) {
    Bins bins;
    bins.top = wt.top, bins.scale = kBinsPerNat / t, bins.lo = bins.hi = 0, bins.shift = 0;
    const bool by_value = fabsf(wt.top) < INFINITY && bins.scale > 0.0f && bins.scale < INFINITY;
    if (!by_value) bins.whole_row(top_key);
    quick = quick && bound && by_value;  // the bound's gather goes by values
    bool counting = by_k;
    unsigned n_above = 0;     // tokens above the interval
    u64 base = 0;             // their weight
    u64 total = 0, want = 0;  // by weight: ranks before which less than `want` lies are kept
    bool known = false;       // total and want are
    float factor = 0.0f;      // by weight: estimated over exact weight, as last seen (0: not yet)
    int b_min = 0, b_max = kBins - 1;  // by weight: the border's bin is in here
    bool alone = false;                // the window is the border's bin alone
    bool counted = false;              // the interval's histogram is at hand
    auto want_of = [&](u64 sum) {
      const double lim = top_p > 0.0f ? (double)top_p * (double)sum : 0.0;
      const u64 w = (u64)__double2ll_ru(lim);
      return w < 1 ? 1 : w > sum ? sum : w;
    };
    auto whole_interval = [&] {
      counted = counted && !bins.lo;
      n_above = 0, base = 0, bins.lo = 0, factor = 0.0f, b_min = 0, b_max = kBins - 1;
      if (!by_value) bins.whole_row(top_key);
    };
    for (bool found = false; !found;) {
      Border at{-1, 0, 0, 0.0f};
      u64 sum = 0;
      int b0 = 0, b1 = 0;
      bool gather = true;
      unsigned outside = 0;  // tokens above the window
      if (threadIdx.x == 0) sm.gathered = Gathered{0, 0, 0, 0xffffffffu, 0};
      if (!quick) {
        // The histogram of the interval.
        const bool weigh = !counting && !known;
        u64 w = 0;
        const bool fresh = !counted || weigh;
        if (fresh) {
          for (int i = threadIdx.x; i < kBins; i += kThreads) sm.counts[i] = 0;
          __syncthreads();
          constexpr float kDeep = 8388608.0f + (kBins - 1);
          const uint32_t counts0 = smem_u32(sm.counts) - 4u * 0x4b000000u;
          if (bins.lo) {
            rd.each(v0, v1, [&](float f, int) {
              const uint32_t k = key_of(f);
              if (weigh && k) w += wt.whole(f);
              if (k >= bins.lo && k <= bins.hi) atomicAdd(&sm.counts[bins.of_key(k)], 1u);
            });
          } else if (weigh && wt.plain) {
            rd.batches(v0, v1, [&](const float(&f)[16], int) {
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                count_if(counts0, bins.place(f[k]), kDeep);
                w += wt.whole_any(f[k]);
              }
            });
          } else {
            rd.batches(v0, v1, [&](const float(&f)[16], int) {
#pragma unroll
              for (int k = 0; k < 16; ++k) count_if(counts0, bins.place(f[k]), kDeep);
            });
            if (weigh) rd.each(v0, v1, [&](float f, int) { w += f > -INFINITY ? wt.whole(f) : 0; });
          }
        }
        counted = true;
        if (weigh) block_incl(w, sm.scratch, &sum);
        cl.sync();
        // CTA r adds up the C histograms over its share of the bins, each warp over consecutive ones.
        constexpr int steps = kBins / kThreads / C;
        const int first = (rank * kWarps + warp) * 32 * steps + lane;
        const float per_nat = 1.0f / t;
        unsigned mine = 0, over = n_above;
        float mine_e = 0.0f, before_e = 0.0f, all_e = 0.0f;
#pragma unroll 4
        for (int j = 0; j < steps; ++j) {
          unsigned n = 0;
          if (C > 1 && fresh) {
#pragma unroll
            for (int i = 0; i < C; ++i) n += cl.map_shared_rank(sm.counts, i)[first + 32 * j];
            sm.counts[first + 32 * j] = n;  // nobody else reads this share here
          } else {
            n = sm.counts[first + 32 * j];
          }
          mine += n;
          if (!counting && n) mine_e += (float)n * bins.middle(first + 32 * j, per_nat);
        }
        mine = __reduce_add_sync(0xffffffffu, mine);
        for (int i = 16; i; i >>= 1) mine_e += __shfl_xor_sync(0xffffffffu, mine_e, i);
        if (lane == 0) sm.warp_n[warp] = mine, sm.warp_e[warp] = mine_e, sm.reached_in[warp].bin = sm.last_in[warp].bin = -1;
        __syncthreads();
        unsigned n_share = 0;
        float e_share = 0.0f;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
          if (i < warp) over += sm.warp_n[i], before_e += sm.warp_e[i];
          n_share += sm.warp_n[i], e_share += sm.warp_e[i];
        }
        if (threadIdx.x == 0) sm.share = Share{sum, n_share, e_share};
        cl.sync();
        {
          Share x{0, 0, 0.0f};
          if (lane < C) x = *cl.map_shared_rank(&sm.share, lane);
          over += __shfl_sync(0xffffffffu, warp_incl(x.n) - x.n, rank);
          if (!counting) {
            const float ei = warp_incl(x.e);
            before_e += __shfl_sync(0xffffffffu, ei - x.e, rank);
            all_e = __shfl_sync(0xffffffffu, ei, 31);
            if (!known) total = __shfl_sync(0xffffffffu, warp_incl(x.total), 31), want = want_of(total), known = true;
            // What is estimated adds up to the total, unless the interval is a part of the row.
            if (factor == 0.0f) factor = base || bins.lo > 1 ? (float)wt.unit : (float)((double)all_e / (double)total);
          }
        }
        const float goal = (float)(want - base) * factor;
        if (!counting || (over < (unsigned)top_k && over + mine >= (unsigned)top_k))
          for (int j = 0; j < steps; ++j) {
            const int bin = first + 32 * j;
            const unsigned n = sm.counts[bin], ni = warp_incl(n);
            const float e = !counting && n ? (float)n * bins.middle(bin, per_nat) : 0.0f, ei = counting ? 0.0f : warp_incl(e);
            const bool in = n && bin >= b_min && bin <= b_max;
            const unsigned hit = __ballot_sync(0xffffffffu, in && (counting ? over + ni >= (unsigned)top_k : before_e + ei >= goal));
            const unsigned some = __ballot_sync(0xffffffffu, in);
            const Border mark{bin, over + ni - n, n, before_e + ei - e};
            if (hit && lane == __ffs(hit) - 1) sm.reached_in[warp] = mark;
            if (some && lane == 31 - __clz(some)) sm.last_in[warp] = mark;
            if (hit) break;
            over += __shfl_sync(0xffffffffu, ni, 31);
            before_e += __shfl_sync(0xffffffffu, ei, 31);
          }
        __syncthreads();
        if (threadIdx.x < C) {  // thread i tells CTA i
          Border reached{-1, 0, 0, 0.0f}, last = reached;
          for (int i = kWarps - 1; i >= 0; --i) {
            if (sm.reached_in[i].bin >= 0) reached = sm.reached_in[i];
            if (last.bin < 0) last = sm.last_in[i];
          }
          Shared *const to = cl.map_shared_rank(&sm, threadIdx.x);
          to->reached[rank] = reached, to->last[rank] = last;
        }
        cl.sync();
        // The first bin where the border is reached; by weight, where the estimate misses it, the last.
#pragma unroll
        for (int i = 0; i < C; ++i) {
          if (at.bin < 0 && sm.reached[i].bin >= 0) at = sm.reached[i];
        }
        if (at.bin < 0 && !counting)
#pragma unroll
          for (int i = 0; i < C; ++i)
            if (sm.last[i].bin >= 0) at = sm.last[i];
        if (at.bin < 0) {
          if (!bins.lo) {  // the border lies below the counted bins
            whole_interval();
            bins.whole_row(top_key);
            counted = false;
            continue;
          }
          if (!counting) break;  // not reached: the weights add up to the total
          by_k = counting = false;  // fewer tokens than top_k
          whole_interval();
          if (!by_p) break;
          continue;
        }
        // The window: the border's bin, by weight the next one too, and all above where they are few.
        gather = at.pop <= kList;
        b1 = counting || !gather || alone || at.bin == kBins - 1 ? at.bin : at.bin + 1;
        b0 = gather && at.over - n_above + 2 * at.pop <= kList ? 0 : at.bin;
        outside = b0 ? at.over : n_above;
      }
      __syncthreads();
      const bool need = outside && (by_p || gather);  // the weight of those above it
      // Few enough to queue up. Measured (never / by the rule / always), 256 rows of 131071 f32: top_k 1000 211 / 171 / 162 us;
      // top_p 0.9 over logits of spread 4 253 / 222 / 218, of spread 2 270 / 273 / 308, of spread 1 408 / 411 / 672.
      const bool few = outside < (unsigned)p.vocab / 16;
      if (lane == 0) sm.waiting[warp] = 0;
      __syncwarp();
      s = Sums{0, 0, 0}, add_up = 0;
      u64 in_window = 0;
      auto note = [&](float f) {  // a token above the window
        const u64 x = wt.whole(f);
        add_up += x;
        if (passes(f)) s.w += x, ++s.n;
      };
      auto take = [&](float f, int i) {  // one in the window
        const uint32_t k = key_of(f);
        if (gather) {
          const unsigned place = atomicAdd(&sm.gathered.n, 1u);
          if (place < kList) sm.list[place] = (u64)k << 32 | (0xffffffffu - (unsigned)i);
        } else {
          atomicMin(&sm.gathered.key_min, k), atomicMax(&sm.gathered.key_max, k);
          if (!counting) in_window += wt.whole(f);
        }
      };
      if (bins.lo) {
        rd.each(v0, v1, [&](float f, int i) {
          const uint32_t k = key_of(f);
          if (k < bins.lo) return;
          const int b = k > bins.hi ? -1 : bins.of_key(k);
          if (b > b1) return;
          if (b >= b0) take(f, i);
          else if (need) note(f);
        });
      } else {
        // place() of a token, or its negative for the bound: above the window below `a`, in it up to `z`.
        const float g_top = quick ? 0.0f : wt.top, g_scale = quick ? 1.0f : bins.scale, g_bias = quick ? 0.0f : 8388608.0f;
        const float a = quick ? -INFINITY : g_bias + (float)b0, z = quick ? -logit_of(bound) : g_bias + (float)b1;
        rd.batches(v0, v1, [&](const float(&f)[16], int v) {
          auto at = [&](int k) { return fmaf(g_top - f[k], g_scale, g_bias); };
          float least = INFINITY;
#pragma unroll
          for (int k = 0; k < 16; ++k) least = fminf(least, at(k));
          if (!__any_sync(0xffffffffu, least <= z)) return;
          unsigned up = 0, in = 0;  // of the 16: those above the window, those in it
          bool doubt = false;       // whether one of those above passes min_p takes its weight to tell
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float x = at(k);
            const bool over = need && x < a;
            up |= over ? 1u << k : 0u;
            in |= x <= z && !(x < a) ? 1u << k : 0u;
            doubt |= over && f[k] >= far && !(f[k] >= sure);
          }
          // The rare tokens are read again, one at a time: a branch for each of the 16 is code that the first warps wait for.
          auto next = [&](unsigned &set) {
            const int k = __ffs(set) - 1;
            set &= set - 1;
            return rd.index(v + 32 * (k / Reader<DT>::VE)) + k % Reader<DT>::VE;
          };
          if (need && few) {  // they queue up for exponentials of 32 at once
            while (up) sm.queue[warp][atomicAdd(&sm.waiting[warp], 1u)] = rd.one(next(up));
            __syncwarp();
            unsigned n = sm.waiting[warp];
            if (n >= 32) {
              for (; n >= 32; n -= 32) note(sm.queue[warp][n - 32 + lane]);
              __syncwarp();
              if (lane == 0) sm.waiting[warp] = n;
              __syncwarp();
            }
          } else if (need && wt.plain && !doubt) {
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              // without a branch, so that the exponentials overlap
              const unsigned over = up >> k & 1, pass = over & (unsigned)(f[k] >= sure);
              const u64 w = wt.whole_any(f[k]);
              add_up += w & (0 - (u64)over);
              s.w += w & (0 - (u64)pass), s.n += pass;
            }
          } else {
            while (up) note(rd.one(next(up)));
          }
          while (in) {
            const int i = next(in);
            take(rd.one(i), i);
          }
        });
      }
      if (lane < (int)sm.waiting[warp]) note(sm.queue[warp][lane]);
      u64 sum_in = 0;
      sum = 0;
      if (need) block_incl(add_up, sm.scratch, &sum);
      if (!gather && !counting) block_incl(in_window, sm.scratch, &sum_in);
      __syncthreads();
      if (threadIdx.x == 0) sm.gathered.above = sum, sm.gathered.in = sum_in;
      cl.sync();
      Gathered got{0, 0, 0, 0xffffffffu, 0};
      if (lane < C) got = *cl.map_shared_rank(&sm.gathered, lane);
      const unsigned listed = warp_incl(got.n);  // in CTAs 0..lane
      const unsigned m = __shfl_sync(0xffffffffu, listed, 31);
      const u64 above = __shfl_sync(0xffffffffu, warp_incl(got.above), 31);
      const u64 in = __shfl_sync(0xffffffffu, warp_incl(got.in), 31);
      const uint32_t kmin = __reduce_min_sync(0xffffffffu, got.key_min), kmax = __reduce_max_sync(0xffffffffu, got.key_max);
      // The estimate missed the border: look on above or below the window, by what the exact weights say.
      auto move = [&](bool up) {
        if (up) b_max = at.bin - 1;
        else b_min = b1 + 1;
        if (above > base && at.e > 0.0f) factor = at.e / (float)(above - base);
      };
      if (!gather) {
        if (!counting && (want <= above || want > above + in)) {
          move(want <= above);
          cl.sync();
          continue;
        }
        if (kmin < kmax) {  // cut the bin again by its keys
          bins.lo = kmin, bins.hi = kmax, bins.shift = 0, counted = false;
          while (((kmax - kmin) >> bins.shift) >= kBins) ++bins.shift;
          n_above = outside, base = above, factor = 0.0f, b_min = 0, b_max = kBins - 1;
          cl.sync();
          continue;
        }
        // More equal logits than the list holds.
        const u64 each = wt.whole(logit_of(kmin));
        key = kmin, ties = at.pop, found = true;
        if (counting) {
          ties = (unsigned)top_k - outside;
          if (by_p) total = above + ties * each, want = want_of(total);
        }
        if (counting && by_p && want <= above) {  // top-p's border lies above top-k's
          found = false, counting = false, known = true;
          whole_interval();
        } else if (by_p && each) {
          ties = (unsigned)min((u64)ties, (want - above + each - 1) / each);
        }
        cl.sync();
        continue;
      }
      // The first CTA finds the border among the gathered tokens.
      if (rank == 0) {
        for (int i = warp; i < C; i += kWarps) {
          const int end = (int)__shfl_sync(0xffffffffu, listed, i), size = (int)__shfl_sync(0xffffffffu, got.n, i);
          const u64 *from = cl.map_shared_rank(sm.list, i);
          for (int j = lane; j < size; j += 32)
            if (end - size + j < kList) sm.all[end - size + j] = from[j];
        }
        const int lim = counting ? min((int)m, (int)((unsigned)top_k - outside)) : (int)m;
        Verdict v{0, 0, 0, 0};
        if (m <= kList) {
          // A thread per token, its rank and the weight before it by comparison with every other.
          u64 *const q = sm.q;
          u64 me = 0, w = 0;
          __syncthreads();
          if (threadIdx.x < m) {
            me = sm.all[threadIdx.x];
            w = wt.whole(logit_of((uint32_t)(me >> 32)));
            q[threadIdx.x] = w;
          }
          __syncthreads();
          int rank_of = 0;
          u64 before = above;
          for (int j = 0; j < (int)m; ++j)
            if (sm.all[j] > me) ++rank_of, before += q[j];
          const bool in_k = threadIdx.x < m && rank_of < lim;
          block_incl(in_k ? w : 0, sm.scratch, &sum);
          if (counting && by_p) total = above + sum, want = want_of(total);
          v.total = total;
          v.next = !by_p ? 0 : want <= above ? (counting ? 3 : 1) : want > above + sum ? 2 : 0;
          bool kept = in_k && (!by_p || before < want);
          if (outside == 0 && v.next == 0) {
            // 4. The kept set is among the gathered tokens: the draw in the order of the indices.
            const float f = logit_of((uint32_t)(me >> 32));
            kept = kept && passes(f);
            if (threadIdx.x < m && !kept) q[threadIdx.x] = 0;
            const int n_kept = __syncthreads_count(kept);
            u64 upto = 0;
            sum = 0;
            for (int j = 0; j < (int)m; ++j) {
              const u64 x = q[j];
              sum += x;
              if ((uint32_t)sm.all[j] > (uint32_t)me) upto += x;  // a lower index
            }
            const u64 d = draw_of(sum);
            if (kept && upto <= d && d < upto + w) {
              p.token[row] = (int32_t)(0xffffffffu - (uint32_t)me);
              if (p.prob) p.prob[row] = (float)(wt.weight(f) / ((double)sum * wt.unit));
            }
            if (threadIdx.x == 0 && p.kept) p.kept[row] = n_kept;
          } else if (v.next == 0) {
            const int n_kept = __syncthreads_count(kept);
            if (kept && rank_of == n_kept - 1) sm.key_min = (uint32_t)(me >> 32);
            __syncthreads();
            v.key = sm.key_min;
            v.ties = (unsigned)__syncthreads_count(kept && (uint32_t)(me >> 32) == v.key);
          }
        }
        if (threadIdx.x == 0) sm.verdict = v;
      }
      cl.sync();
      if (m > kList) {  // more than expected: by a histogram, or without the next bin
        if (!quick) alone = true;
        quick = false;
        continue;
      }
      const Verdict v = *cl.map_shared_rank(&sm.verdict, 0);
      cl.sync();
      quick = false;
      if (v.next == 0 && outside == 0) return;  // the first CTA has drawn
      if (v.next == 0) {
        key = v.key, ties = v.ties, found = summed = true;
      } else if (v.next == 3) {  // top-p's border lies above top-k's
        counting = false, known = true, total = v.total, want = want_of(total);
        whole_interval();
      } else {
        move(v.next == 1);
      }
    }
  }

  // 4. Every warp's kept weight, and the one that the draw falls into.
  const float at_key = key ? logit_of(key) : __int_as_float(0x7fffffff);  // none: NaN
  const float low = fmaxf(fmaxf(key ? at_key : -INFINITY, far), -3.402823466e38f);  // tokens below are not kept
  {
    auto add = [&](float f) {
      double a, b;
      wt.parts(f, a, b);
      if (min_p > 0.0f && f != wt.top && a * b * wt.unit < (double)min_p) return;
      s.w += (u64)__double_as_longlong(fma(a, b, 4503599627370496.0)) - kMagicBits;
      ++s.n;
    };
    if (!summed) s = Sums{0, 0, 0};
    if (summed) {
      // The tokens above the window are in the sums; the kept ones in it follow below.
    } else if (!key && !(min_p > 0.0f) && wt.plain) {  // the whole row
      rd.each(v0, v1, [&](float f, int) {
        s.w += wt.whole_any(f);
        s.n += f > -INFINITY;
      });
    } else {
      rd.each(v0, v1, [&](float f, int) {
        if (!(f >= low)) return;
        if (f == at_key) ++s.ties;
        else add(f);
      });
    }
#pragma unroll
    for (int m = 16; m; m >>= 1) {
      s.w += __shfl_xor_sync(0xffffffffu, s.w, m);
      s.n += __shfl_xor_sync(0xffffffffu, s.n, m);
      s.ties += __shfl_xor_sync(0xffffffffu, s.ties, m);
    }
    if (lane == 0) sm.sums[warp] = s;
  }
  if (summed) {
    __syncthreads();
    for (unsigned j = threadIdx.x; j < sm.gathered.n; j += kThreads) {
      const u64 x = sm.list[j];
      const float f = logit_of((uint32_t)(x >> 32));
      if (!(f >= low)) continue;
      Sums &to = sm.sums[(((int)(0xffffffffu - (uint32_t)x) + rd.mis) / Reader<DT>::VE - rank * per_cta) / per_warp];
      if (f == at_key) atomicAdd(&to.ties, 1u);
      else if (passes(f)) atomicAdd(&to.w, wt.whole(f)), atomicAdd(&to.n, 1u);
    }
  }
  cl.sync();
  for (int i = threadIdx.x; i < C * kWarps; i += kThreads) sm.every[i] = cl.map_shared_rank(sm.sums, i / kWarps)[i % kWarps];
  __syncthreads();
  const u64 tie_w = key ? wt.whole(logit_of(key)) : 0;
  if (key && !passes(at_key)) ties = 0;
  // Every warp walks the stretches, lane by lane of 32, and finds the one that the draw falls into.
  constexpr int kRounds = (C * kWarps + 31) / 32;
  u64 total = 0, from[kRounds], own[kRounds];
  unsigned kept = 0, tie_at = 0, ties_from[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    Sums s{0, 0, 0};
    if (32 * i + lane < C * kWarps) s = sm.every[32 * i + lane];
    const unsigned tie_incl = tie_at + warp_incl(s.ties);
    ties_from[i] = tie_incl - s.ties;
    const unsigned take = min(ties, tie_incl) - min(ties, ties_from[i]);
    own[i] = s.w + take * tie_w;
    const u64 incl = total + warp_incl(own[i]);
    from[i] = incl - own[i];
    const unsigned n = warp_incl(s.n + take);
    total = __shfl_sync(0xffffffffu, incl, 31);
    kept += __shfl_sync(0xffffffffu, n, 31);
    tie_at = __shfl_sync(0xffffffffu, tie_incl, 31);
  }
  if (rank == 0 && threadIdx.x == 0 && p.kept) p.kept[row] = (int32_t)kept;
  const u64 d = draw_of(total);
  int stretch = 0;
  u64 before = 0;
  unsigned tie_before = 0;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const unsigned hit = __ballot_sync(0xffffffffu, from[i] <= d && d < from[i] + own[i]);
    if (!hit) continue;
    stretch = 32 * i + __ffs(hit) - 1;
    before = __shfl_sync(0xffffffffu, from[i], __ffs(hit) - 1);
    tie_before = __shfl_sync(0xffffffffu, ties_from[i], __ffs(hit) - 1);
  }
  if (stretch / kWarps == rank) {
    // The block takes the stretch in pieces, one per thread, then the warp of the piece with the draw takes that, one
    // token per lane. (One warp alone on the stretch waited for its exponentials longer than the rest of the row's work
    // took: 57 000 of 97 000 cycles at 131071 tokens.)
    auto weight_of = [&](float f) -> u64 {  // of a token that is not a tie
      if (!(f >= low) || !(f >= sure || passes(f))) return 0;
      return wt.whole(f);
    };
    const int s0 = min(c1, rank * per_cta + stretch % kWarps * per_warp), s1 = min(c1, s0 + per_warp);
    const int piece = (s1 - s0 + kThreads - 1) / kThreads;
    const int p0 = min(s1, s0 + (int)threadIdx.x * piece), p1 = min(s1, p0 + piece);
    u64 w = 0, all;
    unsigned eq = 0, all_eq;
    for (int v = p0; v < p1; ++v) {
      constexpr int VE = Reader<DT>::VE;
      float f[VE];
      rd.load(v, f);
      if (wt.plain) {
#pragma unroll
        for (int k = 0; k < VE; ++k) {
          const u64 x = wt.whole_any(f[k]);
          if (f[k] == at_key) ++eq;
          else if (f[k] >= low && (f[k] >= sure || passes(f[k]))) w += x;
        }
      } else {
#pragma unroll
        for (int k = 0; k < VE; ++k) {
          if (f[k] == at_key) ++eq;
          else w += weight_of(f[k]);
        }
      }
    }
    unsigned tie = tie_before + block_incl(eq, sm.warp_n, &all_eq) - eq;
    u64 at = before + block_incl(w, sm.scratch, &all) - w + (min(ties, tie) - min(ties, tie_before)) * tie_w;
    w += (min(ties, tie + eq) - min(ties, tie)) * tie_w;
    const unsigned hit = __ballot_sync(0xffffffffu, at <= d && d < at + w);
    if (hit) {
      const int owner = __ffs(hit) - 1;
      at = __shfl_sync(0xffffffffu, at, owner), tie = __shfl_sync(0xffffffffu, tie, owner);
      const int end = min(p.vocab, rd.index(__shfl_sync(0xffffffffu, p1, owner)));
      for (int i = max(0, rd.index(__shfl_sync(0xffffffffu, p0, owner))); i < end; i += 32) {
        const float f = i + lane < end ? rd.one(i + lane) : -INFINITY;
        const unsigned ties_in = __ballot_sync(0xffffffffu, f == at_key);
        u64 q = 0;
        if (f == at_key) q = tie + __popc(ties_in & ((1u << lane) - 1)) < ties ? tie_w : 0;
        else q = weight_of(f);
        const u64 incl = at + warp_incl(q);
        if (incl - q <= d && d < incl) {
          p.token[row] = i + lane;
          if (p.prob) p.prob[row] = (float)(wt.weight(f) / ((double)total * wt.unit));
        }
        at = __shfl_sync(0xffffffffu, incl, 31);
        if (at > d) break;
        tie += __popc(ties_in);
      }
    }
  }
  cl.sync();
}

template <int DT, int C>
int launch_cluster(mpc_device *dev, const SampleParams &p, int rows, cudaStream_t st) {
  static bool configured[64] = {};
  const int ord = dev->ordinal & 63;
  if (!configured[ord]) {
    MPC_CUDA(dev, cudaFuncSetAttribute(sample_kernel<DT, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared)));
    configured[ord] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)rows * C), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = sizeof(Shared), cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C, at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  MPC_CUDA(dev, cudaLaunchKernelEx(&cfg, sample_kernel<DT, C>, p));
  dev->launches++;
  return MPC_OK;
}

// CTAs per row: up to 4 an SM and at least 1024 tokens each. More than the two that an SM holds, so that the rows under
// way at a time stay in L2 for the later passes: 256 rows of 131071 f32 with mixed settings at 2, 4 and 8 CTAs a row 186,
// 175 and 173 us, 4 rows of 50257 bf16 19.1, 15.2 and 14.7 us. Measured with bounds of 1, 4 and 16 an SM, top_p 0.9 and
// top_k 50 alone: 300 x 131071 389, 305, 404 and 118, 101, 189 us; 300 x 50257 173, 163, 274 and 51, 57, 153 us. At 64 to
// 148 rows the bound of 1 is ahead where all rows have the same setting: 148 x 50257 64, 142, 142 and 24, 80, 80 us; 64 x
// 131071 67, 88, 87 and 25, 41, 41 us.
template <int DT>
int launch_sample(mpc_device *dev, const SampleParams &p, int rows, cudaStream_t st) {
  int c = 1;
  while (c < kMaxCluster && (long long)rows * c <= 4ll * dev->prop.multiProcessorCount && p.vocab >= 2 * c * 1024) c *= 2;
  if (c == 8) return launch_cluster<DT, 8>(dev, p, rows, st);
  if (c == 4) return launch_cluster<DT, 4>(dev, p, rows, st);
  if (c == 2) return launch_cluster<DT, 2>(dev, p, rows, st);
  return launch_cluster<DT, 1>(dev, p, rows, st);
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
  if (d->rows > INT32_MAX || d->vocab > (1 << 20))
    return fail(MPC_ERR_UNSUPPORTED, "mpc_sample: more than 2^31 - 1 rows or 2^20 tokens");
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
