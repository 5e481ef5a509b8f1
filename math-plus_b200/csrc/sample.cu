// Sampling (mpc_sample): one token per row of logits by temperature, top-k, top-p and min-p from one
// uniform number. It stands beside softmax, sort and argmax of the op set; the reference has no
// sampler.
//
// All three filters keep a prefix of the tokens ranked by (logit descending, index ascending), so the
// kept set is "every token above a threshold logit, and the first r tokens equal to it". Logits map to
// 32-bit keys of the same order, and the threshold is found by radix selection: histograms of counts
// and weights over 8 key bits at a time, from the top. No sort.
//
// Weights w = exp((l - max) / T) in f64 are held as integers of 2^-shift (shift = 62 - log2 of the row's
// length), so that sums are exact whatever their order: the same row always gives the same token, and
// the borders of top-p and of the drawn interval move by less than 1e-12 of the total.
//
// One CTA of 1024 threads per row; the row is read again by each pass, from L2.
#include "kv_cache.cuh"
#include "mpc_internal.h"

namespace mpc {
namespace {

constexpr int kThreads = 1024;

struct SampleParams {
  const void *logits;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t *top_k;
  int32_t *token, *kept;
  float *prob;
  long long stride;
  int vocab, dt, d_top_k, shift;
  float d_temperature, d_top_p, d_min_p;
};

// Keys of the logits' order; NaN and -inf share the lowest, 0 (they are never kept).
__device__ __forceinline__ uint32_t key_of(float f) {
  const uint32_t b = __float_as_uint(f == 0.0f ? 0.0f : f);  // -0 ties with 0
  return !(f > -INFINITY) ? 0u : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

struct Row {
  const void *x;
  int dt;
  float top;     // the largest logit
  double inv_t;
  int shift;
  __device__ float logit(int i) const { return load_f32(x, dt, i); }
  __device__ double weight(float f) const {
    if (f == top) return 1.0;
    const double d = ((double)f - (double)top) * inv_t;
    return f > -INFINITY && d > -800.0 ? exp(d) : 0.0;
  }
  __device__ unsigned long long whole(double w) const { return (unsigned long long)__double2ll_rn(ldexp(w, shift)); }
};

template <typename T>
__device__ T block_sum(T v, T *sm) {
#pragma unroll
  for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  T all = 0;
  for (int i = 0; i < kThreads / 32; ++i) all += sm[i];
  return all;
}

// Exclusive prefix sum over the threads.
template <typename T>
__device__ T block_before(T v, T *sm) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  T incl = v;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const T u = __shfl_up_sync(0xffffffffu, incl, m);
    if (lane >= m) incl += u;
  }
  __syncthreads();
  if (lane == 31) sm[w] = incl;
  __syncthreads();
  T before = 0;
  for (int i = 0; i < w; ++i) before += sm[i];
  return before + incl - v;
}

struct Shared {
  unsigned long long w[256], sum[32];
  unsigned n[256], cnt[32];
  unsigned long long w_above;
  unsigned n_above, prefix, n_at;
};

// The key at which the ranked tokens' running count (or, with BY_WEIGHT, weight) reaches `want`:
// sm.prefix, with sm.n_above tokens of weight sm.w_above above it and sm.n_at equal to it.
template <bool BY_WEIGHT>
__device__ void select(const Row &r, int vocab, unsigned long long want, Shared &sm) {
  if (threadIdx.x == 0) sm.prefix = 0, sm.n_above = 0, sm.w_above = 0;
  for (int bits = 24; bits >= 0; bits -= 8) {
    for (int i = threadIdx.x; i < 256; i += kThreads) sm.n[i] = 0, sm.w[i] = 0;
    __syncthreads();
    const uint32_t prefix = sm.prefix;
    for (int i = threadIdx.x; i < vocab; i += kThreads) {
      const float f = r.logit(i);
      const uint32_t k = key_of(f);
      if (k == 0 || (bits < 24 && (k >> (bits + 8)) != prefix)) continue;
      atomicAdd(&sm.n[(k >> bits) & 255], 1u);
      atomicAdd(&sm.w[(k >> bits) & 255], r.whole(r.weight(f)));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      unsigned n = sm.n_above;
      unsigned long long w = sm.w_above;
      int last = 0;
      for (int i = 255; i >= 0; --i) {
        if (!sm.n[i]) continue;
        last = i;
        if (BY_WEIGHT ? w + sm.w[i] >= want : n + sm.n[i] >= want) break;
        n += sm.n[i], w += sm.w[i];
      }
      if (BY_WEIGHT ? w + sm.w[last] < want : n + sm.n[last] < want) n -= sm.n[last], w -= sm.w[last];  // all of them
      sm.n_above = n, sm.w_above = w, sm.prefix = prefix << 8 | last, sm.n_at = sm.n[last];
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleParams p) {
  __shared__ Shared sm;
  const int row = blockIdx.x, V = p.vocab;
  Row r;
  r.dt = p.dt;
  r.x = static_cast<const uint8_t *>(p.logits) + (long long)row * p.stride * (p.dt == MPC_F32 ? 4 : 2);
  r.shift = p.shift;
  const float t = p.temperature ? p.temperature[row] : p.d_temperature;
  const float top_p = p.top_p ? p.top_p[row] : p.d_top_p;
  const float min_p = p.min_p ? p.min_p[row] : p.d_min_p;
  const int top_k = p.top_k ? p.top_k[row] : p.d_top_k;

  // The largest logit and its lowest index, as the pair (key, ~index).
  unsigned long long best = 0;
  for (int i = threadIdx.x; i < V; i += kThreads) {
    const unsigned long long c = (unsigned long long)key_of(r.logit(i)) << 32 | (0xffffffffu - (unsigned)i);
    best = c > best ? c : best;
  }
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    const unsigned long long o = __shfl_xor_sync(0xffffffffu, best, m);
    best = o > best ? o : best;
  }
  if ((threadIdx.x & 31) == 0) sm.sum[threadIdx.x >> 5] = best;
  __syncthreads();
  for (int i = 0; i < kThreads / 32; ++i) best = sm.sum[i] > best ? sm.sum[i] : best;
  const uint32_t top_key = (uint32_t)(best >> 32);
  const int top_at = (int)(0xffffffffu - (uint32_t)best);
  if (top_key == 0 || !(t > 0.0f)) {
    if (threadIdx.x == 0) {
      p.token[row] = top_key ? top_at : -1;
      if (p.prob) p.prob[row] = top_key ? 1.0f : 0.0f;
      if (p.kept) p.kept[row] = top_key ? 1 : 0;
    }
    return;
  }
  r.top = r.logit(top_at);
  r.inv_t = 1.0 / (double)t;
  __syncthreads();

  // Kept: keys above `key`, and the first `ties` tokens of that key.
  uint32_t key = 0;
  unsigned ties = 0;
  unsigned long long total = 0;
  const bool by_k = top_k > 0 && top_k < V, by_p = top_p < 1.0f;
  if (by_k) {
    select<false>(r, V, (unsigned long long)top_k, sm);
    key = sm.prefix;
    ties = min(sm.n_at, (unsigned)top_k - sm.n_above);
    const uint32_t b = (key & 0x80000000u) ? (key & 0x7fffffffu) : ~key;
    total = sm.w_above + ties * r.whole(r.weight(__uint_as_float(b)));
    __syncthreads();
  } else if (by_p) {
    unsigned long long w = 0;
    for (int i = threadIdx.x; i < V; i += kThreads) w += r.whole(r.weight(r.logit(i)));
    total = block_sum(w, sm.sum);
    __syncthreads();
  }
  if (by_p) {
    // The ranks before which less than top_p * total lies: those whose preceding weight is < want.
    const double lim = top_p > 0.0f ? (double)top_p * (double)total : 0.0;
    unsigned long long want = (unsigned long long)__double2ll_ru(lim);
    if (want < 1) want = 1;
    if (want > total) want = total;
    select<true>(r, V, want, sm);
    const uint32_t at = sm.prefix;
    const uint32_t b = (at & 0x80000000u) ? (at & 0x7fffffffu) : ~at;
    const unsigned long long w = r.whole(r.weight(__uint_as_float(b)));
    unsigned n = sm.n_at;
    if (w > 0) {
      const unsigned long long need = (want - sm.w_above + w - 1) / w;
      if (need < n) n = (unsigned)need;
    }
    if (at > key || (at == key && n < ties)) key = at, ties = n;
    __syncthreads();
  }

  // Thread i's tokens are [i c, (i + 1) c): the kept weight and number before them give the place of the draw.
  const int c = (V + kThreads - 1) / kThreads;
  const int i0 = min(V, (int)threadIdx.x * c), i1 = min(V, i0 + c);
  unsigned at_key = 0;
  if (key)
    for (int i = i0; i < i1; ++i) at_key += key_of(r.logit(i)) == key;
  unsigned tie = block_before(at_key, sm.cnt);
  const unsigned tie0 = tie;
  unsigned long long mine = 0;
  unsigned count = 0;
  auto keeps = [&](float f, double w) {
    const uint32_t k = key_of(f);
    if (k == 0 || k < key) return false;
    if (k == key && tie++ >= ties) return false;
    return k == top_key || !(w < (double)min_p);
  };
  for (int i = i0; i < i1; ++i) {
    const float f = r.logit(i);
    const double w = r.weight(f);
    if (keeps(f, w)) mine += r.whole(w), ++count;
  }
  __syncthreads();
  count = block_sum(count, sm.cnt);
  __syncthreads();
  total = block_sum(mine, sm.sum);
  __syncthreads();
  const unsigned long long before = block_before(mine, sm.sum);
  const float u = fminf(fmaxf(p.u[row], 0.0f), 1.0f);
  unsigned long long want = (unsigned long long)__double2ll_rd((double)u * (double)total);
  if (want >= total) want = total - 1;
  if (before <= want && want < before + mine) {
    tie = tie0;
    unsigned long long sum = before;
    for (int i = i0; i < i1; ++i) {
      const float f = r.logit(i);
      const double w = r.weight(f);
      if (!keeps(f, w)) continue;
      sum += r.whole(w);
      if (sum > want) {
        p.token[row] = i;
        if (p.prob) p.prob[row] = (float)(w / ldexp((double)total, -r.shift));
        break;
      }
    }
  }
  if (threadIdx.x == 0 && p.kept) p.kept[row] = (int32_t)count;
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
  p.token = token, p.kept = kept, p.prob = prob, p.stride = d->row_stride, p.vocab = (int)d->vocab, p.dt = d->dtype;
  p.d_top_k = d->top_k, p.d_temperature = d->temperature, p.d_top_p = d->top_p, p.d_min_p = d->min_p;
  int log2v = 0;
  while ((int64_t(1) << log2v) < d->vocab) ++log2v;
  p.shift = 62 - log2v;  // V weights of at most 2^shift stay below 2^63
  sample_kernel<<<(unsigned)d->rows, kThreads, 0, stream_of(dev, s)>>>(p);
  dev->launches++;
  return check_launch(dev, "mpc_sample");
}
