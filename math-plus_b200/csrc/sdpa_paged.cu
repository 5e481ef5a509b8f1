// Attention of one new token per sequence over the paged key/value cache (mpc_sdpa_paged): the serving
// form of mpc_sdpa (Backend.sdpa, packages/tensor-cpu/src/index.ts:821-840), Lq = 1.
//
// With s_j = scale * q.k_j for j < length: o = sum_j 2^(s'_j - m) v_j / sum_j 2^(s'_j - m), s' = s log2 e, m any
// upper reference of s' (the running maximum). Every K/V row is read once and used for the query
// heads that share it, so the cache's bytes bound the time and the work is split along the cache:
//
// Split. An item is (sequence, K/V head, tile of its query heads); its keys are cut into chunks of 64.
// The chunks of all items, in order, are dealt to the CTAs in equal runs: CTA i of n takes chunks
// [T i / n, T (i + 1) / n). Each CTA finds its run from the lengths on the device, so ragged batches and a
// single long sequence balance alike and the launch depends on host-known sizes alone (it can be
// captured into a graph). A run that covers an item wholly writes the output; otherwise the (at
// most two) cut items of a CTA leave (m, l, O) in the workspace and a second kernel joins them in
// CTA order, so the result does not depend on timing.
//
// CUDA-core kernel (f32 rows, and any head dim <= 256 or alignment): 8 lanes per key, 4 keys a warp, each
// group of 8 lanes with its own running maximum, sum and O; the 16 groups of a CTA meet once per item.
#include <cfloat>

#include "kv_cache.cuh"
#include "mpc_internal.h"

namespace mpc {
namespace paged {

constexpr int kChunk = 64;     // keys of one unit of the split
constexpr int kThreads = 128;  // 4 warps
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Params {
  const void *q, *kp, *vp;
  const uint8_t *ks, *vs;
  const int32_t *table, *lengths;
  void *out;
  float *lse, *ws;
  int *err;
  long long qs[2], os[2], max_pages, cap;  // cap: max_pages * page_size
  int B, H, hk, group, gt, qt;  // query heads per K/V head, per tile, tiles per K/V head
  int d, dv, page_size, n_pages, dt, dt_pages;
  float scale_log2;
};

// The run of chunks of one CTA, found from the lengths.
struct Run {
  long long total, g0, g1;  // all chunks; this CTA's [g0, g1)
  int n;                    // CTAs that have a run
};
struct Item {
  int b, head;        // head: K/V head * qt + query tile
  long long chunk, chunks;
};

__device__ __forceinline__ long long length_of(const Params &p, int b) {
  const long long len = p.lengths[b];
  return len < 0 ? 0 : len > p.cap ? p.cap : len;
}
__device__ __forceinline__ long long chunks_of(const Params &p, int b) {
  return (length_of(p, b) + kChunk - 1) / kChunk;
}

// Block-wide inclusive scan of one value a thread (kThreads threads); *sum: the block's total.
__device__ __forceinline__ long long scan(long long v, long long *sm, long long *sum) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, m);
    if (lane >= m) v += u;
  }
  __syncthreads();
  if (lane == 31) sm[w] = v;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) {
    if (i < w) before += sm[i];
    all += sm[i];
  }
  *sum = all;
  return v + before;
}

__device__ __forceinline__ Run run_of(const Params &p, int cta, int ctas, long long *sm) {
  long long total = 0;
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    long long sum;
    scan(b < p.B ? chunks_of(p, b) : 0, sm, &sum);
    total += sum;
  }
  Run r;
  r.total = total * (p.hk * p.qt);
  r.n = (int)(r.total < ctas ? r.total : ctas);
  if (cta >= r.n) {
    r.g0 = r.g1 = 0;
  } else {
    r.g0 = r.total * cta / r.n;
    r.g1 = r.total * (cta + 1) / r.n;
  }
  return r;
}

// The item of chunk g (0 <= g < total) and g's place in it.
__device__ __forceinline__ Item item_of(const Params &p, long long g, long long *sm, long long *found) {
  const long long heads = p.hk * p.qt;
  long long before = 0;
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    const long long c = b < p.B ? chunks_of(p, b) : 0;
    long long sum;
    const long long incl = before + scan(c, sm, &sum);
    if (g >= (incl - c) * heads && g < incl * heads) found[0] = b, found[1] = incl - c;
    before += sum;
  }
  __syncthreads();
  Item it;
  it.b = (int)found[0];
  const long long rem = g - found[1] * heads;
  it.chunks = chunks_of(p, it.b);
  it.head = (int)(rem / it.chunks);
  it.chunk = rem - it.head * it.chunks;
  return it;
}

// (m, l, O) of one query over part of an item, in the workspace: m, the exponent O refers to, l, one
// unused, then O.
__device__ __forceinline__ float *slot(const Params &p, int cta, bool first, int g) {
  return p.ws + ((long long)(2 * cta + (first ? 1 : 0)) * p.gt + g) * (p.dv + 4);
}

__device__ __forceinline__ float guard_exp2(float x, float ref) { return x == -INFINITY ? 0.0f : exp2f(x - ref); }

// Sequences without keys: zeros and -inf; lengths outside the table are recorded.
__device__ __forceinline__ void empty_rows(const Params &p) {
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    const long long len = p.lengths[b];
    if (threadIdx.x == 0 && (len < 0 || len > p.cap)) report_bad_page(p.err, kBadLength, b);
    if (len > 0 && p.cap > 0) continue;
    for (int i = threadIdx.x; i < p.H * p.dv; i += kThreads) {
      const int h = i / p.dv;
      store_f32(p.out, p.dt, b * p.os[0] + h * p.os[1] + (i - h * p.dv), 0.0f);
    }
    if (p.lse)
      for (int h = threadIdx.x; h < p.H; h += kThreads) p.lse[(long long)b * p.H + h] = -INFINITY;
  }
}

// ---- CUDA-core kernel ---------------------------------------------------------------------------
template <int NI, int GT, bool VEC>
__global__ void __launch_bounds__(kThreads) simt_kernel(const Params p) {
  constexpr int W = NI * 64;  // padded head dim: lane j of 8 holds values i * 64 + j * 8 ..+7
  __shared__ float sq[GT][W];
  __shared__ float so[kThreads / 32][GT][W];
  __shared__ float sml[kThreads / 32][GT][2];
  __shared__ long long sm[kThreads / 32], found[2];
  empty_rows(p);
  const Run run = run_of(p, blockIdx.x, gridDim.x, sm);
  if (run.g0 >= run.g1) return;
  Item it = item_of(p, run.g0, sm, found);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j8 = (lane & 7) * 8;
  for (long long g = run.g0; g < run.g1;) {
    const long long c1 = min(it.chunks, it.chunk + (run.g1 - g));
    const int kvh = it.head / p.qt, h0 = kvh * p.group + (it.head % p.qt) * GT;
    const int nq = min(GT, (kvh + 1) * p.group - h0);
    __syncthreads();  // the last item's shared arrays are free
    for (int i = threadIdx.x; i < GT * W; i += kThreads) {
      const int q = i / W, e = i % W;
      sq[q][e] = q < nq && e < p.d ? load_f32(p.q, p.dt, it.b * p.qs[0] + (h0 + q) * p.qs[1] + e) : 0.0f;
    }
    __syncthreads();
    float m[GT], l[GT], o[GT][NI * 8];
#pragma unroll
    for (int q = 0; q < GT; ++q) {
      m[q] = -INFINITY, l[q] = 0.0f;
#pragma unroll
      for (int e = 0; e < NI * 8; ++e) o[q][e] = 0.0f;
    }
    const long long end = min(length_of(p, it.b), c1 * kChunk);
    for (long long k0 = it.chunk * kChunk; k0 < end; k0 += kThreads / 8) {
      const long long key = k0 + (threadIdx.x >> 3);
      long long row = -1;
      if (key < end) {
        const long long col = key / p.page_size;
        const int pg = p.table[it.b * p.max_pages + col];
        if (pg >= 0 && pg < p.n_pages) row = ((long long)pg * p.hk + kvh) * p.page_size + (key - col * p.page_size);
        else if ((lane & 7) == 0) report_bad_page(p.err, kBadAttend, it.b);
      }
      float s[GT], x[8];
#pragma unroll
      for (int q = 0; q < GT; ++q) s[q] = 0.0f;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int at = i * 64 + j8;
        if (row >= 0 && at < p.d) {
          load8<VEC>(p.kp, p.dt_pages, row * p.d + at, p.d - at, x);
#pragma unroll
          for (int q = 0; q < GT; ++q)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[q] = fmaf(sq[q][at + e], x[e], s[q]);
        }
      }
#pragma unroll
      for (int q = 0; q < GT; ++q)
#pragma unroll
        for (int k = 4; k; k >>= 1) s[q] += __shfl_xor_sync(0xffffffffu, s[q], k);
      if (row < 0) continue;
      const float f = p.scale_log2 * (p.dt_pages == MPC_E4M3 ? scale_value(p.ks[row]) : 1.0f);
#pragma unroll
      for (int q = 0; q < GT; ++q) {
        s[q] *= f;
        const float top = fmaxf(m[q], s[q]);
        const float keep = guard_exp2(m[q], top);
        s[q] = guard_exp2(s[q], top);
        m[q] = top;
        l[q] = fmaf(l[q], keep, s[q]);
#pragma unroll
        for (int e = 0; e < NI * 8; ++e) o[q][e] *= keep;
      }
      const float fv = p.dt_pages == MPC_E4M3 ? scale_value(p.vs[row]) : 1.0f;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int at = i * 64 + j8;
        if (at < p.dv) {
          load8<VEC>(p.vp, p.dt_pages, row * p.dv + at, p.dv - at, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float v = x[e] * fv;
#pragma unroll
            for (int q = 0; q < GT; ++q) o[q][i * 8 + e] = fmaf(s[q], v, o[q][i * 8 + e]);
          }
        }
      }
    }
    // The 4 groups of a warp meet by shuffles, the warps in shared memory.
#pragma unroll
    for (int q = 0; q < GT; ++q) {
      float top = m[q];
#pragma unroll
      for (int k = 8; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
      const float keep = guard_exp2(m[q], top);
      l[q] *= keep;
#pragma unroll
      for (int k = 8; k < 32; k <<= 1) l[q] += __shfl_xor_sync(0xffffffffu, l[q], k);
#pragma unroll
      for (int e = 0; e < NI * 8; ++e) {
        float v = o[q][e] * keep;
#pragma unroll
        for (int k = 8; k < 32; k <<= 1) v += __shfl_xor_sync(0xffffffffu, v, k);
        if (lane < 8) so[warp][q][(e >> 3) * 64 + j8 + (e & 7)] = v;
      }
      if (lane == 0) sml[warp][q][0] = top, sml[warp][q][1] = l[q];
    }
    __syncthreads();
    const bool whole = it.chunk == 0 && c1 == it.chunks;
    for (int i = threadIdx.x; i < nq * W; i += kThreads) {
      const int q = i / W, e = i % W;
      float top = -INFINITY, sum = 0.0f, v = 0.0f;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) top = fmaxf(top, sml[w][q][0]);
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
        const float keep = guard_exp2(sml[w][q][0], top);
        sum = fmaf(sml[w][q][1], keep, sum);
        v = fmaf(so[w][q][e], keep, v);
      }
      if (whole) {
        if (e < p.dv)
          store_f32(p.out, p.dt, it.b * p.os[0] + (h0 + q) * p.os[1] + e, sum != 0.0f ? v / sum : 0.0f);
        if (p.lse && e == 0) p.lse[(long long)it.b * p.H + h0 + q] = sum != 0.0f ? fmaf(top, kLn2, logf(sum)) : -INFINITY;
      } else {
        float *ws = slot(p, blockIdx.x, it.chunk == 0, q);
        if (e < p.dv) ws[4 + e] = v;
        if (e == 0) ws[0] = ws[1] = top, ws[2] = sum;
      }
    }
    g += c1 - it.chunk;
    it.chunk = 0;
    if (++it.head == p.hk * p.qt) {
      it.head = 0;
      if (g < run.g1)
        do it.chunks = chunks_of(p, ++it.b);
        while (it.chunks == 0);
    }
  }
}

// ---- join -----------------------------------------------------------------------------------------
// Block (i, q) joins the item that starts in CTA i and ends in a later one, query q of its tile.
__global__ void __launch_bounds__(kThreads) join_kernel(const Params p, int ctas) {
  __shared__ long long sm[kThreads / 32], found[2];
  const int cta = blockIdx.x, q = blockIdx.y;
  const Run run = run_of(p, cta, ctas, sm);
  if (run.g0 >= run.g1) return;
  const Item it = item_of(p, run.g1 - 1, sm, found);
  const long long start = run.g1 - 1 - it.chunk, end = start + it.chunks;
  if (start < run.g0 || end <= run.g1) return;
  const int kvh = it.head / p.qt, h = kvh * p.group + (it.head % p.qt) * p.gt + q;
  if (h >= (kvh + 1) * p.group) return;
  const int last = (int)((end * run.n - 1) / run.total);  // the CTA of chunk end - 1
  float top = -INFINITY, otop = -INFINITY, sum = 0.0f;
  for (int c = cta; c <= last; ++c) {
    const float *ws = slot(p, c, c == cta, q);
    top = fmaxf(top, ws[0]);
    otop = fmaxf(otop, ws[1]);
  }
  for (int c = cta; c <= last; ++c) {
    const float *ws = slot(p, c, c == cta, q);
    sum = fmaf(ws[2], guard_exp2(ws[0], top), sum);
  }
  for (int e = threadIdx.x; e < p.dv; e += kThreads) {
    float v = 0.0f;
    for (int c = cta; c <= last; ++c) {
      const float *ws = slot(p, c, c == cta, q);
      v = fmaf(ws[4 + e], guard_exp2(ws[1], otop), v);
    }
    v = sum != 0.0f ? v * exp2f(otop - top) / sum : 0.0f;
    store_f32(p.out, p.dt, it.b * p.os[0] + h * p.os[1] + e, v);
  }
  if (p.lse && threadIdx.x == 0)
    p.lse[(long long)it.b * p.H + h] = sum != 0.0f ? fmaf(top, kLn2, logf(sum)) : -INFINITY;
}

// ---- host -------------------------------------------------------------------------------------------
struct Plan {
  int gt, qt, ctas;
  size_t ws_bytes;
};

static int plan_of(mpc_device *dev, const mpc_kv_desc *c, const mpc_sdpa_paged_desc *d, Plan *pl) {
  int rc = kv_check("mpc_sdpa_paged", c);
  if (rc) return rc;
  if (d->b < 0 || d->h <= 0 || d->max_pages < 0 || d->max_pages > INT32_MAX)
    return fail(MPC_ERR_INVALID, "mpc_sdpa_paged: bad extents b=%lld h=%lld max_pages=%lld", (long long)d->b,
                (long long)d->h, (long long)d->max_pages);
  if (d->h % c->hk)
    return fail(MPC_ERR_INVALID, "mpc_sdpa_paged: h=%lld is not a multiple of hk=%lld", (long long)d->h,
                (long long)c->hk);
  if (d->b > INT32_MAX || d->h > (1 << 20))
    return fail(MPC_ERR_UNSUPPORTED, "mpc_sdpa_paged: more than 2^31 - 1 sequences or 2^20 heads");
  if (d->dtype < MPC_F32 || d->dtype > MPC_BF16 || (c->dtype != MPC_E4M3 && c->dtype != d->dtype))
    return fail(MPC_ERR_INVALID, "mpc_sdpa_paged: queries of dtype %d over a cache of dtype %d", d->dtype, c->dtype);
  for (int64_t s : {d->q_stride[0], d->q_stride[1], d->o_stride[0], d->o_stride[1]})
    if (s < 0) return fail(MPC_ERR_INVALID, "mpc_sdpa_paged: negative stride");
  const int64_t group = d->h / c->hk;
  pl->gt = group >= 4 ? 4 : group >= 2 ? 2 : 1;
  pl->qt = (int)((group + pl->gt - 1) / pl->gt);
  // As many CTAs as are resident, fewer where even the longest lengths give fewer chunks.
  const long long per = (d->max_pages * c->page_size + kChunk - 1) / kChunk;
  const long long sms = (long long)dev->prop.multiProcessorCount * 3;
  const long long heads = c->hk * pl->qt;
  long long ctas = sms;
  if (d->b > 0 && per > 0 && per <= sms / heads / d->b) ctas = per * heads * d->b;
  pl->ctas = (int)(ctas < 1 ? 1 : ctas);
  pl->ws_bytes = (size_t)pl->ctas * 2 * pl->gt * (c->dv + 4) * sizeof(float);
  return MPC_OK;
}

template <int NI, bool VEC>
static void launch_simt(const Params &p, int ctas, cudaStream_t st) {
  if (p.gt == 4) simt_kernel<NI, 4, VEC><<<ctas, kThreads, 0, st>>>(p);
  else if (p.gt == 2) simt_kernel<NI, 2, VEC><<<ctas, kThreads, 0, st>>>(p);
  else simt_kernel<NI, 1, VEC><<<ctas, kThreads, 0, st>>>(p);
}

}  // namespace paged
}  // namespace mpc

using namespace mpc;

extern "C" {

int mpc_sdpa_paged_workspace(mpc_device *dev, const mpc_kv_desc *cache, const mpc_sdpa_paged_desc *desc, size_t *bytes) {
  int rc = enter(dev);
  if (rc) return rc;
  if (!cache || !desc || !bytes) return fail(MPC_ERR_INVALID, "mpc_sdpa_paged_workspace: null argument");
  paged::Plan pl;
  if ((rc = paged::plan_of(dev, cache, desc, &pl))) return rc;
  *bytes = pl.ws_bytes;
  return MPC_OK;
}

int mpc_sdpa_paged(mpc_device *dev, const mpc_kv_desc *cache, const void *k_pages, const void *v_pages,
                   const uint8_t *k_scale, const uint8_t *v_scale, const mpc_sdpa_paged_desc *desc, const void *Q,
                   const int32_t *table, const int32_t *lengths, void *O, float *LSE, void *workspace,
                   size_t workspace_bytes, mpc_stream s) {
  using namespace paged;
  int rc = enter(dev);
  if (rc) return rc;
  if (!cache || !desc) return fail(MPC_ERR_INVALID, "mpc_sdpa_paged: null descriptor");
  Plan pl;
  if ((rc = plan_of(dev, cache, desc, &pl))) return rc;
  if (desc->b == 0) return MPC_OK;
  if (!Q || !O || !lengths || (desc->max_pages > 0 && !table) ||
      (cache->n_pages > 0 && (!k_pages || !v_pages || (cache->dtype == MPC_E4M3 && (!k_scale || !v_scale)))))
    return fail(MPC_ERR_INVALID, "mpc_sdpa_paged: null pointer");
  cudaStream_t st = stream_of(dev, s);
  Scratch own;
  if (workspace) {
    if (workspace_bytes < pl.ws_bytes || ((uintptr_t)workspace & 15))
      return fail(MPC_ERR_INVALID, "mpc_sdpa_paged: a workspace of %zu bytes at %p (%zu, 16-byte aligned, needed)",
                  workspace_bytes, workspace, pl.ws_bytes);
  } else {
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    MPC_CUDA(dev, cudaStreamIsCapturing(st, &cs));
    if (cs != cudaStreamCaptureStatusNone)
      return fail(MPC_ERR_INVALID, "mpc_sdpa_paged: a captured call needs a workspace of its own");
    if ((rc = own.get(dev, st, pl.ws_bytes))) return rc;
    workspace = own.ptr;
  }
  Params p{};
  p.q = Q, p.kp = k_pages, p.vp = v_pages, p.ks = k_scale, p.vs = v_scale, p.table = table, p.lengths = lengths;
  p.out = O, p.lse = LSE, p.ws = static_cast<float *>(workspace), p.err = dev->d_err;
  for (int i = 0; i < 2; ++i) p.qs[i] = desc->q_stride[i], p.os[i] = desc->o_stride[i];
  p.max_pages = desc->max_pages, p.cap = desc->max_pages * cache->page_size;
  p.B = (int)desc->b, p.H = (int)desc->h, p.hk = (int)cache->hk, p.group = p.H / p.hk, p.gt = pl.gt, p.qt = pl.qt;
  p.d = (int)cache->d, p.dv = (int)cache->dv, p.page_size = (int)cache->page_size, p.n_pages = (int)cache->n_pages;
  p.dt = desc->dtype, p.dt_pages = cache->dtype, p.scale_log2 = desc->scale * kLog2e;
  const bool vec = p.d % 8 == 0 && p.dv % 8 == 0 && (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0;
  const int dm = p.d > p.dv ? p.d : p.dv;
  if (dm <= 64) vec ? launch_simt<1, true>(p, pl.ctas, st) : launch_simt<1, false>(p, pl.ctas, st);
  else if (dm <= 128) vec ? launch_simt<2, true>(p, pl.ctas, st) : launch_simt<2, false>(p, pl.ctas, st);
  else vec ? launch_simt<4, true>(p, pl.ctas, st) : launch_simt<4, false>(p, pl.ctas, st);
  dev->launches++;
  if ((rc = check_launch(dev, "mpc_sdpa_paged"))) return rc;
  join_kernel<<<dim3(pl.ctas, pl.gt), kThreads, 0, st>>>(p, pl.ctas);
  dev->launches++;
  return check_launch(dev, "mpc_sdpa_paged join");
}

}  // extern "C"
