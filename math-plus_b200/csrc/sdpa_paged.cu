// Attention of one new token per sequence over the paged key/value cache (mpc_sdpa_paged): the serving
// form of mpc_sdpa (Backend.sdpa, packages/tensor-cpu/src/index.ts:821-840), Lq = 1.
//
// With s_j = scale * q.k_j for j < length: o = sum_j 2^(s'_j - m) v_j / sum_j 2^(s'_j - m), s' = s log2 e, m any
// upper reference of s' (the running maximum). A K/V row is read once for each tile of the query heads that share
// it: 16 on the tensor cores (8 at head dims above 128, or with f32 queries over 8 bits), 4 on the CUDA cores. With one
// tile the cache's bytes bound the time, and the work is split along the cache:
//
// Split. An item is (sequence, K/V head, tile of its query heads); its keys are cut into tiles (16 or 32; more
// where a table could hold 2^30 of them). The
// tiles of all items, in order, with kItemCost more for every item (an item's start and end take about
// as long as that many tiles), are dealt to the warps in equal runs: warp i of n takes units [T i / n,
// T (i + 1) / n). The runs are found from the lengths on the device, so ragged batches and a single long
// sequence balance alike and the launch depends on host-known sizes alone (it can be captured into a
// graph). A warp that has an item wholly writes the output. Otherwise the (at most two) cut items of
// a warp leave (m, l, O) in the workspace, one for the block where all its warps are inside one item, and
// count themselves there; the block that counts an item's last part joins them all, in their order, so the
// result does not depend on timing. The counters are zero between calls: who joins puts them back.
//
// CUDA-core kernel (f32 rows, and any head dim <= 256 or alignment): 8 lanes per key, 4 keys at a time, each
// group of 8 lanes with its own running maximum, sum and O, which meet once per item.
//
// Measured (GPU time of a replayed call): 32 sequences of 500..8191 keys, 32 heads over 8 of 128, f16: 98 us, 5.8 TB/s
// (a copy: 6.55), bound by HBM; 99999 and 131072 keys, 64 heads over 8 of 128, 8 bits: 109 us, 4.4 TB/s, bound by the
// instructions that widen the codes (f32 queries 115 us a call, f16 111); 64 sequences of 1..1024 keys, 12 heads of 64,
// bf16: 25.5 us, 4.0 TB/s, bound by the items' starts and joins; one of 1024 keys 9.9 us and, in f32 on the CUDA cores, 7 of
// 3..2050 keys with 10 heads over 5 of 80 / 72 22 us, both bound by latency. Wider groups than a tile: 8 x 8192 keys, 32
// heads over 2 of 256, bf16, 71 us (two tiles; the bytes 20.5); in f32, four tiles, 843 us (41), with heads of 128 259 (20.5).
#include <cfloat>

#include "kv_cache.cuh"
#include "mpc_internal.h"

namespace mpc {
namespace paged {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kMaxCtas = 4;  // resident on an SM, at most
// Measured (3, 5, 8, 12 tiles an item): 64 sequences of 1..1024 keys, 12 heads of 64, bf16: 23.5, 24.2, 25.2, 26.4 us; 32
// sequences of 500..8191 keys, 8 heads of 128, f16: 100.5, 100.2, 99.0, 98.5 us; 2 of ~115k keys in 8 bits: 113, 111, 108,
// 100 us. (0 against 8 with the joins left out, of an earlier form: 35, 109 and 103 against 27, 98 and 91 us.)
constexpr int kItemCost = 8;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Params {
  const void *q, *kp, *vp;
  const uint8_t *ks, *vs;
  const int32_t *table, *lengths;
  void *out;
  float *lse, *ws;
  int *counters;  // per warp: the warps that have left their part of the item that it starts
  unsigned long long *report;
  long long qs[2], os[2], max_pages, cap;  // cap: max_pages * page_size
  int B, H, hk, group, gt, qt, tile;  // query heads per K/V head, per query tile; tiles per K/V head; keys of a tile
  int d, dv, page_size, n_pages, dt, dt_pages;
  uint32_t page_mul, page_shift;  // key / page_size = key * page_mul >> page_shift for keys below 2^31
  int q_vec;  // queries in aligned pieces of 8 values
  float scale_log2;
  __device__ __forceinline__ unsigned page_of(unsigned key) const { return (unsigned)((uint64_t)key * page_mul >> page_shift); }
};

// A warp's place in an item. All units of a call are fewer than 2^31 (plan_of).
struct Item {
  int b, head;       // head: K/V head * qt + query tile
  int start, units;  // the item's first unit and its units: kItemCost, then one per tile
};

__device__ __forceinline__ int length_of(const Params &p, int b) {
  const int len = p.lengths[b];
  return len < 0 ? 0 : len > p.cap ? (int)p.cap : len;
}
__device__ __forceinline__ int units_of(const Params &p, int b) {
  const int len = length_of(p, b);
  return len ? (int)((unsigned)(len - 1) / (unsigned)p.tile) + 1 + kItemCost : 0;
}

// `total` units dealt to n warps: the first `more` have each + 1.
struct Deal {
  int total, n, each, more;
  __device__ __forceinline__ void set(int units, int warps) {
    total = units, n = min(units, warps);
    each = n ? (unsigned)total / (unsigned)n : 0;
    more = total - each * n;
  }
  __device__ __forceinline__ int start(int warp) const { return warp * each + min(warp, more); }
  __device__ __forceinline__ int warp_of(int unit) const {
    const int cut = more * (each + 1);
    return unit < cut ? (unsigned)unit / (unsigned)(each + 1) : more + (unsigned)(unit - cut) / (unsigned)each;
  }
};

// Block-wide inclusive scan of one value a thread; *sum: the block's total.
__device__ __forceinline__ int scan(int v, int *sm, int *sum) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, m);
    if (lane >= m) v += u;
  }
  __syncthreads();
  if (lane == 31) sm[w] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < w) before += sm[i];
    all += sm[i];
  }
  *sum = all;
  return v + before;
}

// The deal and the item of the block's first unit, by a scan of the lengths, kThreads sequences at a time: once
// where that is all of them. sm: kWarps + 2. Returns whether the block has a run.
__device__ __forceinline__ bool find_run(const Params &p, int *sm, Deal &deal, Item &it) {
  const int heads = p.hk * p.qt;
  int own = threadIdx.x < p.B ? units_of(p, threadIdx.x) * heads : 0, sum;
  int incl = scan(own, sm, &sum), total = sum;
  for (int b0 = kThreads; b0 < p.B; b0 += kThreads) {
    int more;
    scan(b0 + (int)threadIdx.x < p.B ? units_of(p, b0 + threadIdx.x) * heads : 0, sm, &more);
    total += more;
  }
  deal.set(total, gridDim.x * kWarps);
  const int w0 = blockIdx.x * kWarps;
  if (w0 >= deal.n) return false;
  const int c0 = deal.start(w0);
  int before = 0;
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    if (b0) {
      own = b0 + (int)threadIdx.x < p.B ? units_of(p, b0 + threadIdx.x) * heads : 0;
      incl = before + scan(own, sm, &sum);
    }
    if (c0 >= incl - own && c0 < incl) sm[kWarps] = b0 + threadIdx.x, sm[kWarps + 1] = incl - own;
    before += sum;
  }
  __syncthreads();
  it.b = sm[kWarps];
  it.units = units_of(p, it.b);
  const int rem = c0 - sm[kWarps + 1];
  it.head = (unsigned)rem / (unsigned)it.units;
  it.start = c0 - (rem - it.head * it.units);
  return true;
}

__device__ __forceinline__ void advance(const Params &p, Item &it) {
  it.start += it.units;
  if (++it.head == p.hk * p.qt) {
    it.head = 0;
    do it.units = units_of(p, ++it.b);
    while (it.units == 0);  // only called where a later unit exists
  }
}

// (m, l, O) of one query over part of an item, in the workspace: m, the exponent O refers to, l, one
// unused, then O, in whole 16 bytes. A warp's part at the item's start and one further on have a place each.
__host__ __device__ __forceinline__ int slot_floats(int dv) { return (dv + 3) / 4 * 4 + 4; }
__device__ __forceinline__ float *slot(const Params &p, int warp, bool first, int q) {
  return p.ws + (long long)((2 * warp + (first ? 1 : 0)) * p.gt + q) * slot_floats(p.dv);
}

__device__ __forceinline__ float guard_exp2(float x, float ref) { return x == -INFINITY ? 0.0f : exp2f(x - ref); }

// Sequences without keys: zeros and -inf; lengths outside the table are recorded.
__device__ __forceinline__ void empty_rows(const Params &p) {
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    const int len = p.lengths[b];
    if (threadIdx.x == 0 && (len < 0 || len > p.cap)) report_bad_page(p.report, kBadLength, b);
    if (len > 0 && p.cap > 0) continue;
    for (int i = threadIdx.x; i < p.H * p.dv; i += kThreads) {
      const int h = i / p.dv;
      store_f32(p.out, p.dt, b * p.os[0] + h * p.os[1] + (i - h * p.dv), 0.0f);
    }
    if (p.lse)
      for (int h = threadIdx.x; h < p.H; h += kThreads) p.lse[(long long)b * p.H + h] = -INFINITY;
  }
}

// Column e of (sequence, head), and with it the row's log-sum-exp: f = 2^(otop - top) / sum.
__device__ __forceinline__ float factor_of(float sum, float top, float otop) {
  return sum != 0.0f ? exp2f(otop - top) / sum : 0.0f;
}
__device__ __forceinline__ void put(const Params &p, int b, int h, int e, float v, float f, float sum, float top) {
  store_f32(p.out, p.dt, b * p.os[0] + h * p.os[1] + e, sum != 0.0f ? v * f : 0.0f);
  if (p.lse && e == 0) p.lse[(long long)b * p.H + h] = sum != 0.0f ? fmaf(top, kLn2, logf(sum)) : -INFINITY;
}

// Column e of query q over the results of SRC warps: (m, the exponent O refers to, l) in sml[src][q], O in so[src][q].
template <int SRC, int GT, int PITCH>
__device__ __forceinline__ void combine(const float (*so)[GT][PITCH], const float (*sml)[GT][3], int q, int e, float &v,
                                        float &sum, float &top, float &otop) {
  top = otop = -INFINITY, sum = v = 0.0f;
#pragma unroll
  for (int w = 0; w < SRC; ++w) top = fmaxf(top, sml[w][q][0]), otop = fmaxf(otop, sml[w][q][1]);
#pragma unroll
  for (int w = 0; w < SRC; ++w) {
    sum = fmaf(sml[w][q][2], guard_exp2(sml[w][q][0], top), sum);
    v = fmaf(so[w][q][e], guard_exp2(sml[w][q][1], otop), v);
  }
}

// Sends tiles [t0, t1) of an item on: to the output where that is all of it, else to the workspace. The
// results of SRC warps are in shared memory; `threads` threads of which this is `id` do it for warp `gw`.
template <int SRC, int GT, int PITCH>
__device__ __forceinline__ void finish(const Params &p, const Item &it, int t0, int t1, int gw,
                                       const float (*so)[GT][PITCH], const float (*sml)[GT][3], int id, int threads) {
  const int kvh = it.head / p.qt, h0 = kvh * p.group + (it.head % p.qt) * GT;
  const int nq = min(GT, (kvh + 1) * p.group - h0);
  const bool whole = t0 == 0 && t1 == it.units - kItemCost;
  const int w4 = (p.dv + 31) / 32 * 32;  // whole warps per query
  for (int i = id; i < nq * w4; i += threads) {
    const int q = i / w4, e = i - q * w4;
    if (e >= p.dv) continue;
    float top, otop, sum, v;
    combine<SRC>(so, sml, q, e, v, sum, top, otop);
    if (whole) {
      put(p, it.b, h0 + q, e, v, factor_of(sum, top, otop), sum, top);
    } else {
      float *ws = slot(p, gw, t0 == 0, q);
      ws[4 + e] = v;
      if (e == 0) *reinterpret_cast<float4 *>(ws) = make_float4(top, otop, sum, 0.0f);
    }
  }
}

// An item whose parts are all in the workspace: those of warps first..last.
struct Join {
  Item it;
  int first, last;
};

// Whether a block's run is inside one item, so that its warps leave one part, in its first warp's place.
__device__ __forceinline__ bool meets(const Deal &all, const Item &it, int block) {
  const int w0 = block * kWarps;
  return all.start(w0) >= it.start && all.start(min(w0 + kWarps, all.n)) <= it.start + it.units;
}

__device__ __forceinline__ void fence_gpu() { asm volatile("fence.acq_rel.gpu;" ::: "memory"); }

// Counts `warps` more warps' part of a cut item (the caller has fenced its stores); true for the last part.
__device__ __forceinline__ bool last_part(const Params &p, const Deal &all, const Item &it, int warps, Join &j) {
  const int wf = all.warp_of(it.start + kItemCost);  // the warp of the first tile; warps before it have no part
  j.it = it;
  j.first = meets(all, it, wf / kWarps) ? wf / kWarps * kWarps : wf;
  j.last = all.warp_of(it.start + it.units - 1);
  if (atomicAdd(p.counters + j.first, warps) + warps != j.last - j.first + 1) return false;
  p.counters[j.first] = 0;
  fence_gpu();
  return true;
}

// One warp joins query q of an item: lanes hold the parts' headers and weights, 32 at a time, then each lane columns
// 4 lane ..+3 (WIDE: + 128 too) of their O, eight parts' loads in flight. (A single warp's instructions bound this,
// so a part costs few.) Places that a lane has no column or a round no part for repeat another with weight 0.
template <bool WIDE>
__device__ __forceinline__ void join(const Params &p, const Deal &all, const Join &j, int q) {
  constexpr int E = WIDE ? 2 : 1;
  const int lane = threadIdx.x & 31;
  const int kvh = j.it.head / p.qt, h = kvh * p.group + (j.it.head % p.qt) * p.gt + q;
  const int row = slot_floats(p.dv) / 4, step = 2 * p.gt * row;  // float4s from a place to the next, of a warp to the next
  const float4 *const places = reinterpret_cast<const float4 *>(p.ws) + (long long)j.first * step + q * row;
  const int start = p.gt * row;  // the first part is in its warp's second place
  int col[E];
#pragma unroll
  for (int e = 0; e < E; ++e) col[e] = 128 * e + 4 * lane < p.dv ? 1 + 32 * e + lane : 1;
  float top = -INFINITY, otop = -INFINITY, sum = 0.0f;
  float4 v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = make_float4(0, 0, 0, 0);
  // The parts: the first block's warps from j.first on (or one, where they met), one of every block inside the
  // item, the last block's warps up to j.last (or one).
  const int b0 = j.first / kWarps, b1 = j.last / kWarps;
  const int n0 = meets(all, j.it, b0) ? 1 : min((b0 + 1) * kWarps, j.last + 1) - j.first;
  const int n1 = b1 > b0 ? n0 + b1 - b0 - 1 : n0;
  const int parts = b1 == b0 ? n0 : n1 + (meets(all, j.it, b1) ? 1 : j.last - b1 * kWarps + 1);
  auto warp_of = [&](int i) {  // less j.first
    return i < n0 ? i : (i < n1 ? (b0 + 1 + i - n0) * kWarps : b1 * kWarps + i - n1) - j.first;
  };
  for (int base = 0; base < parts; base += 32) {
    const int mine = warp_of(min(base + lane, parts - 1));
    float4 x = make_float4(-INFINITY, -INFINITY, 0, 0);
    if (base + lane < parts) x = __ldcg(places + (long long)mine * step + (mine ? 0 : start));
    float up = x.x, oup = x.y;
#pragma unroll
    for (int k = 16; k; k >>= 1) {
      up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, k));
      oup = fmaxf(oup, __shfl_xor_sync(0xffffffffu, oup, k));
    }
    up = fmaxf(up, top), oup = fmaxf(oup, otop);
    const float keep = guard_exp2(otop, oup);
    float l = x.z * guard_exp2(x.x, up);
    const float f = guard_exp2(x.y, oup);
#pragma unroll
    for (int k = 16; k; k >>= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
    sum = fmaf(sum, guard_exp2(top, up), l);
    top = up, otop = oup;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e].x *= keep, v[e].y *= keep, v[e].z *= keep, v[e].w *= keep;
    unsigned left = __ballot_sync(0xffffffffu, f != 0.0f);
    while (left) {
      float4 z[8][E];
      float wt[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = left ? __ffs(left) - 1 : 0;
        wt[k] = __shfl_sync(0xffffffffu, f, i);
        if (!left) wt[k] = 0.0f;
        const int at = __shfl_sync(0xffffffffu, mine, i);
        const float4 *y = places + (long long)at * step + (at ? 0 : start);
        left &= left - 1;
#pragma unroll
        for (int e = 0; e < E; ++e) z[k][e] = __ldcg(y + col[e]);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          v[e].x = fmaf(z[k][e].x, wt[k], v[e].x), v[e].y = fmaf(z[k][e].y, wt[k], v[e].y);
          v[e].z = fmaf(z[k][e].z, wt[k], v[e].z), v[e].w = fmaf(z[k][e].w, wt[k], v[e].w);
        }
    }
  }
  const float f = factor_of(sum, top, otop);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float y[4] = {v[e].x, v[e].y, v[e].z, v[e].w};
#pragma unroll 1
    for (int k = 0; k < 4; ++k) {
      const int at = 128 * e + 4 * lane + k;
      if (at < p.dv) put(p, j.it.b, h, at, k < 2 ? (k ? y[1] : y[0]) : (k == 2 ? y[2] : y[3]), f, sum, top);
    }
  }
}

// Walks a warp's run: body(sequence, head tile, t0, t1) leaves its part of each item in shared memory. The place
// in the run is in shared memory too, while the body has the registers.
template <int GT, int PITCH, typename Body>
__device__ __forceinline__ void walk(const Params &p, float (*so)[GT][PITCH], float (*sml)[GT][3], Body body) {
  struct Place {
    Item it;
    int u, u1;  // the unit the warp is at, the end of its run
  };
  __shared__ int sm[kWarps + 2];
  __shared__ Place places[kWarps];
  __shared__ Deal all;
  __shared__ Item cut[kWarps][2];  // a warp's run cuts two items at most
  __shared__ Join joins[2 * kWarps];
  __shared__ int n_joins;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gw = blockIdx.x * kWarps + warp;
  volatile Place *const here = &places[warp];
  bool meet = false;  // the block is inside one item: its warps meet at the end
  bool go = false;
  int cuts = 0;
  {
    Deal deal;
    Item it{};
    int u0 = 0, u1 = 0;
    if (find_run(p, sm, deal, it)) {
      meet = meets(deal, it, blockIdx.x);
      if (gw < deal.n) u0 = deal.start(gw), u1 = deal.start(gw + 1);
      go = u0 < u1 || meet;
      if (!meet && go)
        while (it.start + it.units <= u0) advance(p, it);
    }
    if (lane == 0) {
      places[warp].it = it, places[warp].u = u0, places[warp].u1 = u1;
      if (warp == 0) all = deal, n_joins = 0;
    }
  }
  __syncthreads();
  while (go) {
    int u = here->u, end = min(here->u1, here->it.start + here->it.units), base = here->it.start + kItemCost;
    if (meet || end > base) body(here->it.b, here->it.head, max(0, u - base), max(0, end - base));
    __syncwarp();
    Item it;
    it.b = here->it.b, it.head = here->it.head, it.start = here->it.start, it.units = here->it.units;
    const int u1 = here->u1, w0 = gw - warp;
    u = here->u, end = min(u1, it.start + it.units), base = it.start + kItemCost;
    int from = max(0, u - base), to = max(0, end - base);
    if (meet) {
      __syncthreads();
      from = max(0, all.start(w0) - base), to = max(0, all.start(min(w0 + kWarps, all.n)) - base);
      if (to > from) finish<kWarps, GT, PITCH>(p, it, from, to, w0, so, sml, threadIdx.x, kThreads);
      __syncthreads();
    } else if (to > from) {
      finish<1, GT, PITCH>(p, it, from, to, gw, so + warp, sml + warp, lane, 32);
    }
    __syncwarp();
    if ((!meet || warp == 0) && to > from && to - from < it.units - kItemCost) {
      if (lane == 0) cut[warp][cuts] = it;
      ++cuts;
    }
    go = !meet && end < u1;
    if (go) {
      advance(p, it);
      if (lane == 0) places[warp].it = it, places[warp].u = end;
      __syncwarp();
    }
  }
  // The parts are counted once the run is done: one fence, and the two items' counters at once.
  __syncwarp();
  if (lane < cuts) {
    fence_gpu();
    Join j;
    const int w0 = gw - warp;
    if (last_part(p, all, cut[warp][lane], meet ? min(kWarps, all.n - w0) : 1, j)) joins[atomicAdd(&n_joins, 1)] = j;
  }
  empty_rows(p);
  __syncthreads();
  const int queries = min(GT, p.group);
  for (int i = warp; i < n_joins * queries; i += kWarps) {
    const Join j = joins[i / queries];
    const int q = i % queries;
    if (q >= p.group - (j.it.head % p.qt) * GT) continue;
    if (p.dv > 128) join<true>(p, all, j, q);
    else join<false>(p, all, j, q);
  }
}

// ---- CUDA-core kernel ---------------------------------------------------------------------------
template <int NI, int GT, bool VEC>
__global__ void __launch_bounds__(kThreads) simt_kernel(const Params p) {
  constexpr int W = NI * 64;  // padded head dim: lane j of 8 holds values i * 64 + j * 8 ..+7
  __shared__ float sq[kWarps][GT][W];
  __shared__ float so[kWarps][GT][W];
  __shared__ float sml[kWarps][GT][3];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j8 = (lane & 7) * 8;
  walk<GT, W>(p, so, sml, [&](int b, int head, int t0, int t1) {
    const int kvh = head / p.qt, h0 = kvh * p.group + (head % p.qt) * GT;
    const int nq = min(GT, (kvh + 1) * p.group - h0);
    for (int i = lane; i < GT * W; i += 32) {
      const int q = i / W, e = i % W;
      sq[warp][q][e] = q < nq && e < p.d ? load_f32(p.q, p.dt, b * p.qs[0] + (h0 + q) * p.qs[1] + e) : 0.0f;
    }
    __syncwarp();
    float m[GT], l[GT], o[GT][NI * 8];
#pragma unroll
    for (int q = 0; q < GT; ++q) {
      m[q] = -INFINITY, l[q] = 0.0f;
#pragma unroll
      for (int e = 0; e < NI * 8; ++e) o[q][e] = 0.0f;
    }
    const unsigned end = (unsigned)min((long long)length_of(p, b), (long long)t1 * p.tile);  // lengths are below 2^31
    // The row of this group's key, k0 + lane / 8; -1: none (behind the end, or a page outside the cache).
    auto row_at = [&](unsigned k0) -> long long {
      const unsigned key = k0 + (lane >> 3);
      if (key >= end) return -1;
      const unsigned col = p.page_of(key);
      const int pg = p.table[(long long)b * p.max_pages + col];
      if (pg >= 0 && pg < p.n_pages) return ((long long)pg * p.hk + kvh) * p.page_size + (key - col * (unsigned)p.page_size);
      if ((lane & 7) == 0) report_bad_page(p.report, kBadAttend, b);
      return -1;
    };
    // Where the registers allow, a key's V and the next step's row are under way with its K.
    constexpr bool AHEAD = VEC && NI * GT <= 4;
    unsigned k0 = (unsigned)t0 * (unsigned)p.tile;
    long long row = row_at(k0);
    for (; k0 < end; k0 += 4) {
      float s[GT], x[8];
      Raw8 k_raw[AHEAD ? NI : 1], v_raw[AHEAD ? NI : 1];
      if constexpr (AHEAD) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          if (row >= 0 && i * 64 + j8 < p.d) load_raw8(p.kp, p.dt_pages, row * p.d + i * 64 + j8, k_raw[i]);
          if (row >= 0 && i * 64 + j8 < p.dv) load_raw8(p.vp, p.dt_pages, row * p.dv + i * 64 + j8, v_raw[i]);
        }
      }
      const long long next = row_at(k0 + 4);
#pragma unroll
      for (int q = 0; q < GT; ++q) s[q] = 0.0f;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int at = i * 64 + j8;
        if (row >= 0 && at < p.d) {
          if constexpr (AHEAD) widen8(k_raw[i], p.dt_pages, x);
          else load8<VEC>(p.kp, p.dt_pages, row * p.d + at, p.d - at, x);
#pragma unroll
          for (int q = 0; q < GT; ++q)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[q] = fmaf(sq[warp][q][at + e], x[e], s[q]);
        }
      }
#pragma unroll
      for (int q = 0; q < GT; ++q)
#pragma unroll
        for (int k = 4; k; k >>= 1) s[q] += __shfl_xor_sync(0xffffffffu, s[q], k);
      if (row >= 0) {
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
            if constexpr (AHEAD) widen8(v_raw[i], p.dt_pages, x);
            else load8<VEC>(p.vp, p.dt_pages, row * p.dv + at, p.dv - at, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float v = x[e] * fv;
#pragma unroll
              for (int q = 0; q < GT; ++q) o[q][i * 8 + e] = fmaf(s[q], v, o[q][i * 8 + e]);
            }
          }
        }
      }
      row = next;
    }
    // The 4 groups of the warp meet by shuffles.
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
      if (lane == 0) sml[warp][q][0] = sml[warp][q][1] = top, sml[warp][q][2] = l[q];
    }
  });
}

// ---- tensor-core kernel ---------------------------------------------------------------------------
// 16-bit and 8-bit rows. A warp takes 16 keys at a time and forms S^T = K Q^T and O^T += V^T P^T with
// m16n8k16 products, the keys (or V's columns) as rows and up to 8 query heads as columns: one new
// token per sequence fills 8 columns at most, far from the 128 rows of a tcgen05 tile, and the
// products' rate is not what bounds the kernel. The fragments' k order is free as long as both
// operands share it, so every lane loads 8 adjacent values of a row and the loads go from global
// memory straight to the registers that feed the products: no shared memory, no barrier in the loop,
// every warp on its own. The next tile's K is loaded once S has used the present one, the next V after
// the present product.
//   K: lane (r = lane / 4, c = lane % 4) holds values 32 j + 8 c ..+7 of keys r and r + 8; their pairs
//      are the k-slots of two products.
//   V: the lane holds values 64 j + 8 r ..+7 of keys 2c, 2c+1, 2c+8, 2c+9; the pairs of neighbouring keys
//      that the products want are byte permutes of two such registers.
// Weights: S^T's layout transposed (movmatrix) is P^T's. A weight goes in as the sum of two numbers of the
// type (its rounding and the rest), which leaves 2^-16 (bf16) or 2^-22 (f16, the type over 8-bit rows) of it; one
// number alone would leave 2^-8 or 2^-11, of sum p |v| and not of the output, which is smaller where V cancels.
// The reference m of the exponentials is only raised when a score passes it by more than 2^kSlack: a warp
// vote per tile in the common case, the row maximum by shuffles and a rescaling of O else. It is set 2^kHead
// below the maximum so that small weights stay clear of f16's subnormals.
// 8-bit rows: codes convert exactly to f16; Q is scaled by a power of two per row to [2^14, 2^15), where any
// 16-bit q is exact in f16 down to 2^-28 of the row's largest. An f32 q goes in as two f16, 22 of its 24 bits: the 2^-23
// that is left is no more than the f32 sum of the products rounds. K's scale multiplies the
// score. V's joins the weight: w = 2^(s' + e_v - M) with a reference M of its own, so that rows far below
// the largest scale keep their precision.
constexpr float kHead = 6.0f, kSlack = 14.0f;
constexpr float kNoRef = -3e38f;  // the reference before any score; 2^(-inf - kNoRef) is 0
constexpr uint32_t kNoRow = 0xffffffffu;
enum { kF16, kBF16, kE4M3 };

template <bool BF>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  if constexpr (BF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}

// 2^x, 0 for -inf.
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 8 values of a row as loaded: 4 registers of 16-bit pairs, or 2 of 8-bit codes. Zero from the start, they stay so
// where the row is shorter (`in` never changes).
template <int KIND>
struct Chunk {
  static constexpr int N = KIND == kE4M3 ? 2 : 4;
  uint32_t r[N];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = 0;
  }
  __device__ __forceinline__ void load(const uint8_t *at, bool in) {
    if constexpr (KIND == kE4M3) {
      if (in) {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(at));
        r[0] = v.x, r[1] = v.y;
      }
    } else {
      if (in) {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(at));
        r[0] = v.x, r[1] = v.y, r[2] = v.z, r[3] = v.w;
      }
    }
  }
  // Values 0, 1 | 2, 3 | 4, 5 | 6, 7 as pairs.
  __device__ __forceinline__ void pairs(uint32_t (&x)[4]) const {
    if constexpr (KIND == kE4M3) {
      e4m3x4_to_f16x4(r[0], x[0], x[1]);
      e4m3x4_to_f16x4(r[1], x[2], x[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = r[i];
    }
  }
};
// Value 2i (a0) and 2i + 1 (a1) of two neighbouring keys, as pairs (key, next key).
template <int KIND>
__device__ __forceinline__ void key_pairs(const Chunk<KIND> &x, const Chunk<KIND> &y, int i, uint32_t &a0, uint32_t &a1) {
  if constexpr (KIND == kE4M3) {
    e4m3x4_to_f16x4(prmt(x.r[i >> 1], y.r[i >> 1], (i & 1) ? 0x7362u : 0x5140u), a0, a1);
  } else {
    a0 = prmt(x.r[i], y.r[i], 0x5410u);
    a1 = prmt(x.r[i], y.r[i], 0x7632u);
  }
}

// DP: head dims padded to 64, 128 or 256; NT: tiles of 8 query heads; QS: numbers per query value. TPI tiles of 16 keys
// at a time: 32 keys where their rows fit the registers that 16 longer ones take. Blocks per SM as the registers allow;
// over 8-bit rows of 128 two blocks of 32 keys a warp (108 us at 2 x ~115k keys) beat three of 16 (118 us).
template <int KIND, int DP>
constexpr int tiles_at_once() { return DP == 64 || (DP == 128 && KIND == kE4M3) ? 2 : 1; }
constexpr int blocks_per_sm(bool e4m3, int dp, int heads) { return dp == 256 || heads == 16 || (dp == 128 && e4m3) ? 2 : 3; }

template <int KIND, int DP, int NT, int QS>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(KIND == kE4M3, DP, 8 * NT)) mma_kernel(const Params p) {
  constexpr bool BF = KIND == kBF16, Q8 = KIND == kE4M3;
  constexpr int KC = DP / 32, VC = DP / 64, GT = 8 * NT, PITCH = DP + 8, TPI = tiles_at_once<KIND, DP>(), KEYS = 16 * TPI;
  __shared__ alignas(16) float so[kWarps][GT][PITCH];  // written as pairs
  __shared__ float sml[kWarps][GT][3];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;

  walk<GT, PITCH>(p, so, sml, [&](int b, int head, int t0, int t1) {
    const int kvh = head / p.qt, h0 = kvh * p.group + (head % p.qt) * GT;
    const int nq = min(GT, (kvh + 1) * p.group - h0);
    const unsigned end = (unsigned)min((long long)length_of(p, b), (long long)t1 * p.tile);  // lengths are below 2^31
    const int32_t *table = p.table + (long long)b * p.max_pages;

    // The row of this lane's key (lane % KEYS) in the tile of keys from k0 on.
    auto row_at = [&](unsigned k0) -> uint32_t {
      const unsigned key = k0 + (lane & (KEYS - 1));
      if (key >= end) return kNoRow;
      const unsigned col = p.page_of(key);
      const int pg = __ldg(table + col);
      if (pg < 0 || pg >= p.n_pages) {
        report_bad_page(p.report, kBadAttend, b);
        return kNoRow;
      }
      return ((unsigned)pg * (unsigned)p.hk + kvh) * (unsigned)p.page_size + (key - col * (unsigned)p.page_size);
    };
    // Keys without a row load row 0 of the pages instead: S is masked, V set to zero where a tile has such keys.
    constexpr int EB = Q8 ? 1 : 2;
    Chunk<KIND> kf[TPI][2][KC], vf[TPI][4][VC];
    uint32_t ks = 127, vs = 127;  // scale bytes of this lane's key
    auto load_k = [&](uint32_t row) {
#pragma unroll
      for (int t = 0; t < TPI; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t from = __shfl_sync(0xffffffffu, row == kNoRow ? 0 : row, 16 * t + 8 * k + r);
          const uint8_t *at = static_cast<const uint8_t *>(p.kp) + ((size_t)from * p.d + 8 * c) * EB;
#pragma unroll
          for (int j = 0; j < KC; ++j) kf[t][k][j].load(at + 32 * EB * j, 32 * j + 8 * c < p.d);
        }
      if constexpr (Q8) ks = p.ks[row == kNoRow ? 0 : row];
    };
    auto load_v = [&](uint32_t row) {
#pragma unroll
      for (int t = 0; t < TPI; ++t)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t from = __shfl_sync(0xffffffffu, row == kNoRow ? 0 : row, 16 * t + 2 * c + (k & 1) + (k >> 1) * 8);
          const uint8_t *at = static_cast<const uint8_t *>(p.vp) + ((size_t)from * p.dv + 8 * r) * EB;
#pragma unroll
          for (int j = 0; j < VC; ++j) vf[t][k][j].load(at + 64 * EB * j, 64 * j + 8 * r < p.dv);
        }
      if constexpr (Q8) vs = p.vs[row == kNoRow ? 0 : row];
    };
#pragma unroll
    for (int t = 0; t < TPI; ++t) {
#pragma unroll
      for (int j = 0; j < KC; ++j) kf[t][0][j].zero(), kf[t][1][j].zero();
#pragma unroll
      for (int j = 0; j < VC; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) vf[t][k][j].zero();
    }

    unsigned k0 = (unsigned)t0 * (unsigned)p.tile;
    uint32_t row = row_at(k0), next = row_at(k0 + KEYS);
    load_k(row);
    load_v(row);

    // Q^T: lane (r, c) holds values 32 j + 8 c ..+7 of query head r of each tile.
    uint32_t qf[NT][QS][KC][4];
    float qscale[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bool live = n * 8 + r < nq;
      const long long base = b * p.qs[0] + (h0 + n * 8 + r) * p.qs[1] + 8 * c;
      if constexpr (!Q8) {
#pragma unroll
        for (int j = 0; j < KC; ++j) {
          uint4 x = make_uint4(0, 0, 0, 0);
          if (live && 32 * j + 8 * c < p.d) {
            const uint16_t *q = static_cast<const uint16_t *>(p.q) + base + 32 * j;
            if (p.q_vec) x = *reinterpret_cast<const uint4 *>(q);
            else x = make_uint4(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16, q[4] | (uint32_t)q[5] << 16, q[6] | (uint32_t)q[7] << 16);
          }
          qf[n][0][j][0] = x.x, qf[n][0][j][1] = x.y, qf[n][0][j][2] = x.z, qf[n][0][j][3] = x.w;
        }
        qscale[n][0] = qscale[n][1] = p.scale_log2;
      } else {
        float x[KC][8];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < KC; ++j) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[j][i] = 0.0f;
          if (live && 32 * j + 8 * c < p.d) {
            if (p.q_vec) load8<true>(p.q, p.dt, base + 32 * j, 8, x[j]);
            else load8<false>(p.q, p.dt, base + 32 * j, 8, x[j]);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t a = __float_as_uint(x[j][i]) & 0x7fffffffu;
            if (a < 0x7f800000u) top = max(top, a);
          }
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int eq = max(1, min((int)(top >> 23), 253)) - 127;  // the row's largest is in [2^eq, 2^(eq + 1))
        // x 2^(14 - eq) in two exact steps, either of which may pass f32's range alone
        const float f0 = __uint_as_float((uint32_t)(127 + (14 - eq) / 2) << 23);
        const float f1 = __uint_as_float((uint32_t)(127 + (14 - eq) - (14 - eq) / 2) << 23);
#pragma unroll
        for (int j = 0; j < KC; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x0 = x[j][2 * i] * f0 * f1, x1 = x[j][2 * i + 1] * f0 * f1;
            qf[n][0][j][i] = f32_to_f16x2(x0, x1);
            if constexpr (QS == 2) {
              const float2 h = f16x2_to_f32(qf[n][0][j][i]);
              qf[n][1][j][i] = f32_to_f16x2(x0 - h.x, x1 - h.y);
            }
          }
        // The scores' factor of heads 2c and 2c + 1 of the tile: scale * log2 e * 2^(eq - 14).
        const float mine = ldexpf(p.scale_log2, eq - 14);
        qscale[n][0] = __shfl_sync(0xffffffffu, mine, (2 * c) * 4);
        qscale[n][1] = __shfl_sync(0xffffffffu, mine, (2 * c + 1) * 4);
      }
    }

    float o[NT][VC][4][4], m[NT][2], mo[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) m[n][i] = mo[n][i] = kNoRef, l[n][i] = 0.0f;
#pragma unroll
      for (int j = 0; j < VC; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][j][i][e] = 0.0f;
    }

    for (; k0 < end; k0 += KEYS) {
      // S^T: s[t][n][0..1] key 16 t + r, heads 2c, 2c + 1; s[t][n][2..3] key 16 t + r + 8.
      float s[TPI][NT][4], ev[TPI][2];
#pragma unroll
      for (int t = 0; t < TPI; ++t) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[t][n][e] = 0.0f;
#pragma unroll
        for (int j = 0; j < KC; ++j) {
          uint32_t x[4], y[4];
          kf[t][0][j].pairs(x);
          kf[t][1][j].pairs(y);
#pragma unroll
          for (int i = 0; i < 4; i += 2)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int q = 0; q < QS; ++q) mma<BF>(s[t][n], x[i], y[i], x[i + 1], y[i + 1], qf[n][q][j][i], qf[n][q][j][i + 1]);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int from = 16 * t + r + 8 * k;
          const bool see = __shfl_sync(0xffffffffu, row, from) != kNoRow;
          float fk = 1.0f;
          ev[t][k] = 0.0f;
          if constexpr (Q8) {
            fk = scale_value(__shfl_sync(0xffffffffu, ks, from));
            ev[t][k] = (float)((int)__shfl_sync(0xffffffffu, vs, from) - 127);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) s[t][n][2 * k + i] = see ? s[t][n][2 * k + i] * (qscale[n][i] * fk) : -INFINITY;
        }
      }
      load_k(next);

      bool raise = false;
      float top[NT][2], otop[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          top[n][i] = otop[n][i] = -INFINITY;
#pragma unroll
          for (int t = 0; t < TPI; ++t) {
            top[n][i] = fmaxf(top[n][i], fmaxf(s[t][n][i], s[t][n][2 + i]));
            if constexpr (Q8) otop[n][i] = fmaxf(otop[n][i], fmaxf(s[t][n][i] + ev[t][0], s[t][n][2 + i] + ev[t][1]));
          }
          raise |= top[n][i] > m[n][i] + kSlack;
          if constexpr (Q8) raise |= otop[n][i] > mo[n][i] + kSlack;
        }
      if (!__all_sync(0xffffffffu, row != kNoRow)) {  // the last tile of a sequence, or a bad page
#pragma unroll
        for (int t = 0; t < TPI; ++t)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (__shfl_sync(0xffffffffu, row, 16 * t + 2 * c + (k & 1) + (k >> 1) * 8) == kNoRow)
#pragma unroll
              for (int j = 0; j < VC; ++j) vf[t][k][j].zero();
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int k = 4; k < 32; k <<= 1) top[n][i] = fmaxf(top[n][i], __shfl_xor_sync(0xffffffffu, top[n][i], k));
            const float up = fmaxf(m[n][i], top[n][i] - kHead);
            float keep = ex2(m[n][i] - up);
            l[n][i] *= keep;
            m[n][i] = up;
            if constexpr (Q8) {
#pragma unroll
              for (int k = 4; k < 32; k <<= 1) otop[n][i] = fmaxf(otop[n][i], __shfl_xor_sync(0xffffffffu, otop[n][i], k));
              const float oup = fmaxf(mo[n][i], otop[n][i] - kHead);
              keep = ex2(mo[n][i] - oup);
              mo[n][i] = oup;
            }
#pragma unroll
            for (int j = 0; j < VC; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[n][j][e][i] *= keep, o[n][j][e][2 + i] *= keep;
          }
      }
#pragma unroll
      for (int t = 0; t < TPI; ++t) {
        // P^T: b0 keys 2c, 2c + 1 and b1 keys 2c + 8, 2c + 9 of head r, as two numbers each.
        uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[e] = ex2(s[t][n][e] - m[n][e & 1]);
            l[n][e & 1] += w[e];
            if constexpr (Q8) w[e] = ex2(s[t][n][e] - (mo[n][e & 1] - ev[t][e >> 1]));
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t h = BF ? f32_to_bf16x2(w[2 * k], w[2 * k + 1]) : f32_to_f16x2(w[2 * k], w[2 * k + 1]);
            const float2 f = BF ? bf16x2_to_f32(h) : f16x2_to_f32(h);
            const float x = w[2 * k] - f.x, y = w[2 * k + 1] - f.y;
            hi[n][k] = transpose8x8(h);
            lo[n][k] = transpose8x8(BF ? f32_to_bf16x2(x, y) : f32_to_f16x2(x, y));
          }
        }
#pragma unroll
        for (int j = 0; j < VC; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t a0, a1, a2, a3;
            key_pairs<KIND>(vf[t][0][j], vf[t][1][j], i, a0, a1);
            key_pairs<KIND>(vf[t][2][j], vf[t][3][j], i, a2, a3);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma<BF>(o[n][j][i], a0, a1, a2, a3, hi[n][0], hi[n][1]);
              mma<BF>(o[n][j][i], a0, a1, a2, a3, lo[n][0], lo[n][1]);
            }
          }
      }
      load_v(next);
      row = next;
      next = row_at(k0 + 2 * KEYS);
    }

    // o[n][j][i]: columns 64 j + 8 r + 2 i (e < 2) and + 1, heads 2c, 2c + 1.
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], k);
        const int q = n * 8 + 2 * c + i;
        if (r == 0) sml[warp][q][0] = m[n][i], sml[warp][q][1] = Q8 ? mo[n][i] : m[n][i], sml[warp][q][2] = l[n][i];
#pragma unroll
        for (int j = 0; j < VC; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<float2 *>(&so[warp][q][64 * j + 8 * r + 2 * e]) = make_float2(o[n][j][e][i], o[n][j][e][2 + i]);
      }
  });
}

// ---- host -------------------------------------------------------------------------------------------
struct Plan {
  int gt, qt, ctas, tile;
  int dp;  // padded head dim of the tensor-core kernel, 0: the CUDA cores
  size_t counters_bytes, ws_bytes;
};

static int plan_of(mpc_device *dev, const mpc_kv_desc *c, const mpc_sdpa_paged_desc *d, bool aligned, Plan *pl) {
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
  const int64_t group = d->h / c->hk, dm = c->d > c->dv ? c->d : c->dv;
  // The tensor cores take rows of 16 and 8 bits in aligned pieces of 8 values, their numbers in 32 bits.
  const bool tc = aligned && c->dtype != MPC_F32 && c->n_pages > 0 && c->d % 8 == 0 && c->dv % 8 == 0 &&
                  c->n_pages * c->page_size < (int64_t)kNoRow / c->hk;
  const bool two = c->dtype == MPC_E4M3 && d->dtype == MPC_F32;  // two f16 per query value: no registers for 16 heads
  pl->dp = !tc ? 0 : dm <= 64 ? 64 : dm <= 128 ? 128 : 256;
  pl->gt = tc ? (group > 8 && pl->dp < 256 && !two ? 16 : 8) : group >= 4 ? 4 : group >= 2 ? 2 : 1;
  pl->qt = (int)((group + pl->gt - 1) / pl->gt);
  pl->tile = tc && (pl->dp == 64 || (pl->dp == 128 && c->dtype == MPC_E4M3)) ? 32 : 16;  // tiles_at_once
  // Fewer than 2^31 units (and half of that for the sums of their parts), by longer tiles where a table could hold more.
  while ((double)d->b * c->hk * pl->qt * (double)(d->max_pages * c->page_size / pl->tile + 1 + kItemCost) >= (double)(1 << 30)) {
    if (pl->tile >= (1 << 30)) return fail(MPC_ERR_UNSUPPORTED, "mpc_sdpa_paged: too many sequences and heads");
    pl->tile *= 2;
  }
  // CTAs: as many as are resident on the tensor cores, three an SM on the CUDA cores (their registers, 118 to 254 a
  // thread, would let two to four be resident); fewer where even the longest lengths give fewer tiles than warps.
  const long long per = (d->max_pages * c->page_size + kWarps * pl->tile - 1) / (kWarps * pl->tile);
  const long long sms = (long long)dev->prop.multiProcessorCount * (tc ? blocks_per_sm(c->dtype == MPC_E4M3, pl->dp, pl->gt) : 3);
  const long long heads = c->hk * pl->qt;
  long long ctas = sms;
  if (d->b > 0 && per > 0 && per <= sms / heads / d->b) ctas = per * heads * d->b;
  pl->ctas = (int)(ctas < 1 ? 1 : ctas);
  // The counters' room depends on the device alone, so that calls of any shape may follow one another in a workspace.
  pl->counters_bytes = (size_t)dev->prop.multiProcessorCount * kMaxCtas * kWarps * sizeof(int);
  pl->ws_bytes = pl->counters_bytes + (size_t)pl->ctas * kWarps * 2 * pl->gt * slot_floats((int)c->dv) * sizeof(float);
  return MPC_OK;
}

template <int NI, bool VEC>
static void launch_simt(const Params &p, int ctas, cudaStream_t st) {
  if (p.gt == 4) simt_kernel<NI, 4, VEC><<<ctas, kThreads, 0, st>>>(p);
  else if (p.gt == 2) simt_kernel<NI, 2, VEC><<<ctas, kThreads, 0, st>>>(p);
  else simt_kernel<NI, 1, VEC><<<ctas, kThreads, 0, st>>>(p);
}

template <int KIND, int QS>
static void launch_mma(const Params &p, const Plan &pl, cudaStream_t st) {
  constexpr int NT = QS == 2 ? 1 : 2;
  auto run = [&](auto kern) { kern<<<pl.ctas, kThreads, 0, st>>>(p); };
  if (pl.dp == 64) pl.gt == 16 ? run(mma_kernel<KIND, 64, NT, QS>) : run(mma_kernel<KIND, 64, 1, QS>);
  else if (pl.dp == 128) pl.gt == 16 ? run(mma_kernel<KIND, 128, NT, QS>) : run(mma_kernel<KIND, 128, 1, QS>);
  else run(mma_kernel<KIND, 256, 1, QS>);
}

}  // namespace paged
}  // namespace mpc

using namespace mpc;

extern "C" {

int mpc_sdpa_paged_workspace(mpc_device *dev, const mpc_kv_desc *cache, const mpc_sdpa_paged_desc *desc, size_t *bytes) {
  int rc = enter(dev);
  if (rc) return rc;
  if (!cache || !desc || !bytes) return fail(MPC_ERR_INVALID, "mpc_sdpa_paged_workspace: null argument");
  paged::Plan a, b;
  if ((rc = paged::plan_of(dev, cache, desc, true, &a)) || (rc = paged::plan_of(dev, cache, desc, false, &b))) return rc;
  *bytes = a.ws_bytes > b.ws_bytes ? a.ws_bytes : b.ws_bytes;
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
  const bool aligned = (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0;
  Plan pl;
  if ((rc = plan_of(dev, cache, desc, aligned, &pl))) return rc;
  if (desc->b == 0) return MPC_OK;
  if (!Q || !O || !lengths || (desc->max_pages > 0 && !table) ||
      (cache->n_pages > 0 && (!k_pages || !v_pages || (cache->dtype == MPC_E4M3 && (!k_scale || !v_scale)))))
    return fail(MPC_ERR_INVALID, "mpc_sdpa_paged: null pointer");
  cudaStream_t st = stream_of(dev, s);
  Scratch own;
  int *counters = dev->d_counters;  // the device stream's, whose calls follow one another
  if (workspace) {
    if (workspace_bytes < pl.ws_bytes || ((uintptr_t)workspace & 15))
      return fail(MPC_ERR_INVALID, "mpc_sdpa_paged: a workspace of %zu bytes at %p (%zu, 16-byte aligned, needed)",
                  workspace_bytes, workspace, pl.ws_bytes);
    counters = static_cast<int *>(workspace);
  } else {
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    MPC_CUDA(dev, cudaStreamIsCapturing(st, &cs));
    if (cs != cudaStreamCaptureStatusNone)
      return fail(MPC_ERR_INVALID, "mpc_sdpa_paged: a captured call needs a workspace of its own");
    if ((rc = own.get(dev, st, pl.ws_bytes))) return rc;
    workspace = own.ptr;
    if (st != dev->stream || pl.counters_bytes > kCounterBytes) {
      counters = static_cast<int *>(workspace);
      MPC_CUDA(dev, cudaMemsetAsync(counters, 0, pl.counters_bytes, st));
    }
  }
  Params p{};
  p.q = Q, p.kp = k_pages, p.vp = v_pages, p.ks = k_scale, p.vs = v_scale, p.table = table, p.lengths = lengths;
  p.out = O, p.lse = LSE, p.tile = pl.tile, p.counters = counters;
  p.ws = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + pl.counters_bytes);
  if ((rc = report_word(dev, st, &p.report))) return rc;
  for (int i = 0; i < 2; ++i) p.qs[i] = desc->q_stride[i], p.os[i] = desc->o_stride[i];
  p.max_pages = desc->max_pages, p.cap = desc->max_pages * cache->page_size;
  p.B = (int)desc->b, p.H = (int)desc->h, p.hk = (int)cache->hk, p.group = p.H / p.hk, p.gt = pl.gt, p.qt = pl.qt;
  p.d = (int)cache->d, p.dv = (int)cache->dv, p.page_size = (int)cache->page_size, p.n_pages = (int)cache->n_pages;
  const size_t qb = dtype_size(desc->dtype);
  p.q_vec = (((uintptr_t)Q | desc->q_stride[0] * qb | desc->q_stride[1] * qb) & 15) == 0;
  // With 2^(l-1) < page_size <= 2^l and page_mul = ceil(2^(31+l) / page_size) (below 2^32), page_mul * page_size exceeds
  // 2^(31+l) by less than 2^l, so the quotient is exact for keys below 2^31.
  int l = 0;
  while ((1 << l) < p.page_size) ++l;
  p.page_shift = 31 + l, p.page_mul = (uint32_t)(((1ull << (31 + l)) + p.page_size - 1) / p.page_size);
  p.dt = desc->dtype, p.dt_pages = cache->dtype, p.scale_log2 = desc->scale * kLog2e;
  const bool vec = aligned && p.d % 8 == 0 && p.dv % 8 == 0;
  const int dm = p.d > p.dv ? p.d : p.dv;
  if (pl.dp && cache->dtype == MPC_F16) launch_mma<kF16, 1>(p, pl, st);
  else if (pl.dp && cache->dtype == MPC_BF16) launch_mma<kBF16, 1>(p, pl, st);
  else if (pl.dp && desc->dtype == MPC_F32) launch_mma<kE4M3, 2>(p, pl, st);
  else if (pl.dp) launch_mma<kE4M3, 1>(p, pl, st);
  else if (dm <= 64) vec ? launch_simt<1, true>(p, pl.ctas, st) : launch_simt<1, false>(p, pl.ctas, st);
  else if (dm <= 128) vec ? launch_simt<2, true>(p, pl.ctas, st) : launch_simt<2, false>(p, pl.ctas, st);
  else vec ? launch_simt<4, true>(p, pl.ctas, st) : launch_simt<4, false>(p, pl.ctas, st);
  dev->launches++;
  return check_launch(dev, "mpc_sdpa_paged");
}

}  // extern "C"
