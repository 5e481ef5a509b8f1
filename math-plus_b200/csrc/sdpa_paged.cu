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
// type (its rounding and the rest), which leaves 2^-16 (bf16) or less of it; one number alone would add
// as much error as the output's own rounding.
// The reference m of the exponentials is only raised when a score passes it by more than 2^kSlack: a warp
// vote per tile in the common case, the row maximum by shuffles and a rescaling of O else. It is set 2^kHead
// below the maximum so that small weights stay clear of f16's subnormals.
// 8-bit rows: codes convert exactly to f16; Q is scaled by a power of two per row to [2^14, 2^15), where any
// 16-bit q is exact in f16 down to 2^-28 of the row's largest (f32 q as two f16). K's scale multiplies the
// score. V's joins the weight: w = 2^(s' + e_v - M) with a reference M of its own, so that rows far below
// the largest scale keep their precision.
constexpr float kHead = 6.0f, kSlack = 14.0f;
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

// 8 values of a row as loaded: 4 registers of 16-bit pairs, or 2 of 8-bit codes.
template <int KIND>
struct Chunk {
  static constexpr int N = KIND == kE4M3 ? 2 : 4;
  uint32_t r[N];
  __device__ __forceinline__ void load(const void *base, uint32_t row, int d, int at) {
    const bool there = row != kNoRow && at < d;
    if constexpr (KIND == kE4M3) {
      uint2 v = make_uint2(0, 0);
      if (there) v = __ldg(reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(base) + (size_t)row * d + at));
      r[0] = v.x, r[1] = v.y;
    } else {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (there) v = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + (size_t)row * d + at));
      r[0] = v.x, r[1] = v.y, r[2] = v.z, r[3] = v.w;
    }
  }
  // Values 2i and 2i + 1 as a pair.
  __device__ __forceinline__ uint32_t pair(int i) const {
    if constexpr (KIND == kE4M3) return e4m3x2_to_f16x2((i & 1) ? r[i >> 1] >> 16 : r[i >> 1] & 0xffffu);
    else return r[i];
  }
};
// Value 2i (a0) and 2i + 1 (a1) of two neighbouring keys, as pairs (key, next key).
template <int KIND>
__device__ __forceinline__ void key_pairs(const Chunk<KIND> &x, const Chunk<KIND> &y, int i, uint32_t &a0, uint32_t &a1) {
  if constexpr (KIND == kE4M3) {
    const uint32_t t = prmt(x.r[i >> 1], y.r[i >> 1], (i & 1) ? 0x7362u : 0x5140u);
    a0 = e4m3x2_to_f16x2(t & 0xffffu);
    a1 = e4m3x2_to_f16x2(t >> 16);
  } else {
    a0 = prmt(x.r[i], y.r[i], 0x5410u);
    a1 = prmt(x.r[i], y.r[i], 0x7632u);
  }
}

// DP: head dims padded to 64, 128 or 256; NT: tiles of 8 query heads; QS: numbers per query value.
template <int KIND, int DP, int NT, int QS>
__global__ void __launch_bounds__(kThreads, DP == 256 || NT == 2 ? 2 : 3) mma_kernel(const Params p) {
  constexpr bool BF = KIND == kBF16, Q8 = KIND == kE4M3;
  constexpr int KC = DP / 32, VC = DP / 64, GT = 8 * NT, PITCH = DP + 8, WARPS = kThreads / 32;
  __shared__ float so[WARPS][GT][PITCH];
  __shared__ float sml[WARPS][GT][3];
  __shared__ long long sm[WARPS], found[2];
  empty_rows(p);
  const Run run = run_of(p, blockIdx.x, gridDim.x, sm);
  if (run.g0 >= run.g1) return;
  Item it = item_of(p, run.g0, sm, found);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;

  for (long long g = run.g0; g < run.g1;) {
    const long long c1 = min(it.chunks, it.chunk + (run.g1 - g));
    const int kvh = it.head / p.qt, h0 = kvh * p.group + (it.head % p.qt) * GT;
    const int nq = min(GT, (kvh + 1) * p.group - h0);
    const unsigned end = (unsigned)min(length_of(p, it.b), c1 * kChunk);  // lengths are below 2^31
    const int32_t *table = p.table + it.b * p.max_pages;

    // The row of this lane's key (lane % 16) in the tile of keys from k0 on.
    auto row_at = [&](unsigned k0) -> uint32_t {
      const unsigned key = k0 + (lane & 15);
      if (key >= end) return kNoRow;
      const unsigned col = key / (unsigned)p.page_size;
      const int pg = __ldg(table + col);
      if (pg < 0 || pg >= p.n_pages) {
        report_bad_page(p.err, kBadAttend, it.b);
        return kNoRow;
      }
      return ((unsigned)pg * (unsigned)p.hk + kvh) * (unsigned)p.page_size + (key - col * (unsigned)p.page_size);
    };
    Chunk<KIND> kf[2][KC], vf[4][VC];
    uint32_t ks = 127, vs = 127;  // scale bytes of this lane's key
    auto load_k = [&](uint32_t row) {
      const uint32_t ra = __shfl_sync(0xffffffffu, row, r), rb = __shfl_sync(0xffffffffu, row, r + 8);
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        kf[0][j].load(p.kp, ra, p.d, 32 * j + 8 * c);
        kf[1][j].load(p.kp, rb, p.d, 32 * j + 8 * c);
      }
      if constexpr (Q8) ks = row != kNoRow ? p.ks[row] : 127;
    };
    auto load_v = [&](uint32_t row) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t rk = __shfl_sync(0xffffffffu, row, 2 * c + (k & 1) + (k >> 1) * 8);
#pragma unroll
        for (int j = 0; j < VC; ++j) vf[k][j].load(p.vp, rk, p.dv, 64 * j + 8 * r);
      }
      if constexpr (Q8) vs = row != kNoRow ? p.vs[row] : 127;
    };

    unsigned k0 = (unsigned)(it.chunk * kChunk) + warp * 16;
    uint32_t row = row_at(k0), next = row_at(k0 + 16 * WARPS);
    load_k(row);
    load_v(row);

    // Q^T: lane (r, c) holds values 32 j + 8 c ..+7 of query head r of each tile.
    uint32_t qf[NT][QS][KC][4];
    float qscale[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bool live = n * 8 + r < nq;
      const long long base = it.b * p.qs[0] + (h0 + n * 8 + r) * p.qs[1];
      if constexpr (!Q8) {
#pragma unroll
        for (int j = 0; j < KC; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = 32 * j + 8 * c + 2 * i;
            const uint16_t *q = static_cast<const uint16_t *>(p.q) + base + at;
            qf[n][0][j][i] = live && at < p.d ? (uint32_t)q[0] | (uint32_t)q[1] << 16 : 0u;
          }
        qscale[n][0] = qscale[n][1] = p.scale_log2;
      } else {
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < KC; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int at = 32 * j + 8 * c + i;
            if (live && at < p.d) {
              const uint32_t a = __float_as_uint(load_f32(p.q, p.dt, base + at)) & 0x7fffffffu;
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
            const int at = 32 * j + 8 * c + 2 * i;
            float x0 = 0.0f, x1 = 0.0f;
            if (live && at < p.d) x0 = load_f32(p.q, p.dt, base + at) * f0 * f1, x1 = load_f32(p.q, p.dt, base + at + 1) * f0 * f1;
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
      for (int i = 0; i < 2; ++i) m[n][i] = mo[n][i] = -INFINITY, l[n][i] = 0.0f;
#pragma unroll
      for (int j = 0; j < VC; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][j][i][e] = 0.0f;
    }

    for (; k0 < end; k0 += 16 * WARPS) {
      // S^T: s[n][0..1] key r, heads 2c, 2c + 1; s[n][2..3] key r + 8.
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
#pragma unroll
      for (int j = 0; j < KC; ++j)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const uint32_t a0 = kf[0][j].pair(i), a1 = kf[1][j].pair(i), a2 = kf[0][j].pair(i + 1), a3 = kf[1][j].pair(i + 1);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int q = 0; q < QS; ++q) mma<BF>(s[n], a0, a1, a2, a3, qf[n][q][j][i], qf[n][q][j][i + 1]);
        }
      const bool see[2] = {__shfl_sync(0xffffffffu, row, r) != kNoRow, __shfl_sync(0xffffffffu, row, r + 8) != kNoRow};
      float fk[2] = {1.0f, 1.0f}, ev[2] = {0.0f, 0.0f};
      if constexpr (Q8) {
        fk[0] = scale_value(__shfl_sync(0xffffffffu, ks, r)), fk[1] = scale_value(__shfl_sync(0xffffffffu, ks, r + 8));
        ev[0] = (float)((int)__shfl_sync(0xffffffffu, vs, r) - 127), ev[1] = (float)((int)__shfl_sync(0xffffffffu, vs, r + 8) - 127);
      }
      load_k(next);

      bool raise = false;
      float top[NT][2], otop[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = see[e >> 1] ? s[n][e] * (qscale[n][e & 1] * fk[e >> 1]) : -INFINITY;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          top[n][i] = fmaxf(s[n][i], s[n][2 + i]);
          raise |= top[n][i] > m[n][i] + kSlack;
          if constexpr (Q8) {
            otop[n][i] = fmaxf(s[n][i] + ev[0], s[n][2 + i] + ev[1]);
            raise |= otop[n][i] > mo[n][i] + kSlack;
          }
        }
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int k = 4; k < 32; k <<= 1) top[n][i] = fmaxf(top[n][i], __shfl_xor_sync(0xffffffffu, top[n][i], k));
            const float up = fmaxf(m[n][i], top[n][i] - kHead);
            l[n][i] *= guard_exp2(m[n][i], up);
            float keep = guard_exp2(m[n][i], up);
            m[n][i] = up;
            if constexpr (Q8) {
#pragma unroll
              for (int k = 4; k < 32; k <<= 1) otop[n][i] = fmaxf(otop[n][i], __shfl_xor_sync(0xffffffffu, otop[n][i], k));
              const float oup = fmaxf(mo[n][i], otop[n][i] - kHead);
              keep = guard_exp2(mo[n][i], oup);
              mo[n][i] = oup;
            }
#pragma unroll
            for (int j = 0; j < VC; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[n][j][e][i] *= keep, o[n][j][e][2 + i] *= keep;
          }
      }
      // P^T: b0 keys 2c, 2c + 1 and b1 keys 2c + 8, 2c + 9 of head r, as two numbers each.
      uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = guard_exp2(s[n][e], m[n][e & 1]);
          l[n][e & 1] += w[e];
          if constexpr (Q8) w[e] = guard_exp2(s[n][e], mo[n][e & 1] - ev[e >> 1]);
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
          key_pairs<KIND>(vf[0][j], vf[1][j], i, a0, a1);
          key_pairs<KIND>(vf[2][j], vf[3][j], i, a2, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma<BF>(o[n][j][i], a0, a1, a2, a3, hi[n][0], hi[n][1]);
            mma<BF>(o[n][j][i], a0, a1, a2, a3, lo[n][0], lo[n][1]);
          }
        }
      load_v(next);
      row = next;
      next = row_at(k0 + 2 * 16 * WARPS);
    }

    // The warps meet in shared memory. o[n][j][i]: columns 64 j + 8 r + 2 i (e < 2) and + 1, heads 2c, 2c + 1.
    __syncthreads();  // the last item's shared arrays are free
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
    __syncthreads();
    const bool whole = it.chunk == 0 && c1 == it.chunks;
    for (int i = threadIdx.x; i < nq * DP; i += kThreads) {
      const int q = i / DP, e = i % DP;
      float top = -INFINITY, otop = -INFINITY, sum = 0.0f, v = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sml[w][q][0]), otop = fmaxf(otop, sml[w][q][1]);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        sum = fmaf(sml[w][q][2], guard_exp2(sml[w][q][0], top), sum);
        v = fmaf(so[w][q][e], guard_exp2(sml[w][q][1], otop), v);
      }
      if (whole) {
        if (e < p.dv)
          store_f32(p.out, p.dt, it.b * p.os[0] + (h0 + q) * p.os[1] + e, sum != 0.0f ? v * exp2f(otop - top) / sum : 0.0f);
        if (p.lse && e == 0) p.lse[(long long)it.b * p.H + h0 + q] = sum != 0.0f ? fmaf(top, kLn2, logf(sum)) : -INFINITY;
      } else {
        float *ws = slot(p, blockIdx.x, it.chunk == 0, q);
        if (e < p.dv) ws[4 + e] = v;
        if (e == 0) ws[0] = top, ws[1] = otop, ws[2] = sum;
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
  int dp;  // padded head dim of the tensor-core kernel, 0: the CUDA cores
  size_t ws_bytes;
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
  const bool tc = aligned && c->dtype != MPC_F32 && c->d % 8 == 0 && c->dv % 8 == 0 &&
                  c->n_pages * c->page_size < (int64_t)kNoRow / c->hk;
  const bool two = c->dtype == MPC_E4M3 && d->dtype == MPC_F32;  // two f16 per query value: no registers for 16 heads
  pl->dp = !tc ? 0 : dm <= 64 ? 64 : dm <= 128 ? 128 : 256;
  pl->gt = tc ? (group > 8 && pl->dp < 256 && !two ? 16 : 8) : group >= 4 ? 4 : group >= 2 ? 2 : 1;
  pl->qt = (int)((group + pl->gt - 1) / pl->gt);
  // As many CTAs as are resident, fewer where even the longest lengths give fewer chunks.
  const long long per = (d->max_pages * c->page_size + kChunk - 1) / kChunk;
  const long long sms = (long long)dev->prop.multiProcessorCount * (tc && (pl->dp == 256 || pl->gt == 16) ? 2 : 3);
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
  if ((rc = check_launch(dev, "mpc_sdpa_paged"))) return rc;
  join_kernel<<<dim3(pl.ctas, pl.gt), kThreads, 0, st>>>(p, pl.ctas);
  dev->launches++;
  return check_launch(dev, "mpc_sdpa_paged join");
}

}  // extern "C"
