// The paged key/value cache: writing tokens into it (mpc_kv_append) and reading them back
// (mpc_kv_read). It has no counterpart in the reference, whose MultiheadAttention recomputes K and V of
// the whole sequence (packages/tensor-autograd/src/transformer.ts:173-242).
//
// Layout: K pages [n_pages, hk, page_size, d], V pages [n_pages, hk, page_size, dv]; one page of one
// head is one contiguous block, so attention over the cache streams it. Token t of sequence seq[t]
// at position pos[t] lives in page table[seq[t], pos[t] / page_size], row pos[t] % page_size.
//
// 8-bit rows (MPC_E4M3): with a = max |x_d| over the row's finite values, e the least integer in
// [-126, 127] with a <= 448 * 2^e, the row is stored as e4m3(x_d * 2^-e) (round to nearest even,
// saturating, NaN kept) and the byte e + 127. A power of two makes the scaling exact both ways:
// the only rounding is the 8-bit one, at most 2^-4 of the value (2^-10 * 2^e below 2^-6 * 2^e), and a
// row that is read and appended again keeps its values. One byte per row costs 1/d of the codes,
// a 32-bit scale four times that.
//
// Both directions are bound by HBM. A row of up to 256 values is one group of 8, 16 or 32 lanes,
// 8 values (16 bytes of a 16-bit type) per lane, so that the row's maximum is a few shuffles and the
// row is read once; a group keeps its token's place over the heads it walks.
//
// Measured (GPU time of a replayed call): 32768 tokens of 8 heads of 128, bf16 to 8 bits, 38.3 us (5.1 TB/s); 49152
// such tokens from 8 bits to bf16 54.4 us (5.6 TB/s), of a measured copy rate of 6.55; 8 tokens of 12 heads of 64, bf16,
// 2.5 us, where a chain of latencies bounds it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "kv_cache.cuh"
#include "mpc_internal.h"

namespace mpc {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ void store_raw8(void *p, int dt, long long i, const Raw8 &x, bool zero) {
  Raw8 y;
#pragma unroll
  for (int k = 0; k < 8; ++k) y.r[k] = zero ? 0u : x.r[k];
  if (dt == MPC_F32) {
    uint4 *q = reinterpret_cast<uint4 *>(static_cast<float *>(p) + i);
    q[0] = make_uint4(y.r[0], y.r[1], y.r[2], y.r[3]);
    q[1] = make_uint4(y.r[4], y.r[5], y.r[6], y.r[7]);
  } else {
    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p) + i) = make_uint4(y.r[0], y.r[1], y.r[2], y.r[3]);
  }
}

struct KvParams {
  void *pages[2];      // K, V
  uint8_t *scales[2];  // one byte per row (MPC_E4M3), else null
  void *rows[2];       // the tokens' dense K, V rows (source of an append, destination of a read)
  long long ts[2], hs[2];  // element strides of the rows' token and head axes
  const int32_t *table, *seq, *pos;
  unsigned long long *report;
  int d[2];
  int n, n_seq, hk, page_size, n_pages, dt_rows, dt_pages;
  long long max_pages;
};

template <bool VEC>
__device__ __forceinline__ void store8(void *p, int dt, long long i, int n, const float (&x)[8]) {
  if constexpr (VEC) {
    if (dt == MPC_F32) {
      float4 *q = reinterpret_cast<float4 *>(static_cast<float *>(p) + i);
      q[0] = make_float4(x[0], x[1], x[2], x[3]);
      q[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else if (dt == MPC_E4M3) {
      *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(p) + i) =
          make_uint2(f32_to_e4m3x4(x), f32_to_e4m3x4(x + 4));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        w[k] = dt == MPC_BF16 ? f32_to_bf16x2(x[2 * k], x[2 * k + 1]) : f32_to_f16x2(x[2 * k], x[2 * k + 1]);
      *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) store_f32(p, dt, i + k, x[k]);
  }
}

// The scale byte of a row: the least e with amax <= 448 * 2^e = 1.75 * 2^(e + 8), biased by 127 and
// clamped to the exponents whose power of two and its inverse are normal numbers.
__device__ __forceinline__ int scale_byte(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < 1 ? 1 : e;
}

// Where token t lives, or false: padding (pos < 0, nothing recorded), or a sequence, position or
// page outside the cache (recorded in the device's error words, the token left out).
__device__ __forceinline__ bool locate(const KvParams &p, long long t, long long *page, int *off, bool first) {
  const int pos = p.pos[t];
  if (pos < 0) return false;
  const int seq = p.seq ? p.seq[t] : (int)t;
  const long long col = pos / p.page_size;
  int pg = -1;
  if (seq >= 0 && seq < p.n_seq && col < p.max_pages) pg = p.table[(long long)seq * p.max_pages + col];
  if (pg < 0 || pg >= p.n_pages) {
    if (first) report_bad_page(p.report, kBadAppendRead, (int)t);
    return false;
  }
  *page = pg;
  *off = pos - (int)col * p.page_size;
  return true;
}

// The largest magnitude of a row's finite values, as f32 bits, over the LPR lanes of its group. Magnitudes compare as
// their bits, two 16-bit ones at a time; a row with a NaN or an infinity (the largest bits of all) is gone through again.
template <int LPR>
__device__ __forceinline__ uint32_t row_amax(const Raw8 &v, int dt, bool mine) {
  uint32_t m = 0, end;  // from `end` on: not finite
  if (dt == MPC_F32) {
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, v.r[k] & 0x7fffffffu);
    end = 0x7f800000u;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) m = __vmaxu2(m, v.r[k] & 0x7fff7fffu);
    m = max(m & 0xffffu, m >> 16);
    end = dt == MPC_BF16 ? 0x7f80u : 0x7c00u;
  }
  if (!mine) m = 0;
#pragma unroll
  for (int i = LPR / 2; i; i >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, i));
  if (__any_sync(0xffffffffu, m >= end)) {
    m = 0;
    if (mine) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t a = dt == MPC_F32 ? v.r[k] & 0x7fffffffu : (v.r[k >> 1] >> (16 * (k & 1))) & 0x7fffu;
        if (a < end) m = max(m, a);
      }
    }
#pragma unroll
    for (int i = LPR / 2; i; i >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, i));
  }
  return dt == MPC_F32 ? m : dt == MPC_BF16 ? m << 16 : __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
}

// One group of LPR lanes per token, walking the heads blockIdx.y, + gridDim.y, .. With VEC the K and V rows of H heads
// are loaded before any is used, whether the token is written or not.
// DR, DP: the types of the rows and the pages; kAny: as the parameters say (the fixed ones save a third of the
// instructions, which bound the 8-bit forms next to HBM).
constexpr int kAny = -1;
template <int LPR, bool VEC, int H, bool APPEND, int DR, int DP>
__global__ void __launch_bounds__(kThreads) kv_rows_kernel(const KvParams p) {
  const int dt_rows = DR == kAny ? p.dt_rows : DR, dt_pages = DP == kAny ? p.dt_pages : DP;
  const int lane = threadIdx.x % LPR;
  const int groups = kThreads / LPR;
  for (long long t0 = (long long)blockIdx.x * groups; t0 < p.n; t0 += (long long)gridDim.x * groups) {
    const long long t = t0 + threadIdx.x / LPR;  // lanes of a group agree; a group past the end only shuffles
    long long page = 0;
    int off = 0;
    const bool live = t < p.n;
    const bool ok = live && locate(p, t, &page, &off, lane == 0 && blockIdx.y == 0);
    const long long row0 = page * p.hk * p.page_size + off;  // of head 0
    const bool any = APPEND || p.n_pages > 0;                // an empty cache has no row to read in place of a bad one
    const long long tt = live ? t : p.n - 1;
    // This lane's 8 values of head h: rows_at + h * hs, pages_at + h * step.
    long long rows_at[2], pages_at[2];
    int step[2];
    bool mine[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      mine[w] = lane * 8 < p.d[w];
      const int at = mine[w] ? lane * 8 : 0;
      rows_at[w] = tt * p.ts[w] + at, pages_at[w] = row0 * p.d[w] + at, step[w] = p.page_size * p.d[w];
    }
    for (int h0 = blockIdx.y; h0 < p.hk; h0 += H * gridDim.y) {
      Raw8 raw[H][2];
      uint32_t byte[H][2];
      if constexpr (VEC) {
#pragma unroll
        for (int u = 0; u < H; ++u)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int h = H == 1 ? h0 : min(h0 + u * (int)gridDim.y, p.hk - 1);
            if (APPEND) {
              load_raw8(p.rows[w], dt_rows, rows_at[w] + h * p.hs[w], raw[u][w]);
            } else if (any) {
              load_raw8(p.pages[w], dt_pages, pages_at[w] + (long long)h * step[w], raw[u][w]);
              if (dt_pages == MPC_E4M3) byte[u][w] = p.scales[w][row0 + (long long)h * p.page_size];
            }
          }
      }
#pragma unroll
      for (int u = 0; u < H; ++u) {
        const int h = h0 + u * (int)gridDim.y;
        if (H > 1 && h >= p.hk) break;  // the same for the whole block
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int n = p.d[w] - lane * 8;
          const long long in_rows = rows_at[w] + h * p.hs[w], in_pages = pages_at[w] + (long long)h * step[w];
          if constexpr (VEC) {
            if (dt_pages == dt_rows) {  // as they are
              if (APPEND ? ok && mine[w] : live && mine[w])
                store_raw8(APPEND ? p.pages[w] : p.rows[w], dt_rows, APPEND ? in_pages : in_rows, raw[u][w], !ok);
              continue;
            }
          }
          float x[8];
          if constexpr (APPEND) {
            if constexpr (!VEC) {
#pragma unroll
              for (int k = 0; k < 8; ++k) x[k] = 0.0f;
              if (ok && mine[w]) load8<false>(p.rows[w], dt_rows, in_rows, n, x);
            }
            if (dt_pages == MPC_E4M3) {
              uint32_t amax = 0;
              if constexpr (VEC) {
                amax = row_amax<LPR>(raw[u][w], dt_rows, mine[w]);
                widen8(raw[u][w], dt_rows, x);
              } else {
                Raw8 v;
#pragma unroll
                for (int k = 0; k < 8; ++k) v.r[k] = __float_as_uint(x[k]);
                amax = row_amax<LPR>(v, MPC_F32, mine[w]);
              }
              const int sb = scale_byte(amax);
              const float inv = __uint_as_float((uint32_t)(254 - sb) << 23);  // 2^-(sb - 127): sb in 1..247
#pragma unroll
              for (int k = 0; k < 8; ++k) x[k] *= inv;
              if (ok && lane == 0) p.scales[w][row0 + (long long)h * p.page_size] = (uint8_t)sb;
            }
            if (ok && mine[w]) store8<VEC>(p.pages[w], dt_pages, in_pages, n, x);
          } else {
            if constexpr (VEC) {
              widen8(raw[u][w], dt_pages, x);
              const float s = dt_pages == MPC_E4M3 ? scale_value(byte[u][w]) : 1.0f;
#pragma unroll
              for (int k = 0; k < 8; ++k) x[k] = ok ? x[k] * s : 0.0f;
            } else {
#pragma unroll
              for (int k = 0; k < 8; ++k) x[k] = 0.0f;
              if (ok && mine[w]) {
                load8<false>(p.pages[w], dt_pages, in_pages, n, x);
                const float s = dt_pages == MPC_E4M3 ? scale_value(p.scales[w][row0 + (long long)h * p.page_size]) : 1.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] *= s;
              }
            }
            if (live && mine[w]) store8<VEC>(p.rows[w], dt_rows, in_rows, n, x);
          }
        }
      }
    }
  }
}

template <bool APPEND>
int kv_run(mpc_device *dev, const char *what, const mpc_kv_desc *c, void *k_pages, void *v_pages, uint8_t *k_scale,
           uint8_t *v_scale, const mpc_kv_tokens *t, void *k, void *v, const int32_t *table, const int32_t *seq,
           const int32_t *pos, cudaStream_t st) {
  if (!c || !t) return fail(MPC_ERR_INVALID, "%s: null descriptor", what);
  int rc = kv_check(what, c);
  if (rc) return rc;
  if (t->dtype < MPC_F32 || t->dtype > MPC_BF16)
    return fail(MPC_ERR_INVALID, "%s: rows of dtype %d (f32, f16 or bf16)", what, t->dtype);
  if (APPEND && c->dtype != MPC_E4M3 && c->dtype != t->dtype)
    return fail(MPC_ERR_INVALID, "%s: rows of dtype %d into a cache of dtype %d", what, t->dtype, c->dtype);
  if (t->n < 0 || t->n_seq < 0 || t->max_pages < 0 || t->n > INT32_MAX || t->n_seq > INT32_MAX ||
      t->max_pages > INT32_MAX)
    return fail(MPC_ERR_INVALID, "%s: bad extents n=%lld n_seq=%lld max_pages=%lld", what, (long long)t->n,
                (long long)t->n_seq, (long long)t->max_pages);
  for (int64_t s : {t->k_stride[0], t->k_stride[1], t->v_stride[0], t->v_stride[1]})
    if (s < 0) return fail(MPC_ERR_INVALID, "%s: negative stride", what);
  if (!seq && t->n > t->n_seq)
    return fail(MPC_ERR_INVALID, "%s: %lld tokens for %lld sequences need their sequence indices", what,
                (long long)t->n, (long long)t->n_seq);
  if (t->n == 0) return MPC_OK;
  if (!k || !v || !k_pages || !v_pages || !table || !pos) return fail(MPC_ERR_INVALID, "%s: null pointer", what);
  if (c->dtype == MPC_E4M3 && (!k_scale || !v_scale))
    return fail(MPC_ERR_INVALID, "%s: an 8-bit cache needs its scale pages", what);
  KvParams p{};
  p.pages[0] = k_pages, p.pages[1] = v_pages, p.scales[0] = k_scale, p.scales[1] = v_scale;
  p.rows[0] = k, p.rows[1] = v;
  p.ts[0] = t->k_stride[0], p.hs[0] = t->k_stride[1], p.ts[1] = t->v_stride[0], p.hs[1] = t->v_stride[1];
  p.table = table, p.seq = seq, p.pos = pos;
  if ((rc = report_word(dev, st, &p.report))) return rc;
  p.d[0] = (int)c->d, p.d[1] = (int)c->dv;
  p.n = (int)t->n, p.n_seq = (int)t->n_seq, p.hk = (int)c->hk, p.page_size = (int)c->page_size;
  p.n_pages = (int)c->n_pages, p.max_pages = t->max_pages, p.dt_rows = t->dtype, p.dt_pages = c->dtype;
  const size_t eb = dtype_size(t->dtype);
  bool vec = c->d % 8 == 0 && c->dv % 8 == 0;
  for (int w = 0; w < 2; ++w)
    vec = vec && ((p.ts[w] * eb) | (p.hs[w] * eb) | (uintptr_t)p.rows[w] | (uintptr_t)p.pages[w]) % 16 == 0;
  const int64_t dm = c->d > c->dv ? c->d : c->dv;
  const int lpr = dm <= 64 ? 8 : dm <= 128 ? 16 : 32;
  const long long per = kThreads / lpr;
  const long long gx = (t->n + per - 1) / per;
  // Two waves of eight resident blocks an SM; few tokens spread over the heads instead.
  const long long want = (long long)dev->prop.multiProcessorCount * 16;
  const unsigned bx = (unsigned)(gx < want ? gx : want);
  long long gy = want / bx;
  gy = gy > c->hk ? c->hk : gy;
  const dim3 grid(bx, (unsigned)(gy < 1 ? 1 : gy > 65535 ? 65535 : gy));
  const bool two = vec && 2ll * grid.y <= c->hk;  // a block walks several heads: two at a time
  auto run = [&](auto kern) { kern<<<grid, kThreads, 0, st>>>(p); };
  auto pick = [&](auto width) {
    constexpr int LPR = decltype(width)::value;
    auto fixed = [&](auto rows, auto pages) {
      constexpr int R = decltype(rows)::value, P = decltype(pages)::value;
      two ? run(kv_rows_kernel<LPR, true, 2, APPEND, R, P>) : run(kv_rows_kernel<LPR, true, 1, APPEND, R, P>);
    };
    using std::integral_constant;
    const integral_constant<int, MPC_F32> f32;
    const integral_constant<int, MPC_F16> f16;
    const integral_constant<int, MPC_BF16> bf16;
    const integral_constant<int, MPC_E4M3> e4m3;
    const integral_constant<int, kAny> any;
    if (!vec) run(kv_rows_kernel<LPR, false, 1, APPEND, kAny, kAny>);
    else if (t->dtype == c->dtype) t->dtype == MPC_F32 ? fixed(f32, f32) : fixed(bf16, bf16);  // a copy: f16 alike
    else if (c->dtype != MPC_E4M3) fixed(any, any);
    else if (t->dtype == MPC_F32) fixed(f32, e4m3);
    else if (t->dtype == MPC_F16) fixed(f16, e4m3);
    else fixed(bf16, e4m3);
  };
  if (lpr == 8) pick(std::integral_constant<int, 8>());
  else if (lpr == 16) pick(std::integral_constant<int, 16>());
  else pick(std::integral_constant<int, 32>());
  dev->launches++;
  return check_launch(dev, what);
}

}  // namespace

int kv_check(const char *what, const mpc_kv_desc *c) {
  if (c->n_pages < 0 || c->page_size <= 0 || c->hk <= 0 || c->d <= 0 || c->dv <= 0)
    return fail(MPC_ERR_INVALID, "%s: bad cache n_pages=%lld page_size=%lld hk=%lld d=%lld dv=%lld", what,
                (long long)c->n_pages, (long long)c->page_size, (long long)c->hk, (long long)c->d, (long long)c->dv);
  if (c->d > 256 || c->dv > 256) return fail(MPC_ERR_UNSUPPORTED, "%s: head dim above 256", what);
  if (c->n_pages > INT32_MAX || c->page_size > (1 << 20) || c->hk > 65535)
    return fail(MPC_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 pages, 2^20 rows a page or 65535 heads", what);
  if (c->dtype < MPC_F32 || (c->dtype > MPC_BF16 && c->dtype != MPC_E4M3))
    return fail(MPC_ERR_INVALID, "%s: cache of dtype %d (f32, f16, bf16 or e4m3)", what, c->dtype);
  return MPC_OK;
}

}  // namespace mpc

using namespace mpc;

extern "C" {

int mpc_kv_append(mpc_device *dev, const mpc_kv_desc *cache, void *k_pages, void *v_pages, uint8_t *k_scale,
                  uint8_t *v_scale, const mpc_kv_tokens *tokens, const void *k, const void *v, const int32_t *table,
                  const int32_t *seq, const int32_t *pos, mpc_stream s) {
  int rc = enter(dev);
  if (rc) return rc;
  return kv_run<true>(dev, "mpc_kv_append", cache, k_pages, v_pages, k_scale, v_scale, tokens, const_cast<void *>(k),
                      const_cast<void *>(v), table, seq, pos, stream_of(dev, s));
}

int mpc_kv_read(mpc_device *dev, const mpc_kv_desc *cache, const void *k_pages, const void *v_pages,
                const uint8_t *k_scale, const uint8_t *v_scale, const mpc_kv_tokens *tokens, void *k, void *v,
                const int32_t *table, const int32_t *seq, const int32_t *pos, mpc_stream s) {
  int rc = enter(dev);
  if (rc) return rc;
  return kv_run<false>(dev, "mpc_kv_read", cache, const_cast<void *>(k_pages), const_cast<void *>(v_pages),
                       const_cast<uint8_t *>(k_scale), const_cast<uint8_t *>(v_scale), tokens, k, v, table, seq, pos,
                       stream_of(dev, s));
}

}  // extern "C"
