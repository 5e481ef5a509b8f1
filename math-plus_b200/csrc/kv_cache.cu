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
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kv_cache.cuh"
#include "mpc_internal.h"

namespace mpc {
namespace {

constexpr int kThreads = 256;

struct KvParams {
  void *pages[2];      // K, V
  uint8_t *scales[2];  // one byte per row (MPC_E4M3), else null
  void *rows[2];       // the tokens' dense K, V rows (source of an append, destination of a read)
  long long ts[2], hs[2];  // element strides of the rows' token and head axes
  const int32_t *table, *seq, *pos;
  int *err;
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
    if (first) report_bad_page(p.err, kBadAppendRead, (int)t);
    return false;
  }
  *page = pg;
  *off = pos - (int)col * p.page_size;
  return true;
}

// One group of LPR lanes per token, walking the heads blockIdx.y, + gridDim.y, ..
template <int LPR, bool VEC, bool APPEND>
__global__ void __launch_bounds__(kThreads) kv_rows_kernel(const KvParams p) {
  const int lane = threadIdx.x % LPR;
  const int groups = kThreads / LPR;
  for (long long t0 = (long long)blockIdx.x * groups; t0 < p.n; t0 += (long long)gridDim.x * groups) {
    const long long t = t0 + threadIdx.x / LPR;  // lanes of a group agree; a group past the end only shuffles
    long long page = 0;
    int off = 0;
    const bool live = t < p.n;
    const bool ok = live && locate(p, t, &page, &off, lane == 0 && blockIdx.y == 0);
    for (int h = blockIdx.y; h < p.hk; h += gridDim.y) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int d = p.d[w];
        const bool mine = lane * 8 < d;
        const long long row = (page * p.hk + h) * p.page_size + off;
        const long long at = row * d + lane * 8;
        const long long src = t * p.ts[w] + h * p.hs[w] + lane * 8;
        float x[8];
        if constexpr (APPEND) {
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = 0.0f;
          if (ok && mine) load8<VEC>(p.rows[w], p.dt_rows, src, d - lane * 8, x);
          if (p.dt_pages == MPC_E4M3) {
            uint32_t amax = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint32_t a = __float_as_uint(x[k]) & 0x7fffffffu;
              if (a < 0x7f800000u) amax = max(amax, a);
            }
#pragma unroll
            for (int m = LPR / 2; m; m >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, m));
            const int sb = scale_byte(amax);
            const float inv = __uint_as_float((uint32_t)(254 - sb) << 23);  // 2^-(sb - 127): sb in 1..247
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] *= inv;
            if (ok && lane == 0) p.scales[w][row] = (uint8_t)sb;
          }
          if (ok && mine) store8<VEC>(p.pages[w], p.dt_pages, at, d - lane * 8, x);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = 0.0f;
          if (ok && mine) {
            load8<VEC>(p.pages[w], p.dt_pages, at, d - lane * 8, x);
            if (p.dt_pages == MPC_E4M3) {
              const float s = scale_value(p.scales[w][row]);
#pragma unroll
              for (int k = 0; k < 8; ++k) x[k] *= s;
            }
          }
          if (live && mine) store8<VEC>(p.rows[w], p.dt_rows, src, d - lane * 8, x);
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
  p.table = table, p.seq = seq, p.pos = pos, p.err = dev->d_err;
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
  auto run = [&](auto kern) { kern<<<grid, kThreads, 0, st>>>(p); };
  if (lpr == 8) vec ? run(kv_rows_kernel<8, true, APPEND>) : run(kv_rows_kernel<8, false, APPEND>);
  else if (lpr == 16) vec ? run(kv_rows_kernel<16, true, APPEND>) : run(kv_rows_kernel<16, false, APPEND>);
  else vec ? run(kv_rows_kernel<32, true, APPEND>) : run(kv_rows_kernel<32, false, APPEND>);
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
