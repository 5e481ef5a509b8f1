// What the kernels over the paged key/value cache share: the 8-bit format, element access and the
// record of a block-table entry outside the cache.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "../../include/mathplus_cuda.h"

namespace mpc {

// Checks of a cache descriptor (kv_cache.cu).
int kv_check(const char *what, const mpc_kv_desc *c);

// A report of a place outside the cache: the kind above the token or sequence, in one word, so that it is left and
// taken (mpc_runtime.cu) whole. A stream's first one stays until a synchronisation takes it.
enum : int { kBadAppendRead = 1, kBadAttend = 2, kBadLength = 3 };

__device__ __forceinline__ void report_bad_page(unsigned long long *report, int kind, int which) {
  atomicCAS(report, 0ull, (unsigned long long)kind << 32 | (unsigned)which);
}

// Two e4m3 numbers (low byte first) as f16x2, exactly.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
  uint32_t r;
  asm("{\n .reg .b16 t;\n cvt.u16.u32 t, %1;\n cvt.rn.f16x2.e4m3x2 %0, t;\n}\n" : "=r"(r) : "r"(two));
  return r;
}
// Four of them, as two f16x2.
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t four, uint32_t &lo, uint32_t &hi) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(four));
}
__device__ __forceinline__ float2 f16x2_to_f32(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
__device__ __forceinline__ float2 bf16x2_to_f32(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ uint32_t f32_to_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t f32_to_bf16x2(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void e4m3x4_to_f32(uint32_t v, float *x) {
  uint32_t lo, hi;
  e4m3x4_to_f16x4(v, lo, hi);
  const float2 a = f16x2_to_f32(lo), b = f16x2_to_f32(hi);
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}
// Round to nearest even, saturating at 448; NaN gives NaN.
__device__ __forceinline__ uint32_t f32_to_e4m3x2(float lo, float hi) {
  uint32_t r;
  asm("{\n .reg .b16 t;\n cvt.rn.satfinite.e4m3x2.f32 t, %2, %1;\n cvt.u32.u16 %0, t;\n}\n" : "=r"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ uint32_t f32_to_e4m3x4(const float *x) {
  return f32_to_e4m3x2(x[0], x[1]) | f32_to_e4m3x2(x[2], x[3]) << 16;
}
// 2^(byte - 127); the append writes 1..247, so 0 and 255 come only from pages filled elsewhere.
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte ? byte << 23 : 0x00400000u);
}

__device__ __forceinline__ float load_f32(const void *p, int dt, long long i) {
  switch (dt) {
    case MPC_F32:
      return static_cast<const float *>(p)[i];
    case MPC_BF16:
      return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    case MPC_F16:
      return __half2float(static_cast<const __half *>(p)[i]);
    default:
      return f16x2_to_f32(e4m3x2_to_f16x2(static_cast<const uint8_t *>(p)[i])).x;
  }
}
__device__ __forceinline__ void store_f32(void *p, int dt, long long i, float v) {
  switch (dt) {
    case MPC_F32:
      static_cast<float *>(p)[i] = v;
      break;
    case MPC_BF16:
      static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16(v);
      break;
    case MPC_F16:
      static_cast<__half *>(p)[i] = __float2half(v);
      break;
    default:
      static_cast<uint8_t *>(p)[i] = (uint8_t)f32_to_e4m3x2(v, 0.0f);
  }
}

// 8 values from index i of a row as stored, and as f32; with VEC the address is a multiple of 8 values.
struct Raw8 {
  uint32_t r[8];
};
__device__ __forceinline__ void load_raw8(const void *p, int dt, long long i, Raw8 &x) {
  if (dt == MPC_F32) {
    const uint4 *q = reinterpret_cast<const uint4 *>(static_cast<const float *>(p) + i);
    const uint4 a = q[0], b = q[1];
    x.r[0] = a.x, x.r[1] = a.y, x.r[2] = a.z, x.r[3] = a.w, x.r[4] = b.x, x.r[5] = b.y, x.r[6] = b.z, x.r[7] = b.w;
  } else if (dt == MPC_E4M3) {
    const uint2 v = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(p) + i);
    x.r[0] = v.x, x.r[1] = v.y;
  } else {
    const uint4 v = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i);
    x.r[0] = v.x, x.r[1] = v.y, x.r[2] = v.z, x.r[3] = v.w;
  }
}
__device__ __forceinline__ void widen8(const Raw8 &v, int dt, float (&x)[8]) {
  if (dt == MPC_F32) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = __uint_as_float(v.r[k]);
  } else if (dt == MPC_E4M3) {
    e4m3x4_to_f32(v.r[0], x);
    e4m3x4_to_f32(v.r[1], x + 4);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = dt == MPC_BF16 ? bf16x2_to_f32(v.r[k]) : f16x2_to_f32(v.r[k]);
      x[2 * k] = f.x, x[2 * k + 1] = f.y;
    }
  }
}
template <bool VEC>
__device__ __forceinline__ void load8(const void *p, int dt, long long i, int n, float (&x)[8]) {
  if constexpr (VEC) {
    Raw8 v;
    load_raw8(p, dt, i, v);
    widen8(v, dt, x);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = k < n ? load_f32(p, dt, i + k) : 0.0f;
  }
}

}  // namespace mpc
