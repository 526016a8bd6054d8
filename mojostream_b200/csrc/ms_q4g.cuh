// ms_q4g.cuh -- device helpers shared by the kernels of group-scaled 4-bit
// products (ms_q4g.cu, ms_q4g_tc.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ms_common.cuh"
#include "ms_q4g.h"

namespace ms {

__device__ __forceinline__ float u16_scale(uint32_t u, int bf) {
  return bf ? __uint_as_float(u << 16) : __half2float(__ushort_as_half((unsigned short)u));
}

// Shared-memory loads by 32-bit address.
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  uint32_t v;
  asm volatile("{\n .reg .u16 h;\n ld.shared.u16 h, [%1];\n cvt.u32.u16 %0, h;\n}" : "=r"(v) : "r"(a));
  return v;
}

// Eight consecutive values of a row (zeros past K, a multiple of 32).
__device__ __forceinline__ void load8(const Q4gRows& a, int m, int k, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = 0.f;
  if (k >= a.K) return;
  if (a.type == kQgF32) {
    const float* x = reinterpret_cast<const float*>(a.a) + (size_t)m * a.lda + k;
    if (a.vec) {
      const float4 y = __ldcg(reinterpret_cast<const float4*>(x));
      const float4 z = __ldcg(reinterpret_cast<const float4*>(x) + 1);
      v[0] = y.x; v[1] = y.y; v[2] = y.z; v[3] = y.w;
      v[4] = z.x; v[5] = z.y; v[6] = z.z; v[7] = z.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __ldcg(x + j);
    }
  } else {
    const unsigned short* x = reinterpret_cast<const unsigned short*>(a.a) + (size_t)m * a.lda + k;
    uint32_t u[8];
    if (a.vec) {
      const uint4 y = __ldcg(reinterpret_cast<const uint4*>(x));
      const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = (w[j / 2] >> (16 * (j & 1))) & 0xffffu;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = __ldcg(x + j);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = a.type == kQgBf16 ? __uint_as_float(u[j] << 16)
                               : __half2float(__ushort_as_half((unsigned short)u[j]));
  }
}

// SiLU: g / (1 + e^-g); GELU: (1 + tanh u) / 2 = 1 / (1 + e^-2u), without
// cancellation for negative u.
__device__ __forceinline__ float act_arg(float g, int act) {
  return act == 0 ? g : 2.f * 0.7978845608028654f * (g + 0.044715f * g * g * g);
}
__device__ __forceinline__ float act_wide(float g, int act) { return g / (1.f + expf(-act_arg(g, act))); }
// For results of 16 bits: the approximate exponential (2^-22; of an argument x
// with up to four roundings, |x| 2^-24 relative each: 2^-15 before the result
// vanishes) and reciprocal (2^-23).  A 16-bit result has steps of 2^-8 or 2^-11.
__device__ __forceinline__ float act_narrow(float g, int act) {
  float e, r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * act_arg(g, act)));
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return g * r;
}

__device__ __forceinline__ float load_out(const void* p, size_t i, int type) {
  if (type == kQgF32) return reinterpret_cast<const float*>(p)[i];
  if (type == kQgBf16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_out(void* p, size_t i, int type, float v) {
  if (type == kQgF32)
    reinterpret_cast<float*>(p)[i] = v;
  else if (type == kQgBf16)
    reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else
    reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}

// A finished sum v (gated: gate v, up u) of row m, column n.
__device__ __forceinline__ void finish(const Q4gParams& p, int m, int n, float v, float u) {
  if (n >= p.w.N) return;
  if (p.w2) v = (p.a.type == kQgF32 ? act_wide(v, p.act) : act_narrow(v, p.act)) * u;
  const size_t at = (size_t)m * p.ldo + n;
  if (p.accumulate) v += load_out(p.out, at, p.a.type);
  store_out(p.out, at, p.a.type, v);
}

__device__ __forceinline__ void add4(float4& a, const float4& b) {
  a.x += b.x;
  a.y += b.y;
  a.z += b.z;
  a.w += b.w;
}

// finish() of four neighbouring columns, in one store where they are aligned.
__device__ __forceinline__ void finish4(const Q4gParams& p, int m, int n, const float4& v,
                                        const float4& u) {
  const size_t at = (size_t)m * p.ldo + n;
  const int bytes = p.a.type == kQgF32 ? 16 : 8;
  uint8_t* d = reinterpret_cast<uint8_t*>(p.out) + at * (bytes / 4);
  float x[4] = {v.x, v.y, v.z, v.w};
  if (n + 4 > p.w.N || ((uintptr_t)d & (bytes - 1)) || p.accumulate) {
    const float y[4] = {u.x, u.y, u.z, u.w};
#pragma unroll 1
    for (int e = 0; e < 4; ++e) {
      const float xe = e == 0 ? x[0] : e == 1 ? x[1] : e == 2 ? x[2] : x[3];
      const float ye = e == 0 ? y[0] : e == 1 ? y[1] : e == 2 ? y[2] : y[3];
      finish(p, m, n + e, xe, ye);
    }
    return;
  }
  if (p.w2) {
    if (p.a.type == kQgF32) {
#pragma unroll 1  // (its code is long: the loop turns the four through one place)
      for (int e = 0; e < 4; ++e) {
        const float y = act_wide(x[0], p.act);
        x[0] = x[1];
        x[1] = x[2];
        x[2] = x[3];
        x[3] = y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = act_narrow(x[e], p.act);
    }
    x[0] *= u.x;
    x[1] *= u.y;
    x[2] *= u.z;
    x[3] *= u.w;
  }
  if (p.a.type == kQgF32) {
    *reinterpret_cast<float4*>(d) = make_float4(x[0], x[1], x[2], x[3]);
  } else if (p.a.type == kQgBf16) {
    __nv_bfloat162 h[2] = {__floats2bfloat162_rn(x[0], x[1]), __floats2bfloat162_rn(x[2], x[3])};
    *reinterpret_cast<uint2*>(d) = *reinterpret_cast<const uint2*>(h);
  } else {
    __half2 h[2] = {__floats2half2_rn(x[0], x[1]), __floats2half2_rn(x[2], x[3])};
    *reinterpret_cast<uint2*>(d) = *reinterpret_cast<const uint2*>(h);
  }
}

// Eight columns of a product that is only rounded and stored, 16-byte aligned.
__device__ __forceinline__ void store8(const Q4gParams& p, int m, int n, const float4& a,
                                       const float4& b) {
  const size_t at = (size_t)m * p.ldo + n;
  if (p.a.type == kQgF32) {
    float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at);
    d[0] = a;
    d[1] = b;
    return;
  }
  uint4 o;
  if (p.a.type == kQgBf16) {
    const __nv_bfloat162 h[4] = {__floats2bfloat162_rn(a.x, a.y), __floats2bfloat162_rn(a.z, a.w),
                                 __floats2bfloat162_rn(b.x, b.y), __floats2bfloat162_rn(b.z, b.w)};
    o = *reinterpret_cast<const uint4*>(h);
  } else {
    const __half2 h[4] = {__floats2half2_rn(a.x, a.y), __floats2half2_rn(a.z, a.w),
                          __floats2half2_rn(b.x, b.y), __floats2half2_rn(b.z, b.w)};
    o = *reinterpret_cast<const uint4*>(h);
  }
  *reinterpret_cast<uint4*>(reinterpret_cast<unsigned short*>(p.out) + at) = o;
}

}  // namespace ms
