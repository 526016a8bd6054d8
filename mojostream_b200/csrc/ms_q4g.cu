// ms_q4g.cu -- products with group-scaled 4-bit weights (layout: ms_q4g.h):
//   C[m][n] (+)= sum_k A[m][k] (q[k][n] - z) s,   H = act(A Wg) * (A Wu).
//
// Mathematics.  q - z is an integer of at most 5 bits: exact in bfloat16
// ((0x4300 | q) is the bfloat16 128 + q; subtracting 128 + z leaves q - z).
// An activation is cut into bfloat16 limbs that add up to it exactly (fp32:
// 8 + 8 + 8 bits, fp16: 8 + 3, bfloat16: itself), so every product of the
// mma.m16n8k16 is exact and its fp32 accumulator holds the sum of one group;
// the group's scale is applied in fp32 when the group ends.  All limbs of a
// row add into the same accumulator.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ms_common.cuh"
#include "ms_kernels.h"
#include "ms_q4g.h"

namespace ms {
namespace {

__device__ __forceinline__ float u16_scale(uint32_t u, int bf) {
  return bf ? __uint_as_float(u << 16) : __half2float(__ushort_as_half((unsigned short)u));
}

// ------------------------------------------------------------- repack --
// One thread per word of nibbles, then one per scale of the piece.
__global__ void q4g_repack_kernel(uint8_t* __restrict__ out, const Q4gView v,
                                  const uint8_t* __restrict__ src,
                                  const uint16_t* __restrict__ scales,
                                  const uint8_t* __restrict__ zeros, int* bad) {
  const int ng = kQgBlockK / v.group;
  const size_t pieces = (size_t)q4g_quads(v.N) * v.nkb * kQgQuad;
  const int per = 256 + ng * kQgTile;
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < pieces * per;
       i += (size_t)gridDim.x * blockDim.x) {
    const size_t piece = i / per;
    const int e = (int)(i % per);
    const int tile = (int)(piece / ((size_t)v.nkb * kQgQuad)) * kQgQuad + (int)(piece % kQgQuad);
    const int kb = (int)(piece / kQgQuad % v.nkb);
    uint8_t* dst = out + piece * v.block_bytes;
    if (e < 256) {
      // e = (half * 32 + lane) * 4 + s
      const int s = e & 3, lane = (e >> 2) & 31, half = e >> 7;
      const int r = lane >> 2, t = lane & 3;
      const int k0 = kb * kQgBlockK + half * 64 + 32 * (s >> 1) + 8 * t + 4 * (s & 1);
      uint32_t word = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int hi = j >> 2, jj = j & 3;
        const int n = tile * kQgTile + r + ((jj & 1) ? 8 : 0);
        const int k = k0 + hi + ((jj & 2) ? 2 : 0);
        uint32_t nib = 8;
        if (n < v.N && k < v.K) {
          const uint8_t b = src[(size_t)k * (v.N / 2) + (n >> 1)];
          nib = (n & 1) ? (b >> 4) : (b & 15);
        }
        word |= nib << (4 * jj + 16 * hi);
      }
      reinterpret_cast<uint32_t*>(dst)[e] = word;
    } else {
      const int j = (e - 256) / kQgTile, c = (e - 256) % kQgTile;  // group, column
      const int n = tile * kQgTile + c, kg = kb * ng + j;
      const bool in = n < v.N && kg < v.K / v.group;
      const int at = (j * 8 + (c & 7)) * 2 + (c >> 3);
      reinterpret_cast<uint16_t*>(dst + kQgNibbles)[at] = in ? scales[(size_t)kg * v.N + n] : 0;
      if (v.zeros) {
        uint8_t z = in ? zeros[(size_t)kg * v.N + n] : 8;
        if (z > 15) {
          atomicExch(bad, 1);
          z = 15;
        }
        dst[kQgNibbles + ng * 32 + at] = z;
      }
    }
  }
}

// -------------------------------------------------------------- planes --
// v = hi + mid + lo exactly: each limb is the leading 8 bits of what is left
// (truncated, so nothing can round up to infinity).  An infinity or a NaN
// stays in the first limb alone.
__device__ __forceinline__ void limbs3(float v, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  const uint32_t u = __float_as_uint(v);
  hi = u & 0xffff0000u;
  float r = v - __uint_as_float(hi);
  if ((u & 0x7f800000u) == 0x7f800000u) {
    if (u & 0x007fffffu) hi |= 0x00400000u;  // a NaN whose payload sits in the low bits
    r = 0.f;
  }
  mid = __float_as_uint(r) & 0xffff0000u;
  lo = __float_as_uint(r - __uint_as_float(mid));  // at most 8 bits: exact
}

// Thread: 8 k of one row.  Grid x over k / 32 pieces of 4 threads, y over rows
// of the padded row blocks.
__global__ void __launch_bounds__(256) q4g_planes_kernel(const Q4gPlanes p) {
  pdl_wait();     // the activations are an earlier kernel's output, and the
  pdl_trigger();  // planes may still be read by the product before this one
  const int k8 = blockIdx.x * blockDim.x + threadIdx.x;
  if (k8 * 8 >= p.kpad) return;
  for (int m = blockIdx.y; m < p.M; m += gridDim.y) {
    float v[8];
    const int k0 = k8 * 8;
    if (k0 >= p.K) {  // K is a multiple of 32: a piece is inside or outside
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    } else if (p.type == kQgF32) {
      const float* a = reinterpret_cast<const float*>(p.a) + (size_t)m * p.lda + k0;
      if (p.vec) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(a));
        const float4 y = __ldcg(reinterpret_cast<const float4*>(a) + 1);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
        v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __ldcg(a + j);
      }
    } else {
      const unsigned short* a = reinterpret_cast<const unsigned short*>(p.a) + (size_t)m * p.lda + k0;
      uint32_t u[8];
      if (p.vec) {
        const uint4 x = __ldcg(reinterpret_cast<const uint4*>(a));
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = (w[j / 2] >> (16 * (j & 1))) & 0xffffu;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = __ldcg(a + j);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = p.type == kQgBf16 ? __uint_as_float(u[j] << 16)
                                 : __half2float(__ushort_as_half((unsigned short)u[j]));
    }
    uint32_t l[3][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (p.limbs == 1)
        l[0][j] = __float_as_uint(v[j]);
      else
        limbs3(v[j], l[0][j], l[1][j], l[2][j]);
    }
    const int rb = m / p.mb, r = m % p.mb;
    const int rows = min(p.mb, p.M - rb * p.mb);
    uint8_t* base = p.planes + (size_t)rb * p.mb * p.limbs * p.kpad * 2;
    for (int i = 0; i < p.limbs; ++i) {
      const uint32_t* s = i == 0 ? l[0] : i == 1 ? l[1] : l[2];
      uint4 o;
      o.x = __byte_perm(s[0], s[1], 0x7632);
      o.y = __byte_perm(s[2], s[3], 0x7632);
      o.z = __byte_perm(s[4], s[5], 0x7632);
      o.w = __byte_perm(s[6], s[7], 0x7632);
      *reinterpret_cast<uint4*>(
          base + (((size_t)(k0 / 32) * p.limbs + i) * rows + r) * 64 + (k8 & 3) * 16) = o;
    }
  }
}

// ----------------------------------------------------- streaming kernel --
// Decode rows.  A warp owns T tiles (T x 16 columns) over its share of the
// 128-k blocks; the kw warps that share a tile set split K, and their sums
// are added in k order through shared memory at the end (the same bits on
// every run).  Each warp streams its own pieces through a private ring of
// bulk copies: the weight pieces of a block and the same block of the limb
// planes, one mbarrier per stage and no CTA barrier inside the loop.  The
// first stages' weights are issued before the previous kernel has finished
// (nothing writes them); activations and results wait for it.
constexpr int kQgMaxWarps = 16;
constexpr int kQgMaxStages = 8;
constexpr size_t kQgSmemMax = 208 * 1024;

__device__ __forceinline__ float act_fn(float g, int act) {
  if (act == 0) return g / (1.f + expf(-g));
  // (1 + tanh u) / 2 = 1 / (1 + e^-2u): no cancellation for negative u
  const float u = 0.7978845608028654f * (g + 0.044715f * g * g * g);
  return g / (1.f + expf(-2.f * u));
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

template <int T, int NB>
__global__ void __launch_bounds__(kQgMaxWarps* kWarp, T* NB <= 2 ? 2 : 1) q4g_stream_kernel(const Q4gParams p) {
  extern __shared__ __align__(128) uint8_t dsm[];
  __shared__ __align__(8) uint64_t s_full[kQgMaxWarps * kQgMaxStages];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, t = lane & 3;
  const int ks = warp % p.kw;
  const int set = blockIdx.x * p.tw + warp / p.kw;
  const int n_sets = (q4g_quads(p.w.N) * kQgQuad) / (p.w2 ? T / 2 : T);
  const int nkb = p.w.nkb, bb = p.w.block_bytes, ng = kQgBlockK / p.w.group;
  const int row0 = blockIdx.y * p.mb, rows = min(p.mb, p.M - row0);
  const int L = p.limbs;
  const int a_bytes = rows * L * 256;
  const int stage_bytes = T * bb + p.mb * L * 256;
  const int kb0 = (int)((long long)nkb * ks / p.kw), kb1 = (int)((long long)nkb * (ks + 1) / p.kw);
  const int n = set < n_sets ? kb1 - kb0 : 0;  // blocks of this warp
  uint8_t* ring = dsm + (size_t)warp * p.stages * stage_bytes;
  uint64_t* full = s_full + warp * kQgMaxStages;

  if (lane == 0) {
    for (int s = 0; s < p.stages; ++s) mbar_init(&full[s], 1);
    mbar_fence_init();
  }
  __syncwarp();
  pdl_trigger();

  // the pieces of tiles set * T .. (gated: T / 2 of the gate, then of the up)
  const int per = p.w2 ? T / 2 : T;
  const int tile0 = set * per;
  const size_t w_off = ((size_t)(tile0 / kQgQuad) * nkb * kQgQuad + tile0 % kQgQuad) * bb;
  const uint8_t* a_src = p.planes + (size_t)row0 * L * nkb * 256;
  auto issue_w = [&](int i) {
    uint8_t* st = ring + (size_t)(i % p.stages) * stage_bytes;
    uint64_t* bar = &full[i % p.stages];
    const size_t off = w_off + (size_t)(kb0 + i) * kQgQuad * bb;
    mbar_expect_tx(bar, T * bb + a_bytes);
    bulk_g2s(st, p.w.w + off, per * bb, bar);
    if (p.w2) bulk_g2s(st + per * bb, p.w2 + off, per * bb, bar);
  };
  auto issue_a = [&](int i) {
    bulk_g2s(ring + (size_t)(i % p.stages) * stage_bytes + T * bb, a_src + (size_t)(kb0 + i) * a_bytes,
             a_bytes, &full[i % p.stages]);
  };
  const int first = min(n, p.stages);
  if (lane == 0)
    for (int i = 0; i < first; ++i) issue_w(i);
  pdl_wait();
  if (lane == 0)
    for (int i = 0; i < first; ++i) issue_a(i);

  float acc[T][NB][4];
#pragma unroll
  for (int i = 0; i < T; ++i)
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][b][j] = 0.f;

  const int flush_mask = p.w.group / 32 - 1;  // a group ends after 32-k step h if (h & mask) == mask
  bool ok = true;
  for (int i = 0; i < n; ++i) {
    const int slot = i % p.stages;
    if (!mbar_wait(&full[slot], (i / p.stages) & 1)) {
      if (lane == 0) atomicOr(p.err, kErrWaitTimeout);
      // let the other copies land before the CTA can exit
      for (int j = i + 1; j < min(n, i + p.stages); ++j)
        mbar_wait(&full[j % p.stages], (j / p.stages) & 1);
      ok = false;
      break;
    }
    const uint8_t* st = ring + (size_t)slot * stage_bytes;
    const uint8_t* sa = st + T * bb;
    float c[T][NB][4];
    uint32_t bias[T][2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {  // 64-k halves
      uint4 wv[T];
#pragma unroll
      for (int j = 0; j < T; ++j)
        wv[j] = lds_u4(reinterpret_cast<const uint4*>(st + j * bb + q * 512) + lane);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {  // 32-k steps
        const int h = 2 * q + hh;
        const int grp = h / (flush_mask + 1);
        if ((h & flush_mask) == 0) {  // a group begins
#pragma unroll
          for (int j = 0; j < T; ++j) {
            uint32_t lo = 0x43084308u, hi = 0x43084308u;  // 128 + 8
            if (p.w.zeros) {
              const uint32_t z = *reinterpret_cast<const uint16_t*>(st + j * bb + kQgNibbles +
                                                                    ng * 32 + (grp * 8 + r) * 2);
              lo = (0x4300u | (z & 0xffu)) * 0x10001u;
              hi = (0x4300u | (z >> 8)) * 0x10001u;
            }
            bias[j][0] = lo;
            bias[j][1] = hi;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
              for (int e = 0; e < 4; ++e) c[j][b][e] = 0.f;
          }
        }
        uint32_t a[T][2][4];
#pragma unroll
        for (int j = 0; j < T; ++j)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const uint32_t w = hh == 0 ? (s == 0 ? wv[j].x : wv[j].y) : (s == 0 ? wv[j].z : wv[j].w);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t v = ((w >> (4 * e)) & 0x000F000Fu) | 0x43004300u;
              asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(a[j][s][e]) : "r"(v), "r"(bias[j][e & 1]));
            }
          }
        for (int l = 0; l < L; ++l) {
          uint4 bv[NB];
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const int m = b * 8 + r;
            bv[b] = make_uint4(0u, 0u, 0u, 0u);
            if (m < rows)
              bv[b] = lds_u4(reinterpret_cast<const uint4*>(sa + ((h * L + l) * rows + m) * 64) + t);
          }
#pragma unroll
          for (int j = 0; j < T; ++j)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              mma_bf16_16816(c[j][b], a[j][0], bv[b].x, bv[b].y);
              mma_bf16_16816(c[j][b], a[j][1], bv[b].z, bv[b].w);
            }
        }
        if ((h & flush_mask) == flush_mask) {  // it ends
#pragma unroll
          for (int j = 0; j < T; ++j) {
            const uint32_t s2 = *reinterpret_cast<const uint32_t*>(st + j * bb + kQgNibbles +
                                                                   (grp * 8 + r) * 4);
            const float lo = u16_scale(s2 & 0xffffu, p.w.bf_scale);
            const float hi = u16_scale(s2 >> 16, p.w.bf_scale);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              acc[j][b][0] = fmaf(lo, c[j][b][0], acc[j][b][0]);
              acc[j][b][1] = fmaf(lo, c[j][b][1], acc[j][b][1]);
              acc[j][b][2] = fmaf(hi, c[j][b][2], acc[j][b][2]);
              acc[j][b][3] = fmaf(hi, c[j][b][3], acc[j][b][3]);
            }
          }
        }
      }
    }
    __syncwarp();  // every lane has read the stage
    if (lane == 0 && i + p.stages < n) {
      issue_w(i + p.stages);
      issue_a(i + p.stages);
    }
  }

  // sums over the kw warps of a tile set, in k order; columns fastest
  constexpr int kCols = T * kQgTile, kLd = kCols + 4;
  __syncthreads();  // the rings are free
  float* red = reinterpret_cast<float*>(dsm);
  if (ok && n > 0) {
    float* mine = red + (size_t)warp * (NB * 8) * kLd;
#pragma unroll
    for (int j = 0; j < T; ++j)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float* d = mine + (b * 8 + 2 * t) * kLd + j * kQgTile + r;
        d[0] = acc[j][b][0];
        d[kLd] = acc[j][b][1];
        d[8] = acc[j][b][2];
        d[kLd + 8] = acc[j][b][3];
      }
  }
  if (__syncthreads_or(!ok)) return;  // nothing is written after a wait that ran out
  const int live = min(p.kw, nkb);    // warps past that had no blocks
  const int cols = per * kQgTile;     // result columns of a tile set
  for (int i = threadIdx.x; i < p.tw * rows * cols; i += blockDim.x) {
    const int col = i % cols, m = i / cols % rows, ts = i / (cols * rows);
    const int set_i = blockIdx.x * p.tw + ts;
    const int nn = set_i * cols + col;
    if (set_i >= n_sets || nn >= p.w.N) continue;
    const float* src = red + ((size_t)ts * p.kw * (NB * 8) + m) * kLd + col;
    float v = 0.f, u = 0.f;
    for (int k = 0; k < p.kw; ++k) {
      // block ranges nkb k / kw .. nkb (k + 1) / kw: empty where kw > nkb
      if (live < p.kw && (long long)nkb * k / p.kw == (long long)nkb * (k + 1) / p.kw) continue;
      v += src[(size_t)k * (NB * 8) * kLd];
      if (p.w2) u += src[(size_t)k * (NB * 8) * kLd + cols];
    }
    if (p.w2) v = act_fn(v, p.act) * u;
    const size_t at = (size_t)(row0 + m) * p.ldo + nn;
    if (p.accumulate) v += load_out(p.out, at, p.type);
    store_out(p.out, at, p.type, v);
  }
}

template <int T, int NB>
cudaError_t launch_stream_t(const Q4gParams& p0, int sm_count, cudaStream_t s) {
  Q4gParams p = p0;
  const int per = p.w2 ? T / 2 : T;
  const int sets = q4g_quads(p.w.N) * kQgQuad / per;
  const int row_blocks = (p.M + p.mb - 1) / p.mb;
  // 16 warps, fewer where three stages of theirs would not fit; as many tile
  // sets as still leave two CTAs for each SM, the rest of the warps split K
  const size_t stage = (size_t)T * p.w.block_bytes + (size_t)p.mb * p.limbs * 256;
  int warps = kQgMaxWarps;
  while (warps > 2 && 3 * stage * warps > kQgSmemMax) warps /= 2;
  int tw = warps;
  while (tw > 1 && (long long)(sets + tw - 1) / tw * row_blocks < 2LL * sm_count) tw /= 2;
  const int kw = warps / tw;
  p.tw = tw;
  p.kw = kw;
  size_t budget = kQgSmemMax / 2;  // two CTAs per SM where three stages fit
  if (3 * stage * warps > budget) budget = kQgSmemMax;
  int st = (int)(budget / (stage * warps));
  const int longest = (p.w.nkb + kw - 1) / kw;
  st = st > kQgMaxStages ? kQgMaxStages : st;
  st = st > longest ? longest : st;
  if (st < 1) return cudaErrorInvalidConfiguration;
  p.stages = st;
  size_t smem = (size_t)st * stage * warps;
  const size_t red = (size_t)warps * NB * 8 * (T * kQgTile + 4) * sizeof(float);
  if (red > smem) smem = red;
  if (smem > kQgSmemMax) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((sets + tw - 1) / tw, row_blocks, 1);
  cfg.blockDim = dim3(warps * kWarp);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, q4g_stream_kernel<T, NB>, p);
}

template <int T, int NB>
cudaError_t prepare_t() {
  return cudaFuncSetAttribute(q4g_stream_kernel<T, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              (int)kQgSmemMax);
}

}  // namespace

cudaError_t launch_q4g_repack(uint8_t* out, const Q4gView& v, const uint8_t* src, const void* scales,
                              const uint8_t* zeros, int* bad, cudaStream_t s) {
  const size_t n = (size_t)q4g_quads(v.N) * v.nkb * kQgQuad * (256 + kQgBlockK / v.group * kQgTile);
  const size_t blocks = (n + 255) / 256;
  q4g_repack_kernel<<<(unsigned)(blocks < 148 * 64 ? blocks : 148 * 64), 256, 0, s>>>(
      out, v, src, reinterpret_cast<const uint16_t*>(scales), zeros, bad);
  return cudaGetLastError();
}

cudaError_t launch_q4g_planes(const Q4gPlanes& p, cudaStream_t s) {
  const int k8 = p.kpad / 8;
  const int threads = k8 < 256 ? (k8 + 31) / 32 * 32 : 256;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((k8 + threads - 1) / threads, p.M < 65535 ? p.M : 65535, 1);
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, q4g_planes_kernel, p);
}

cudaError_t launch_q4g_stream(const Q4gParams& p, int T, int NB, int sm_count, cudaStream_t s) {
  if (p.mb > NB * 8 || p.mb <= 0 || (p.w2 && T < 2)) return cudaErrorInvalidValue;
  if (NB == 1 && T == 1) return launch_stream_t<1, 1>(p, sm_count, s);
  if (NB == 1 && T == 2) return launch_stream_t<2, 1>(p, sm_count, s);
  if (NB == 1 && T == 4) return launch_stream_t<4, 1>(p, sm_count, s);
  if (NB == 2 && T == 2) return launch_stream_t<2, 2>(p, sm_count, s);
  return cudaErrorInvalidValue;
}

cudaError_t prepare_q4g() {
  cudaError_t e = prepare_t<1, 1>();
  if (e == cudaSuccess) e = prepare_t<2, 1>();
  if (e == cudaSuccess) e = prepare_t<4, 1>();
  if (e == cudaSuccess) e = prepare_t<2, 2>();
  return e;
}

}  // namespace ms
