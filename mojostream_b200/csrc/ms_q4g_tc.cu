// ms_q4g_tc.cu -- products with group-scaled 4-bit weights for many rows, on
// the 5th-generation tensor cores (layout: ms_q4g.h):
//   C[m][n] (+)= sum_k A[m][k] (q[k][n] - z) s,   H = act(A Wg) * (A Wu).
//
// Mathematics.  q - z is an integer of at most 5 bits: exact in bfloat16
// ((0x4300 | q) is the bfloat16 128 + q; subtracting 128 + z leaves q - z).
// An activation is cut into bfloat16 limbs that add up to it exactly (fp32:
// 8 + 8 + 8 bits, fp16: 8 + 3, bfloat16: itself), so every product of a
// tcgen05.mma is exact and its fp32 accumulator in tensor memory holds the sum
// of one group of k over all limbs; when the group ends its scale is applied
// and it is added to fp32 sums in registers.
//
// CTA: 128 weight columns on the MMA's M side (gated: 64 of the gate, 64 of
// the up weight) x NT rows on its N side x a share of the k blocks.  Warp 0
// streams weight pieces with bulk copies; one thread of warp 1 issues the MMAs; warps 2-9 unpack a 64-k half of the weights into the A
// operand, then take the groups that the half before completed out of tensor
// memory (a thread owns one weight column and half of the rows); warp 10
// streams the limb planes.  Weights,
// A operand, B operand and accumulators have rings of their own, so unpacking,
// MMAs and sums of neighbouring halves overlap.  A cluster's CTAs share k; the
// sums are added in k order through distributed shared memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ms_common.cuh"
#include "ms_kernels.h"
#include "ms_q4g.h"
#include "ms_q4g.cuh"
#include "ms_tc.cuh"

namespace ms {
namespace {

constexpr int kTqWorkers = 8;
constexpr int kTqThreads = (3 + kTqWorkers) * kWarp;
constexpr int kTqLboA = 2048 + 32;  // k cores of A: 32 bytes apart in the banks
constexpr int kTqA = 8 * kTqLboA;   // a 64-k half of 128 columns, bfloat16
constexpr int kTqStagesA = 3;
constexpr int kTqMaxB = 12, kTqMaxW = 4, kTqMaxD = 4;
constexpr size_t kTqSmemMax = 224 * 1024;
constexpr int kTqMaxCluster = 8;

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

// Planes [row tile][64-k half][limb][8 k cores][NT rows][16 bytes]: the B
// operand's core matrices.  Thread: 8 k (a core) of one row; rows past M are
// left as they are (their columns of the product are not used).
__global__ void __launch_bounds__(256) q4g_planes_kernel(const Q4gRows a, int limbs, int NT) {
  pdl_wait();     // the rows are an earlier kernel's output, and the planes
  pdl_trigger();  // may still be read by the product before this one
  // eight neighbouring threads: the eight rows of a core matrix; then k
  const int cores = a.nkb * 16;
  for (int m8 = blockIdx.y; m8 < (a.M + 7) / 8; m8 += gridDim.y) {
    const int m = m8 * 8 + (threadIdx.x & 7), core = blockIdx.x * 32 + (threadIdx.x >> 3);
    if (m >= a.M || core >= cores) continue;
    float v[8];
    load8(a, m, core * 8, v);
    uint32_t l[3][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (limbs == 1)
        l[0][j] = __float_as_uint(v[j]);
      else
        limbs3(v[j], l[0][j], l[1][j], l[2][j]);
    }
    const int rt = m / NT, r = m % NT;
    uint8_t* dst = a.records + (((size_t)rt * a.nkb * 2 + (core >> 3)) * limbs * 8 + (core & 7)) * NT * 16 + r * 16;
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < limbs)
        *reinterpret_cast<uint4*>(dst + (size_t)i * 8 * NT * 16) = make_uint4(
            __byte_perm(l[i][0], l[i][1], 0x7632), __byte_perm(l[i][2], l[i][3], 0x7632),
            __byte_perm(l[i][4], l[i][5], 0x7632), __byte_perm(l[i][6], l[i][7], 0x7632));
  }
}

// ------------------------------------------------------------- product --
struct TcShape {
  int limbs, nB, nW, nD, cs, row_tiles;
};

// Four bfloat16 pairs of one column: k 0..7 of a core from the words x, y.
__device__ __forceinline__ uint4 unpack8(uint32_t x, uint32_t y, int shift, uint32_t bias) {
  uint32_t o[4];
  const uint32_t w[4] = {x >> shift, x >> (8 + shift), y >> shift, y >> (8 + shift)};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t v = (w[e] & 0x000F000Fu) | 0x43004300u;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(o[e]) : "r"(v), "r"(bias));
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}
__device__ __forceinline__ void sts128(uint32_t a, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

// NC: rows per worker thread (the tile has NT = 2 NC); G: 32-k steps per group.
template <int NC, int G>
__global__ void __launch_bounds__(kTqThreads, NC <= 32 ? 2 : 1)
    q4g_tc_kernel(const Q4gParams p, const TcShape c) {
  constexpr int NT = 2 * NC;
  extern __shared__ __align__(1024) uint8_t dsm[];
  __shared__ __align__(8) uint64_t full_w[kTqMaxW], empty_w[kTqMaxW], full_a[kTqStagesA],
      empty_a[kTqStagesA], full_b[kTqMaxB], empty_b[kTqMaxB], full_d[kTqMaxD], empty_d[kTqMaxD], done;
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_bad;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nkb = p.w.nkb, bb = p.w.block_bytes;
  const int rank = blockIdx.x % c.cs, tile = blockIdx.x / c.cs, rt = blockIdx.y;
  const int kb0 = nkb * rank / c.cs, kb1 = nkb * (rank + 1) / c.cs;
  const int steps = (kb1 - kb0) * 2;  // 64-k halves
  constexpr int kUnitB = NT * 128;    // a limb of a half
  const int stage_w = 2 * kQgQuad * bb;
  uint8_t* ring_a = dsm;
  uint8_t* ring_b = ring_a + kTqStagesA * kTqA;
  uint8_t* ring_w = ring_b + c.nB * kUnitB;
  constexpr uint32_t kColsD = NT;

  if (threadIdx.x == 0) {
    s_bad = 0;
    for (int s = 0; s < c.nW; ++s) {
      mbar_init(&full_w[s], 1);
      mbar_init(&empty_w[s], kTqWorkers);
    }
    for (int s = 0; s < kTqStagesA; ++s) {
      mbar_init(&full_a[s], kTqWorkers);
      mbar_init(&empty_a[s], 1);
    }
    for (int s = 0; s < c.nB; ++s) {
      mbar_init(&full_b[s], 1);
      mbar_init(&empty_b[s], 1);
    }
    for (int s = 0; s < c.nD; ++s) {
      mbar_init(&full_d[s], 1);
      mbar_init(&empty_d[s], kTqWorkers);
    }
    mbar_init(&done, 1);
    mbar_fence_init();
  }
  // columns: a power of two of at least 32
  uint32_t cols = 32;
  while (cols < c.nD * kColsD) cols *= 2;
  if (warp == 1) {
    tmem_alloc(&s_tmem, cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  pdl_trigger();

  auto fail = [&]() {
    atomicOr(p.err, kErrWaitTimeout);
    s_bad = 1;
  };

  float acc[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) acc[i] = 0.f;
  const int wk = warp - 2;              // worker
  const int quad = warp & 3;            // tensor-memory lanes 32 quad ..
  const int half_n = wk >> 2;           // rows half_n * NC ..
  const int col = quad * kWarp + lane;  // the thread's weight column

  if (warp == 0) {
    // -------------------------------------------------------- producer --
    if (lane == 0) {
      const uint8_t* w0;
      const uint8_t* w1;  // the tile's two quads (the second may not exist)
      const size_t quad_bytes = (size_t)nkb * kQgQuad * bb;
      int second = 1;
      if (p.w2) {
        w0 = p.w.w + (size_t)tile * quad_bytes;
        w1 = p.w2 + (size_t)tile * quad_bytes;
      } else {
        w0 = p.w.w + (size_t)tile * 2 * quad_bytes;
        w1 = w0 + quad_bytes;
        second = tile * 2 + 1 < q4g_quads(p.w.N);
      }
      w0 += (size_t)kb0 * kQgQuad * bb;
      w1 += (size_t)kb0 * kQgQuad * bb;
      const int n = kb1 - kb0;
      int i = 0;
      for (; i < n; ++i) {  // no kernel writes the weights: no wait for the previous one
        const int s = i % c.nW;
        if (i >= c.nW && !mbar_wait(&empty_w[s], ((i / c.nW) - 1) & 1)) break;
        uint8_t* st = ring_w + s * stage_w;
        mbar_expect_tx(&full_w[s], kQgQuad * bb * (1 + second));
        bulk_g2s(st, w0 + (size_t)i * kQgQuad * bb, kQgQuad * bb, &full_w[s]);
        if (second) bulk_g2s(st + kQgQuad * bb, w1 + (size_t)i * kQgQuad * bb, kQgQuad * bb, &full_w[s]);
      }
      if (i < n) fail();
      // the copies issued last land before the CTA can exit
      for (int j = max(0, i - c.nW); j < i; ++j) mbar_wait(&full_w[j % c.nW], (j / c.nW) & 1);
    }
  } else if (warp == 2 + kTqWorkers) {
    // ------------------------------------------------- planes producer --
    if (lane == 0) {
      const uint8_t* b0 = p.a.records + ((size_t)rt * nkb + kb0) * 2 * c.limbs * kUnitB;
      const int n = steps * c.limbs;
      pdl_wait();
      int i = 0;
      for (; i < n; ++i) {
        const int s = i % c.nB;
        if (i >= c.nB && !mbar_wait(&empty_b[s], ((i / c.nB) - 1) & 1)) break;
        mbar_expect_tx(&full_b[s], kUnitB);
        bulk_g2s(ring_b + s * kUnitB, b0 + (size_t)i * kUnitB, kUnitB, &full_b[s]);
      }
      if (i < n) fail();
      for (int j = max(0, i - c.nB); j < i; ++j) mbar_wait(&full_b[j % c.nB], (j / c.nB) & 1);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------ MMA issuer --
    if (lane == 0) {
      const uint32_t idesc = idesc_bf16(128, NT);
      const uint32_t a_base = smem_u32(ring_a), b_base = smem_u32(ring_b);
      int d = -1;  // accumulators used so far - 1
      for (int j = 0; j < steps; ++j) {
        const int sa = j % kTqStagesA;
        bool ok = mbar_wait(&full_a[sa], (j / kTqStagesA) & 1);
        for (int l = 0; l < c.limbs && ok; ++l) {
          const int ub = j * c.limbs + l;
          ok = mbar_wait(&full_b[ub % c.nB], (ub / c.nB) & 1);
        }
        // groups inside this half (two of 32, one of 64, or half of one of 128)
        constexpr int kSub = G == 1 ? 2 : 1, kK16 = 4 / kSub;
        for (int g = 0; g < kSub && ok; ++g) {
          const bool begins = G < 4 || (j & 1) == 0;
          if (begins) {
            ++d;
            if (d >= c.nD) ok = mbar_wait(&empty_d[d % c.nD], ((d / c.nD) - 1) & 1);
            if (!ok) break;
          }
          tc_fence_after();
          const uint32_t dt = tmem + (uint32_t)(d % c.nD) * kColsD;
          for (int l = 0; l < c.limbs; ++l) {
            const uint32_t b = b_base + ((j * c.limbs + l) % c.nB) * kUnitB;
#pragma unroll
            for (int k = 0; k < kK16; ++k) {
              const int k16 = g * kK16 + k;
              umma_bf16(dt, umma_desc(a_base + sa * kTqA + 2 * k16 * kTqLboA, kTqLboA, 128),
                        umma_desc(b + 2 * k16 * NT * 16, NT * 16, 128), idesc,
                        !(begins && l == 0 && k == 0));
            }
          }
          if (G < 4 || (j & 1)) umma_commit(&full_d[d % c.nD]);
        }
        if (!ok) {
          fail();
          break;
        }
        umma_commit(&empty_a[sa]);
        for (int l = 0; l < c.limbs; ++l) umma_commit(&empty_b[(j * c.limbs + l) % c.nB]);
      }
      umma_commit(&done);  // arrives when every MMA issued above has finished
    }
  } else {
    // --------------------------------------- unpacking and group sums --
    const int r = lane >> 2, t = lane & 3;
    const uint32_t ring_a_s = smem_u32(ring_a), ring_w_s = smem_u32(ring_w);
    constexpr int ng = 4 / G, kSub = G == 1 ? 2 : 1;
    const bool live = p.w2 || wk < 4 || tile * 2 + 1 < q4g_quads(p.w.N);  // the tile's quad exists
    float sc[kSub] = {};  // scales of the groups of the half before
    int d = 0;
    // the group sums of accumulator d, scaled
    auto take = [&](float s) -> bool {
      const int sd = d % c.nD;
      if (!mbar_wait(&full_d[sd], (d / c.nD) & 1)) return false;
      tc_fence_after();
      const uint32_t ta = tmem + ((uint32_t)(quad * kWarp) << 16) + (uint32_t)(sd * (int)kColsD + half_n * NC);
#pragma unroll
      for (int i = 0; i < NC; i += 16) {
        uint32_t v[16];
        tmem_ld16(ta + i, v);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i + e] = fmaf(s, __uint_as_float(v[e]), acc[i + e]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_d[sd]);
      ++d;
      return true;
    };
    bool ok = true;
    for (int j = 0; j < steps && ok; ++j) {
      const int kb = j >> 1, half = j & 1, sw = kb % c.nW, sa = j % kTqStagesA;
      ok = mbar_wait(&full_w[sw], (kb / c.nW) & 1) &&
           (j < kTqStagesA || mbar_wait(&empty_a[sa], ((j / kTqStagesA) - 1) & 1));
      if (!ok) break;
      const uint32_t st = ring_w_s + sw * stage_w;
      // warp wk unpacks tile wk of the 128 columns
      const uint32_t pc = st + wk * bb;
      const uint32_t dst = ring_a_s + sa * kTqA + t * kTqLboA + wk * 256 + r * 16;
      if (live) {
        const uint4 w = lds128(pc + half * 512 + lane * 16);
        uint32_t lo[2], hi[2];  // biases of the half's two 32-k steps
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          lo[hh] = hi[hh] = 0x43084308u;  // 128 + 8
          if (p.w.zeros) {
            const uint32_t z = lds16(pc + kQgNibbles + ng * 32 + ((2 * half + hh) / G * 8 + r) * 2);
            lo[hh] = (0x4300u | (z & 0xffu)) * 0x10001u;
            hi[hh] = (0x4300u | (z >> 8)) * 0x10001u;
          }
        }
        sts128(dst, unpack8(w.x, w.y, 0, lo[0]));
        sts128(dst + 128, unpack8(w.x, w.y, 4, hi[0]));
        sts128(dst + 4 * kTqLboA, unpack8(w.z, w.w, 0, lo[1]));
        sts128(dst + 4 * kTqLboA + 128, unpack8(w.z, w.w, 4, hi[1]));
      }
      // scales of this half's groups for the thread's column
      float sn[kSub];
#pragma unroll
      for (int g = 0; g < kSub; ++g) {
        const int grp = G == 1 ? 2 * half + g : half * 2 / G;
        const uint32_t at = st + (col >> 4) * bb + kQgNibbles + ((grp * 8 + (col & 7)) * 2 + ((col >> 3) & 1)) * 2;
        sn[g] = u16_scale(lds16(at), p.w.bf_scale);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&full_a[sa]);
        if (half) mbar_arrive(&empty_w[sw]);
      }
      if (j > 0) {
#pragma unroll
        for (int g = 0; g < kSub; ++g)
          if (ok && (G < 4 || half == 0)) ok = take(sc[g]);
      }
#pragma unroll
      for (int g = 0; g < kSub; ++g) sc[g] = sn[g];
    }
#pragma unroll
    for (int g = 0; g < kSub; ++g)
      if (ok) ok = take(sc[g]);
    if (!ok && lane == 0) fail();
    if (!mbar_wait(&done, 0) && lane == 0) fail();  // no MMA is in flight
  }

  // ------------------------------------------------------------- results --
  // rows m of this tile, the thread's column: straight to memory (32 columns
  // of a row per warp), or, gated and in a cluster, by way of shared memory
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, cols);
  const int row0 = rt * NT, rows = min(NT, p.a.M - row0);
  int bad = s_bad;
  constexpr int kLd = 128 + 4;
  float* S = reinterpret_cast<float*>(dsm);  // [NT][kLd]
  const bool staged = p.w2 || c.cs > 1;
  if (wk >= 0 && wk < kTqWorkers) {
    pdl_wait();  // results may overwrite what the previous kernel still reads
    if (!staged) {
      const int n = tile * 128 + col;
      if (!bad && n < p.w.N) {
#pragma unroll
        for (int i = 0; i < NC; ++i)
          if (half_n * NC + i < rows) finish(p, row0 + half_n * NC + i, n, acc[i], 0.f);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NC; ++i) S[(half_n * NC + i) * kLd + col] = acc[i];
    }
  }
  if (!staged) return;
  __syncthreads();
  if (c.cs > 1) {
    cluster_arrive();
    cluster_wait();
    const uint32_t bad0 = smem_u32(const_cast<int*>(&s_bad));
    for (int k = 0; k < c.cs; ++k) bad |= ld_dsmem_s32(dsmem_addr(bad0, (uint32_t)k));
  }
  if (!bad) {
    pdl_wait();
    const int out_cols = p.w2 ? 64 : 128, sh = p.w2 ? 6 : 7;
    // the rows of this rank: m = rank, rank + cs, ...
    const int mine = rank < rows ? (rows - rank + c.cs - 1) / c.cs : 0;
    for (int i = threadIdx.x; i < mine << sh; i += kTqThreads) {
      const int m = rank + (i >> sh) * c.cs, n0 = i & (out_cols - 1);
      float v = 0.f, u = 0.f;
      if (c.cs > 1) {
        const uint32_t at = smem_u32(S + m * kLd + n0);
        for (int k = 0; k < c.cs; ++k) v += ld_dsmem(dsmem_addr(at, (uint32_t)k));
        if (p.w2)
          for (int k = 0; k < c.cs; ++k) u += ld_dsmem(dsmem_addr(at + 256, (uint32_t)k));
      } else {
        v = S[m * kLd + n0];
        u = S[m * kLd + n0 + 64];
      }
      finish(p, row0 + m, tile * out_cols + n0, v, u);
    }
  }
  if (c.cs > 1) {  // the other CTAs have read this one's sums
    cluster_arrive();
    cluster_wait();
  }
}

struct TcPlan {
  int NC, tiles;
  TcShape c;
  size_t smem;
};

int tc_limbs(int type) { return type == kQgF32 ? 3 : type == kQgF16 ? 2 : 1; }

TcPlan plan_tc(const Q4gParams& p, int sm_count) {
  TcPlan o{};
  o.c.limbs = tc_limbs(p.a.type);
  // rows per tile: as few tiles as fit (256 rows of one limb, 128 of more),
  // all of about the same size
  const int most = o.c.limbs == 1 ? 256 : 128;
  const int tiles = (p.a.M + most - 1) / most, each = (p.a.M + tiles - 1) / tiles;
  const int widths[5] = {16, 32, 64, 96, 128};
  o.NC = 128;
  for (int i = 4; i >= 0; --i)
    if (each <= 2 * widths[i]) o.NC = widths[i];
  o.c.row_tiles = (p.a.M + 2 * o.NC - 1) / (2 * o.NC);
  o.tiles = p.w2 ? q4g_quads(p.w.N) : (q4g_quads(p.w.N) + 1) / 2;
  // k shared by a cluster while the CTAs do not fill the GPU
  o.c.cs = 1;
  while (o.c.cs < kTqMaxCluster && (long long)o.tiles * o.c.row_tiles * o.c.cs * 2 <= sm_count * 5 / 4 &&
         p.w.nkb >= 4 * o.c.cs)
    o.c.cs *= 2;
  o.c.nD = o.NC <= 64 ? 4 : 2;
  const size_t limit = o.NC <= 32 ? 112 * 1024 : kTqSmemMax;
  const size_t stage_w = 2 * (size_t)kQgQuad * p.w.block_bytes, unit = (size_t)o.NC * 256;
  o.c.nW = 2;
  o.c.nB = 2 * o.c.limbs;
  size_t smem = kTqStagesA * kTqA + o.c.nW * stage_w + o.c.nB * unit;
  // what is left: more stages of the weights, then of the planes
  while (o.c.nW < kTqMaxW && smem + stage_w <= limit) {
    ++o.c.nW;
    smem += stage_w;
  }
  while (o.c.nB + o.c.limbs <= kTqMaxB && smem + o.c.limbs * unit <= limit) {
    o.c.nB += o.c.limbs;
    smem += o.c.limbs * unit;
  }
  const size_t staged = p.w2 || o.c.cs > 1 ? (size_t)2 * o.NC * 132 * 4 : 0;
  o.smem = staged > smem ? staged : smem;
  return o;
}

template <int NC, int G>
cudaError_t launch_tc_t(const Q4gParams& p, const TcPlan& o, cudaStream_t s) {
  if (o.smem > kTqSmemMax) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(o.tiles * o.c.cs, o.c.row_tiles, 1);
  cfg.blockDim = dim3(kTqThreads);
  cfg.dynamicSmemBytes = o.smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (o.c.cs > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)o.c.cs;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, q4g_tc_kernel<NC, G>, p, o.c);
}

template <int NC>
cudaError_t launch_tc_g(const Q4gParams& p, const TcPlan& o, cudaStream_t s) {
  switch (p.w.group) {
    case 32: return launch_tc_t<NC, 1>(p, o, s);
    case 64: return launch_tc_t<NC, 2>(p, o, s);
    default: return launch_tc_t<NC, 4>(p, o, s);
  }
}

template <int NC, int G>
cudaError_t prepare_tc_t() {
  return cudaFuncSetAttribute(q4g_tc_kernel<NC, G>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              (int)kTqSmemMax);
}
template <int NC>
cudaError_t prepare_tc_g() {
  cudaError_t e = prepare_tc_t<NC, 1>();
  if (e == cudaSuccess) e = prepare_tc_t<NC, 2>();
  if (e == cudaSuccess) e = prepare_tc_t<NC, 4>();
  return e;
}

}  // namespace

size_t q4g_planes_bytes(const Q4gParams& p, int sm_count) {
  const TcPlan o = plan_tc(p, sm_count);
  return (size_t)o.c.row_tiles * 2 * o.NC * p.w.nkb * kQgBlockK * 2 * o.c.limbs;
}

cudaError_t launch_q4g_tc(const Q4gParams& p, int sm_count, cudaStream_t s) {
  const TcPlan o = plan_tc(p, sm_count);
  const int m8 = (p.a.M + 7) / 8;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.w.nkb * 16 + 31) / 32, m8 < 65535 ? m8 : 65535, 1);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, q4g_planes_kernel, p.a, o.c.limbs, 2 * o.NC);
  if (e != cudaSuccess) return e;
  switch (o.NC) {
    case 16: return launch_tc_g<16>(p, o, s);
    case 32: return launch_tc_g<32>(p, o, s);
    case 64: return launch_tc_g<64>(p, o, s);
    case 96: return launch_tc_g<96>(p, o, s);
    case 128: return launch_tc_g<128>(p, o, s);
  }
  return cudaErrorInvalidValue;
}

cudaError_t prepare_q4g_tc() {
  cudaError_t e = prepare_tc_g<16>();
  if (e == cudaSuccess) e = prepare_tc_g<32>();
  if (e == cudaSuccess) e = prepare_tc_g<64>();
  if (e == cudaSuccess) e = prepare_tc_g<96>();
  if (e == cudaSuccess) e = prepare_tc_g<128>();
  return e;
}

}  // namespace ms
