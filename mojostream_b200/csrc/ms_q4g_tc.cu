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
// the up weight) x NT rows on its N side x a share of the k blocks.  Roles, in
// warpgroups of four warps that split the register file between them:
//   0      weight pieces and limb planes by bulk copy; the MMAs
//   1, 2   unpack the weights of one 64-k half each into the A operand
//   3, 4   take finished groups out of tensor memory (a thread owns one weight
//          column and half of the rows)
// Packed weights, operand stages (HS 64-k halves of A and of every limb of B)
// and accumulators have rings of their own.  With unpacking and sums on the
// same eight warps a 128-k block took 2700 cycles against 1024 of MMAs (256
// rows); with separate rings for A and B the issuing warp's waits took 2200.
// A cluster's CTAs share k; their sums are added in k order through
// distributed shared memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ms_common.cuh"
#include "ms_kernels.h"
#include "ms_q4g.h"
#include "ms_q4g.cuh"
#include "ms_tc.cuh"

namespace ms {
namespace {

constexpr int kTqThreads = 20 * kWarp;
constexpr int kTqLboA = 2048 + 32;  // k cores of A: 32 bytes apart in the banks
constexpr int kTqA = 8 * kTqLboA;   // a 64-k half of 128 columns, bfloat16
constexpr int kTqMaxS = 6, kTqMaxW = 4, kTqMaxD = 4;
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
// Position in a ring of n slots; phase counts the rounds (its parity is the one
// to wait for).
struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int n, int by = 1) {  // by <= n
    slot += by;
    if (slot >= n) {
      slot -= n;
      phase ^= 1;
    }
  }
};

struct TcShape {
  int limbs, nS, nW, nD, cs, row_tiles;
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
// One lane of a converged warp, the same on every call: the compiler then
// keeps what that lane hands to the tensor core in uniform registers (behind
// lane == 0 an MMA took 125 cycles to issue).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void sts128(uint32_t a, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

// Registers a thread of warpgroups 0-2 and of 3-4 holds after the split.  The
// launch gives every thread `kLaunch` (the register file over 20 warps, or
// over 40 where two CTAs share an SM); 12 x low + 8 x high <= 20 x kLaunch.
constexpr __host__ __device__ int halves_per_stage(int NC) { return NC <= 16 ? 2 : 1; }
template <int NC>
struct Regs {
  static constexpr int kCtas = NC <= 32 ? 2 : 1;
  static constexpr int kLaunch = NC <= 32 ? 48 : 96;
  static constexpr int kLow = NC <= 32 ? 40 : 48;
  static constexpr int kHigh = NC <= 16 ? 56 : NC <= 32 ? 56 : 168;
  static_assert(12 * kLow + 8 * kHigh <= 20 * kLaunch, "register split");
};
template <int N>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// NC: rows per thread that takes sums (the tile has NT = 2 NC); G: 32-k steps
// per group.
template <int NC, int G>
__global__ void __launch_bounds__(kTqThreads, Regs<NC>::kCtas)
    q4g_tc_kernel(const Q4gParams p, const TcShape c) {
  constexpr int NT = 2 * NC, HS = halves_per_stage(NC);
  extern __shared__ __align__(1024) uint8_t dsm[];
  __shared__ __align__(8) uint64_t full_w[kTqMaxW], empty_w[kTqMaxW], full_s[kTqMaxS],
      empty_s[kTqMaxS], full_d[kTqMaxD], empty_d[kTqMaxD], done;
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_bad;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int nkb = p.w.nkb, bb = p.w.block_bytes;
  const int rank = blockIdx.x % c.cs, tile = blockIdx.x / c.cs, rt = blockIdx.y;
  const int kb0 = nkb * rank / c.cs, kb1 = nkb * (rank + 1) / c.cs;
  const int blocks = kb1 - kb0, stages = blocks * 2 / HS;
  constexpr int kUnitB = NT * 128;  // a limb of a half
  const int stage_w = 2 * kQgQuad * bb;
  // operand stage: HS halves of A, then [HS][limb] units of B
  const int stage_s = HS * (kTqA + c.limbs * kUnitB);
  uint8_t* ring_s = dsm;
  uint8_t* ring_w = dsm + c.nS * stage_s;
  constexpr uint32_t kColsD = NT;

  if (threadIdx.x == 0) {
    s_bad = 0;
    for (int s = 0; s < c.nW; ++s) {
      mbar_init(&full_w[s], 1);
      mbar_init(&empty_w[s], 8);
    }
    for (int s = 0; s < c.nS; ++s) {
      mbar_init(&full_s[s], 4 * HS + 1);  // the unpacking warps, and the planes' bytes
      mbar_init(&empty_s[s], 1);
    }
    for (int s = 0; s < c.nD; ++s) {
      mbar_init(&full_d[s], 1);
      mbar_init(&empty_d[s], 8);
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
  // the tile's quads of columns (the second may not exist)
  const size_t quad_bytes = (size_t)nkb * kQgQuad * bb;
  const uint8_t* w0 = p.w.w + (size_t)tile * (p.w2 ? 1 : 2) * quad_bytes;
  const uint8_t* w1 = p.w2 ? p.w2 + (size_t)tile * quad_bytes : w0 + quad_bytes;
  const bool second = p.w2 || tile * 2 + 1 < q4g_quads(p.w.N);

  const int row0 = rt * NT, rows = min(NT, p.a.M - row0);
  constexpr int kLd = 128 + 4;
  float* S = reinterpret_cast<float*>(dsm);  // [NT][kLd]: staged sums

  if (warp < 4) {
    reg_dec<Regs<NC>::kLow>();
    if (warp == 0) {
    // ------------------------------------------------ weight producer --
    if (lane == 0) {
      const uint8_t* x0 = w0 + (size_t)kb0 * kQgQuad * bb;
      const uint8_t* x1 = w1 + (size_t)kb0 * kQgQuad * bb;
      const int n = blocks, run = kQgQuad * bb;
      Ring w;
      int i = 0;
      for (; i < n; ++i, w.next(c.nW)) {  // no kernel writes the weights: no wait for the previous one
        if (i >= c.nW && !mbar_wait(&empty_w[w.slot], w.phase ^ 1)) break;
        uint8_t* st = ring_w + w.slot * stage_w;
        mbar_expect_tx(&full_w[w.slot], run * (1 + second));
        bulk_g2s(st, x0, run, &full_w[w.slot]);
        if (second) bulk_g2s(st + run, x1, run, &full_w[w.slot]);
        x0 += run;
        x1 += run;
      }
      if (i < n) fail();
      // the copies issued last land before the CTA can exit
      for (int j = max(0, i - c.nW); j < i; ++j) mbar_wait(&full_w[j % c.nW], (j / c.nW) & 1);
    }
    } else if (warp == 2) {
    // ------------------------------------------------- planes producer --
    if (lane == 0) {
      const int bytes = HS * c.limbs * kUnitB;
      const uint8_t* b0 = p.a.records + ((size_t)rt * nkb + kb0) * 2 * c.limbs * kUnitB;
      pdl_wait();
      Ring u;
      int i = 0;
      for (; i < stages; ++i, u.next(c.nS)) {
        if (i >= c.nS && !mbar_wait(&empty_s[u.slot], u.phase ^ 1)) break;
        mbar_expect_tx(&full_s[u.slot], bytes);
        bulk_g2s(ring_s + u.slot * stage_s + HS * kTqA, b0, bytes, &full_s[u.slot]);
        b0 += bytes;
      }
      if (i < stages) {
        fail();
        // (the copies that were issued: bounded, the unpacking may have stopped)
        for (int j = max(0, i - c.nS); j < i; ++j) mbar_wait(&full_s[j % c.nS], (j / c.nS) & 1);
      }
    }
    } else if (warp == 1) {
    // ------------------------------------------------------ MMA issuer --
    // (the whole warp walks the loop, one lane issues)
    const uint32_t idesc = idesc_bf16(128, NT);
    const uint64_t desc_a = umma_desc(smem_u32(ring_s), kTqLboA, 128);
    const uint64_t desc_b = umma_desc(smem_u32(ring_s) + HS * kTqA, NT * 16, 128);
    constexpr uint32_t kStepA = 2 * kTqLboA / 16, kStepB = 2 * NT;  // 16 k, in 16-byte units
    // groups that a half completes (32: two, 64: one, 128: every second half one)
    constexpr int kSub = G == 1 ? 2 : 1, kK16 = 4 / kSub;
    Ring rs, rd;
    int used = 0;  // accumulators begun
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t phase) {
      return __all_sync(0xffffffffu, mbar_wait(bar, phase)) != 0;
    };
    for (int j = 0; j < stages && ok; ++j, rs.next(c.nS)) {
      ok = wait(&full_s[rs.slot], rs.phase);
      const uint64_t da = desc_a + (uint32_t)(rs.slot * stage_s / 16);
      const uint64_t db = desc_b + (uint32_t)(rs.slot * stage_s / 16);
      tc_fence_after();
#pragma unroll
      for (int h = 0; h < HS; ++h) {
        const bool odd = HS == 2 ? h == 1 : (j & 1) != 0;
#pragma unroll
        for (int g = 0; g < kSub; ++g) {
          const bool begins = G < 4 || !odd, ends = G < 4 || odd;
          if (begins) {
            if (used >= c.nD) {
              ok = ok && wait(&empty_d[rd.slot], rd.phase ^ 1);
              tc_fence_after();
            }
            ++used;
          }
          const uint32_t dt = tmem + (uint32_t)rd.slot * kColsD;
          if (ok && elect_one()) {
            for (int l = 0; l < c.limbs; ++l) {
              const uint64_t dbl = db + (uint32_t)((h * c.limbs + l) * (kUnitB / 16));
#pragma unroll
              for (int k = 0; k < kK16; ++k)
                umma_bf16(dt, da + h * (kTqA / 16) + (g * kK16 + k) * kStepA, dbl + (g * kK16 + k) * kStepB,
                          idesc, k != 0 || l != 0 || !begins);
            }
            if (ends) umma_commit(&full_d[rd.slot]);
            if (h == HS - 1 && g == kSub - 1) umma_commit(&empty_s[rs.slot]);
          }
          if (ends) rd.next(c.nD);
        }
      }
    }
    if (!ok && lane == 0) fail();
    if (elect_one()) umma_commit(&done);  // arrives when every MMA issued above has finished
    __syncwarp();
    }
  } else if (warp < 12) {
    // ----------------------------------------------------- unpacking --
    // warps 4-7 the first half of each block, 8-11 the second; two tiles each
    reg_dec<Regs<NC>::kLow>();
    const int half = (warp - 4) >> 2, i = warp & 3;
    const int r = lane >> 2, t = lane & 3;
    const uint32_t ring_a = smem_u32(ring_s), ring_w_s = smem_u32(ring_w);
    constexpr int ng = 4 / G;
    const bool live = second || i < 2;  // the tiles exist
    Ring rs, rw;
    if (HS == 1) rs.next(c.nS, half);
    for (int kb = 0; kb < blocks; ++kb) {
      if (!mbar_wait(&full_w[rw.slot], rw.phase)) {
        if (lane == 0) fail();
        break;
      }
      const uint32_t pc = ring_w_s + rw.slot * stage_w + 2 * i * bb;
      const uint4 x[2] = {lds128(pc + half * 512 + lane * 16), lds128(pc + bb + half * 512 + lane * 16)};
      uint32_t z[2][2] = {{0x0808u, 0x0808u}, {0x0808u, 0x0808u}};
      if (p.w.zeros)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh)
            z[j][hh] = lds16(pc + j * bb + kQgNibbles + ng * 32 + ((2 * half + hh) / G * 8 + r) * 2);
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_w[rw.slot]);
      rw.next(c.nW);
      if ((HS == 1 ? 2 * kb + half : kb) >= c.nS && !mbar_wait(&empty_s[rs.slot], rs.phase ^ 1)) {
        if (lane == 0) fail();
        break;
      }
      if (live) {
        const uint32_t dst = ring_a + rs.slot * stage_s + (HS == 2 ? half * kTqA : 0) + t * kTqLboA +
                             2 * i * 256 + r * 16;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t l0 = (0x4300u | (z[j][0] & 0xffu)) * 0x10001u, h0 = (0x4300u | (z[j][0] >> 8)) * 0x10001u;
          const uint32_t l1 = (0x4300u | (z[j][1] & 0xffu)) * 0x10001u, h1 = (0x4300u | (z[j][1] >> 8)) * 0x10001u;
          sts128(dst + j * 256, unpack8(x[j].x, x[j].y, 0, l0));
          sts128(dst + j * 256 + 128, unpack8(x[j].x, x[j].y, 4, h0));
          sts128(dst + j * 256 + 4 * kTqLboA, unpack8(x[j].z, x[j].w, 0, l1));
          sts128(dst + j * 256 + 4 * kTqLboA + 128, unpack8(x[j].z, x[j].w, 4, h1));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full_s[rs.slot]);
      rs.next(c.nS, HS == 1 ? 2 : 1);
    }
  } else {
    // ----------------------------------------------------- group sums --
    reg_inc<Regs<NC>::kHigh>();
    const int quad = warp & 3;                  // tensor-memory lanes 32 quad ..
    const int half_n = (warp - 12) >> 2;        // rows half_n * NC ..
    const int col = quad * kWarp + lane;        // the thread's weight column
    float2 acc[NC / 2];
#pragma unroll
    for (int i = 0; i < NC / 2; ++i) acc[i] = make_float2(0.f, 0.f);
    // the column's scales, a block ahead, from the weight's pieces (in L2)
    constexpr int ng = 4 / G;
    const bool exists = second || quad < 2;
    const uint8_t* scales = (quad < 2 ? w0 : w1) + (size_t)kb0 * kQgQuad * bb + ((col & 63) >> 4) * bb +
                            kQgNibbles + ((col & 7) * 2 + ((col >> 3) & 1)) * 2;
    unsigned short sn[ng];
    auto fetch = [&]() {
#pragma unroll
      for (int g = 0; g < ng; ++g)
        sn[g] = exists ? __ldg(reinterpret_cast<const unsigned short*>(scales + g * 32)) : 0;
      scales += kQgQuad * bb;
    };
    fetch();
    Ring rd;
    bool ok = true;
    for (int kb = 0; kb < blocks && ok; ++kb) {
      float sc[ng];
#pragma unroll
      for (int g = 0; g < ng; ++g) sc[g] = u16_scale(sn[g], p.w.bf_scale);
      if (kb + 1 < blocks) fetch();
#pragma unroll
      for (int g = 0; g < ng; ++g) {
        ok = ok && mbar_wait(&full_d[rd.slot], rd.phase);
        if (!ok) break;
        tc_fence_after();
        const uint32_t ta = tmem + ((uint32_t)(quad * kWarp) << 16) + (uint32_t)(rd.slot * (int)kColsD + half_n * NC);
        const float2 s2 = make_float2(sc[g], sc[g]);
#pragma unroll
        for (int i = 0; i < NC; i += 16) {
          uint32_t v[16];
          tmem_ld16(ta + i, v);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 8; ++e)
            fma2(acc[i / 2 + e], make_float2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), s2);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty_d[rd.slot]);
        rd.next(c.nD);
      }
    }
    if (!ok && lane == 0) fail();
    if (!mbar_wait(&done, 0) && lane == 0) fail();  // no MMA is in flight
    tc_fence_before();
    __syncthreads();
    // --------------------------------------------------------- results --
    // by way of shared memory (every copy into it has landed: the MMAs and the
    // unpacking waited for them), rows of 128 columns, four to a thread
    int bad = s_bad;
    pdl_wait();  // results may overwrite what the previous kernel still reads
#pragma unroll
    for (int i = 0; i < NC; ++i)
      S[(half_n * NC + i) * kLd + col] = i & 1 ? acc[i / 2].y : acc[i / 2].x;
    if (c.cs > 1) {
      cluster_arrive();
      cluster_wait();
      const uint32_t bad0 = smem_u32(const_cast<int*>(&s_bad));
      for (int k = 0; k < c.cs; ++k) bad |= ld_dsmem_s32(dsmem_addr(bad0, (uint32_t)k));
    } else {
      bar_sync_n(1, 8 * kWarp);
    }
    if (!bad) {  // no results after a wait that ran out
      const int out_cols = p.w2 ? 64 : 128, sh = p.w2 ? 4 : 5;
      // the rows of this rank: m = rank, rank + cs, ...
      const int mine = rank < rows ? (rows - rank + c.cs - 1) / c.cs : 0;
      for (int i = threadIdx.x - 12 * kWarp; i < mine << sh; i += 8 * kWarp) {
        const int m = rank + (i >> sh) * c.cs, n0 = 4 * (i & ((1 << sh) - 1));
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f), u = v;
        const float* at = S + m * kLd + n0;
        if (c.cs > 1) {
          for (int k = 0; k < c.cs; ++k) add4(v, ld_dsmem4(dsmem_addr(smem_u32(at), (uint32_t)k)));
          if (p.w2)
            for (int k = 0; k < c.cs; ++k) add4(u, ld_dsmem4(dsmem_addr(smem_u32(at + 64), (uint32_t)k)));
        } else {
          v = *reinterpret_cast<const float4*>(at);
          if (p.w2) u = *reinterpret_cast<const float4*>(at + 64);
        }
        finish4(p, row0 + m, tile * out_cols + n0, v, u);
      }
    }
    if (c.cs > 1) {  // the other CTAs have read this one's sums
      cluster_arrive();
      cluster_wait();
    }
    return;
  }
  // warps 0-11 (few registers): the takers' barriers, and the tensor memory back
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, cols);
  if (c.cs > 1) {
    cluster_arrive();
    cluster_wait();
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
  const size_t limit = o.NC <= 32 ? kTqSmemMax / 2 : kTqSmemMax;
  const size_t stage_w = 2 * (size_t)kQgQuad * p.w.block_bytes, unit = (size_t)o.NC * 256;
  const int hs = halves_per_stage(o.NC);
  const size_t stage_s = hs * (kTqA + o.c.limbs * unit);
  o.c.nS = 2;
  o.c.nW = 2;
  size_t smem = o.c.nS * stage_s + o.c.nW * stage_w;
  while (o.c.nS < kTqMaxS && smem + stage_s <= limit) {
    ++o.c.nS;
    smem += stage_s;
  }
  while (o.c.nW < kTqMaxW && smem + stage_w <= limit) {
    ++o.c.nW;
    smem += stage_w;
  }
  const size_t staged = (size_t)2 * o.NC * 132 * 4;
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
