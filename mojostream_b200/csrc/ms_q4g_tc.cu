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
//   1-2    unpack the weights into the A operand (1-4 for 32-row tiles, where
//          the weights' stream is the bound)
//   last 2 take finished groups out of tensor memory: a thread owns one weight
//          column and half of the rows (one warpgroup and all rows for 32)
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

// Shape of a kernel for tiles of NT rows.  Registers: the launch gives every
// thread kLaunch; then warpgroup 0 and the unpacking ones keep kLow, those
// that hold sums take kHigh.
template <int NT>
struct Tile {
  static constexpr int kCtas = NT <= 64 ? 2 : 1;    // CTAs per SM
  static constexpr int HS = NT <= 32 ? 2 : 1;       // 64-k halves of an operand stage
  static constexpr int kUnpackWg = NT <= 32 ? 4 : 2, kTakeWg = NT <= 32 ? 1 : 2;
  static constexpr int kWg = 1 + kUnpackWg + kTakeWg;
  static constexpr int kThreads = kWg * 4 * kWarp;
  static constexpr int kTakeWarp0 = 4 * (1 + kUnpackWg);
  static constexpr int TC = NT / kTakeWg;           // rows per thread that holds sums
  static constexpr int kLaunch = NT <= 32 ? 40 : NT <= 64 ? 48 : 96;
  static constexpr int kLow = NT <= 32 ? 32 : NT <= 64 ? 40 : 48;
  static constexpr int kHigh = NT <= 32 ? 80 : NT <= 64 ? 56 : 168;
  static_assert((1 + kUnpackWg) * kLow + kTakeWg * kHigh <= kWg * kLaunch, "register split");
  static_assert(kCtas * kThreads * kLaunch <= 65536, "register file");
};
template <int N>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// NT: rows of the tile; G: 32-k steps per group.
template <int NT, int G>
__global__ void __launch_bounds__(Tile<NT>::kThreads, Tile<NT>::kCtas)
    q4g_tc_kernel(const Q4gParams p, const TcShape c) {
  using S_ = Tile<NT>;
  constexpr int HS = S_::HS;
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
      mbar_init(&empty_w[s], 4 * S_::kUnpackWg);
    }
    for (int s = 0; s < c.nS; ++s) {
      mbar_init(&full_s[s], 2 * HS * S_::kUnpackWg + 1);  // the unpacking warps, and the planes' bytes
      mbar_init(&empty_s[s], 1);
    }
    for (int s = 0; s < c.nD; ++s) {
      mbar_init(&full_d[s], 1);
      mbar_init(&empty_d[s], 4 * S_::kTakeWg);
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
    reg_dec<S_::kLow>();
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
    // a wait costs this warp as much as two MMAs, so those of the next stage are
    // taken while half of this one's MMAs are still to issue; with an accumulator
    // to wait for in every half that would hold MMAs back for the sums' warps
    // (groups of 32, 2048 rows: 222 us, and 255 us so), so only for groups of 128
    constexpr bool kAhead = G == 4;
    Ring rs, rd;
    int used = 0;  // accumulators begun
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t phase) {
      return __all_sync(0xffffffffu, mbar_wait(bar, phase)) != 0;
    };
    // stage rs, and the accumulator rd if its first group begins one there
    auto ready = [&](bool begins) {
      return wait(&full_s[rs.slot], rs.phase) &&
             (!begins || used < c.nD || wait(&empty_d[rd.slot], rd.phase ^ 1));
    };
    if (kAhead) ok = ready(true);
    for (int j = 0; j < stages && ok; ++j) {
      if (!kAhead) ok = wait(&full_s[rs.slot], rs.phase);
      const uint64_t da = desc_a + (uint32_t)(rs.slot * stage_s / 16);
      const uint64_t db = desc_b + (uint32_t)(rs.slot * stage_s / 16);
      const int slot = rs.slot;
      rs.next(c.nS);
      tc_fence_after();
#pragma unroll
      for (int h = 0; h < HS; ++h) {
        const bool odd = HS == 2 ? h == 1 : (j & 1) != 0;
#pragma unroll
        for (int g = 0; g < kSub; ++g) {
          const bool begins = G < 4 || !odd, ends = G < 4 || odd;
          const bool last = h == HS - 1 && g == kSub - 1;
          if (begins) {
            if (!kAhead && used >= c.nD) {
              ok = ok && wait(&empty_d[rd.slot], rd.phase ^ 1);
              tc_fence_after();
            }
            ++used;
          }
          const uint32_t dt = tmem + (uint32_t)rd.slot * kColsD;
          auto issue = [&](int l, int k) {
            umma_bf16(dt, da + h * (kTqA / 16) + (g * kK16 + k) * kStepA,
                      db + (uint32_t)((h * c.limbs + l) * (kUnitB / 16)) + (g * kK16 + k) * kStepB, idesc,
                      k != 0 || l != 0 || !begins);
          };
          constexpr int kNow = kAhead ? kK16 / 2 : kK16;  // of a stage's last limb before the waits
          if (ok && elect_one()) {
            for (int l = 0; l + 1 < c.limbs; ++l)
#pragma unroll
              for (int k = 0; k < kK16; ++k) issue(l, k);
#pragma unroll
            for (int k = 0; k < (last ? kNow : kK16); ++k) issue(c.limbs - 1, k);
            if ((!last || !kAhead) && ends) umma_commit(&full_d[rd.slot]);
            if (last && !kAhead) umma_commit(&empty_s[slot]);
          }
          const int sd = rd.slot;
          if (ends) rd.next(c.nD);
          if (kAhead && last) {
            const bool more = j + 1 >= stages || ready(HS == 2 || odd);
            if (ok && elect_one()) {
#pragma unroll
              for (int k = kNow; k < kK16; ++k) issue(c.limbs - 1, k);
              if (ends) umma_commit(&full_d[sd]);
              umma_commit(&empty_s[slot]);
            }
            ok = ok && more;
          }
        }
      }
    }
    if (!ok && lane == 0) fail();
    if (elect_one()) umma_commit(&done);  // arrives when every MMA issued above has finished
    __syncwarp();
    }
  } else if (warp < S_::kTakeWarp0) {
    // ----------------------------------------------------- unpacking --
    // half of the warps the first half of each block, the others the second;
    // kTiles neighbouring tiles to a warp
    reg_dec<S_::kLow>();
    constexpr int kTiles = 4 / S_::kUnpackWg;
    const int half = (warp - 4) / (2 * S_::kUnpackWg), tile0 = (warp - 4) % (2 * S_::kUnpackWg) * kTiles;
    const int r = lane >> 2, t = lane & 3;
    const uint32_t ring_a = smem_u32(ring_s), ring_w_s = smem_u32(ring_w);
    constexpr int ng = 4 / G;
    const bool live = second || tile0 < 4;  // the tiles exist
    Ring rs, rw;
    if (HS == 1) rs.next(c.nS, half);
    for (int kb = 0; kb < blocks; ++kb) {
      if (!mbar_wait(&full_w[rw.slot], rw.phase)) {
        if (lane == 0) fail();
        break;
      }
      const uint32_t pc = ring_w_s + rw.slot * stage_w + tile0 * bb;
      uint4 x[kTiles];
      uint32_t z[kTiles][2];
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        x[j] = lds128(pc + j * bb + half * 512 + lane * 16);
        z[j][0] = z[j][1] = 0x0808u;
        if (p.w.zeros)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh)
            z[j][hh] = lds16(pc + j * bb + kQgNibbles + ng * 32 + ((2 * half + hh) / G * 8 + r) * 2);
      }
      if ((HS == 1 ? 2 * kb + half : kb) >= c.nS && !mbar_wait(&empty_s[rs.slot], rs.phase ^ 1)) {
        if (lane == 0) fail();
        break;
      }
      if (live) {
        const uint32_t dst = ring_a + rs.slot * stage_s + (HS == 2 ? half * kTqA : 0) + t * kTqLboA +
                             tile0 * 256 + r * 16;
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
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
      if (lane == 0) {
        mbar_arrive(&full_s[rs.slot]);
        // only now: what was unpacked depends on the loads from this slot, which
        // the arrival would not have waited for (the MMAs' reads of shared memory
        // can hold loads up until the next copy has landed)
        mbar_arrive(&empty_w[rw.slot]);
      }
      rw.next(c.nW);
      rs.next(c.nS, HS == 1 ? 2 : 1);
    }
  } else {
    // ----------------------------------------------------- group sums --
    reg_inc<S_::kHigh>();
    constexpr int TC = S_::TC;
    const int quad = warp & 3;                  // tensor-memory lanes 32 quad ..
    const int part = (warp - S_::kTakeWarp0) >> 2;  // rows part * TC ..
    const int col = quad * kWarp + lane;        // the thread's weight column
    float2 acc[TC / 2];
#pragma unroll
    for (int i = 0; i < TC / 2; ++i) acc[i] = make_float2(0.f, 0.f);
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
        const uint32_t ta = tmem + ((uint32_t)(quad * kWarp) << 16) + (uint32_t)(rd.slot * (int)kColsD + part * TC);
        const float2 s2 = make_float2(sc[g], sc[g]);
#pragma unroll
        for (int i = 0; i < TC; i += 16) {
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
    for (int i = 0; i < TC; ++i)
      S[(part * TC + i) * kLd + col] = i & 1 ? acc[i / 2].y : acc[i / 2].x;
    if (c.cs > 1) {
      cluster_arrive();
      cluster_wait();
      const uint32_t bad0 = smem_u32(const_cast<int*>(&s_bad));
      for (int k = 0; k < c.cs; ++k) bad |= ld_dsmem_s32(dsmem_addr(bad0, (uint32_t)k));
    } else {
      bar_sync_n(1, 4 * S_::kTakeWg * kWarp);
    }
    if (!bad) {  // no results after a wait that ran out
      const int out_cols = p.w2 ? 64 : 128, sh = p.w2 ? 4 : 5;
      // the rows of this rank, m = rank, rank + cs, ..., four columns to a thread
      constexpr int kTakers = S_::kTakeWg * 4 * kWarp;
      const int i0 = threadIdx.x - S_::kTakeWarp0 * kWarp, n0 = 4 * (i0 & ((1 << sh) - 1));
      const int step = (kTakers >> sh) * c.cs;
#pragma unroll 2
      for (int m = rank + (i0 >> sh) * c.cs; m < rows; m += step) {
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
  // the other warps (few registers): the takers' barriers, and the tensor memory back
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
  int NT, tiles;
  TcShape c;
  size_t smem;
};

int tc_limbs(int type) { return type == kQgF32 ? 3 : type == kQgF16 ? 2 : 1; }

// Clusters of cs CTAs that run at the same time, with `ctas` CTAs to an SM:
// asked of the driver once (prepare_q4g_tc), or an even spread.
int g_clusters[3][kTqMaxCluster + 1];  // [CTAs per SM][cs]
long long clusters_at_once(int sm_count, int ctas, int cs) {
  const int n = g_clusters[ctas][cs];
  return n > 0 ? n : (long long)ctas * sm_count / cs;
}

TcPlan plan_tc(const Q4gParams& p, int sm_count) {
  TcPlan o{};
  o.c.limbs = tc_limbs(p.a.type);
  // rows per tile: as few tiles as fit (256 rows of one limb, 128 of more),
  // all of about the same size
  const int most = o.c.limbs == 1 ? 256 : 128;
  const int row_tiles = (p.a.M + most - 1) / most, each = (p.a.M + row_tiles - 1) / row_tiles;
  const int sizes[5] = {32, 64, 128, 192, 256};
  o.NT = 256;
  // (with limbs a 32-row tile's stages leave one CTA to an SM: 24 rows fp32, K
  // 2560, N 20480 took 62 us so and 50 us in tiles of 64)
  for (int i = 4; i >= (o.c.limbs > 1 ? 1 : 0); --i)
    if (each <= sizes[i]) o.NT = sizes[i];
  o.c.row_tiles = (p.a.M + o.NT - 1) / o.NT;
  o.tiles = p.w2 ? q4g_quads(p.w.N) : (q4g_quads(p.w.N) + 1) / 2;
  // operand stages: at least two; what is left goes to them, then to the weights
  const size_t limit = o.NT <= 64 ? kTqSmemMax / 2 : kTqSmemMax;
  const size_t stage_w = 2 * (size_t)kQgQuad * p.w.block_bytes;
  const size_t stage_s = (o.NT <= 32 ? 2 : 1) * (kTqA + (size_t)o.c.limbs * o.NT * 128);
  o.c.nS = 2;
  o.c.nW = 2;
  o.c.nD = o.NT <= 128 ? 4 : 2;
  size_t smem = o.c.nS * stage_s + o.c.nW * stage_w;
  const int ctas = smem <= limit && o.NT <= 64 ? 2 : 1;  // per SM
  while (o.c.nS < kTqMaxS && smem + stage_s <= limit) {
    ++o.c.nS;
    smem += stage_s;
  }
  while (o.c.nW < kTqMaxW && smem + stage_w <= limit) {
    ++o.c.nW;
    smem += stage_w;
  }
  const size_t staged = (size_t)o.NT * 132 * 4;
  o.smem = staged > smem ? staged : smem;
  // k shared by the CTAs of a cluster: the split with the least rounds x (blocks
  // of a CTA + what a CTA costs besides, about ten blocks).  A cluster's CTAs
  // share a GPC, so what fits at once is counted in clusters (16 rows, K 13824,
  // N 5120: 40 clusters of seven do not, 39 us; of six they do, 29 us).
  const long long grid = (long long)o.tiles * o.c.row_tiles;
  long long best = 0;
  for (int cs = 1; cs <= kTqMaxCluster && (cs == 1 || p.w.nkb >= 4 * cs); ++cs) {
    const long long slots = clusters_at_once(sm_count, ctas, cs);
    const long long cost = (grid + slots - 1) / slots * ((p.w.nkb + cs - 1) / cs + 10);
    if (cs == 1 || cost < best) {
      best = cost;
      o.c.cs = cs;
    }
  }
  return o;
}

template <int NT, int G>
cudaError_t launch_tc_t(const Q4gParams& p, const TcPlan& o, cudaStream_t s) {
  if (o.smem > kTqSmemMax) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(o.tiles * o.c.cs, o.c.row_tiles, 1);
  cfg.blockDim = dim3(Tile<NT>::kThreads);
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
  return cudaLaunchKernelEx(&cfg, q4g_tc_kernel<NT, G>, p, o.c);
}

template <int NT>
cudaError_t launch_tc_g(const Q4gParams& p, const TcPlan& o, cudaStream_t s) {
  switch (p.w.group) {
    case 32: return launch_tc_t<NT, 1>(p, o, s);
    case 64: return launch_tc_t<NT, 2>(p, o, s);
    default: return launch_tc_t<NT, 4>(p, o, s);
  }
}

template <int NT>
void count_clusters(int ctas) {
  for (int cs = kTqMaxCluster; cs >= 1; --cs) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cs * 1024);
    cfg.blockDim = dim3(Tile<NT>::kThreads);
    cfg.dynamicSmemBytes = kTqSmemMax / ctas;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cs;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, q4g_tc_kernel<NT, 4>, &cfg) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
    g_clusters[ctas][cs] = n;
  }
}

template <int NT, int G>
cudaError_t prepare_tc_t() {
  return cudaFuncSetAttribute(q4g_tc_kernel<NT, G>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              (int)kTqSmemMax);
}
template <int NT>
cudaError_t prepare_tc_g() {
  cudaError_t e = prepare_tc_t<NT, 1>();
  if (e == cudaSuccess) e = prepare_tc_t<NT, 2>();
  if (e == cudaSuccess) e = prepare_tc_t<NT, 4>();
  return e;
}

}  // namespace

size_t q4g_planes_bytes(const Q4gParams& p, int sm_count) {
  const TcPlan o = plan_tc(p, sm_count);
  return (size_t)o.c.row_tiles * o.NT * p.w.nkb * kQgBlockK * 2 * o.c.limbs;
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, q4g_planes_kernel, p.a, o.c.limbs, o.NT);
  if (e != cudaSuccess) return e;
  switch (o.NT) {
    case 32: return launch_tc_g<32>(p, o, s);
    case 64: return launch_tc_g<64>(p, o, s);
    case 128: return launch_tc_g<128>(p, o, s);
    case 192: return launch_tc_g<192>(p, o, s);
    case 256: return launch_tc_g<256>(p, o, s);
  }
  return cudaErrorInvalidValue;
}

cudaError_t prepare_q4g_tc() {
  cudaError_t e = prepare_tc_g<32>();
  if (e == cudaSuccess) e = prepare_tc_g<64>();
  if (e == cudaSuccess) e = prepare_tc_g<128>();
  if (e == cudaSuccess) e = prepare_tc_g<192>();
  if (e == cudaSuccess) e = prepare_tc_g<256>();
  if (e == cudaSuccess && !g_clusters[1][1]) {  // (every GPU of a node is alike)
    count_clusters<64>(2);
    count_clusters<256>(1);
  }
  return e;
}

}  // namespace ms
