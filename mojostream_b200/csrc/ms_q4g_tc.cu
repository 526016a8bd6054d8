// ms_q4g_tc.cu -- products with group-scaled 4-bit weights for many rows, on
// the 5th-generation tensor cores (layout: ms_q4g.h):
//   C[m][n] (+)= sum_k A[m][k] (q[k][n] - z) s,   H = act(A Wg) * (A Wu).
//
// Mathematics.  q - z is an integer of at most 5 bits: exact in bfloat16.  The
// bits of q alone, in bits 0-3 or 4-7, are the bfloat16 q 2^-133 or 16 q 2^-133
// (the numbers up to 2^-125 are evenly spaced), so one fused multiply-add gives
// (q - z) / 128 without a shift; the sums are multiplied by 128 at the end.
// An activation is cut into bfloat16 limbs that add up to it exactly (fp32:
// 8 + 8 + 8 bits, fp16: 8 + 3, bfloat16: itself; bits of fp32 below bfloat16's
// least, 2^-133, are lost, which reaches values under 2^-110), so every product of a
// tcgen05.mma is exact and its fp32 accumulator in tensor memory holds the sum
// of one group of k over all limbs (fp32 rows: of at most 64 k); when it ends the
// group's scale is applied and it is added to fp32 sums in registers.
//
// CTA: tiles of 128 weight columns on the MMA's M side (gated: 64 of the gate,
// 64 of the up weight, in turns of 16) x NT rows on its N side x a share of the
// k blocks.  Roles, in warpgroups of four warps that split the register file
// between them:
//   0      weight pieces and limb planes by bulk copy; the MMAs
//   1-2    unpack the weights into the A operand (1-4 for 32-row tiles, where
//          the weights' stream is the bound)
//   last 2 take finished groups out of tensor memory: a thread owns one weight
//          column and half of the rows (one warpgroup and all rows for 32)
// The A operand lies in tensor memory, written in the weights' fragment order:
// in shared memory its 64 KB of traffic a block and the MMA's own reads were
// the bound (an MMA of 32 rows took 40 cycles so, and takes 17).  That leaves
// 384 of 512 columns for accumulators: tiles of at most 192 rows.
// The roles walk the CTA's tiles without a break, so weights and planes of the
// next tile are there when it begins.  Where there are too few tiles, a
// cluster's CTAs share the k of one; their sums are added in k order through
// distributed shared memory.
// The loops are kept short: with unrolled limbs and the next stage's waits among
// the MMAs 2048 rows (K 2560, N 10240, bfloat16) took 137 us, and take 98 us
// (1095 TFLOP/s; inputs that are not in L2 113 us; 4096 x 5120 x 13824 537 us,
// 1080 TFLOP/s), with the activation's exact division unrolled 519 gated rows took
// 114 us, and take 99.
//
// What bounds it: many rows, the MMAs (at their measured rate 65 of the 98 us)
// and the hand-over between the roles; a quarter of the planes' bytes (58 KB a
// block come from L2) would save 9 us, no writing of results as much.  Few rows:
// a chain of 1.2 us per block of 128 k (an unpacking warp waits for its stage,
// unpacks, stores to tensor memory, waits for the store, arrives and only then
// takes the next block's words), the same in tiles of 32 and of 64 rows though
// there a warp unpacks twice as much (64 gated rows, K 5120, N 13824, 40 blocks
// a CTA: 48 us, issue slots taken for 61 % of the active cycles, the tensor pipe
// for 21 %).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>

#include "ms_common.cuh"
#include "ms_kernels.h"
#include "ms_q4g.h"
#include "ms_q4g.cuh"
#include "ms_tc.cuh"

namespace ms {
namespace {

constexpr int kTqMaxS = 4, kTqMaxW = 8;
// dynamic shared memory of a CTA, alone on its SM or one of two
constexpr size_t kTqSmemMax = 224 * 1024, kTqSmemHalf = 110 * 1024;
constexpr int kTqMaxCluster = 8;
constexpr int kChunk = 32;  // rows of a chunk of results
constexpr int kChunkBytes = 8 * kChunk * (kWarp + 4) * 4;

// -------------------------------------------------------------- planes --
// The next limb of v, the leading 8 bits of what is left (truncated, so nothing
// can round up to infinity).  An infinity or a NaN stays in the first limb alone.
__device__ __forceinline__ uint32_t next_limb(float& v) {
  const uint32_t u = __float_as_uint(v), top = u & 0xffff0000u;
  if ((u & 0x7f800000u) == 0x7f800000u) {
    v = 0.f;
    return u & 0x007fffffu ? top | 0x00400000u : top;  // a NaN's payload may sit in the low bits
  }
  v -= __uint_as_float(top);
  return top;
}

// Planes [row tile][64-k half][limb][NT rows][128 bytes, swizzled]: the B
// operand.  The weights' fragments put k 8 t + 2 j and the one after it, of each
// 32 k, into column 4 j + t of the A operand, so the 16-byte piece j of the 32 k
// holds those pairs for t = 0..3.  Thread: 32 k of one row; rows past M
// are left as they are (their columns of the product are not used).
__global__ void __launch_bounds__(128) q4g_planes_kernel(const Q4gRows a, int limbs, int NT) {
  pdl_wait();     // the rows are an earlier kernel's output, and the planes
  pdl_trigger();  // may still be read by the product before this one
  // eight neighbouring threads: eight rows; then k
  const int spans = a.nkb * 4;
  for (int m8 = blockIdx.y; m8 < (a.M + 7) / 8; m8 += gridDim.y) {
    const int m = m8 * 8 + (threadIdx.x & 7), span = blockIdx.x * 16 + (threadIdx.x >> 3);
    if (m >= a.M || span >= spans) continue;
    float v[4][8];
#pragma unroll
    for (int t = 0; t < 4; ++t) load8(a, m, span * 32 + t * 8, v[t]);
    const int rt = m / NT, r = m % NT;
    uint8_t* dst = a.records +
                   (((size_t)rt * a.nkb * 2 + (span >> 1)) * limbs * NT + r) * 128;
    for (int l = 0; l < limbs; ++l, dst += NT * 128)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t w[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint32_t lo = next_limb(v[t][2 * j]), hi = next_limb(v[t][2 * j + 1]);
          w[t] = __byte_perm(lo, hi, 0x7632);
        }
        *reinterpret_cast<uint4*>(dst + ((((span & 1) * 4 + j) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
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
  int limbs, nS, nW, cs, row_tiles;
  int tiles, units;  // column tiles; tiles in all
};

__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
constexpr uint32_t kUp126 = 0x7E807E80u, kUp122 = 0x7C807C80u;  // pairs of 2^126, 2^122
constexpr uint32_t kMinus8 = 0xBD80BD80u;                       // -8 / 128
// -z / 128 in both halves, z a byte of v (0 or 1)
__device__ __forceinline__ uint32_t bias_of(uint32_t v, int byte) {
  return fma_bf16x2(__byte_perm(v, 0, byte ? 0x4141 : 0x4040), kUp126 | 0x80008000u, 0x80008000u);
}
// k 0..7 of the columns r (low nibbles) and r + 8 in the words x, y as bfloat16
// pairs: r's into the even, the other's into the odd of o.
__device__ __forceinline__ void unpack16(uint32_t x, uint32_t y, uint32_t bias_lo, uint32_t bias_hi,
                                         uint32_t* o) {
  const uint32_t w[4] = {x, x >> 8, y, y >> 8};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    o[2 * e] = fma_bf16x2(w[e] & 0x000F000Fu, kUp126, bias_lo);
    o[2 * e + 1] = fma_bf16x2(w[e] & 0x00F000F0u, kUp122, bias_hi);
  }
}
// Shared to global, both 16-byte aligned, in the thread's open bulk group.
__device__ __forceinline__ void bulk_s2g(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void sts16(uint32_t a, uint32_t v) {
  asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"((unsigned short)v) : "memory");
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

// Shape of a kernel for tiles of NT rows.  Registers: the launch gives every
// thread kLaunch; then warpgroup 0 and the unpacking ones keep kLow, those
// that hold sums take kHigh.
template <int NT>
struct Tile {
  static constexpr int kCtas = NT <= 64 ? 2 : 1;    // CTAs per SM
  static constexpr int HS = NT == 32 || NT == 192 ? 2 : 1;       // 64-k halves of an operand stage
  static constexpr int kUnpackWg = NT <= 32 ? 4 : 2, kTakeWg = NT <= 32 ? 1 : 2;
  static constexpr int kWg = 1 + kUnpackWg + kTakeWg;
  static constexpr int kThreads = kWg * 4 * kWarp;
  // tensor memory: accumulators, then operand stages of 32 columns to a half
  static constexpr int kCols = 512 / kCtas;
  static constexpr int kD = NT == 128 ? 3 : 2;
  static constexpr int kMaxS = (kCols - kD * NT) / (32 * HS);
  static_assert(kMaxS >= 2 && kMaxS <= kTqMaxS, "tensor memory");
  static constexpr bool kWalk = NT >= 128;  // the CTA's tiles one after the other
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

// NT: rows of the tile; G: 32-k steps that an accumulator sums: a group's, or
// (`parts`, fp32 rows) two of a group of four.
template <int NT, int G, bool parts = false>
__global__ void __launch_bounds__(Tile<NT>::kThreads, Tile<NT>::kCtas)
    q4g_tc_kernel(const Q4gParams p, const TcShape c) {
  using S_ = Tile<NT>;
  constexpr int HS = S_::HS;
  extern __shared__ __align__(1024) uint8_t dsm[];
  __shared__ __align__(8) uint64_t full_w[kTqMaxW], empty_w[kTqMaxW], full_s[kTqMaxS],
      empty_s[kTqMaxS], full_d[S_::kD], empty_d[S_::kD], done, full_t, empty_t;
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_bad;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int nkb = p.w.nkb, bb = p.w.block_bytes;
  // this CTA's tiles: unit0, unit0 + step, ... (in a cluster one, shared)
  const int rank = blockIdx.x % c.cs, unit0 = blockIdx.x / c.cs;
  const int step = gridDim.x;
  const int n_units = S_::kWalk && c.cs == 1 ? (c.units - unit0 + step - 1) / step : 1;
  const int kb0 = nkb * rank / c.cs, kb1 = nkb * (rank + 1) / c.cs;
  const int blocks = kb1 - kb0, stages = blocks * 2 / HS;  // of a tile
  constexpr int kUnitB = NT * 128;  // a limb of a half
  const int stage_w = 2 * kQgQuad * bb;
  // operand stage: [HS halves][limb] units of B (A's is in tensor memory)
  const int stage_s = HS * c.limbs * kUnitB;
  uint8_t* ring_s = dsm;
  uint8_t* ring_w = dsm + c.nS * stage_s;
  // results: [warp][kChunk][kLdO], and behind them a tile of 16-bit rows (apart:
  // a warp may be a tile ahead of another)
  float* ring_o = reinterpret_cast<float*>(ring_w + c.nW * stage_w);
  const uint32_t tile_o = smem_u32(ring_o) + kChunkBytes;
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
    for (int s = 0; s < S_::kD; ++s) {
      mbar_init(&full_d[s], 1);
      mbar_init(&empty_d[s], 4 * S_::kTakeWg);
    }
    mbar_init(&done, 1);
    mbar_init(&full_t, 4 * S_::kTakeWg);
    mbar_init(&empty_t, 1);
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(&s_tmem, S_::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem, tmem_a = tmem + S_::kD * NT;
  pdl_trigger();

  auto fail = [&]() {
    atomicOr(p.err, kErrWaitTimeout);
    s_bad = 1;
  };
  // a tile's quads of columns (the second may not exist)
  const size_t quad_bytes = (size_t)nkb * kQgQuad * bb;
  const int quads = q4g_quads(p.w.N), run = kQgQuad * bb;
  struct Unit {
    int tile, rt;
    const uint8_t *w0, *w1;
    bool second;
  };
  auto unit = [&](int n) {
    const int u = unit0 + n * step;
    Unit o;
    o.rt = u / c.tiles;
    o.tile = u - o.rt * c.tiles;
    o.w0 = p.w.w + (size_t)o.tile * (p.w2 ? 1 : 2) * quad_bytes + (size_t)kb0 * run;
    o.w1 = p.w2 ? p.w2 + (size_t)o.tile * quad_bytes + (size_t)kb0 * run : o.w0 + quad_bytes;
    o.second = p.w2 || o.tile * 2 + 1 < quads;
    return o;
  };

  // a tile whose results leave by bulk copies while the next one is made: not
  // the last, only rounded, inside the matrix, aligned (2048 rows: 104 us without,
  // and 99 us; the last tile so, too: 128 rows, K 5120, N 13824 38 and 41 us)
  const bool plain = S_::kWalk && c.cs == 1 && !p.accumulate && !p.w2 && !((uintptr_t)p.out & 15) &&
                     p.ldo * (p.a.type == kQgF32 ? 4 : 2) % 16 == 0;
  auto by_bulk = [&](const Unit& t, int n) {
    return plain && p.a.type != kQgF32 && n + 1 < n_units && t.tile * 128 + 128 <= p.w.N;
  };

  constexpr int kLd = 128 + 4, kLdO = kWarp + 4;
  float* S = reinterpret_cast<float*>(dsm);  // [NT][kLd]: a cluster's staged sums

  if (warp < 4) {
    reg_dec<S_::kLow>();
    if (warp == 0) {
    // ------------------------------------------------ weight producer --
    if (lane == 0) {
      Ring w;
      int i = 0;
      const int total = blocks * n_units;
      for (int n = 0; n < n_units; ++n) {
        const Unit t = unit(n);
        const uint8_t *x0 = t.w0, *x1 = t.w1;
        int b = 0;
        for (; b < blocks; ++b, ++i, w.next(c.nW)) {  // no kernel writes the weights: no wait for the previous one
          if (i >= c.nW && !mbar_wait(&empty_w[w.slot], w.phase ^ 1)) break;
          uint8_t* st = ring_w + w.slot * stage_w;
          mbar_expect_tx(&full_w[w.slot], run * (1 + t.second));
          bulk_g2s(st, x0, run, &full_w[w.slot]);
          if (t.second) bulk_g2s(st + run, x1, run, &full_w[w.slot]);
          x0 += run;
          x1 += run;
        }
        if (b < blocks) break;
      }
      if (i < total) fail();
      // the copies issued last land before the CTA can exit
      for (int j = max(0, i - c.nW); j < i; ++j) mbar_wait(&full_w[j % c.nW], (j / c.nW) & 1);
    }
    } else if (warp == 2) {
    // ------------------------------------------------- planes producer --
    if (lane == 0) {
      const int bytes = HS * c.limbs * kUnitB;
      pdl_wait();
      Ring u;
      int i = 0;
      const int total = stages * n_units;
      for (int n = 0; n < n_units; ++n) {
        const uint8_t* b0 = p.a.records + ((size_t)unit(n).rt * nkb + kb0) * 2 * c.limbs * kUnitB;
        int b = 0;
        for (; b < stages; ++b, ++i, u.next(c.nS)) {
          if (i >= c.nS && !mbar_wait(&empty_s[u.slot], u.phase ^ 1)) break;
          mbar_expect_tx(&full_s[u.slot], bytes);
          bulk_g2s(ring_s + u.slot * stage_s, b0, bytes, &full_s[u.slot]);
          b0 += bytes;
        }
        if (b < stages) break;
      }
      if (i < total) {
        fail();
        // (the copies that were issued: bounded, the unpacking may have stopped)
        for (int j = max(0, i - c.nS); j < i; ++j) mbar_wait(&full_s[j % c.nS], (j / c.nS) & 1);
      }
    }
    } else if (warp == 1) {
    // ------------------------------------------------------ MMA issuer --
    // (the whole warp walks the loop, one lane issues)
    const uint32_t idesc = idesc_bf16(128, NT);
    const uint64_t desc_b = umma_desc_sw128(smem_u32(ring_s));
    constexpr uint32_t kStepB = 2;  // 16 k, in 16-byte units
    // groups that a half completes (32: two, 64: one, 128: every second half one)
    constexpr int kSub = G == 1 ? 2 : 1, kK16 = 4 / kSub;
    Ring rs, rd;
    int used = 0;  // accumulators begun
    bool ok = true;
    const int total = stages * n_units;  // (an even number of halves to a tile)
    for (int j = 0; j < total && ok; ++j) {
      ok = mbar_wait_warp(&full_s[rs.slot], rs.phase);
      const uint32_t da = tmem_a + (uint32_t)(rs.slot * HS * 32);
      const uint64_t db = desc_b + (uint32_t)(rs.slot * stage_s / 16);
      tc_fence_after();
#pragma unroll
      for (int h = 0; h < HS; ++h) {
        const bool odd = HS == 2 ? h == 1 : (j & 1) != 0;
#pragma unroll
        for (int g = 0; g < kSub; ++g) {
          const bool begins = G < 4 || !odd, ends = G < 4 || odd;
          if (begins) {
            if (used >= S_::kD) {
              ok = ok && mbar_wait_warp(&empty_d[rd.slot], rd.phase ^ 1);
              tc_fence_after();
            }
            ++used;
          }
          const uint32_t dt = tmem + (uint32_t)rd.slot * kColsD;
          if (ok && elect_one()) {
            // the smallest limbs first: an MMA cuts its sum off below the
            // accumulator's last place, which costs least while that is small
            for (int l = c.limbs - 1; l >= 0; --l)
#pragma unroll
              for (int k = 0; k < kK16; ++k)
                umma_bf16_ta(dt, da + h * 32 + (g * kK16 + k) * 8,
                             db + (uint32_t)((h * c.limbs + l) * (kUnitB / 16)) +
                                 (g * kK16 + k) * kStepB,
                             idesc, k != 0 || l != c.limbs - 1 || !begins);
            if (ends) umma_commit(&full_d[rd.slot]);
            if (h == HS - 1 && g == kSub - 1) umma_commit(&empty_s[rs.slot]);
          }
          if (ends) rd.next(S_::kD);
        }
      }
      rs.next(c.nS);
    }
    if (!ok && lane == 0) fail();
    if (elect_one()) umma_commit(&done);  // arrives when every MMA issued above has finished
    __syncwarp();
    } else if (plain) {
    // ------------------------------------- whole tiles of 16-bit results --
    pdl_wait();  // they may overwrite what the previous kernel still reads
    int written = 0;
    for (int n = 0; n < n_units; ++n) {
      const Unit t = unit(n);
      if (!by_bulk(t, n)) continue;
      if (!mbar_wait_warp(&full_t, written & 1)) {
        if (lane == 0) fail();
        break;
      }
      const int rows = min(NT, p.a.M - t.rt * NT);
      uint8_t* dst = reinterpret_cast<uint8_t*>(p.out) + ((size_t)t.rt * NT * p.ldo + t.tile * 128) * 2;
      for (int r = lane; r < rows; r += kWarp) bulk_s2g(dst + (size_t)r * p.ldo * 2, tile_o + r * 256, 256);
      bulk_commit();
      bulk_wait_read();
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_t);
      ++written;
    }
    bulk_wait();
    }
  } else if (warp < S_::kTakeWarp0) {
    // ----------------------------------------------------- unpacking --
    // half of the warps the first 64 k of each block, the others the second; of
    // the 32 columns in the warp's quarter of the tensor memory's lanes, kTiles x 16
    reg_dec<S_::kLow>();
    constexpr int kTiles = 4 / S_::kUnpackWg;
    const int quad = warp & 3, wg = (warp - 4) >> 2;
    const int half = wg * kTiles >> 1, j0 = kTiles == 1 ? wg & 1 : 0;
    const int r = lane >> 2;
    const uint32_t ring_w_s = smem_u32(ring_w);
    const uint32_t ta = tmem_a + ((uint32_t)(quad * kWarp + j0 * 16) << 16) + (HS == 2 ? half * 32 : 0);
    // the tiles among a stage's eight
    const int piece = p.w2 ? quad + 4 * j0 : 2 * quad + j0, piece_step = (p.w2 ? 4 : 1) * bb;
    constexpr int ng = parts ? 1 : 4 / G;  // groups of a block
    Ring rs, rw;
    if (HS == 1) rs.next(c.nS, half);
    int n = 0, left = blocks;
    bool live = unit(0).second || quad < 2;  // the tiles exist
    uint4 x[kTiles];
    uint32_t z[kTiles][2];
    auto load = [&]() {  // the tiles of the next block, if it has arrived
      if (!mbar_wait_warp(&full_w[rw.slot], rw.phase)) return false;
      const uint32_t pc = ring_w_s + rw.slot * stage_w + piece * bb;
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        x[j] = lds128(pc + j * piece_step + half * 512 + lane * 16);
        if (p.w.zeros)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh)
            z[j][hh] = lds16(pc + j * piece_step + kQgNibbles + ng * 32 + ((2 * half + hh) * ng / 4 * 8 + r) * 2);
      }
      return true;
    };
    bool ok = load();
    const int total = blocks * n_units;
    for (int kb = 0; kb < total && ok; ++kb, --left) {
      if (left == 0) {
        left = blocks;
        live = unit(++n).second || quad < 2;
      }
      ok = (HS == 1 ? 2 * kb + half : kb) < c.nS || mbar_wait_warp(&empty_s[rs.slot], rs.phase ^ 1);
      if (!ok) break;
      tc_fence_after();
      if (live) {
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          uint32_t o[16];
          if (p.w.zeros) {
            unpack16(x[j].x, x[j].y, bias_of(z[j][0], 0), bias_of(z[j][0], 1), o);
            unpack16(x[j].z, x[j].w, bias_of(z[j][1], 0), bias_of(z[j][1], 1), o + 8);
          } else {
            unpack16(x[j].x, x[j].y, kMinus8, kMinus8, o);
            unpack16(x[j].z, x[j].w, kMinus8, kMinus8, o + 8);
          }
          tmem_st_16x32(ta + rs.slot * (HS * 32) + (j << 20), o);
        }
        tmem_wait_st();
      }
      tc_fence_before();
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
      if (kb + 1 < total) ok = load();
    }
    if (!ok && lane == 0) fail();
  } else {
    // ----------------------------------------------------- group sums --
    reg_inc<S_::kHigh>();
    constexpr int TC = S_::TC, kLoad = TC >= 64 ? 32 : 16;  // rows in all, and taken at once
    const int quad = warp & 3;                  // tensor-memory lanes 32 quad ..
    const int part = (warp - S_::kTakeWarp0) >> 2;  // rows part * TC ..
    // the thread's weight column: of this tile among a stage's eight (gated: of
    // the gate for the lower lanes, the same column of the up weight for the others)
    const int piece = p.w2 ? quad + (lane >> 4) * 4 : quad * 2 + (lane >> 4);
    float* mine = ring_o + (warp - S_::kTakeWarp0) * kChunk * kLdO;
    int written = 0;  // tiles by bulk copies
    constexpr int ng = 4 / G;
    Ring rd;
    bool ok = true;
    float2 acc[TC / 2];
    Unit un = unit(0);
    for (int n_unit = 0; n_unit < n_units; ++n_unit) {
      un = unit(n_unit);
      const int row0 = un.rt * NT + part * TC, rows = p.a.M - row0;  // of this warp
#pragma unroll
      for (int i = 0; i < TC / 2; ++i) acc[i] = make_float2(0.f, 0.f);
      // the column's scales, a block ahead, from the weight's pieces (in L2)
      const bool exists = un.second || piece < 4;
      const uint8_t* scales = (piece < 4 ? un.w0 : un.w1) + (piece & 3) * bb + kQgNibbles +
                              ((lane & 7) * 2 + ((lane >> 3) & 1)) * 2;
      constexpr int second = parts ? 0 : 16;  // (two sums of a group: its scale again)
      uint2 sn = make_uint2(0, 0);  // the scales of the block's ng sums
      auto fetch = [&]() {
        const unsigned short* q = reinterpret_cast<const unsigned short*>(scales);
        if (exists) {
          sn.x = __ldg(q);
          if (ng > 1) sn.x |= (uint32_t)__ldg(q + second) << 16;
          if (ng > 2) sn.y = __ldg(q + 32) | (uint32_t)__ldg(q + 48) << 16;
        }
        scales += run;
      };
      fetch();
      for (int kb = 0; kb < blocks && ok; ++kb) {
        uint2 sb = sn;
        if (kb + 1 < blocks) fetch();
#pragma unroll 1
        for (int g = 0; g < ng; ++g) {
          const float sc = u16_scale((unsigned short)(sb.x & 0xffffu), p.w.bf_scale);
          sb.x = g == 1 ? sb.y : sb.x >> 16;
          ok = ok && mbar_wait_warp(&full_d[rd.slot], rd.phase);
          if (!ok) break;
          tc_fence_after();
          const uint32_t ta = tmem + ((uint32_t)(quad * kWarp) << 16) + (uint32_t)(rd.slot * (int)kColsD + part * TC);
          const float2 s2 = make_float2(sc, sc);
#pragma unroll
          for (int i = 0; i < TC; i += kLoad) {
            uint32_t v[kLoad / 16][16];
#pragma unroll
            for (int q = 0; q < kLoad / 16; ++q) tmem_ld16(ta + i + q * 16, v[q]);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < kLoad / 2; ++e)
              fma2(acc[i / 2 + e],
                   make_float2(__uint_as_float(v[e / 8][2 * (e & 7)]), __uint_as_float(v[e / 8][2 * (e & 7) + 1])), s2);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty_d[rd.slot]);
          rd.next(S_::kD);
        }
      }
      if (!S_::kWalk || c.cs > 1) break;
      // ------------------------------------------------- a tile's results --
      // through this warp's chunk of shared memory
      ok = __all_sync(0xffffffffu, ok && !s_bad);
      if (!ok) break;  // no results after a wait that ran out
      if (n_unit == 0) pdl_wait();  // they may overwrite what the previous kernel still reads
      const int n0 = un.tile * (p.w2 ? 64 : 128) + quad * (p.w2 ? kWarp / 2 : kWarp);  // first column
      const bool fast = plain && n0 + kWarp <= p.w.N;
      if (by_bulk(un, n_unit)) {
        if (written > 0 && !mbar_wait_warp(&empty_t, (written - 1) & 1)) {
          ok = false;
          break;
        }
        const uint32_t at = tile_o + part * TC * 256 + (quad * kWarp + lane) * 2;
#pragma unroll
        for (int i = 0; i < TC; i += 2) {
          const float lo = 128.f * acc[i / 2].x, hi = 128.f * acc[i / 2].y;
          uint32_t v;
          if (p.a.type == kQgBf16)
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
          else
            asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
          sts16(at + i * 256, v);
          sts16(at + i * 256 + 256, v >> 16);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full_t);
        ++written;
        continue;
      }
#pragma unroll 1
      for (int i = 0; i < TC; i += kChunk) {
#pragma unroll
        for (int h = 0; h < TC; h += kChunk)  // (the sums stay in registers)
          if (h == i)
#pragma unroll
            for (int e = 0; e < kChunk; ++e)
              mine[e * kLdO + lane] = 128.f * (e & 1 ? acc[(h + e) / 2].y : acc[(h + e) / 2].x);
        __syncwarp();
        const int e0 = lane >> 2, k4 = 4 * (lane & 3), k8 = 8 * (lane & 3);
        if (p.w2) {
#pragma unroll 2
          for (int e = e0; e < kChunk; e += 8) {
            const float* at = mine + e * kLdO + k4;
            if (i + e < rows)
              finish4(p, row0 + i + e, n0 + k4, *reinterpret_cast<const float4*>(at),
                      *reinterpret_cast<const float4*>(at + 16));
          }
        } else if (fast) {
#pragma unroll
          for (int e = e0; e < kChunk; e += 8) {
            const float* at = mine + e * kLdO + k8;
            if (i + e < rows)
              store8(p, row0 + i + e, n0 + k8, *reinterpret_cast<const float4*>(at),
                     *reinterpret_cast<const float4*>(at + 4));
          }
        } else {
#pragma unroll 1
          for (int e = e0; e < kChunk && i + e < rows; e += 8)
#pragma unroll 1
            for (int k = k8; k < k8 + 8; k += 4) {
              const float4 v = *reinterpret_cast<const float4*>(mine + e * kLdO + k);
              finish4(p, row0 + i + e, n0 + k, v, v);
            }
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) fail();
    if (!mbar_wait_warp(&done, 0) && lane == 0) fail();  // no MMA is in flight
    tc_fence_before();
    __syncthreads();
    if (S_::kWalk && c.cs == 1) return;
    // -------------------------------- results of a CTA's, or cluster's, only tile --
    // by way of shared memory (every copy into it has landed: the MMAs and the
    // unpacking waited for them), rows of 128 columns, four to a thread
    int bad = s_bad;
    const int rows = min(NT, p.a.M - un.rt * NT);
    pdl_wait();  // results may overwrite what the previous kernel still reads
#pragma unroll
    for (int i = 0; i < TC; ++i)
      S[(part * TC + i) * kLd + quad * kWarp + lane] = 128.f * (i & 1 ? acc[i / 2].y : acc[i / 2].x);
    constexpr int kTakers = S_::kTakeWg * 4 * kWarp;
    if (c.cs > 1) {
      cluster_arrive();
      cluster_wait();
      const uint32_t bad0 = smem_u32(const_cast<int*>(&s_bad));
      for (int k = 0; k < c.cs; ++k) bad |= ld_dsmem_s32(dsmem_addr(bad0, (uint32_t)k));
    } else {
      bar_sync_n(1, kTakers);
    }
    if (!bad) {  // no results after a wait that ran out
      const int out_cols = p.w2 ? 64 : 128, sh = p.w2 ? 4 : 5;
      // the rows of this rank, m = rank, rank + cs, ..., four columns to a thread
      const int i0 = threadIdx.x - S_::kTakeWarp0 * kWarp, n0 = 4 * (i0 & ((1 << sh) - 1));
#pragma unroll 1
      for (int m = rank + (i0 >> sh) * c.cs; m < rows; m += (kTakers >> sh) * c.cs) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f), u = v;
        const float* at = S + m * kLd + (p.w2 ? n0 + (n0 & ~15) : n0);
        if (c.cs > 1) {
          for (int k = 0; k < c.cs; ++k) add4(v, ld_dsmem4(dsmem_addr(smem_u32(at), (uint32_t)k)));
          if (p.w2)
            for (int k = 0; k < c.cs; ++k) add4(u, ld_dsmem4(dsmem_addr(smem_u32(at + 16), (uint32_t)k)));
        } else {
          v = *reinterpret_cast<const float4*>(at);
          if (p.w2) u = *reinterpret_cast<const float4*>(at + 16);
        }
        finish4(p, un.rt * NT + m, un.tile * out_cols + n0, v, u);
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
  if (warp == 1) tmem_dealloc(tmem, S_::kCols);
  if (c.cs > 1) {
    cluster_arrive();
    cluster_wait();
    cluster_arrive();
    cluster_wait();
  }
}

struct TcPlan {
  int NT, tiles;
  long long ctas;
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
  // rows per tile: as few tiles as fit (192 rows of one limb, 128 of more),
  // all of about the same size
  const int most = o.c.limbs == 1 ? 192 : 128;
  const int row_tiles = (p.a.M + most - 1) / most, each = (p.a.M + row_tiles - 1) / row_tiles;
  const int sizes[4] = {32, 64, 128, 192};
  for (int i = 3; i >= 0; --i)
    if (each <= sizes[i]) o.NT = sizes[i];
  o.c.row_tiles = (p.a.M + o.NT - 1) / o.NT;
  o.tiles = p.w2 ? q4g_quads(p.w.N) : (q4g_quads(p.w.N) + 1) / 2;
  // operand stages: at least two; what is left goes to them, then to the weights
  const size_t limit = o.NT <= 64 ? kTqSmemHalf : kTqSmemMax;
  const size_t stage_w = 2 * (size_t)kQgQuad * p.w.block_bytes;
  const size_t stage_s = (size_t)(o.NT == 32 || o.NT == 192 ? 2 : 1) * o.c.limbs * o.NT * 128;
  o.c.nS = 2;
  o.c.nW = 2;
  const int max_s = o.NT == 32 ? Tile<32>::kMaxS : o.NT == 64 ? Tile<64>::kMaxS : o.NT == 128 ? Tile<128>::kMaxS
                                                                                 : Tile<192>::kMaxS;
  const size_t chunks = o.NT < 128 ? 0 : kChunkBytes + (o.c.limbs < 3 ? (size_t)o.NT * 256 : 0);
  size_t smem = o.c.nS * stage_s + o.c.nW * stage_w + chunks;
  const int ctas = o.NT <= 64 ? 2 : 1;  // per SM
  while (o.c.nS < max_s && smem + stage_s <= limit) {
    ++o.c.nS;
    smem += stage_s;
  }
  while (o.c.nW < kTqMaxW && smem + stage_w <= limit) {
    ++o.c.nW;
    smem += stage_w;
  }
  // All of it, so that no CTA of another kernel that needs more tensor memory
  // than is left can share the SM: two clusters whose CTAs waited there for each
  // other's tensor memory would not end.
  o.smem = smem <= limit ? limit : 0;
  static_assert((size_t)Tile<192>::kTakeWg * Tile<192>::TC * 132 * 4 <= kTqSmemMax &&
                    (size_t)Tile<64>::kTakeWg * Tile<64>::TC * 132 * 4 <= kTqSmemHalf,
                "a cluster's staged sums");
  o.c.tiles = o.tiles;
  o.c.units = o.tiles * o.c.row_tiles;
  // k shared by the CTAs of a cluster: the split with the least rounds x (blocks
  // of a CTA + what a CTA costs besides, about ten blocks).  A cluster's CTAs
  // share a GPC, so what fits at once is counted in clusters (16 rows, K 13824,
  // N 5120: 40 clusters of seven do not, 36 us; of six they do, 27 us).
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
  const long long slots = clusters_at_once(sm_count, ctas, 1);
  o.ctas = grid * o.c.cs;
  if (o.NT >= 128 && o.c.cs == 1 && o.ctas > slots) o.ctas = slots;
  return o;
}

template <int NT, int G, bool parts = false>
cudaError_t launch_tc_t(const Q4gParams& p, const TcPlan& o, cudaStream_t s) {
  if (!o.smem) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)o.ctas, 1, 1);
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
  return cudaLaunchKernelEx(&cfg, q4g_tc_kernel<NT, G, parts>, p, o.c);
}

template <int NT>
cudaError_t launch_tc_g(const Q4gParams& p, const TcPlan& o, cudaStream_t s) {
  switch (p.w.group) {
    case 32: return launch_tc_t<NT, 1>(p, o, s);
    case 64: return launch_tc_t<NT, 2>(p, o, s);
    default:
      // fp32: two sums of 64 k to a group, so that the low limbs of its second half
      // are not cut off against the first half's sum (the error of 20 rows, K 256:
      // 0.7e-7, with one sum 2.6e-7); never in tiles of 192 rows, which have one limb
      if constexpr (NT <= 128)
        if (o.c.limbs == 3) return launch_tc_t<NT, 2, true>(p, o, s);
      return launch_tc_t<NT, 4>(p, o, s);
  }
}

// Asked with a kernel that has no tensor memory: of one that has, the runtime
// counts one CTA to an SM, while two whose columns fit do run together.
void count_clusters() {
  if (cudaFuncSetAttribute(q4g_planes_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (int)kTqSmemMax) != cudaSuccess)
    cudaGetLastError();
  for (int ctas = 1; ctas <= 2; ++ctas)
    for (int cs = kTqMaxCluster; cs >= 1; --cs) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(cs * 1024);
      cfg.blockDim = dim3(128);
      cfg.dynamicSmemBytes = ctas == 2 ? kTqSmemHalf : kTqSmemMax;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = (unsigned)cs;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;  // unknown: an even spread
      if (cudaOccupancyMaxActiveClusters(&n, q4g_planes_kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
      }
      g_clusters[ctas][cs] = n;
    }
}

template <int NT, int G, bool parts = false>
cudaError_t prepare_tc_t() {
  return cudaFuncSetAttribute(q4g_tc_kernel<NT, G, parts>,
                              cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kTqSmemMax);
}
template <int NT>
cudaError_t prepare_tc_g() {
  cudaError_t e = prepare_tc_t<NT, 1>();
  if (e == cudaSuccess) e = prepare_tc_t<NT, 2>();
  if (e == cudaSuccess) e = prepare_tc_t<NT, 4>();
  if constexpr (NT <= 128)
    if (e == cudaSuccess) e = prepare_tc_t<NT, 2, true>();
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
  cfg.gridDim = dim3((p.w.nkb * 4 + 15) / 16, m8 < 65535 ? m8 : 65535, 1);
  cfg.blockDim = dim3(128);
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
      }
  return cudaErrorInvalidValue;
}

cudaError_t prepare_q4g_tc() {
  cudaError_t e = prepare_tc_g<32>();
  if (e == cudaSuccess) e = prepare_tc_g<64>();
  if (e == cudaSuccess) e = prepare_tc_g<128>();
  if (e == cudaSuccess) e = prepare_tc_g<192>();
  // once (every GPU of a node is alike), and a context of another thread waits for it
  static std::once_flag counted;
  if (e == cudaSuccess) std::call_once(counted, count_clusters);
  return e;
}

}  // namespace ms
