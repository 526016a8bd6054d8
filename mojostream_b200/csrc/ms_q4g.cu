// ms_q4g.cu -- products with group-scaled 4-bit weights (layout: ms_q4g.h):
//   C[m][n] (+)= sum_k A[m][k] (q[k][n] - z) s,   H = act(A Wg) * (A Wu).
//
// Decode rows run on integer tensor cores: activations as signed 8-bit digits
// relative to their group's largest value (ms_q4g.h), so that
//   sum_k (q - z) a = sum_l f_l (sum_k q d_l - z sum_k d_l)
// with exact integer sums per group (|sum| < 2^23, exact in fp32 too); group
// scales, digit factors and groups are applied and added in fp32.  Unpacking
// costs two ANDs for eight weights; the same product with weights expanded to
// bfloat16 took seven shifts and logic operations and four subtractions for
// them, and that, not memory, was its bound (K 2560, N 262144, one row:
// 109 us against 53 us of bytes).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ms_common.cuh"
#include "ms_kernels.h"
#include "ms_q4g.cuh"
#include "ms_q4g.h"

namespace ms {
namespace {

// D = A (16 x 32, unsigned bytes) * B (32 x 8, signed bytes) + C, exact in s32.
__device__ __forceinline__ void mma_u8s8_16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                               uint32_t a3, uint32_t b0, uint32_t b1,
                                               const int (&c)[4]) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]),
        "r"(c[3]));
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

// ----------------------------------------------------- rows to records --
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Byte l of four digit words, k order {0, 2, 1, 3}, for l = 0..3.
__device__ __forceinline__ void transpose4(const uint32_t* d, uint32_t (&w)[4]) {
  const uint32_t lo0 = __byte_perm(d[0], d[2], 0x5140), lo1 = __byte_perm(d[1], d[3], 0x5140);
  const uint32_t hi0 = __byte_perm(d[0], d[2], 0x7362), hi1 = __byte_perm(d[1], d[3], 0x7362);
  w[0] = __byte_perm(lo0, lo1, 0x5410);
  w[1] = __byte_perm(lo0, lo1, 0x7632);
  w[2] = __byte_perm(hi0, hi1, 0x5410);
  w[3] = __byte_perm(hi0, hi1, 0x7632);
}

// Sixteen lanes: 128 k of a row, 8 consecutive ones (v) per lane hl, into
// columns c0 .. c0 + D - 1 of a record with `cols` columns.  Whole warp (two
// rows or blocks at a time); nothing is written where live is false.
//   A group with a NaN gets the factor NaN; one with infinities holds +-1 at
// them, 0 elsewhere and the factor infinity, so that infinity * w comes out
// as it should (NaN for w = 0).  Of several infinities only the sum of their
// weights is seen so: undefined_sum corrects the results that it gets wrong.
template <int D>
__device__ __forceinline__ void convert8(float (&v)[8], int group, int c0, int cols, int hl,
                                         bool live, uint8_t* rec) {
  const int glanes = group / 8, ng = kQgBlockK / group;
  const int c8 = (cols + 7) / 8 * 8;
  uint32_t mx = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) mx = max(mx, __float_as_uint(v[j]) & 0x7fffffffu);
  for (int o = 1; o < glanes; o <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  // exponent of the largest value; groups below 2^-90 share its scale
  constexpr int top = 29;
  const int e = max((int)(mx >> 23) - 127, -90);
  const bool finite = mx < 0x7f800000u;
  constexpr int P = D > 4 ? 2 : 1;
  uint32_t w[P][2][4];  // digit words of the lane's 8 k
  int sum[D / 2];       // digit sums of the lane's, then the group's k
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int x = min(top - e + 15 * p, 126);
    const float up = finite ? pow2(x) : 0.f, down = pow2(-x);
    uint32_t d[8];  // the digits of q: q + 0x80808080 with every byte's top bit flipped
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      int q = __float2int_rn(v[j] * up);
      if (!finite) q = p == 0 && isinf(v[j]) ? (v[j] > 0.f ? 1 : -1) : 0;
      d[j] = ((uint32_t)q + 0x80808080u) ^ 0x80808080u;
      // what is left, exactly: q has no more bits than v where it is not 0
      if (p + 1 < P) v[j] = fmaf(-(float)q, down, v[j]);
    }
    transpose4(d, w[p][0]);
    transpose4(d + 4, w[p][1]);
    // two digits of the first four, l and l + 2, to a word (|sum| <= 2^14); so
    // the last two
    int s[4];
#pragma unroll
    for (int l = 0; l < 4; ++l)
      s[l] = __dp4a((int)w[p][1][l], 0x01010101, __dp4a((int)w[p][0][l], 0x01010101, 0));
    if (p == 0) {
      sum[0] = s[0] + s[2] * 65536;
      sum[1] = s[1] + s[3] * 65536;
    } else {
      sum[D / 2 - 1] = s[0] + s[1] * 65536;
    }
  }
  for (int o = 1; o < glanes; o <<= 1)
#pragma unroll
    for (int i = 0; i < D / 2; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
  if (!live) return;
  // 4 lanes per 32-k step, two steps to a half
  uint8_t* dst = rec + ((hl >> 3) * cols + c0) * 64 + (hl & 3) * 16 + ((hl >> 2) & 1) * 8;
#pragma unroll
  for (int l = 0; l < D; ++l)
    *reinterpret_cast<uint2*>(dst + l * 64) = make_uint2(w[l / 4][0][l & 3], w[l / 4][1][l & 3]);
  if (hl % glanes == 0) {
    const int at = hl / glanes * c8 + c0;
    float* f = reinterpret_cast<float*>(rec + (size_t)cols * 128);
    int2* n = reinterpret_cast<int2*>(reinterpret_cast<int*>(f + ng * c8 / 2) + at);
    const float f0 = finite ? pow2(e - top)
                            : mx > 0x7f800000u ? __uint_as_float(0x7fc00000u) : INFINITY;
    // (an infinity sits in the first digit alone)
    f[at / 2] = f0;
    f[at / 2 + 1] = finite ? f0 * 65536.f : 0.f;
    const int lo02 = (int)(short)sum[0], lo13 = (int)(short)sum[1];
    n[0] = make_int2(lo02, lo13);
    n[1] = make_int2((sum[0] - lo02) >> 16, (sum[1] - lo13) >> 16);
    if (P == 2) {
      f[at / 2 + 2] = finite ? pow2(-min(top - e + 15, 126)) : 0.f;
      const int lo = (int)(short)sum[D / 2 - 1];
      n[2] = make_int2(lo, (sum[D / 2 - 1] - lo) >> 16);
    }
  }
}

// Half a warp per (row, block); grid x over blocks, y over rows.
__global__ void __launch_bounds__(256) q4g_rows_kernel(const Q4gRows a) {
  pdl_wait();     // the rows are an earlier kernel's output, and the records
  pdl_trigger();  // may still be read by the product before this one
  const int kb = blockIdx.x * 16 + (threadIdx.x >> 4), hl = threadIdx.x & 15;
  const int digits = qg_digits(a.type), per = qg_block_rows(a.type, a.M);
  for (int m = blockIdx.y; m < a.M; m += gridDim.y) {
    const int rb = m / per, cols = min(per, a.M - rb * per) * digits;
    float v[8];
    load8(a, m, kb * kQgBlockK + 8 * hl, v);
    uint8_t* rec = a.records + rb * (size_t)a.nkb * qg_record_bytes(per * digits, a.group) +
                   (size_t)kb * qg_record_bytes(cols, a.group);
    if (digits == 6)
      convert8<6>(v, a.group, m % per * 6, cols, hl, kb < a.nkb, rec);
    else
      convert8<4>(v, a.group, m % per * 4, cols, hl, kb < a.nkb, rec);
  }
}

// Whether the sum of row m and column n is NaN by its infinities: one of them
// meets a weight of 0, or two products are infinities of opposite sign.
__device__ __forceinline__ bool undefined_sum(const Q4gParams& p, const uint8_t* w, int m, int n) {
  const int tile = n / kQgTile, c = n % kQgTile, bb = p.w.block_bytes;
  const uint8_t* piece = w + ((size_t)(tile / kQgQuad) * p.w.nkb * kQgQuad + tile % kQgQuad) * bb;
  bool pos = false, neg = false;
#pragma unroll 1
  for (int k = 0; k < p.w.K; ++k) {
    const float x = load_out(p.a.a, (size_t)m * p.a.lda + k, p.a.type);
    if (!isinf(x)) continue;
    const uint8_t* b = piece + (size_t)(k / kQgBlockK) * kQgQuad * bb;
    const int kk = k % 64, g = k % kQgBlockK / p.w.group;
    const int word = (k % kQgBlockK / 64 * 32 + (c & 7) * 4 + kk % 32 / 8) * 4 + kk / 32 * 2 + kk % 8 / 4;
    const int bit = (kk & 2) * 4 + (kk & 1) * 16 + (c >> 3) * 4, at = (g * 8 + (c & 7)) * 2 + (c >> 3);
    const int q = (reinterpret_cast<const uint32_t*>(b)[word] >> bit) & 15u;
    const int z = p.w.zeros ? b[kQgNibbles + kQgBlockK / p.w.group * 32 + at] : 8;
    const float y = (float)(q - z) *
                    u16_scale(reinterpret_cast<const uint16_t*>(b + kQgNibbles)[at], p.w.bf_scale);
    if (!(y > 0.f || y < 0.f)) return true;
    pos |= (x > 0.f) == (y > 0.f);
    neg |= (x > 0.f) != (y > 0.f);
  }
  return pos && neg;
}

// ----------------------------------------------------- streaming kernel --
// Decode rows.  The work is a line of pieces, set by set (a set is T tiles, T x
// 16 columns, of a weight, or T / 2 of the gate and T / 2 of the up weight)
// and inside a set by 128-k block.  The CTAs share the sets evenly, and the 16
// warps of a CTA the pieces of its sets.  A warp streams its pieces through a private ring of
// bulk copies, one mbarrier per stage and no CTA barrier inside the loop.  A
// set that lies in one warp's share is finished by that warp; the sums of
// others meet in shared memory and are added in k order (the same bits on
// every run).  A CTA has whole sets: a split of the line in the middle of sets,
// with the last CTA to arrive adding the parts, was balanced to a piece and
// took 4 us more at every size.
//   The first stages are issued before the previous kernel has finished
// (nothing writes the weights); activations and results wait for it.  For few
// rows the CTA converts the rows into shared memory itself; else their
// records come with each stage of the ring.
constexpr int kQgWarps = 16;
constexpr int kQgMaxStages = 8;
constexpr size_t kQgSmemMax = 208 * 1024;

// n elements in W consecutive parts that differ by one element at most, the
// longer ones first.
struct Split {
  int q, rem;
  __device__ __forceinline__ Split(int n, int W) : q(n / W), rem(n % W) {}
  __device__ __forceinline__ int begin(int w) const { return w * q + min(w, rem); }
  // the part that holds element i
  __device__ __forceinline__ int of(int i) const {
    const int head = rem * (q + 1);
    return i < head ? (int)((unsigned)i / (unsigned)(q + 1))
                    : rem + (int)((unsigned)(i - head) / (unsigned)max(q, 1));
  }
};

// NB: 8-column blocks of digits (two rows of four digits each, or 4/3 rows of
// six); G: 32-k steps per group (1, 2, 4); wide: fp32 rows.
template <int T, int NB, int G, bool wide>
__global__ void __launch_bounds__(kQgWarps* kWarp, T* NB <= 2 ? 2 : 1)
    q4g_stream_kernel(const Q4gParams p) {
  extern __shared__ __align__(128) uint8_t dsm[];
  __shared__ __align__(8) uint64_t s_full[kQgWarps * kQgMaxStages];
  __shared__ int s_bad;
  constexpr int kCols = T * kQgTile;  // columns of a set (gate and up)

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, t = lane & 3;
  const int per = p.w2 ? T / 2 : T;  // tiles of each weight in a set
  const int cols = per * kQgTile;    // result columns of a set
  const int nkb = p.w.nkb, bb = p.w.block_bytes;
  constexpr int ng = 4 / G;
  constexpr int digits = wide ? 6 : 4;
  constexpr int kRows = wide ? NB * 8 / 6 : NB;  // loops over rows of six digits, or blocks
  const int row_block = qg_block_rows(p.a.type, p.a.M);
  const int row0 = blockIdx.y * row_block, rows = min(row_block, p.a.M - row0);
  const int C = rows * digits, rc8 = (C + 7) / 8 * 8;
  const int rec = C * 128 + ng * rc8 * 6;
  const bool own_a = p.a.records == nullptr;
  const int stage_bytes = T * bb + (own_a ? 0 : rec);
  // pieces of the CTA, and of this warp
  const int set0 = blockIdx.x * p.set_q + min((int)blockIdx.x, p.set_rem);
  const int sets = p.set_q + ((int)blockIdx.x < p.set_rem);
  const Split own(sets * nkb, kQgWarps);
  const int p0 = own.begin(warp), n = own.begin(warp + 1) - p0;
  float* slots = reinterpret_cast<float*>(dsm + p.a_smem);  // [warps][2][rows][kCols]
  uint8_t* ring = dsm + p.a_smem + kQgWarps * 2 * rows * kCols * sizeof(float) +
                  (size_t)warp * p.stages * stage_bytes;
  uint64_t* full = s_full + warp * kQgMaxStages;

  if (threadIdx.x == 0) s_bad = 0;
  if (lane == 0) {
    for (int s = 0; s < p.stages; ++s) mbar_init(&full[s], 1);
    mbar_fence_init();
  }
  __syncwarp();
  pdl_trigger();

  // the next piece to copy
  const int first_set = p0 / nkb;
  int i_set = set0 + first_set, i_kb = p0 - first_set * nkb;
  const int i_set0 = i_set, i_kb0 = i_kb;
  size_t i_off = 0;
  auto seek = [&]() {
    const int tile = i_set * per;
    i_off = (((size_t)(tile / kQgQuad) * nkb + i_kb) * kQgQuad + tile % kQgQuad) * bb;
  };
  seek();
  const uint8_t* a_src =
      own_a ? nullptr
            : p.a.records + (size_t)blockIdx.y * nkb * qg_record_bytes(row_block * digits, p.w.group);
  auto issue_w = [&](int slot) {
    uint8_t* st = ring + slot * stage_bytes;
    mbar_expect_tx(&full[slot], stage_bytes);
    bulk_g2s(st, p.w.w + i_off, per * bb, &full[slot]);
    if (p.w2) bulk_g2s(st + per * bb, p.w2 + i_off, per * bb, &full[slot]);
  };
  auto issue_a = [&](int slot, int kb) {
    bulk_g2s(ring + slot * stage_bytes + T * bb, a_src + (size_t)kb * rec, rec, &full[slot]);
  };
  auto advance = [&]() {
    i_off += kQgQuad * bb;
    if (++i_kb == nkb) {
      i_kb = 0;
      ++i_set;
      seek();
    }
  };
  const int first = min(n, p.stages);
  if (lane == 0)
    for (int i = 0; i < first; ++i) {
      issue_w(i);
      advance();
    }
  pdl_wait();
  int set = i_set0, kb = i_kb0;
  if (own_a) {
    // two (row, block) items per warp and round, the next round's loads first
    const int items = rows * nkb, hl = lane & 15;
    int it = warp * 2 + (lane >> 4);
    float v[8], nx[8];
    load8(p.a, row0 + it / nkb, it < items ? it % nkb * kQgBlockK + 8 * hl : p.a.K, v);
    for (; __any_sync(0xffffffffu, it < items); it += 2 * kQgWarps) {
      const int nt = it + 2 * kQgWarps;
      load8(p.a, row0 + nt / nkb, nt < items ? nt % nkb * kQgBlockK + 8 * hl : p.a.K, nx);
      convert8<digits>(v, p.w.group, it / nkb * digits, C, hl, it < items, dsm + (size_t)(it % nkb) * rec);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = nx[j];
    }
    __syncthreads();
  } else if (lane == 0) {
    for (int i = 0; i < first; ++i) issue_a(i, (kb + i) % nkb);
  }

  float acc[T][NB][2];  // columns r and r + 8 of a tile
#pragma unroll
  for (int i = 0; i < T; ++i)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[i][b][0] = acc[i][b][1] = 0.f;
  // The sums of tile j: of row i of six digits, in pairs 3 i .. 3 i + 2 (lane t
  // of column block b has pair 4 b + t), or of row 2 i (lanes t = 0, 1) or
  // 2 i + 1 (t = 2, 3).  `mine`: this lane has a row of its own, m.
  auto row_sums = [&](int j, int i, float& lo, float& hi) {
    if constexpr (wide) {
      lo = hi = 0.f;
#pragma unroll
      for (int q = 3 * i; q < 3 * i + 3; ++q) {
        lo += __shfl_sync(0xffffffffu, acc[j][q >> 2][0], (lane & 28) | (q & 3));
        hi += __shfl_sync(0xffffffffu, acc[j][q >> 2][1], (lane & 28) | (q & 3));
      }
    } else {
      lo = acc[j][i][0] + __shfl_xor_sync(0xffffffffu, acc[j][i][0], 1);
      hi = acc[j][i][1] + __shfl_xor_sync(0xffffffffu, acc[j][i][1], 1);
    }
  };
  auto row_of = [&](int i) { return wide ? i : 2 * i + (t >> 1); };
  auto mine = [&](int i) { return wide ? t == (i & 3) && i < rows : !(t & 1) && 2 * i + (t >> 1) < rows; };

  const uint32_t dsm_s = smem_u32(dsm), ring_s = smem_u32(ring);
  bool ok = true;
  bool odd = false;  // an infinity or a NaN among the sums
  int slot = 0;
  uint32_t phase = 0;
  int begun = kb;  // block of the set that this warp's sum starts at
  for (int i = 0; i < n; ++i) {
    if (!mbar_wait_warp(&full[slot], phase)) {
      if (lane == 0) atomicOr(p.err, kErrWaitTimeout);
      // let the other copies land before the CTA can exit
      for (int j = i + 1; j < min(n, i + p.stages); ++j)
        mbar_wait_warp(&full[j % p.stages], (j / p.stages) & 1);
      ok = false;
      break;
    }
    const uint32_t st = ring_s + slot * stage_bytes;
    const uint32_t sa = own_a ? dsm_s + kb * rec : st + T * bb;
    const uint32_t fac = sa + C * 128 + 4 * t, sums = sa + C * 128 + ng * rc8 * 2 + 8 * t;
    const uint32_t wl = st + lane * 16;
    const uint32_t sc = st + kQgNibbles + r * 4;
    int c[T][NB][4];
    int ci[NB][4];  // -z times the group's digit sums (column r + 8 counts 16-fold)
    uint2 sd[NB];
    float f[NB];
#pragma unroll
    for (int q = 0; q < 2; ++q) {  // 64-k halves
      uint4 bv[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        bv[b] = make_uint4(0u, 0u, 0u, 0u);
        if (b * 8 + r < C) bv[b] = lds128(sa + r * 64 + t * 16 + (q * C + b * 8) * 64);
      }
      uint4 wv[T];
#pragma unroll
      for (int j = 0; j < T; ++j) wv[j] = lds128(wl + j * bb + q * 512);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {  // 32-k steps
        const int h = 2 * q + hh, grp = h / G;
        if (h % G == 0) {  // a group begins
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            f[b] = 0.f;
            sd[b] = make_uint2(0u, 0u);
            if (b * 8 < C) {
              f[b] = __uint_as_float(lds32(fac + (grp * rc8 / 2 + b * 4) * 4));
              sd[b] = lds64(sums + (grp * rc8 + b * 8) * 4);
            }
            ci[b][0] = -8 * (int)sd[b].x;
            ci[b][1] = -8 * (int)sd[b].y;
            ci[b][2] = -128 * (int)sd[b].x;
            ci[b][3] = -128 * (int)sd[b].y;
          }
        }
#pragma unroll
        for (int j = 0; j < T; ++j) {
          if (h % G == 0 && p.w.zeros) {
            const uint32_t z = lds16(st + j * bb + kQgNibbles + ng * 32 + (grp * 8 + r) * 2);
            const int zl = -(int)(z & 0xffu), zh = -16 * (int)(z >> 8);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              ci[b][0] = zl * (int)sd[b].x;
              ci[b][1] = zl * (int)sd[b].y;
              ci[b][2] = zh * (int)sd[b].x;
              ci[b][3] = zh * (int)sd[b].y;
            }
          }
          const uint32_t x0 = hh == 0 ? wv[j].x : wv[j].z, x1 = hh == 0 ? wv[j].y : wv[j].w;
          const uint32_t a0 = x0 & 0x0F0F0F0Fu, a1 = x0 & 0xF0F0F0F0u;
          const uint32_t a2 = x1 & 0x0F0F0F0Fu, a3 = x1 & 0xF0F0F0F0u;
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const uint32_t b0 = hh == 0 ? bv[b].x : bv[b].z, b1 = hh == 0 ? bv[b].y : bv[b].w;
            if (h % G == 0)
              mma_u8s8_16832(c[j][b], a0, a1, a2, a3, b0, b1, ci[b]);
            else
              mma_u8s8_16832(c[j][b], a0, a1, a2, a3, b0, b1, c[j][b]);
          }
        }
        if (h % G == G - 1) {  // it ends: two digits in one integer (|sum| < 2^30)
#pragma unroll
          for (int j = 0; j < T; ++j) {
            const uint32_t s2 = lds32(sc + j * bb + grp * 32);
            const float lo = u16_scale(s2 & 0xffffu, p.w.bf_scale);
            const float hi = 0.0625f * u16_scale(s2 >> 16, p.w.bf_scale);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              acc[j][b][0] = fmaf(lo * f[b], (float)(c[j][b][0] + 256 * c[j][b][1]), acc[j][b][0]);
              acc[j][b][1] = fmaf(hi * f[b], (float)(c[j][b][2] + 256 * c[j][b][3]), acc[j][b][1]);
            }
          }
        }
      }
    }
    // Every lane's loads from the stage have arrived before it is refilled: every
    // tile's and every column block's are in this sum, and a sum is never this
    // NaN (neither a barrier nor a later load's arrival says that an earlier
    // load in flight has arrived)
    float all = acc[T - 1][NB - 1][1];
#pragma unroll
    for (int j = 0; j < T - 1; ++j) all += acc[j][NB - 1][1];
#pragma unroll
    for (int b = 0; b < NB - 1; ++b) all += acc[T - 1][b][1];
    const unsigned read = __ballot_sync(0xffffffffu, __float_as_uint(all) != 0x7fedcba9u);
    if (lane == 0 && read && i + p.stages < n) {
      issue_w(slot);
      if (!own_a) issue_a(slot, i_kb);
      advance();
    }
    if (++slot == p.stages) {
      slot = 0;
      phase ^= 1;
    }
    if (++kb == nkb || i + 1 == n) {  // the warp's share of this set is complete
      if (begun == 0 && kb == nkb) {  // all of it
#pragma unroll
        for (int j = 0; j < T; ++j)
#pragma unroll
          for (int i2 = 0; i2 < kRows; ++i2) {
            float lo, hi, ulo = 0.f, uhi = 0.f;
            if (p.w2 && j >= T / 2) break;
            row_sums(j, i2, lo, hi);
            if (p.w2) row_sums((j + T / 2) % T, i2, ulo, uhi);
            if (mine(i2)) {
              const int m = row0 + row_of(i2);
              odd |= !isfinite(lo + hi) || (p.w2 && !isfinite(ulo + uhi));
              finish(p, m, set * cols + j * kQgTile + r, lo, ulo);
              finish(p, m, set * cols + j * kQgTile + r + 8, hi, uhi);
            }
          }
      } else {
        float* d = slots + (size_t)(warp * 2 + (set != i_set0)) * rows * kCols;
#pragma unroll
        for (int j = 0; j < T; ++j)
#pragma unroll
          for (int i2 = 0; i2 < kRows; ++i2) {
            float lo, hi;
            row_sums(j, i2, lo, hi);
            if (mine(i2)) {
              float* at = d + row_of(i2) * kCols + j * kQgTile + r;
              at[0] = lo;
              at[8] = hi;
            }
          }
      }
#pragma unroll
      for (int j = 0; j < T; ++j)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[j][b][0] = acc[j][b][1] = 0.f;
      if (kb == nkb) {
        kb = 0;
        ++set;
      }
      begun = kb;
    }
  }
  if (!ok) s_bad = 1;
  __syncthreads();
  if (s_bad) return;  // nothing more is written after a wait that ran out

  // sets that no single warp covers: sums over the warps in k order
  const int cl = 31 - __clz(cols);
  for (int i = threadIdx.x; i < sets * rows << cl; i += blockDim.x) {
    const int col = i & (cols - 1), sm = i >> cl, s = rows == 1 ? sm : sm / rows, m = sm - s * rows;
    const int q0 = s * nkb, wa = own.of(q0), wb = own.of(q0 + nkb - 1);
    if (wa == wb) continue;
    // a warp's first set sits in its first slot, its last one in the second
    float v = 0.f, u = 0.f;
#pragma unroll 4
    for (int w = wa; w <= wb; ++w) {
      const float* d = slots + ((w * 2 + (own.begin(w) < q0)) * rows + m) * kCols + col;
      v += d[0];
      if (p.w2) u += d[cols];
    }
    odd |= !isfinite(v) || !isfinite(u);
    finish(p, row0 + m, (set0 + s) * cols + col, v, u);
  }
  // (rare: infinities that may have to be NaN)
  if (!__syncthreads_or(odd)) return;
#pragma unroll 1
  for (int i = threadIdx.x; i < sets * rows << cl; i += blockDim.x) {
    const int col = i & (cols - 1), sm = i >> cl, s = sm / rows, m = row0 + sm - s * rows;
    const int n = (set0 + s) * cols + col;
    const size_t at = (size_t)m * p.ldo + n;
    if (n >= p.w.N || !isinf(load_out(p.out, at, p.a.type))) continue;
    bool nan = false;
#pragma unroll 1
    for (int u = 0; u < (p.w2 ? 2 : 1) && !nan; ++u) nan = undefined_sum(p, u ? p.w2 : p.w.w, m, n);
    if (nan) store_out(p.out, at, p.a.type, __uint_as_float(0x7fc00000u));
  }
}

struct StreamPlan {
  int T, NB, ctas, stages, sets;
  size_t a_smem, smem;
};

StreamPlan plan_stream(const Q4gParams& p, int sm_count) {
  StreamPlan o{};
  const int digits = qg_digits(p.a.type), per = qg_block_rows(p.a.type, p.a.M);  // rows of a block
  const int row_blocks = (p.a.M + per - 1) / per;
  o.NB = (per * digits + 7) / 8;
  // four tiles to a set share a block's loads and loop (one row, K 2560, N
  // 20480 bfloat16: 7.0 us, with two 8.8 us) where the GPU still gets a set per
  // SM; fewer columns fill it better with two (three rows, N 2560: 6.5 us, with
  // four 7.1 us).
  // From five rows (three of fp32) on four tiles' sums do not fit the registers.
  const int quads = q4g_quads(p.w.N) * (p.w2 ? 2 : 1);
  o.T = o.NB <= 2 && quads >= sm_count ? 4 : 2;
  o.sets = quads * kQgQuad / o.T;
  // rows x blocks that 16 warps convert in two rounds (one or two rows: three,
  // more fp32 rows: one); more come converted, a launch more (one row, K 2560, N
  // 20480 bfloat16: 7.0 us, and 7.8 us; four rows, N 2560: 7.5 and 5.5 us; fp32,
  // four rows, K 1280, N 2560: 6.0 and 5.5 us)
  const size_t rec = (size_t)qg_record_bytes(per * digits, p.w.group);
  const size_t a_all = p.w.nkb * rec;
  o.a_smem = row_blocks == 1 && per * p.w.nkb <= (per <= 2 ? 6 : digits == 6 ? 2 : 4) * kQgWarps && a_all <= 64 * 1024 ? a_all : 0;
  const size_t stage = (size_t)o.T * p.w.block_bytes + (o.a_smem ? 0 : rec);
  const size_t fixed = o.a_smem + (size_t)kQgWarps * 2 * per * o.T * kQgTile * sizeof(float);
  // small sets run two CTAs to an SM (64 registers)
  const bool two = o.T * o.NB <= 2 && fixed + 2 * stage * kQgWarps <= kQgSmemMax / 2;
  o.ctas = sm_count * (two ? 2 : 1);
  if (o.sets < o.ctas) o.ctas = o.sets;
  int st = (int)(((two ? kQgSmemMax / 2 : kQgSmemMax) - fixed) / (stage * kQgWarps));
  const long long longest =
      ((long long)(o.sets + o.ctas - 1) / o.ctas * p.w.nkb + kQgWarps - 1) / kQgWarps;
  st = st > kQgMaxStages ? kQgMaxStages : st;
  st = st > longest ? (int)longest : st;
  o.stages = st;
  o.smem = fixed + (size_t)st * stage * kQgWarps;
  return o;
}

template <int T, int NB, int G, bool wide>
cudaError_t launch_stream_t(const Q4gParams& p0, const StreamPlan& o, cudaStream_t s) {
  Q4gParams p = p0;
  p.stages = o.stages;
  p.a_smem = (int)o.a_smem;
  p.set_q = o.sets / o.ctas;
  p.set_rem = o.sets % o.ctas;
  if (o.stages < 1 || o.smem > kQgSmemMax || !p.a.records != (o.a_smem > 0))
    return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  const int per = qg_block_rows(p.a.type, p.a.M);
  cfg.gridDim = dim3(o.ctas, (p.a.M + per - 1) / per, 1);
  cfg.blockDim = dim3(kQgWarps * kWarp);
  cfg.dynamicSmemBytes = o.smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, q4g_stream_kernel<T, NB, G, wide>, p);
}

template <int T, int NB, bool wide>
cudaError_t launch_stream_g(const Q4gParams& p, const StreamPlan& o, cudaStream_t s) {
  switch (p.w.group) {
    case 32: return launch_stream_t<T, NB, 1, wide>(p, o, s);
    case 64: return launch_stream_t<T, NB, 2, wide>(p, o, s);
    default: return launch_stream_t<T, NB, 4, wide>(p, o, s);
  }
}

template <bool wide>
cudaError_t launch_stream_w(const Q4gParams& p, const StreamPlan& o, cudaStream_t s) {
  switch (o.T * 8 + o.NB) {  // the plan's own shape, or nothing
    case 2 * 8 + 1: return launch_stream_g<2, 1, wide>(p, o, s);
    case 4 * 8 + 1: return launch_stream_g<4, 1, wide>(p, o, s);
    case 4 * 8 + 2: return launch_stream_g<4, 2, wide>(p, o, s);
    case 2 * 8 + 2: return launch_stream_g<2, 2, wide>(p, o, s);
    case 2 * 8 + 3: return launch_stream_g<2, 3, wide>(p, o, s);
    case 2 * 8 + 4: return launch_stream_g<2, 4, wide>(p, o, s);
  }
  return cudaErrorInvalidValue;
}

template <int T, int NB, int G>
cudaError_t prepare_t() {
  const cudaError_t e = cudaFuncSetAttribute(
      q4g_stream_kernel<T, NB, G, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kQgSmemMax);
  if (e != cudaSuccess) return e;
  return cudaFuncSetAttribute(q4g_stream_kernel<T, NB, G, true>,
                              cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kQgSmemMax);
}
template <int T, int NB>
cudaError_t prepare_g() {
  cudaError_t e = prepare_t<T, NB, 1>();
  if (e == cudaSuccess) e = prepare_t<T, NB, 2>();
  if (e == cudaSuccess) e = prepare_t<T, NB, 4>();
  return e;
}

}  // namespace

cudaError_t launch_q4g_repack(uint8_t* out, const Q4gView& v, const uint8_t* src, const void* scales,
                              const uint8_t* zeros, int* bad, cudaStream_t s) {
  const size_t n = (size_t)q4g_quads(v.N) * v.nkb * kQgQuad * (256 + kQgBlockK / v.group * kQgTile);
  const size_t blocks = (n + 255) / 256;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(blocks < 148 * 64 ? blocks : 148 * 64));
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  return cudaLaunchKernelEx(&cfg, q4g_repack_kernel, out, v, src,
                            reinterpret_cast<const uint16_t*>(scales), zeros, bad);
}

size_t q4g_records_bytes(const Q4gRows& r) {
  const int per = qg_block_rows(r.type, r.M);
  return (size_t)((r.M + per - 1) / per) * r.nkb *
         qg_record_bytes(per * qg_digits(r.type), r.group);
}

cudaError_t launch_q4g_rows(const Q4gRows& r, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((r.nkb + 15) / 16, r.M < 65535 ? r.M : 65535, 1);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, q4g_rows_kernel, r);
}

bool q4g_stream_converts(const Q4gParams& p, int sm_count) {
  return plan_stream(p, sm_count).a_smem > 0;
}

cudaError_t launch_q4g_stream(const Q4gParams& p, int sm_count, cudaStream_t s) {
  const StreamPlan o = plan_stream(p, sm_count);
  return p.a.type == kQgF32 ? launch_stream_w<true>(p, o, s) : launch_stream_w<false>(p, o, s);
}

cudaError_t prepare_q4g() {
  cudaError_t e = prepare_g<2, 1>();
  if (e == cudaSuccess) e = prepare_g<4, 1>();
  if (e == cudaSuccess) e = prepare_g<4, 2>();
  if (e == cudaSuccess) e = prepare_g<2, 2>();
  if (e == cudaSuccess) e = prepare_g<2, 3>();
  if (e == cudaSuccess) e = prepare_g<2, 4>();
  return e;
}

}  // namespace ms
