// ms_q4g.h -- 4-bit weights with a scale (and a zero point) per group of k:
// the device layout and the parameter block that their kernels share.
// Internal to libmojostream_cuda.so (the public C-ABI is include/mojostream_cuda.h).
//
// w[k][n] = (q - z) s with q a nibble, z (8 without zero points) and s of the
// group k / g, g in {32, 64, 128}.  The matrix is cut into tiles of 16 columns
// and blocks of 128 k, four neighbouring tiles (a quad, 64 columns) to a run:
//   [quad][block][4 tiles] x block_bytes
// A (tile, block) piece is everything a warp needs for its 16 x 128 weights:
//   2 x [32 lanes] uint4   nibbles of two 64-k halves, MMA fragment order
//   [128 / g][8] x 2 x 16-bit    scales of columns c and c + 8
//   [128 / g][8] x 2 x 8-bit     their zero points (only where there are any)
// Word s (0..3) of lane (r = lane / 4, t = lane % 4) of a 64-k half holds the
// nibbles of columns r and r + 8 at k = 32 (s / 2) + 8 t + 4 (s % 2) + {0..3}:
//   bits  0- 3 / 16-19 : column r    , k + 0 / k + 1
//   bits  4- 7 / 20-23 : column r + 8, k + 0 / k + 1
//   bits  8-11 / 24-27 : column r    , k + 2 / k + 3
//   bits 12-15 / 28-31 : column r + 8, k + 2 / k + 3
// so that masking a word with 0x0F0F0F0F gives four bytes q of column r and
// masking it with 0xF0F0F0F0 four bytes 16 q of column r + 8: half of the A
// operand (16 columns x 32 k) of an integer mma.m16n8k32 whose k are permuted
// so that a lane's share of an activation row is 8 values in a row.  Blocks
// past K and columns past N hold nibble 8, zero point 8 and scale 0.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ms {

constexpr int kQgTile = 16;     // columns per tile
constexpr int kQgQuad = 4;      // tiles per quad
constexpr int kQgBlockK = 128;  // k per block
constexpr int kQgNibbles = kQgTile * kQgBlockK / 2;  // 1024 bytes

struct Q4gView {
  const uint8_t* w;
  int K, N;
  int nkb;         // blocks of 128 k
  int group;       // k per scale: 32, 64 or 128
  int zeros;       // zero points stored
  int bf_scale;    // scales are bfloat16 (else IEEE half)
  int block_bytes;
};

__host__ __device__ inline int q4g_block_bytes(int group, int zeros) {
  return kQgNibbles + (kQgBlockK / group) * (zeros ? 48 : 32);
}
__host__ __device__ inline int q4g_quads(int N) { return (N + 63) / 64; }

// Element types of activations and results (MS_F32, MS_BF16, MS_F16).
enum QgType : int { kQgF32 = 0, kQgBf16 = 1, kQgF16 = 2 };

// Decode rows (streaming kernel): activations as signed 8-bit digits.  For a row
// and a group of k with 2^e <= max |a| < 2^(e + 1),
// q = rint(a 2^(29 - e)) = sum_l d_l 256^l, l = 0..3: a value within 2^6 (fp32),
// 2^19 (half) or 2^22 (bfloat16) of its group's largest is held exactly, any
// other to 2^-30 of the largest.  That is enough for results of 16 bits.  fp32
// rows have two more digits, rint(r 2^(44 - e)) of what q leaves of a value, so a
// value within 2^21 of the largest is exact and any other held to 2^-45 of it: a
// large channel whose weights are q = z adds nothing to a result, and must not
// take bits from the channels that do (one of 1e4 beside values around 1 cost
// 3e-6 of the result with four digits, where fp32 itself costs 3e-7).
//   A digit of a row is a column of the MMA: C = rows x digits <= 32, padded to a
// multiple of 8.  Record of a 128-k block:
//   2 x [C] x 64 bytes   the 64-k halves of each column, in fragment order
//   [128 / g][C8 / 2] float  factors of the pairs of digits: 2^(e - 29),
//                            2^(e - 13), fp32: 2^(e - 44)
//   [128 / g][C8] int        sums of the group's digits
constexpr int kQgCols = 32;
__host__ __device__ inline int qg_digits(int type) { return type == kQgF32 ? 6 : 4; }
// Rows of a block (a launch's grid y, a run of records): at most 8, of fp32 5,
// and there about the same in every block.
__host__ __device__ inline int qg_block_rows(int type, int M) {
  if (type != kQgF32) return M < 8 ? M : 8;
  const int blocks = (M + 4) / 5;
  return (M + blocks - 1) / blocks;
}
__host__ __device__ inline int qg_record_bytes(int cols, int group) {
  return cols * 128 + (kQgBlockK / group) * ((cols + 7) / 8 * 8) * 6;
}

struct Q4gRows {
  const void* a;
  long long lda;
  int type, M, K, nkb, group;
  int vec;           // rows start on 16-byte boundaries
  uint8_t* records;  // [row block][128-k block]; many rows: limb planes
};

struct Q4gParams {
  Q4gView w;         // the weight, or the gate
  const uint8_t* w2; // gated: the up weight (same shape and groups), else null
  Q4gRows a;         // records null: the CTAs convert the rows themselves
  void* out;
  long long ldo;
  int accumulate;
  int act;           // gated: 0 SiLU, 1 tanh-GELU
  int* err;
  // launch shape of the streaming kernel: ring stages, bytes of converted
  // rows, sets of a CTA (one more in the first set_rem CTAs)
  int stages, a_smem, set_q, set_rem;
};

cudaError_t launch_q4g_repack(uint8_t* out, const Q4gView& v, const uint8_t* src, const void* scales,
                              const uint8_t* zeros, int* bad, cudaStream_t s);
// Rows to records, in blocks of qg_block_rows.
cudaError_t launch_q4g_rows(const Q4gRows& r, cudaStream_t s);
size_t q4g_records_bytes(const Q4gRows& r);
// Fewer rows than q4g_tc_rows, qg_block_rows at a time.  q4g_stream_converts:
// the launch needs no records.
bool q4g_stream_converts(const Q4gParams& p, int sm_count);
cudaError_t launch_q4g_stream(const Q4gParams& p, int sm_count, cudaStream_t s);
cudaError_t prepare_q4g();
// Many rows on tcgen05 (ms_q4g_tc.cu): two launches; p.a.records is workspace
// of q4g_planes_bytes.
// From how many rows on: 9 bfloat16 rows (K 13824, N 5120: 27 us, two rounds of
// the streaming kernel 37 us; 8 rows 27 and 27 us), 17 half rows, of two limbs
// (K 2560, N 20480: 16 rows 29 and 27 us, 20 rows 29 and 35 us), 9 fp32 rows, of
// three limbs here and six digits there (K 5120, N 13824: 8 rows 32 and 31 us,
// 10 rows 32 and 38 us; K 10240, N 2560: 8 rows 18 and 21 us, 5 rows 18 and 14).
inline int q4g_tc_rows(int type) { return type == kQgF16 ? 17 : 9; }
size_t q4g_planes_bytes(const Q4gParams& p, int sm_count);
cudaError_t launch_q4g_tc(const Q4gParams& p, int sm_count, cudaStream_t s);
cudaError_t prepare_q4g_tc();

}  // namespace ms
