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

// Decode rows (streaming kernel): activations as four signed 8-bit digits.
// For a row and a group of k with 2^e <= max |a| < 2^(e + 1),
// q = rint(a 2^(29 - e)) = sum_l d_l 256^l: a value within 2^6 (fp32) or 2^21
// (bfloat16) of its group's largest is held exactly, any other to 2^-30 of the
// largest.  A digit of a row is a column of the MMA: C = 4 rows, padded to a
// multiple of 8.  Record of a 128-k block:
//   2 x [C] x 64 bytes   the 64-k halves of each column, in fragment order
//   [128 / g][C8 / 2] float  factors 2^(e - 29), 2^(e - 13) of a row's lower
//                            and upper two digits
//   [128 / g][C8] int        sums of the group's digits
constexpr int kQgMaxRows = 8;
constexpr int kQgDigits = 4;
__host__ __device__ inline int qg_record_bytes(int rows, int group) {
  return rows * kQgDigits * 128 + (kQgBlockK / group) * ((rows + 1) / 2 * 8) * 6;
}

struct Q4gRows {
  const void* a;
  long long lda;
  int type, M, K, nkb, group;
  int vec;           // rows start on 16-byte boundaries
  uint8_t* records;  // [row block of 8][128-k block]; many rows: limb planes
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
// Rows to records, blocks of kQgMaxRows rows.
cudaError_t launch_q4g_rows(const Q4gRows& r, cudaStream_t s);
size_t q4g_records_bytes(const Q4gRows& r);
// Any number of rows, kQgMaxRows at a time.  q4g_stream_converts: the launch
// needs no records.
bool q4g_stream_converts(const Q4gParams& p, int sm_count);
cudaError_t launch_q4g_stream(const Q4gParams& p, int sm_count, cudaStream_t s);
cudaError_t prepare_q4g();
// Many rows on tcgen05 (ms_q4g_tc.cu): two launches; p.a.records is workspace
// of q4g_planes_bytes.
// From how many rows on: 9 bfloat16 rows (K 13824, N 5120: 27 us, two rounds of
// the streaming kernel 37 us; 8 rows 27 and 27 us), 17 rows that take two or
// three limbs (K 2560, N 20480 half: 16 rows 29 and 27 us, 20 rows 29 and 35 us;
// K 5120, N 13824 fp32: 34 and 36, 34 and 50 us).
inline int q4g_tc_rows(int type) { return type == kQgBf16 ? 9 : 17; }
size_t q4g_planes_bytes(const Q4gParams& p, int sm_count);
cudaError_t launch_q4g_tc(const Q4gParams& p, int sm_count, cudaStream_t s);
cudaError_t prepare_q4g_tc();

}  // namespace ms
