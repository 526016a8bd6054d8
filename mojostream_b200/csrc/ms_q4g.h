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
// which is the A operand (16 columns x 16 k) of one mma.m16n8k16 with the k of
// the MMA permuted so that a lane's share of an activation row is 8 values in
// a row.  Blocks past K and columns past N hold nibble 8, zero point 8 and
// scale 0.
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
// bfloat16 limbs that hold a value of a type exactly: 24 = 8 + 8 + 8 bits,
// 11 = 8 + 3 bits.
__host__ __device__ inline int qg_limbs(int type) {
  return type == kQgF32 ? 3 : type == kQgF16 ? 2 : 1;
}

struct Q4gParams {
  Q4gView w;         // the weight, or the gate
  const uint8_t* w2; // gated: the up weight (same shape and groups), else null
  // activations as bfloat16 limb planes, row blocks of `mb` rows:
  // [row block][k / 32][limb][row in block][32 k], k padded to 128
  const uint8_t* planes;
  int limbs, M, mb;
  void* out;
  long long ldo;
  int type;          // of out
  int accumulate;
  int act;           // gated: 0 SiLU, 1 tanh-GELU
  int* err;
  // launch shape of the streaming kernel
  int kw, tw, stages;
};

// Activation rows (any type and stride) to limb planes.
struct Q4gPlanes {
  const void* a;
  long long lda;
  int type, M, K, kpad, mb, limbs;
  int vec;           // rows start on 16-byte boundaries
  uint8_t* planes;
};

cudaError_t launch_q4g_repack(uint8_t* out, const Q4gView& v, const uint8_t* src, const void* scales,
                              const uint8_t* zeros, int* bad, cudaStream_t s);
cudaError_t launch_q4g_planes(const Q4gPlanes& p, cudaStream_t s);
cudaError_t launch_q4g_stream(const Q4gParams& p, int T, int NB, int sm_count, cudaStream_t s);
cudaError_t prepare_q4g();

}  // namespace ms
