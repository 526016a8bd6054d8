// ms_rules.h -- parameter block of the logit rules kernel (ms_rules.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ms {

struct RulesParams {
  const void* logits;
  void* out;
  long long ld, ldo;  // elements
  int type;           // 0 fp32, 1 bfloat16, 2 half
  int M, V;
  const int* hist;
  const int* hist_off;  // [M + 1] or null
  int n_hist;
  const float* repetition;  // [M] or null
  const float* presence;
  const float* frequency;
  const int* bias_id;
  const float* bias_val;
  const int* bias_off;  // [M + 1] or null
  int n_bias;
  const uint32_t* mask;  // [n_masks][mask_ld] words, or null
  long long mask_ld;
  int n_masks;
  const int* mask_row;  // [M], or null: row r uses mask r
};

cudaError_t launch_rules(const RulesParams& p, int sm_count, cudaStream_t s);

}  // namespace ms
