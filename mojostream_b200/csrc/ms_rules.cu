// ms_rules.cu -- rules on logits before the sampler: repetition, presence and
// frequency penalties, biases and grammar masks, for every row of a block.
//
// Row r, id j, c = occurrences of j in the row's history:
//   v = logit;  if c > 0:  v = (v > 0 ? v / rep : v * rep) - (pres + freq c)
//   if j is in the row's bias list:  v = v + bias   (the last entry of an id)
//   if the row's mask bit of j is 0: v = -inf
// in fp32, rounded once to the logits' type.
//
// Bound: HBM, one read of the allowed logits and one write of all of them.
// One CTA owns `chunk` columns of a row.  It counts the history's ids and
// finds the last bias entry of its columns in shared memory while the rest is
// a stream: a 32-column word of the mask that allows nothing is written
// without reading its logits, and in place a word that changes nothing is not
// touched.  The ids that the lists name (few) are then rewritten one by one.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ms_common.cuh"
#include "ms_rules.h"

namespace ms {
namespace {

constexpr int kRuThreads = 256;

template <typename E>
struct Elem;
template <>
struct Elem<float> {
  static __device__ float load(const float* p) { return *p; }
  static __device__ float cvt(float v) { return v; }
};
template <>
struct Elem<__nv_bfloat16> {
  static __device__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __nv_bfloat16 cvt(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<__half> {
  static __device__ float load(const __half* p) { return __half2float(*p); }
  static __device__ __half cvt(float v) { return __float2half_rn(v); }
};

struct Span {
  int b, e;
};
__device__ __forceinline__ Span row_span(const int* off, int r, int n) {
  Span s{0, 0};
  if (off) {
    s.b = min(max(off[r], 0), n);
    s.e = min(max(off[r + 1], s.b), n);
  }
  return s;
}

template <typename E>
__global__ void __launch_bounds__(kRuThreads) rules_kernel(const RulesParams p) {
  extern __shared__ uint32_t tab[];  // counts [chunk], then bias entries [chunk]
  const int r = blockIdx.y, tid = threadIdx.x;
  const int lo = blockIdx.x * p.chunk, n = min(p.chunk, p.V - lo);
  const E* in = reinterpret_cast<const E*>(p.logits) + (size_t)r * p.ld + lo;
  E* out = reinterpret_cast<E*>(p.out) + (size_t)r * p.ldo + lo;
  const bool in_place = p.logits == p.out;
  const uint32_t* mask = nullptr;
  if (p.mask) {
    const int k = p.mask_row ? p.mask_row[r] : r;
    if (k >= 0 && k < p.n_masks) mask = p.mask + (size_t)k * p.mask_ld + lo / 32;
  }
  const Span h = row_span(p.hist_off, r, p.n_hist), b = row_span(p.bias_off, r, p.n_bias);
  const bool lists = h.e > h.b || b.e > b.b;
  uint32_t* cnt = tab;
  uint32_t* ent = tab + p.chunk;
  if (lists) {
    for (int i = tid; i < 2 * p.chunk; i += kRuThreads) tab[i] = 0u;
    __syncthreads();
    for (int i = h.b + tid; i < h.e; i += kRuThreads) {
      const long long d = (long long)p.hist[i] - lo;
      if (d >= 0 && d < n) atomicAdd(&cnt[d], 1u);
    }
    for (int i = b.b + tid; i < b.e; i += kRuThreads) {
      const long long d = (long long)p.bias_id[i] - lo;
      if (d >= 0 && d < n) atomicMax(&ent[d], (unsigned)(i - b.b) + 1u);
    }
  }
  // the stream: copy the allowed columns, -inf into the others
  const E ninf = Elem<E>::cvt(-INFINITY);
  for (int j = tid; j < n; j += kRuThreads) {
    const bool keep = !mask || ((mask[j >> 5] >> (j & 31)) & 1u);
    if (!keep)
      out[j] = ninf;
    else if (!in_place)
      out[j] = in[j];
  }
  if (!lists) return;
  __syncthreads();  // counts complete; the stream's writes come before the rewrites
  const float rep = p.repetition ? p.repetition[r] : 1.f;
  const float pres = p.presence ? p.presence[r] : 0.f;
  const float freq = p.frequency ? p.frequency[r] : 0.f;
  auto rewrite = [&](int j) {
    if (mask && !((mask[j >> 5] >> (j & 31)) & 1u)) return;
    float v = Elem<E>::load(in + j);
    const uint32_t c = cnt[j] & 0x7fffffffu, e = ent[j];
    if (c) {
      v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
      v = __fsub_rn(v, __fadd_rn(pres, __fmul_rn(freq, (float)c)));
    }
    if (e) v = __fadd_rn(v, p.bias_val[b.b + (int)e - 1]);
    out[j] = Elem<E>::cvt(v);
  };
  // each id once: the first thread to set the top bit of its count rewrites it
  for (int i = h.b + tid; i < h.e; i += kRuThreads) {
    const long long d = (long long)p.hist[i] - lo;
    if (d >= 0 && d < n && !(atomicOr(&cnt[d], 0x80000000u) >> 31)) rewrite((int)d);
  }
  for (int i = b.b + tid; i < b.e; i += kRuThreads) {
    const long long d = (long long)p.bias_id[i] - lo;
    if (d >= 0 && d < n && !(atomicOr(&cnt[d], 0x80000000u) >> 31)) rewrite((int)d);
  }
}

}  // namespace

cudaError_t launch_rules(const RulesParams& p0, int sm_count, cudaStream_t s) {
  RulesParams p = p0;
  // columns per CTA: 8192 where the rows fill the GPU, fewer for few rows
  int chunk = 8192;
  while (chunk > 1024 && (long long)((p.V + chunk - 1) / chunk) * p.M < 4LL * sm_count) chunk /= 2;
  p.chunk = chunk;
  const dim3 grid((p.V + chunk - 1) / chunk, p.M);
  const size_t smem = (size_t)2 * chunk * sizeof(uint32_t);
  if (p.type == 0)
    rules_kernel<float><<<grid, kRuThreads, smem, s>>>(p);
  else if (p.type == 1)
    rules_kernel<__nv_bfloat16><<<grid, kRuThreads, smem, s>>>(p);
  else
    rules_kernel<__half><<<grid, kRuThreads, smem, s>>>(p);
  return cudaGetLastError();
}

cudaError_t prepare_rules() {
  cudaError_t e = cudaFuncSetAttribute(rules_kernel<float>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(rules_kernel<__nv_bfloat16>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(rules_kernel<__half>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             64 * 1024);
  return e;
}

}  // namespace ms
