// ms_ops.cu -- C-ABI of the operators that stand beside the token loop:
// group-scaled 4-bit products, the gated feed-forward half on them, and the
// rules on logits.  Kernels: ms_q4g.cu, ms_rules.cu.
#include <cuda_runtime.h>

#include <climits>
#include <cstdio>
#include <new>

#include "../../include/mojostream_cuda.h"
#include "ms_internal.h"
#include "ms_overlap.h"
#include "ms_q4g.h"
#include "ms_rules.h"

using namespace ms;

struct ms_q4g_weight {
  int device = 0;
  Q4gView v{};
  size_t bytes = 0;
};

namespace {

#define OPS_FAIL(c, s, ...)                 \
  do {                                      \
    char b_[384];                           \
    snprintf(b_, sizeof b_, __VA_ARGS__);   \
    return ms_fail_((c), (s), b_);          \
  } while (0)

#define OPS_CUDA(c, call)                                                                       \
  do {                                                                                          \
    const cudaError_t e_ = (call);                                                              \
    if (e_ != cudaSuccess) {                                                                    \
      cudaGetLastError(); /* reported here: a later launch must not see it again */             \
      OPS_FAIL((c), e_ == cudaErrorMemoryAllocation ? MS_ERR_OOM : MS_ERR_CUDA, "%s: %s", #call, \
               cudaGetErrorString(e_));                                                         \
    }                                                                                           \
  } while (0)

// The context's device is current inside a call; the caller's comes back after.
struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int device) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != device)
      cudaSetDevice(device);
    else
      prev = -1;
  }
  ~DeviceGuard() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

// Device memory that kernels on `device` can use.
bool on_device(const void* p, int device) {
  cudaPointerAttributes a;
  if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  return (a.type == cudaMemoryTypeDevice && a.device == device) || a.type == cudaMemoryTypeManaged;
}

int type_size(int t) { return t == MS_F32 ? 4 : 2; }

// Work that may still write `src`: everything queued on the device that holds
// it (null: none), pinned host memory counting for the context's device.
cudaError_t wait_for_writers(const void* src, int device) {
  cudaPointerAttributes a;
  if (!src) return cudaSuccess;
  if (cudaPointerGetAttributes(&a, src) != cudaSuccess) {
    cudaGetLastError();
    return cudaSuccess;
  }
  if (a.type != cudaMemoryTypeDevice || a.device == device) return cudaSuccess;  // (waited for already)
  DeviceGuard other(a.device);
  return cudaDeviceSynchronize();
}

// A source matrix on the device: itself, or a copy of host memory.
struct Staged {
  const void* p = nullptr;
  void* owned = nullptr;
  ~Staged() {
    if (owned) cudaFree(owned);
  }
  cudaError_t take(const void* src, size_t bytes, int device) {
    if (on_device(src, device)) {
      p = src;
      return cudaSuccess;
    }
    cudaError_t e = cudaMalloc(&owned, bytes);
    if (e == cudaSuccess) e = cudaMemcpy(owned, src, bytes, cudaMemcpyDefault);
    p = owned;
    return e;
  }
};

// Checks shared by the products; rows of `cols` results, K inputs.
ms_status check_rows_args(ms_ctx* c, const char* what, const ms_q4g_weight* w, const void* out,
                          int64_t ldo, const void* a, int64_t lda, int dtype, int M) {
  if (!c || !w || !out || !a) return c ? ms_fail_(c, MS_ERR_INVALID_ARG, "null argument") : MS_ERR_INVALID_ARG;
  const int dev = ms_device_(c);
  if (w->device != dev)
    OPS_FAIL(c, MS_ERR_STATE, "%s: weight on device %d, context on %d", what, w->device, dev);
  if (dtype != MS_F32 && dtype != MS_BF16 && dtype != MS_F16)
    OPS_FAIL(c, MS_ERR_INVALID_ARG, "%s: dtype %d", what, dtype);
  if (M <= 0) OPS_FAIL(c, MS_ERR_SHAPE, "%s: M=%d", what, M);
  if (lda < w->v.K || ldo < w->v.N)
    OPS_FAIL(c, MS_ERR_SHAPE, "%s: row strides %lld, %lld below K=%d, N=%d", what, (long long)lda,
             (long long)ldo, w->v.K, w->v.N);
  const uintptr_t es = (uintptr_t)type_size(dtype);
  if (((uintptr_t)a % es) || ((uintptr_t)out % es))
    OPS_FAIL(c, MS_ERR_ALIGN, "%s: A and the result must be aligned to their elements", what);
  if (!on_device(a, dev) || !on_device(out, dev))
    OPS_FAIL(c, MS_ERR_INVALID_ARG, "%s: A and the result must be memory of device %d", what, dev);
  if (rows_share((uintptr_t)a, lda * es, w->v.K * es, (uintptr_t)out, ldo * es, w->v.N * es, M))
    OPS_FAIL(c, MS_ERR_INVALID_ARG, "%s: A and the result share memory", what);
  return MS_OK;
}

ms_status run_q4g(ms_ctx* c, const ms_q4g_weight* w, const ms_q4g_weight* w2, int act, void* out,
                  int64_t ldo, const void* a, int64_t lda, int dtype, int M, int accumulate,
                  void* stream) {
  cudaStream_t s = stream ? (cudaStream_t)stream : ms_stream_(c);
  DeviceGuard guard(ms_device_(c));
  Q4gParams p{};
  p.w = w->v;
  p.w2 = w2 ? w2->v.w : nullptr;
  p.a.a = a;
  p.a.lda = lda;
  p.a.type = dtype;
  p.a.M = M;
  p.a.K = w->v.K;
  p.a.nkb = w->v.nkb;
  p.a.group = w->v.group;
  p.a.vec = !((uintptr_t)a & 15) && (lda * type_size(dtype)) % 16 == 0;
  p.out = out;
  p.ldo = ldo;
  p.accumulate = accumulate;
  p.act = act;
  p.err = ms_err_word_(c);
  if (M >= q4g_tc_rows(dtype)) {
    if (M > (1 << 22)) OPS_FAIL(c, MS_ERR_SHAPE, "q4g: M=%d", M);
    void* ws = nullptr;
    const ms_status st = ms_workspace_(c, s, q4g_planes_bytes(p, ms_sm_count_(c)), &ws);
    if (st != MS_OK) return st;
    p.a.records = (uint8_t*)ws;
    OPS_CUDA(c, launch_q4g_tc(p, ms_sm_count_(c), s));
    return MS_OK;
  }
  if (!q4g_stream_converts(p, ms_sm_count_(c))) {
    void* ws = nullptr;
    const ms_status st = ms_workspace_(c, s, q4g_records_bytes(p.a), &ws);
    if (st != MS_OK) return st;
    p.a.records = (uint8_t*)ws;
    OPS_CUDA(c, launch_q4g_rows(p.a, s));
  }
  OPS_CUDA(c, launch_q4g_stream(p, ms_sm_count_(c), s));
  return MS_OK;
}

}  // namespace

extern "C" ms_status ms_q4g_weight_create(ms_ctx* c, const uint8_t* w, const void* scales,
                                          int scale_dtype, const uint8_t* zeros, int K, int N,
                                          int group, ms_q4g_weight** out) {
  if (!c || !w || !scales || !out) return MS_ERR_INVALID_ARG;
  *out = nullptr;
  if (group != 32 && group != 64 && group != 128)
    OPS_FAIL(c, MS_ERR_SHAPE, "ms_q4g_weight_create: group %d (32, 64 or 128)", group);
  if (K <= 0 || N <= 0 || K % group || N % 2 || K > INT_MAX - 128 || N > INT_MAX - 64)
    OPS_FAIL(c, MS_ERR_SHAPE, "ms_q4g_weight_create: K=%d N=%d (need K%%%d==0, N%%2==0)", K, N, group);
  if (scale_dtype != MS_F16 && scale_dtype != MS_BF16)
    OPS_FAIL(c, MS_ERR_INVALID_ARG, "ms_q4g_weight_create: scale type %d (half or bfloat16)",
             scale_dtype);
  if ((uintptr_t)scales & 1) OPS_FAIL(c, MS_ERR_ALIGN, "ms_q4g_weight_create: scales not 2-byte aligned");
  const int dev = ms_device_(c);
  DeviceGuard guard(dev);
  cudaStream_t s = ms_stream_(c);
  Q4gView v{};
  v.K = K;
  v.N = N;
  v.nkb = (K + kQgBlockK - 1) / kQgBlockK;
  v.group = group;
  v.zeros = zeros != nullptr;
  v.bf_scale = scale_dtype == MS_BF16;
  v.block_bytes = q4g_block_bytes(group, v.zeros);
  const size_t bytes = (size_t)q4g_quads(N) * v.nkb * kQgQuad * v.block_bytes;
  const size_t n_groups = (size_t)(K / group) * N;
  // the sources may still be written by work on other streams, host memory by
  // copies out of the device: all of it first, then the copies of them
  OPS_CUDA(c, cudaDeviceSynchronize());
  for (const void* src : {(const void*)w, scales, (const void*)zeros})
    OPS_CUDA(c, wait_for_writers(src, dev));
  Staged sw, ss, sz;
  OPS_CUDA(c, sw.take(w, (size_t)K * (N / 2), dev));
  OPS_CUDA(c, ss.take(scales, n_groups * 2, dev));
  if (zeros) OPS_CUDA(c, sz.take(zeros, n_groups, dev));
  uint8_t* d = nullptr;
  int* bad = nullptr;
  int h_bad = 0;
  cudaError_t e = cudaMalloc((void**)&d, bytes);
  if (e == cudaSuccess) e = cudaMalloc((void**)&bad, sizeof(int));
  if (e == cudaSuccess) e = cudaMemsetAsync(bad, 0, sizeof(int), s);
  if (e == cudaSuccess)
    e = launch_q4g_repack(d, v, (const uint8_t*)sw.p, ss.p, (const uint8_t*)sz.p, bad, s);
  if (e == cudaSuccess) e = cudaMemcpyAsync(&h_bad, bad, sizeof(int), cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  cudaFree(bad);
  ms_q4g_weight* h = e == cudaSuccess && !h_bad ? new (std::nothrow) ms_q4g_weight : nullptr;
  if (!h) cudaFree(d);
  OPS_CUDA(c, e);
  if (h_bad) OPS_FAIL(c, MS_ERR_INVALID_ARG, "ms_q4g_weight_create: a zero point above 15");
  if (!h) OPS_FAIL(c, MS_ERR_OOM, "ms_q4g_weight_create: host memory");
  v.w = d;
  h->device = dev;
  h->v = v;
  h->bytes = bytes;
  *out = h;
  return MS_OK;
}

extern "C" ms_status ms_q4g_weight_destroy(ms_ctx* c, ms_q4g_weight* w) {
  if (!c || !w) return MS_ERR_INVALID_ARG;
  DeviceGuard guard(w->device);
  cudaDeviceSynchronize();  // calls on any stream may still read it
  cudaFree(const_cast<uint8_t*>(w->v.w));
  delete w;
  return MS_OK;
}

extern "C" size_t ms_q4g_weight_bytes(const ms_q4g_weight* w) { return w ? w->bytes : 0; }

extern "C" ms_status ms_q4g_gemm(ms_ctx* c, const ms_q4g_weight* w, void* C, int64_t ldc,
                                 const void* A, int64_t lda, int dtype, int M, int accumulate,
                                 void* stream) {
  const ms_status st = check_rows_args(c, "ms_q4g_gemm", w, C, ldc, A, lda, dtype, M);
  if (st != MS_OK) return st;
  return run_q4g(c, w, nullptr, 0, C, ldc, A, lda, dtype, M, accumulate != 0, stream);
}

extern "C" ms_status ms_q4g_gated(ms_ctx* c, const ms_q4g_weight* gate, const ms_q4g_weight* up,
                                  int act, void* H, int64_t ldh, const void* A, int64_t lda,
                                  int dtype, int M, void* stream) {
  const ms_status st = check_rows_args(c, "ms_q4g_gated", gate, H, ldh, A, lda, dtype, M);
  if (st != MS_OK) return st;
  if (!up) OPS_FAIL(c, MS_ERR_INVALID_ARG, "ms_q4g_gated: null up weight");
  if (act != MS_ACT_SILU && act != MS_ACT_GELU_TANH)
    OPS_FAIL(c, MS_ERR_INVALID_ARG, "ms_q4g_gated: activation %d", act);
  if (up->device != gate->device)
    OPS_FAIL(c, MS_ERR_STATE, "ms_q4g_gated: gate on device %d, up on %d", gate->device, up->device);
  const Q4gView &g = gate->v, &u = up->v;
  if (g.K != u.K || g.N != u.N || g.group != u.group || g.zeros != u.zeros || g.bf_scale != u.bf_scale)
    OPS_FAIL(c, MS_ERR_SHAPE,
             "ms_q4g_gated: gate (K %d, N %d, group %d, zeros %d) and up (K %d, N %d, group %d, "
             "zeros %d) must match, their scale types too",
             g.K, g.N, g.group, g.zeros, u.K, u.N, u.group, u.zeros);
  return run_q4g(c, gate, up, act, H, ldh, A, lda, dtype, M, 0, stream);
}

extern "C" ms_status ms_logit_rules_apply(ms_ctx* c, const void* logits, int64_t ld, void* out,
                                          int64_t ldo, int dtype, int M, int V,
                                          const ms_logit_rules* rules, void* stream) {
  if (!c || !logits || !out || !rules)
    return c ? ms_fail_(c, MS_ERR_INVALID_ARG, "ms_logit_rules_apply: null argument")
             : MS_ERR_INVALID_ARG;
  const char* what = "ms_logit_rules_apply";
  if (dtype != MS_F32 && dtype != MS_BF16 && dtype != MS_F16)
    OPS_FAIL(c, MS_ERR_INVALID_ARG, "%s: dtype %d", what, dtype);
  if (M <= 0 || M > 65535 || V <= 0 || V > INT_MAX - 65536)
    OPS_FAIL(c, MS_ERR_SHAPE, "%s: M=%d V=%d", what, M, V);
  if (ld < V || ldo < V)
    OPS_FAIL(c, MS_ERR_SHAPE, "%s: row strides %lld, %lld below V=%d", what, (long long)ld,
             (long long)ldo, V);
  if (logits == out && ld != ldo)
    OPS_FAIL(c, MS_ERR_SHAPE, "%s: in place needs one row stride, got %lld and %lld", what,
             (long long)ld, (long long)ldo);
  const uintptr_t es = (uintptr_t)type_size(dtype);
  if (((uintptr_t)logits % es) || ((uintptr_t)out % es))
    OPS_FAIL(c, MS_ERR_ALIGN, "%s: logits must be aligned to their elements", what);
  // out either is logits or shares no byte with it
  if (logits != out && rows_share((uintptr_t)logits, ld * es, V * es, (uintptr_t)out, ldo * es, V * es, M))
    OPS_FAIL(c, MS_ERR_INVALID_ARG, "%s: out overlaps logits without being it", what);
  const ms_logit_rules& q = *rules;
  if (!q.hist != !q.hist_off || !q.bias_id != !q.bias_off || !q.bias_id != !q.bias_val)
    OPS_FAIL(c, MS_ERR_INVALID_ARG, "%s: a list and its offsets go together", what);
  if (q.n_hist < 0 || q.n_bias < 0 || (!q.hist && q.n_hist) || (!q.bias_id && q.n_bias))
    OPS_FAIL(c, MS_ERR_INVALID_ARG, "%s: list lengths %d, %d", what, q.n_hist, q.n_bias);
  // (a list is walked in steps of up to 4096 entries, by int)
  if (q.n_hist > INT_MAX - 65536 || q.n_bias > INT_MAX - 65536)
    OPS_FAIL(c, MS_ERR_SHAPE, "%s: list lengths %d, %d", what, q.n_hist, q.n_bias);
  if ((q.repetition || q.presence || q.frequency) && !q.hist)
    OPS_FAIL(c, MS_ERR_INVALID_ARG, "%s: penalties without a history", what);
  if (q.mask) {
    if (q.n_masks <= 0 || q.mask_ld < (V + 31) / 32)
      OPS_FAIL(c, MS_ERR_SHAPE, "%s: %d masks of %lld words for V=%d", what, q.n_masks,
               (long long)q.mask_ld, V);
    if (!q.mask_row && q.n_masks < M)
      OPS_FAIL(c, MS_ERR_SHAPE, "%s: %d masks for %d rows without mask_row", what, q.n_masks, M);
  } else if (q.mask_row) {
    OPS_FAIL(c, MS_ERR_INVALID_ARG, "%s: mask_row without masks", what);
  }
  const int dev = ms_device_(c);
  const void* ptrs[] = {logits,      out,       q.hist,     q.hist_off, q.repetition, q.presence,
                        q.frequency, q.bias_id, q.bias_val, q.bias_off, q.mask,       q.mask_row};
  for (int i = 0; i < 12; ++i) {
    if (!ptrs[i]) continue;
    if (i >= 2 && ((uintptr_t)ptrs[i] & 3))
      OPS_FAIL(c, MS_ERR_ALIGN, "%s: lists and masks must be 4-byte aligned", what);
    if (!on_device(ptrs[i], dev))
      OPS_FAIL(c, MS_ERR_INVALID_ARG, "%s: every buffer must be memory of device %d", what, dev);
  }
  RulesParams p{};
  p.logits = logits;
  p.out = out;
  p.ld = ld;
  p.ldo = ldo;
  p.type = dtype;
  p.M = M;
  p.V = V;
  p.hist = q.hist;
  p.hist_off = q.hist_off;
  p.n_hist = q.n_hist;
  p.repetition = q.repetition;
  p.presence = q.presence;
  p.frequency = q.frequency;
  p.bias_id = q.bias_id;
  p.bias_val = q.bias_val;
  p.bias_off = q.bias_off;
  p.n_bias = q.n_bias;
  p.mask = q.mask;
  p.mask_ld = q.mask_ld;
  p.n_masks = q.n_masks;
  p.mask_row = q.mask_row;
  DeviceGuard guard(dev);
  OPS_CUDA(c, launch_rules(p, ms_sm_count_(c), stream ? (cudaStream_t)stream : ms_stream_(c)));
  return MS_OK;
}
