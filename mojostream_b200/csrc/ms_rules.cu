// ms_rules.cu -- rules on logits before the sampler: repetition, presence and
// frequency penalties, biases and grammar masks, for every row of a block.
//
// Row r, id j, c = occurrences of j in the row's history:
//   v = logit;  if c > 0:  v = (v > 0 ? v / rep : v * rep) - (pres + freq c)
//   if j is in the row's bias list:  v = v + bias   (the last entry of an id)
//   if the row's mask bit of j is 0: v = -inf
// in fp32, rounded once to the logits' type.
//
// Bound: HBM, one read of the allowed logits and one write of all of them.  A
// thread moves 16-byte pieces; a piece that the mask empties is not read, and
// in place only pieces that the mask cuts are written.  The few ids that the
// lists name are rewritten one by one afterwards.
//   Few columns in all: one kernel, whose CTAs count the history's ids of their
// columns in shared memory while their pieces are on the way (one row, V
// 262144: 4.1 us).  Many: every CTA would scan its row's history for a sliver
// of columns, so the stream runs by itself and a second kernel, which starts as
// the first drains, gathers each row's ids in hash tables and rewrites them (64
// rows of V 262144, 4096 ids each, 16 masks: 39 us in one kernel, 26 us in two,
// of them 22 us the stream, 4.5 TB/s).
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
  static constexpr uint32_t kNinf = 0xff800000u;
};
template <>
struct Elem<__nv_bfloat16> {
  static __device__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __nv_bfloat16 cvt(float v) { return __float2bfloat16_rn(v); }
  static constexpr uint32_t kNinf = 0xff80u;
};
template <>
struct Elem<__half> {
  static __device__ float load(const __half* p) { return __half2float(*p); }
  static __device__ __half cvt(float v) { return __float2half_rn(v); }
  static constexpr uint32_t kNinf = 0xfc00u;
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

// f(i, list[i]) for b <= i < e by a CTA of N threads, four ids in flight per
// thread (f is a loop over shared memory: more copies of it cost more in
// instruction fetches than they save).
template <int N, typename F>
__device__ __forceinline__ void scan_ids(const int* list, int b, int e, F f) {
  for (int i0 = b + threadIdx.x; i0 < e; i0 += 4 * N) {
    int x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = i0 + u * N < e ? __ldg(list + i0 + u * N) : -1;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (x[u] >= 0) f(i0 + u * N, x[u]);
  }
}

// A row of the call: its logits, result and mask.
template <typename E>
struct Row {
  static constexpr int VEC = 16 / sizeof(E);
  static constexpr uint32_t kAll = (1u << VEC) - 1;
  const E* in;
  E* out;
  const uint32_t* mask;  // or null
  bool in_place, same;   // `same`: aligned pieces of out are aligned in `in` too
  int V, head;           // columns before out's first 16-byte boundary

  __device__ __forceinline__ Row(const RulesParams& p, int r) {
    const int mk = p.mask ? (p.mask_row ? p.mask_row[r] : r) : -1;
    in = reinterpret_cast<const E*>(p.logits) + (size_t)r * p.ld;
    out = reinterpret_cast<E*>(p.out) + (size_t)r * p.ldo;
    mask = mk >= 0 && mk < p.n_masks ? p.mask + (size_t)mk * p.mask_ld : nullptr;
    in_place = p.logits == p.out;
    same = (((uintptr_t)in ^ (uintptr_t)out) & 15) == 0;
    V = p.V;
    head = min((int)(((16 - ((uintptr_t)out & 15)) & 15) / sizeof(E)), V);
  }
  __device__ __forceinline__ bool keeps(int j) const {
    return !mask || ((__ldg(mask + (j >> 5)) >> (j & 31)) & 1u);
  }
  // allowed columns j .. j + VEC - 1 as bits (columns past V: 0)
  __device__ __forceinline__ uint32_t allowed(int j) const {
    if (j >= V) return 0u;
    uint32_t bits = kAll;
    if (mask) {
      const uint32_t w0 = __ldg(mask + (j >> 5));
      const uint32_t w1 = (j & 31) + VEC > 32 && ((j >> 5) + 1) * 32 < V ? __ldg(mask + (j >> 5) + 1) : 0u;
      bits = __funnelshift_r(w0, w1, j & 31) & kAll;
    }
    return j + VEC <= V ? bits : bits & ((1u << (V - j)) - 1);
  }
  // the piece at column j (a boundary of out) where it has to be read: in place
  // only to be written back around its masked columns
  __device__ __forceinline__ uint4 load(int j, uint32_t ok) const {
    if (!ok || (in_place && ok == kAll)) return make_uint4(0u, 0u, 0u, 0u);
    if (same && j + VEC <= V) return *reinterpret_cast<const uint4*>(in + j);
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if ((ok >> e) & 1u) {
        if (sizeof(E) == 4)
          w[e & 3] = reinterpret_cast<const uint32_t*>(in)[j + e];
        else
          w[(e / 2) & 3] |= (uint32_t)reinterpret_cast<const unsigned short*>(in)[j + e] << (16 * (e & 1));
      }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // the allowed columns copied, -inf in the others
  __device__ __forceinline__ void store(int j, uint32_t ok, const uint4& x) const {
    if (j >= V || (in_place && ok == kAll)) return;
    constexpr uint32_t n1 = Elem<E>::kNinf, n2 = sizeof(E) == 4 ? n1 : n1 | (n1 << 16);
    uint32_t w[4] = {x.x, x.y, x.z, x.w};
    if (j + VEC <= V) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (sizeof(E) == 4) {
          if (!((ok >> k) & 1u)) w[k] = n2;
        } else {
          if (!((ok >> (2 * k)) & 1u)) w[k] = (w[k] & 0xffff0000u) | n1;
          if (!((ok >> (2 * k + 1)) & 1u)) w[k] = (w[k] & 0xffffu) | (n1 << 16);
        }
      }
      *reinterpret_cast<uint4*>(out + j) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (j + e >= V) break;
        const bool keep = (ok >> e) & 1u;
        if (sizeof(E) == 4)
          reinterpret_cast<uint32_t*>(out)[j + e] = keep ? w[e & 3] : n1;
        else
          reinterpret_cast<unsigned short*>(out)[j + e] =
              (unsigned short)(keep ? w[(e / 2) & 3] >> (16 * (e & 1)) : n1);
      }
    }
  }
  // the columns before the first boundary
  __device__ __forceinline__ void store_head(int j) const {
    if (j >= head) return;
    if (!keeps(j))
      out[j] = Elem<E>::cvt(-INFINITY);
    else if (!in_place)
      out[j] = in[j];
  }
};

struct Penalty {
  float rep, pres, freq;
  __device__ __forceinline__ Penalty(const RulesParams& p, int r)
      : rep(p.repetition ? p.repetition[r] : 1.f),
        pres(p.presence ? p.presence[r] : 0.f),
        freq(p.frequency ? p.frequency[r] : 0.f) {}
  // logit v of an id with c occurrences and (ent > 0) the bias entry ent - 1
  __device__ __forceinline__ float apply(float v, uint32_t c, uint32_t ent, const float* bias) const {
    if (c) {
      v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
      v = __fsub_rn(v, __fadd_rn(pres, __fmul_rn(freq, (float)c)));
    }
    return ent ? __fadd_rn(v, bias[ent - 1]) : v;
  }
};

// Stream and lists in one kernel: NV pieces per thread.
template <typename E, int NV>
__global__ void __launch_bounds__(kRuThreads) rules_kernel(const RulesParams p) {
  constexpr int VEC = Row<E>::VEC, kChunk = kRuThreads * NV * VEC, kTab = kChunk + VEC;
  extern __shared__ __align__(16) uint32_t tab[];  // counts, bias entries, ids touched (16 bits)
  __shared__ int s_n;
  const int r = blockIdx.y, tid = threadIdx.x;
  const Row<E> row(p, r);
  const Span h = row_span(p.hist_off, r, p.n_hist), b = row_span(p.bias_off, r, p.n_bias);
  const bool lists = h.e > h.b || b.e > b.b;
  // the columns before the row's first 16-byte boundary belong to the first CTA
  const int first = row.head + blockIdx.x * kChunk;  // first piece
  const int end = min(first + kChunk, p.V);          // columns of this CTA: lo .. end - 1
  const int lo = blockIdx.x == 0 ? 0 : min(first, p.V);

  uint4 x[NV];
  uint32_t ok[NV];
#pragma unroll
  for (int u = 0; u < NV; ++u) ok[u] = row.allowed(first + (u * kRuThreads + tid) * VEC);
#pragma unroll
  for (int u = 0; u < NV; ++u) x[u] = row.load(first + (u * kRuThreads + tid) * VEC, ok[u]);

  uint32_t* cnt = tab;
  uint32_t* ent = tab + kTab;
  uint16_t* ids = reinterpret_cast<uint16_t*>(tab + 2 * kTab);
  if (lists) {
    uint4* z = reinterpret_cast<uint4*>(tab);
    const int nz = (b.e > b.b ? 2 : 1) * kTab / 4;
    for (int i = tid; i < nz; i += kRuThreads) z[i] = make_uint4(0u, 0u, 0u, 0u);
    if (tid == 0) s_n = 0;
    __syncthreads();
    // each id that is met for the first time, in either list, joins `ids`
    scan_ids<kRuThreads>(p.hist, h.b, h.e, [&](int, int id) {
      const unsigned d = (unsigned)id - (unsigned)lo;
      if (id >= lo && id < end && !atomicAdd(&cnt[d], 1u)) ids[atomicAdd(&s_n, 1)] = (uint16_t)d;
    });
  }
#pragma unroll
  for (int u = 0; u < NV; ++u) row.store(first + (u * kRuThreads + tid) * VEC, ok[u], x[u]);
  if (blockIdx.x == 0) row.store_head(tid);
  if (!lists) return;

  __syncthreads();  // counts complete
  if (b.e > b.b) {
    scan_ids<kRuThreads>(p.bias_id, b.b, b.e, [&](int i, int id) {
      const unsigned d = (unsigned)id - (unsigned)lo;
      if (id >= lo && id < end && !atomicMax(&ent[d], (unsigned)(i - b.b) + 1u) && !cnt[d])
        ids[atomicAdd(&s_n, 1)] = (uint16_t)d;
    });
    __syncthreads();
  }
  const Penalty pen(p, r);
  for (int i = tid; i < s_n; i += kRuThreads) {
    const int d = ids[i], j = lo + d;
    if (row.keeps(j))
      row.out[j] = Elem<E>::cvt(pen.apply(Elem<E>::load(row.in + j), cnt[d], b.e > b.b ? ent[d] : 0u,
                                          p.bias_val + b.b));
  }
}

// The stream alone.  A warp takes 1024 columns: one coalesced load brings their
// 32 mask words, a shuffle hands each piece its bits, and all pieces are on
// the way before the first is stored.
template <typename E>
__global__ void __launch_bounds__(kRuThreads, 5) rules_stream_kernel(const RulesParams p) {
  constexpr int VEC = Row<E>::VEC, kSteps = 32 / VEC;
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const Row<E> row(p, blockIdx.y);
  const int c0 = row.head + (blockIdx.x * (kRuThreads / 32) + (threadIdx.x >> 5)) * 1024;
  if (blockIdx.x == 0) row.store_head(threadIdx.x);
  if (c0 >= p.V) return;  // (whole warps)
  const int mine = c0 + 32 * lane;  // this lane's 32 columns of the mask
  uint32_t bits = 0xffffffffu;
  if (row.mask) {
    const int k = c0 >> 5, words = (p.V + 31) >> 5;
    const uint32_t w = k + lane < words ? __ldg(row.mask + k + lane) : 0u;
    uint32_t next = __shfl_down_sync(0xffffffffu, w, 1);
    if (lane == 31) next = (c0 & 31) && k + 32 < words ? __ldg(row.mask + k + 32) : 0u;
    bits = __funnelshift_r(w, next, c0 & 31);
  }
  if (mine + 32 > p.V) bits = mine < p.V ? bits & ((1u << (p.V - mine)) - 1) : 0u;
  uint4 x[kSteps];
  uint32_t ok = 0;  // VEC bits per piece
#pragma unroll
  for (int u = 0; u < kSteps; ++u) {
    const uint32_t o = (__shfl_sync(0xffffffffu, bits, u * VEC + lane * VEC / 32) >>
                        (lane * VEC % 32)) & Row<E>::kAll;
    ok |= o << (u * VEC);
    x[u] = row.load(c0 + (u * 32 + lane) * VEC, o);
  }
#pragma unroll
  for (int u = 0; u < kSteps; ++u)
    row.store(c0 + (u * 32 + lane) * VEC, (ok >> (u * VEC)) & Row<E>::kAll, x[u]);
}

// The lists alone, after the stream.  CTA s of a row's S = 2^sb takes the ids
// with id % S == s: an open-addressing table of ids, counts and last bias entries.  A
// table in which an id finds no slot within kHsProbe steps is emptied and its
// ids are taken in two halves (id / S even or odd), each halved again as often
// as it takes: the classes are walked as a binary tree, (m, q) being the ids
// with id / S % m == q.  (A class of kHsProbe ids always fits.)
constexpr int kHsThreads = 1024, kHsBits = 11, kHsSlots = 1 << kHsBits, kHsProbe = 64;
constexpr uint32_t kHsFree = 0xffffffffu;

template <typename E>
__global__ void __launch_bounds__(kHsThreads) rules_lists_kernel(const RulesParams p, int sb) {
  __shared__ uint32_t key[kHsSlots], cnt[kHsSlots], ent[kHsSlots];
  __shared__ volatile int s_full;
  const uint32_t key_s = smem_u32(key), cnt_s = smem_u32(cnt), ent_s = smem_u32(ent);
  const int r = blockIdx.y, tid = threadIdx.x;
  const uint32_t part = blockIdx.x;
  const Span h = row_span(p.hist_off, r, p.n_hist), b = row_span(p.bias_off, r, p.n_bias);
  const Row<E> row(p, r);
  const Penalty pen(p, r);
  bool waited = false;
  uint32_t m = 1, q = 0;
  if (h.e > h.b || b.e > b.b)
    for (;;) {
      for (int i = tid; i < kHsSlots; i += kHsThreads) {
        key[i] = kHsFree;
        cnt[i] = 0u;
        ent[i] = 0u;
      }
      if (tid == 0) s_full = 0;
      __syncthreads();
      // the slot of an id of the class, or -1
      auto slot = [&](int id) -> int {
        if (id < 0 || id >= p.V || ((uint32_t)id & ((1u << sb) - 1)) != part) return -1;
        const uint32_t w = (uint32_t)id >> sb;
        if ((w & (m - 1)) != q || s_full) return -1;
        uint32_t at = (w * 0x9E3779B1u) >> (32 - kHsBits);
        for (int n = 0; n < kHsProbe; ++n, at = (at + 1) & (kHsSlots - 1)) {
          uint32_t old;
          asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(old) : "r"(key_s + at * 4) : "memory");
          if (old == kHsFree)
            asm volatile("atom.shared.cas.b32 %0, [%1], %2, %3;"
                         : "=r"(old)
                         : "r"(key_s + at * 4), "r"(kHsFree), "r"((uint32_t)id)
                         : "memory");
          if (old == kHsFree || old == (uint32_t)id) return (int)at;
        }
        s_full = 1;
        return -1;
      };
      scan_ids<kHsThreads>(p.hist, h.b, h.e, [&](int, int id) {
        const int at = slot(id);
        if (at >= 0)
          asm volatile("red.shared.add.u32 [%0], %1;" ::"r"(cnt_s + at * 4), "r"(1u) : "memory");
      });
      scan_ids<kHsThreads>(p.bias_id, b.b, b.e, [&](int i, int id) {
        const int at = slot(id);
        if (at >= 0)
          asm volatile("red.shared.max.u32 [%0], %1;" ::"r"(ent_s + at * 4), "r"((uint32_t)(i - b.b) + 1u)
                       : "memory");
      });
      __syncthreads();
      if (s_full) {
        m *= 2;
        __syncthreads();  // read before it is reset
        continue;
      }
      if (!waited) pdl_wait();  // the stream has written
      waited = true;
      constexpr int kPer = kHsSlots / kHsThreads;
      int j[kPer];
      float v[kPer];
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        j[u] = (int)key[u * kHsThreads + tid];
        if (j[u] >= 0 && !row.keeps(j[u])) j[u] = -1;
      }
#pragma unroll
      for (int u = 0; u < kPer; ++u) v[u] = j[u] >= 0 ? Elem<E>::load(row.in + j[u]) : 0.f;
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        const int i = u * kHsThreads + tid;
        if (j[u] >= 0)
          row.out[j[u]] = Elem<E>::cvt(pen.apply(v[u], cnt[i], ent[i], p.bias_val + b.b));
      }
      while (m > 1 && q >= m / 2) {  // the next class
        q -= m / 2;
        m /= 2;
      }
      if (m == 1) break;
      q += m / 2;
      __syncthreads();  // the table is free
    }
  if (!waited) pdl_wait();
}

template <typename E, int NV>
constexpr size_t rules_smem() {
  constexpr size_t n = kRuThreads * NV * (16 / sizeof(E)) + 16 / sizeof(E);
  return n * 10;
}

template <typename E, int NV>
cudaError_t launch_t(const RulesParams& p, cudaStream_t s) {
  constexpr int chunk = kRuThreads * NV * (16 / (int)sizeof(E));
  const bool lists = p.n_hist > 0 || p.n_bias > 0;
  cudaLaunchConfig_t cfg = {};  // (the launch's own status, not an older call's)
  cfg.gridDim = dim3((p.V + chunk - 1) / chunk, p.M);
  cfg.blockDim = dim3(kRuThreads);
  cfg.dynamicSmemBytes = lists ? rules_smem<E, NV>() : 0;
  cfg.stream = s;
  return cudaLaunchKernelEx(&cfg, rules_kernel<E, NV>, p);
}

// One kernel, 1024 columns (16-bit types: 2048) per CTA, or two or four times
// as many where the rows still give every SM two CTAs; from 4096 columns for
// each of 4 x the SMs on, or with long lists, the stream and the lists apart.
template <typename E>
cudaError_t launch_e(const RulesParams& p, int sm_count, cudaStream_t s) {
  constexpr int kMax = 4096 / (kRuThreads * 16 / sizeof(E));  // 4 pieces of fp32, 2 of 16 bits
  const bool lists = p.n_hist > 0 || p.n_bias > 0;
  const long long n = (long long)p.M * p.V / 4096;
  if (n < 4LL * sm_count && ((long long)p.n_hist + p.n_bias) / p.M <= 8192) {
    if (n >= 2LL * sm_count) return launch_t<E, kMax>(p, s);
    if (kMax > 2 && n >= sm_count) return launch_t<E, (kMax + 1) / 2>(p, s);
    return launch_t<E, 1>(p, s);
  }
  const bool stream = p.mask || p.logits != p.out;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = s;
  if (stream) {
    constexpr int kCols = kRuThreads * 32;
    cfg.gridDim = dim3((p.V + kCols - 1) / kCols, p.M);
    cfg.blockDim = dim3(kRuThreads);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, rules_stream_kernel<E>, p);
    if (e != cudaSuccess) return e;
  }
  if (!lists) return cudaSuccess;
  // CTAs per row: enough for the GPU, and for about 1000 list entries each
  const long long each = ((long long)p.n_hist + p.n_bias) / p.M;
  int sb = 0;
  while (sb < 6 && (((long long)p.M << sb) < sm_count || each >> sb > 1024)) ++sb;
  cfg.gridDim = dim3(1u << sb, p.M, 1);
  cfg.blockDim = dim3(kHsThreads);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = stream ? 1 : 0;  // (alone it must wait for the kernel that wrote its inputs)
  return cudaLaunchKernelEx(&cfg, rules_lists_kernel<E>, p, sb);
}

}  // namespace

cudaError_t launch_rules(const RulesParams& p, int sm_count, cudaStream_t s) {
  if (p.type == 0) return launch_e<float>(p, sm_count, s);
  if (p.type == 1) return launch_e<__nv_bfloat16>(p, sm_count, s);
  return launch_e<__half>(p, sm_count, s);
}

}  // namespace ms
