// Distillation from a teacher's top logits.  Per row of student logits s [V] and teacher entries (id_j, t_j), j < K:
//
//     q = softmax_j(t / tau)         p = softmax_v(s / tau)         L = sum_j q_j (log q_j - log p[id_j])
//     dL/ds_v = (p_v - sum_{j: id_j = v} q_j) / tau
//
// An entry with t = -inf is no entry, nor is one whose id lies outside the vocabulary; a row without entries has L = 0
// and a zero gradient whatever its logits hold, and so has a row of weight 0.  The same id may come several times.
//
// Three kernels:
//   distill_row_kernel    the row stays in the registers of a thread-block cluster: one read of the logits gives the
//                         loss, the statistics and (optionally) the gradient, which may overwrite the logits
//   distill_stats_kernel  a row of any length, or the local part of a vocabulary that is sharded over ranks:
//                         max, sum of exponentials and the student's logits at the teacher's ids
//   distill_grad_kernel   the gradient from finished statistics (backward pass; sharded or very long rows)
//
// Statistics of a row: {top, sum, max t, sum of exp((t - max t) / tau)}.  With c = log2(e) / tau, `top` is the rounded
// c * max s and `sum` that of 2^(c s - top), so that c * max s is rounded once and cancels; the last number is 0 for a
// row without entries.  All sums are fp32; the logits' gradient is rounded once.
//
// Memory bound: the logits are read once and the gradient written once; two exponentials per element.
#include "common.cuh"

namespace stb {

constexpr int kDsThreads = 256;
constexpr int kDsMaxEntries = 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct DistillParams {
  const void* logits;
  void* grad;
  const void* ids;              // [T][K] int64 or int32
  const float* teacher;         // [T][K]
  const float* weight;          // [T] or nullptr (1)
  float* loss;                  // [T] or nullptr
  float4* stats;                // [T] or nullptr
  float* picked;                // stats kernel: [T][K] student logit at each id, 0 where it is not in this shard
  long long ld, ldg, ld_ids, ld_t;
  long long vocab_start, vocab_total;
  int V, K, T;
  int ids64;
  float inv_tau;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 bytes of logits <-> fp32
template <typename T> struct Lane;
template <> struct Lane<__nv_bfloat16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void widen(const uint4& u, float (&f)[8]) {
    f[0] = bf16_lo(u.x); f[1] = bf16_hi(u.x); f[2] = bf16_lo(u.y); f[3] = bf16_hi(u.y);
    f[4] = bf16_lo(u.z); f[5] = bf16_hi(u.z); f[6] = bf16_lo(u.w); f[7] = bf16_hi(u.w);
  }
  static __device__ __forceinline__ uint4 narrow(const float (&f)[8]) {
    return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
  }
  static __device__ __forceinline__ uint32_t bits(const __nv_bfloat16* p) {
    return *reinterpret_cast<const uint16_t*>(p);
  }
  static __device__ __forceinline__ void put(uint4& u, int j, uint32_t b) {
    uint32_t* w = &u.x;
    const int sh = 16 * (j & 1);
    w[j >> 1] = (w[j >> 1] & ~(0xFFFFu << sh)) | (b << sh);
  }
  static __device__ __forceinline__ float value(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
  static constexpr uint32_t kMinusInf = 0xFF80u;
};
template <> struct Lane<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void widen(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 narrow(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ uint32_t bits(const float* p) { return __float_as_uint(*p); }
  static __device__ __forceinline__ void put(uint4& u, int j, uint32_t b) { (&u.x)[j] = b; }
  static __device__ __forceinline__ float value(const float* p) { return *p; }
  static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
  static constexpr uint32_t kMinusInf = 0xFF800000u;
};

// A row as 16-byte granules: granule g covers elements [g*n - lead, g*n - lead + n), where `lead` elements lie between
// the 16-byte boundary below the row's first element and that element.  Granules that the row fills are moved as
// vectors, the first and last one element by element, so that nothing outside the row is touched whatever the
// alignment of its start.
template <typename T>
struct Granules {
  int lead, count;
  __device__ __forceinline__ Granules(const T* row, int V) {
    lead = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
    count = (lead + V + Lane<T>::n - 1) / Lane<T>::n;
  }
};
template <typename T>
__device__ __forceinline__ uint4 load_granule(const T* row, int g, int lead, int V) {
  constexpr int n = Lane<T>::n;
  const int a = g * n - lead;
  uint4 u;
  if (a >= 0 && a + n <= V) {
    // read once: not kept in L1.  Not the read-only path, because the gradient may be written over the logits
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(row + a) : "memory");
  } else {
    u = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < n; ++j)
      Lane<T>::put(u, j, (a + j >= 0 && a + j < V) ? Lane<T>::bits(row + a + j) : Lane<T>::kMinusInf);
  }
  return u;
}
// The gradient's n elements of a granule; `aligned`: they are one aligned vector there as well.
template <typename TO, int n>
__device__ __forceinline__ bool granules_aligned(const TO* row, int lead) {
  return ((reinterpret_cast<uintptr_t>(row) - lead * sizeof(TO)) & (n * sizeof(TO) - 1)) == 0;
}
template <typename TO, int n>
__device__ __forceinline__ void store_granule(TO* row, int g, int lead, int V, bool aligned, const float (&f)[n]) {
  const int a = g * n - lead;
  if (aligned && a >= 0 && a + n <= V) {
    if constexpr (n == Lane<TO>::n) {
      *reinterpret_cast<uint4*>(row + a) = Lane<TO>::narrow(f);
    } else {                                // fp32 logits, bf16 gradient
      *reinterpret_cast<uint2*>(row + a) = make_uint2(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < n; ++j)
      if (a + j >= 0 && a + j < V) Lane<TO>::store(row + a + j, f[j]);
  }
}

// (m, s) <- the pair that stands for both, s being relative to exp2(m).  -inf: nothing seen yet.
__device__ __forceinline__ void merge(float& m, float& s, float om, float os) {
  const float top = fmaxf(m, om);
  const float a = m == top ? s : s * ex2(m - top);
  const float b = om == top ? os : os * ex2(om - top);
  m = top;
  s = a + b;
}

// Teacher entries of a row in shared memory, filled by warp 0.
struct Entries {
  float q[kDsMaxEntries];      // probability, 0 where there is no entry
  float s[kDsMaxEntries];      // the student's logit there (0 where the id is not in this shard)
  int id[kDsMaxEntries];       // local id, -1 where there is no entry in this shard
  float tmax, tsum;            // tsum = 0: no entry at all
};

__device__ __forceinline__ long long entry_id(const DistillParams& p, long long row, int j) {
  return p.ids64 ? static_cast<const long long*>(p.ids)[row * p.ld_ids + j]
                 : static_cast<long long>(static_cast<const int*>(p.ids)[row * p.ld_ids + j]);
}

// q of an entry from the row's teacher statistics; the same expression in every kernel, so that a backward pass
// subtracts exactly what the forward pass used
__device__ __forceinline__ float entry_q(float t, float tmax, float inv_tsum, float c) {
  return ex2((t - tmax) * c) * inv_tsum;
}

template <typename T>
__device__ __forceinline__ void load_entries(const DistillParams& p, const T* row_ptr, long long row, Entries& e, int lane) {
  const float c = p.inv_tau * kLog2e;
  float tmax = -INFINITY;
  bool bad = false;            // fmaxf drops a NaN; it has to reach the loss
  for (int j = lane; j < p.K; j += 32) {
    const long long id = entry_id(p, row, j);
    const bool in = id >= 0 && id < p.vocab_total;
    const float t = in ? p.teacher[row * p.ld_t + j] : -INFINITY;
    const long long local = id - p.vocab_start;
    const bool here = in && t != -INFINITY && local >= 0 && local < p.V;
    e.q[j] = t;
    e.id[j] = here ? static_cast<int>(local) : -1;
    e.s[j] = here ? Lane<T>::value(row_ptr + local) : 0.f;
    tmax = fmaxf(tmax, t);
    bad |= t != t;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) tmax = fmaxf(tmax, __shfl_xor_sync(0xffffffffu, tmax, o));
  if (__any_sync(0xffffffffu, bad)) tmax = __uint_as_float(0x7FC00000u);
  float tsum = 0.f;
  if (tmax != -INFINITY) {
    for (int j = lane; j < p.K; j += 32) tsum += ex2((e.q[j] - tmax) * c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) tsum += __shfl_xor_sync(0xffffffffu, tsum, o);
  }
  const float inv = tmax != -INFINITY ? __fdiv_rn(1.f, tsum) : 0.f;
  for (int j = lane; j < p.K; j += 32) e.q[j] = tmax != -INFINITY ? entry_q(e.q[j], tmax, inv, c) : 0.f;
  if (lane == 0) { e.tmax = tmax; e.tsum = tsum; }
}

// One term q (log2 q - log2 p) of the loss, the difference of logarithms taken before the sum over the entries, so
// that a small divergence is not the difference of two large sums.
__device__ __forceinline__ float loss_term(float q, float t, float s, float c, const float4& st, float log_sum,
                                           float log_tsum) {
  if (q == 0.f) return 0.f;
  return q * (((t - st.z) * c - log_tsum) - (fmaf(s, c, -st.x) - log_sum));
}
__device__ __forceinline__ float warp_total(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Gradient at the ids that `mine(local id)` says are this CTA's: written once more over the dense p, from the logit
// kept in shared memory, with the q of equal ids added in order.  The caller has a barrier between the dense writes
// and this.
template <typename TO, typename Mine>
__device__ __forceinline__ void write_entries(const DistillParams& p, const Entries& e, TO* grad_row, const float4& st,
                                              float w, Mine mine) {
  const float c = p.inv_tau * kLog2e, g = w * p.inv_tau, inv = __fdiv_rn(1.f, st.y);
  for (int j = threadIdx.x; j < p.K; j += blockDim.x) {
    const int id = e.id[j];
    if (id < 0 || !mine(id)) continue;
    bool first = true;
    float q = 0.f;
    for (int i = 0; i < p.K; ++i) {
      if (e.id[i] != id) continue;
      if (i < j) { first = false; break; }
      q += e.q[i];
    }
    if (first) Lane<TO>::store(grad_row + id, (ex2(fmaf(e.s[j], c, -st.x)) * inv - q) * g);
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void store_remote(const void* local, uint32_t rank, float a, float b) {
  uint32_t addr;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(a), "f"(b) : "memory");
}

// (top, sum) of the CTA's threads, known to every thread afterwards; ends behind a block barrier.
template <int THREADS>
__device__ __forceinline__ void block_merge(float& m, float& s, float2* red) {
  constexpr int kWarps = THREADS / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    merge(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
  if (lane == 0) red[warp] = make_float2(m, s);
  __syncthreads();
  m = red[lane & (kWarps - 1)].x;
  s = red[lane & (kWarps - 1)].y;
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1)
    merge(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
}

// ------------------------------------------------------------------------------------------- row in registers
// A cluster of C CTAs holds a row: CTA r of the cluster takes granules (i * C + r) * 256 + thread, i < NV.
template <typename T, typename TO, int C, int NV>
__global__ void __launch_bounds__(kDsThreads)
distill_row_kernel(const DistillParams p) {
  constexpr int n = Lane<T>::n;
  __shared__ Entries e;
  __shared__ float2 red[kDsThreads / 32];
  __shared__ float2 part[8];               // (top, sum) of every CTA of the cluster
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = C > 1 ? static_cast<int>(cluster_rank()) : 0;
  const long long row = blockIdx.x / C;
  if constexpr (C > 1) cluster_arrive();   // "running": awaited before the first store into another CTA
  const T* src = static_cast<const T*>(p.logits) + row * p.ld;
  const Granules<T> gr(src, p.V);
  uint4 v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int g = (i * C + rank) * kDsThreads + threadIdx.x;
    if (g < gr.count) v[i] = load_granule<T>(src, g, gr.lead, p.V);
  }
  if (warp == 0) load_entries<T>(p, src, row, e, lane);
  const float c = p.inv_tau * kLog2e;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if ((i * C + rank) * kDsThreads + threadIdx.x >= gr.count) continue;
    float f[n];
    Lane<T>::widen(v[i], f);
#pragma unroll
    for (int j = 0; j < n; ++j) m = fmaxf(m, f[j]);
  }
  // a thread that has seen nothing but -inf adds exp2(-inf) = 0
  float top = m * c, sum = 0.f;
  const float base = m == -INFINITY ? 0.f : top;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if ((i * C + rank) * kDsThreads + threadIdx.x >= gr.count) continue;
    float f[n];
    Lane<T>::widen(v[i], f);
#pragma unroll
    for (int j = 0; j < n; ++j) sum += ex2(fmaf(f[j], c, -base));
  }
  block_merge<kDsThreads>(top, sum, red);
  if constexpr (C > 1) {
    cluster_wait();
    if (threadIdx.x < C) store_remote(&part[rank], threadIdx.x, top, sum);
    __syncwarp();
    cluster_arrive();                      // also: every CTA has read the logits at the teacher's ids
    cluster_wait();
    top = part[lane & (C - 1)].x;
    sum = part[lane & (C - 1)].y;
#pragma unroll
    for (int o = C / 2; o > 0; o >>= 1)
      merge(top, sum, __shfl_xor_sync(0xffffffffu, top, o), __shfl_xor_sync(0xffffffffu, sum, o));
  }
  const float4 st = make_float4(top, sum, e.tmax, e.tsum);
  if (rank == 0 && warp == 0) {
    if (p.loss != nullptr) {
      const float log_sum = log2f(st.y), log_tsum = st.w == 0.f ? 0.f : log2f(st.w);
      float l = 0.f;
      for (int j = lane; j < p.K; j += 32)
        l += e.q[j] == 0.f ? 0.f : loss_term(e.q[j], p.teacher[row * p.ld_t + j], e.s[j], c, st, log_sum, log_tsum);
      l = warp_total(l) * kLn2;
      if (lane == 0) p.loss[row] = l;
    }
    if (p.stats != nullptr && lane == 0) p.stats[row] = st;
  }
  if (p.grad == nullptr) return;

  TO* dst = static_cast<TO*>(p.grad) + row * p.ldg;
  const bool aligned = granules_aligned<TO, n>(dst, gr.lead);
  const float w = p.weight != nullptr ? p.weight[row] : 1.f;
  const bool zero = st.w == 0.f || w == 0.f;   // no entries, or a token that does not count: whatever the logits hold
  const float g = w * p.inv_tau * __fdiv_rn(1.f, st.y);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = (i * C + rank) * kDsThreads + threadIdx.x;
    if (k >= gr.count) continue;
    float f[n];
    Lane<T>::widen(v[i], f);
#pragma unroll
    for (int j = 0; j < n; ++j) f[j] = zero ? 0.f : ex2(fmaf(f[j], c, -top)) * g;
    store_granule<TO, n>(dst, k, gr.lead, p.V, aligned, f);
  }
  if (zero) return;
  __syncthreads();
  write_entries<TO>(p, e, dst, st, w, [&](int id) { return ((id + gr.lead) / n / kDsThreads) % C == rank; });
}

// ------------------------------------------------------------------------------------------- statistics, any row
constexpr int kDsStatsThreads = 512;

template <typename T>
__global__ void __launch_bounds__(kDsStatsThreads)
distill_stats_kernel(const DistillParams p) {
  constexpr int n = Lane<T>::n;
  __shared__ Entries e;
  __shared__ float2 red[kDsStatsThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row = blockIdx.x;
  const T* src = static_cast<const T*>(p.logits) + row * p.ld;
  const Granules<T> gr(src, p.V);
  const float c = p.inv_tau * kLog2e;
  if (warp == 0) {
    load_entries<T>(p, src, row, e, lane);
    for (int j = lane; j < p.K; j += 32) p.picked[row * p.K + j] = e.s[j];
  }
  float top = -INFINITY, sum = 0.f;
  constexpr int kUnroll = 4;
  for (int g0 = threadIdx.x; g0 < gr.count; g0 += kDsStatsThreads * kUnroll) {
    uint4 v[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      if (g0 + i * kDsStatsThreads < gr.count) v[i] = load_granule<T>(src, g0 + i * kDsStatsThreads, gr.lead, p.V);
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      if (g0 + i * kDsStatsThreads >= gr.count) continue;
      float f[n];
      Lane<T>::widen(v[i], f);
      float m = f[0];
#pragma unroll
      for (int j = 1; j < n; ++j) m = fmaxf(m, f[j]);
      m *= c;
      if (m > top) {
        sum *= ex2(top - m);
        top = m;
      }
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int j = 0; j < n; ++j) sum += ex2(fmaf(f[j], c, -base));
    }
  }
  block_merge<kDsStatsThreads>(top, sum, red);
  if (threadIdx.x == 0) p.stats[row] = make_float4(top, sum, e.tmax, e.tsum);
}

// Loss from the statistics of whole rows and the student's logits at the teacher's ids; one warp per row.
__global__ void __launch_bounds__(256)
distill_loss_kernel(const DistillParams p) {
  const int lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= p.T) return;
  const float c = p.inv_tau * kLog2e;
  const float4 st = p.stats[row];
  float l = 0.f;
  if (st.w != 0.f) {
    const float inv = __fdiv_rn(1.f, st.w), log_sum = log2f(st.y), log_tsum = log2f(st.w);
    for (int j = lane; j < p.K; j += 32) {
      const long long id = entry_id(p, row, j);
      if (id < 0 || id >= p.vocab_total) continue;
      const float t = p.teacher[row * p.ld_t + j];
      l += loss_term(entry_q(t, st.z, inv, c), t, p.picked[row * p.K + j], c, st, log_sum, log_tsum);
    }
  }
  l = warp_total(l) * kLn2;
  if (lane == 0) p.loss[row] = l;
}

// ------------------------------------------------------------------------------------------- gradient from statistics
// A CTA takes 256 * kGradVec granules of one row.
constexpr int kGradVec = 8;

template <typename T, typename TO>
__global__ void __launch_bounds__(kDsThreads)
distill_grad_kernel(const DistillParams p, int chunks) {
  constexpr int n = Lane<T>::n;
  __shared__ Entries e;
  const long long row = blockIdx.x / chunks;
  const int g0 = static_cast<int>(blockIdx.x % chunks) * (kDsThreads * kGradVec);
  const T* src = static_cast<const T*>(p.logits) + row * p.ld;
  TO* dst = static_cast<TO*>(p.grad) + row * p.ldg;
  const Granules<T> gr(src, p.V);
  const bool aligned = granules_aligned<TO, n>(dst, gr.lead);
  const float4 st = p.stats[row];
  const float w = p.weight != nullptr ? p.weight[row] : 1.f;
  const bool zero = st.w == 0.f || w == 0.f;
  const float c = p.inv_tau * kLog2e;
  uint4 v[kGradVec];
  if (!zero) {
#pragma unroll
    for (int i = 0; i < kGradVec; ++i) {
      const int g = g0 + i * kDsThreads + threadIdx.x;
      if (g < gr.count) v[i] = load_granule<T>(src, g, gr.lead, p.V);
    }
    // the entries that fall into this chunk, their logits read before they may be overwritten
    const long long first = static_cast<long long>(g0) * n - gr.lead, last = first + kDsThreads * kGradVec * n;
    const float inv = __fdiv_rn(1.f, st.w);
    for (int j = threadIdx.x; j < p.K; j += kDsThreads) {
      const long long id = entry_id(p, row, j), local = id - p.vocab_start;
      const bool here = id >= 0 && id < p.vocab_total && local >= 0 && local < p.V && local >= first && local < last;
      const float t = here ? p.teacher[row * p.ld_t + j] : -INFINITY;
      e.id[j] = t != -INFINITY ? static_cast<int>(local) : -1;
      e.q[j] = t != -INFINITY ? entry_q(t, st.z, inv, c) : 0.f;
      e.s[j] = t != -INFINITY ? Lane<T>::value(src + local) : 0.f;
    }
    __syncthreads();
  }
  const float g = w * p.inv_tau * __fdiv_rn(1.f, st.y);
#pragma unroll
  for (int i = 0; i < kGradVec; ++i) {
    const int k = g0 + i * kDsThreads + threadIdx.x;
    if (k >= gr.count) continue;
    float f[n];
    if (!zero) Lane<T>::widen(v[i], f);
#pragma unroll
    for (int j = 0; j < n; ++j) f[j] = zero ? 0.f : ex2(fmaf(f[j], c, -st.x)) * g;
    store_granule<TO, n>(dst, k, gr.lead, p.V, aligned, f);
  }
  if (zero) return;
  __syncthreads();
  write_entries<TO>(p, e, dst, st, w, [](int) { return true; });
}

// ------------------------------------------------------------------------------------------- launchers
template <typename T, typename TO, int C, int NV>
static cudaError_t launch_row(const DistillParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.T) * C);
  cfg.blockDim = dim3(kDsThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, distill_row_kernel<T, TO, C, NV>, p);
}
constexpr int kDsMostVec = 20;     // granules per thread with clusters of 8
constexpr int kDsGoodVec = 12;     // and with smaller ones, where a larger cluster is still to be had

template <typename T, typename TO, int C>
static cudaError_t launch_row_nv(const DistillParams& p, int nv, cudaStream_t stream) {
  if (nv <= 1) return launch_row<T, TO, C, 1>(p, stream);
  if (nv <= 2) return launch_row<T, TO, C, 2>(p, stream);
  if (nv <= 4) return launch_row<T, TO, C, 4>(p, stream);
  if (nv <= 8) return launch_row<T, TO, C, 8>(p, stream);
  if (nv <= 10) return launch_row<T, TO, C, 10>(p, stream);
  if constexpr (C < 8) {
    return launch_row<T, TO, C, kDsGoodVec>(p, stream);
  } else {
    if (nv <= kDsGoodVec) return launch_row<T, TO, C, kDsGoodVec>(p, stream);
    if (nv <= 16) return launch_row<T, TO, C, 16>(p, stream);
    return launch_row<T, TO, C, kDsMostVec>(p, stream);
  }
}

// Granules of a row whose start may lie anywhere in its first granule.
static long long max_granules(int V, int n) { return (static_cast<long long>(V) + 2 * (n - 1)) / n; }

// CTAs per row: the fewest that hold the row with at most 12 granules per thread, more (up to 8) while the rows alone
// do not fill the SMs.
static int row_cluster(int T, int V, int n) {
  const long long g = max_granules(V, n);
  int c = 1;
  while (c < 8 && g > static_cast<long long>(c) * kDsThreads * kDsGoodVec) c *= 2;
  while (c < 8 && static_cast<long long>(T) * c < sm_count() && g > static_cast<long long>(c) * kDsThreads) c *= 2;
  return c;
}

template <typename T, typename TO>
static cudaError_t run_row(const DistillParams& p, cudaStream_t stream) {
  const long long g = max_granules(p.V, Lane<T>::n);
  const int c = row_cluster(p.T, p.V, Lane<T>::n);
  const int nv = static_cast<int>((g + static_cast<long long>(c) * kDsThreads - 1) / (static_cast<long long>(c) * kDsThreads));
  switch (c) {
    case 1: return launch_row_nv<T, TO, 1>(p, nv, stream);
    case 2: return launch_row_nv<T, TO, 2>(p, nv, stream);
    case 4: return launch_row_nv<T, TO, 4>(p, nv, stream);
    default: return launch_row_nv<T, TO, 8>(p, nv, stream);
  }
}

}  // namespace stb

using namespace stb;

// Longest row that stb_distill_row takes, for 2- or 4-byte logits.
extern "C" int stb_distill_row_limit(int elem_bytes) {
  const int n = 16 / elem_bytes;
  return 8 * kDsThreads * kDsMostVec * n - 2 * (n - 1);
}

static bool distill_args_ok(const DistillParams& p) {
  return p.T > 0 && p.T <= 0x0FFFFFFF && p.V > 0 && p.K >= 0 && p.K <= kDsMaxEntries && p.inv_tau > 0.f;
}

// The gradient has the logits' type, or is bf16 for fp32 logits.
static bool distill_types_ok(int elem_bytes, int grad_bytes) {
  return (elem_bytes == 2 && grad_bytes == 2) || (elem_bytes == 4 && (grad_bytes == 4 || grad_bytes == 2));
}

// Loss, statistics and (grad != null) gradient of whole rows in one pass; grad may be the logits where the types are equal.
extern "C" int stb_distill_row(const void* logits, long long ld, void* grad, long long ldg, const void* ids, int ids64,
                               long long ld_ids, const float* teacher, long long ld_t, const float* weight, float* loss,
                               float* stats, int T, int V, int K, float inv_tau, int elem_bytes, int grad_bytes,
                               cudaStream_t stream) {
  if (T == 0) return 0;
  DistillParams p{};
  p.logits = logits; p.ld = ld; p.grad = grad; p.ldg = ldg; p.ids = ids; p.ids64 = ids64; p.ld_ids = ld_ids;
  p.teacher = teacher; p.ld_t = ld_t; p.weight = weight; p.loss = loss; p.stats = reinterpret_cast<float4*>(stats);
  p.T = T; p.V = V; p.K = K; p.vocab_start = 0; p.vocab_total = V; p.inv_tau = inv_tau;
  if (!distill_args_ok(p) || !distill_types_ok(elem_bytes, grad_bytes) || V > stb_distill_row_limit(elem_bytes))
    return -kErrBadArgument;
  cudaError_t e;
  if (elem_bytes == 2) e = run_row<__nv_bfloat16, __nv_bfloat16>(p, stream);
  else if (grad_bytes == 4) e = run_row<float, float>(p, stream);
  else e = run_row<float, __nv_bfloat16>(p, stream);
  return -static_cast<int>(e);
}

// Statistics [T][4] of the columns [vocab_start, vocab_start + V) and picked [T][K], the logits at the ids that fall there.
extern "C" int stb_distill_stats(const void* logits, long long ld, const void* ids, int ids64, long long ld_ids,
                                 const float* teacher, long long ld_t, float* stats, float* picked, int T, int V, int K,
                                 long long vocab_start, long long vocab_total, float inv_tau, int elem_bytes,
                                 cudaStream_t stream) {
  if (T == 0) return 0;
  DistillParams p{};
  p.logits = logits; p.ld = ld; p.ids = ids; p.ids64 = ids64; p.ld_ids = ld_ids; p.teacher = teacher; p.ld_t = ld_t;
  p.stats = reinterpret_cast<float4*>(stats); p.picked = picked; p.T = T; p.V = V; p.K = K;
  p.vocab_start = vocab_start; p.vocab_total = vocab_total; p.inv_tau = inv_tau;
  if (!distill_args_ok(p) || (elem_bytes != 2 && elem_bytes != 4)) return -kErrBadArgument;
  if (elem_bytes == 2) distill_stats_kernel<__nv_bfloat16><<<T, kDsStatsThreads, 0, stream>>>(p);
  else distill_stats_kernel<float><<<T, kDsStatsThreads, 0, stream>>>(p);
  return -static_cast<int>(cudaGetLastError());
}

// Loss [T] from the statistics of whole rows and the logits at all ids.
extern "C" int stb_distill_loss(const void* ids, int ids64, long long ld_ids, const float* teacher, long long ld_t,
                                const float* stats, const float* picked, float* loss, int T, int K, long long vocab_total,
                                float inv_tau, cudaStream_t stream) {
  if (T == 0) return 0;
  DistillParams p{};
  p.ids = ids; p.ids64 = ids64; p.ld_ids = ld_ids; p.teacher = teacher; p.ld_t = ld_t; p.loss = loss;
  p.stats = reinterpret_cast<float4*>(const_cast<float*>(stats)); p.picked = const_cast<float*>(picked);
  p.T = T; p.V = 1; p.K = K; p.vocab_total = vocab_total; p.inv_tau = inv_tau;
  if (!distill_args_ok(p)) return -kErrBadArgument;
  distill_loss_kernel<<<(T + 7) / 8, 256, 0, stream>>>(p);
  return -static_cast<int>(cudaGetLastError());
}

// Gradient of columns [vocab_start, vocab_start + V) from the statistics of whole rows; grad may be the logits.
extern "C" int stb_distill_grad(const void* logits, long long ld, void* grad, long long ldg, const void* ids, int ids64,
                                long long ld_ids, const float* teacher, long long ld_t, const float* weight,
                                const float* stats, int T, int V, int K, long long vocab_start, long long vocab_total,
                                float inv_tau, int elem_bytes, int grad_bytes, cudaStream_t stream) {
  if (T == 0) return 0;
  DistillParams p{};
  p.logits = logits; p.ld = ld; p.grad = grad; p.ldg = ldg; p.ids = ids; p.ids64 = ids64; p.ld_ids = ld_ids;
  p.teacher = teacher; p.ld_t = ld_t; p.weight = weight; p.stats = reinterpret_cast<float4*>(const_cast<float*>(stats));
  p.T = T; p.V = V; p.K = K; p.vocab_start = vocab_start; p.vocab_total = vocab_total; p.inv_tau = inv_tau;
  if (!distill_args_ok(p) || grad == nullptr || !distill_types_ok(elem_bytes, grad_bytes)) return -kErrBadArgument;
  const int n = 16 / elem_bytes;
  const long long chunks = (max_granules(V, n) + kDsThreads * kGradVec - 1) / (kDsThreads * kGradVec);
  if (chunks * T > 0x7FFFFFFFll) return -kErrBadArgument;
  const unsigned grid = static_cast<unsigned>(chunks * T);
  const int ch = static_cast<int>(chunks);
  if (elem_bytes == 2) distill_grad_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, kDsThreads, 0, stream>>>(p, ch);
  else if (grad_bytes == 4) distill_grad_kernel<float, float><<<grid, kDsThreads, 0, stream>>>(p, ch);
  else distill_grad_kernel<float, __nv_bfloat16><<<grid, kDsThreads, 0, stream>>>(p, ch);
  return -static_cast<int>(cudaGetLastError());
}
