// Distillation from a teacher's top logits.  Per row of student logits s [V] and teacher entries (id_j, t_j), j < K:
//
//     q = softmax_j(t / tau)         p = softmax_v(s / tau)         L = sum_j q_j (log q_j - log p[id_j])
//     dL/ds_v = (p_v - sum_{j: id_j = v} q_j) / tau
//
// An entry with t = -inf is no entry, nor is one whose id lies outside the vocabulary; a row without entries has L = 0
// and a zero gradient whatever its logits hold, and so has a row of weight 0.  The same id may come several times.
//
// Three kernels:
//   distill_row_kernel    a row on a thread-block cluster, its logits in shared memory as far as they fit and for the
//                         rest once more from L2: one read of the logits from DRAM gives the loss, the statistics and
//                         (optionally) the gradient, which may overwrite the logits
//   distill_stats_kernel  a row of any length, or the local part of a vocabulary that is sharded over ranks:
//                         max, sum of exponentials and the student's logits at the teacher's ids
//   distill_grad_kernel   the gradient from finished statistics (backward pass of few rows; sharded or very long rows)
//
// Statistics of a row: {top, sum, max t, sum of exp((t - max t) / tau)}.  With c = log2(e) / tau, `top` is the rounded
// c * max s and `sum` that of 2^(c s - top), so that c * max s is rounded once and cancels; the last number is 0 for a
// row without entries.  All sums are fp32; the logits' gradient is rounded once.
//
// Large rows.  The rounding of c * max s cancels as long as 2 to its power is in range, and c * s may leave the range
// altogether (a row masked with the type's lowest value).  From |c max s| = 2^31 on neighbouring numbers of that size are
// 128 apart in the exponent, so that p is the same for all elements that equal the maximum and 0 elsewhere: the exponent
// is then taken with a power of two instead of c, for which products and differences are exact.  In the statistics such a
// row, and wherever sums are joined such a part of one, has {max s, -(number of elements that equal it)}.
//
// Memory bound: the logits are read once and the gradient written once; two exponentials per element.
#include "common.cuh"

#include <atomic>

namespace stb {

constexpr int kDsThreads = 256;              // gradient kernel
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
  const float4* given;          // row kernel: finished statistics, only the gradient is wanted
  float* picked;                // stats kernel: [T][K] student logit at each id, 0 where it is not in this shard
  long long ld, ldg, ld_ids, ld_t;
  long long vocab_start, vocab_total;
  int V, K, T;
  int ids64;
  float inv_tau;
  int* status;                  // row kernel: error word of its bounded waits
};

// 2 units in the last place, results below 2^-126 as 0: p is off by 1e-7 of itself, and what is flushed lies 2^-126 below a
// row's largest probability.  Tenfold instructions for the last bit would make bf16 rows wait for arithmetic.
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

// The exponents of a row: fma(s, c, -top).  `sum` is negative for a large row or part of one, whose `top` is its maximum m:
// the power of two takes m to [2^31, 2^32) (m is above 2^31 / c > 2^10, so that it is a normal number).
constexpr float kLarge = 2147483648.f;
struct Exponent { float c, top; };
__device__ __forceinline__ Exponent exponent_of(float top, float& sum, float c) {
  if (!(sum < 0.f)) return {c, top};
  sum = -sum;
  const float pw = __uint_as_float((285u - ((__float_as_uint(top) >> 23) & 255u)) << 23);
  return {pw, top * pw};
}
// log2 of 2^(c (s - max)), times 2^-32, so that no finite logit leaves the range.
constexpr float kDown = 1.f / 4294967296.f;
__device__ __forceinline__ float log_weight(float s, float c, const Exponent& e) {
  if (e.c == c) return fmaf(s * kDown, c, -e.top * kDown);
  return (s * kDown - e.top * __frcp_rn(e.c) * kDown) * c;
}

// (top, sum) of a thread's logits whose largest scaled one is outside (-2^31, 2^31), from another look at them.
template <typename T>
struct LargePart {
  float m = -INFINITY, equal = 0.f;
  bool bad = false;
  __device__ __forceinline__ void add(float x) {
    bad |= x != x;
    if (x > m) { m = x; equal = 0.f; }
    if (x == m) equal += 1.f;
  }
  __device__ __forceinline__ void add(const uint4& u) {
    float f[Lane<T>::n];
    Lane<T>::widen(u, f);
#pragma unroll
    for (int j = 0; j < Lane<T>::n; ++j) add(f[j]);
  }
  __device__ __forceinline__ void result(float& top, float& sum) const {
    top = m;                                       // infinite logits are not scaled
    sum = bad || m == INFINITY ? __uint_as_float(0x7FC00000u) : m == -INFINITY ? 0.f : -equal;
  }
};

// Large parts beside others.  `keys`: c * max (infinite for a large part) and a large part's maximum; their maxima over the
// parts say what the whole is and what each part adds to it.
__device__ __forceinline__ float2 large_keys(float m, float s) {
  return s < 0.f ? make_float2(copysignf(INFINITY, m), m) : make_float2(m, -INFINITY);
}
__device__ __forceinline__ bool large_whole(float2 keys) { return isinf(keys.x) && keys.y > -INFINITY; }
__device__ __forceinline__ float large_part(float m, float s, float2 keys) {
  if (s != s) return s;                            // a NaN stays visible
  if (large_whole(keys)) return s < 0.f && m == keys.y ? -s : 0.f;
  return s < 0.f || m == -INFINITY ? fmaxf(s, 0.f) : s * ex2(m - keys.x);
}

// (m, s) <- the pair that stands for both, s being relative to exp2(m).  -inf: nothing seen yet.
__device__ __forceinline__ void merge(float& m, float& s, float om, float os) {
  if (s < 0.f || os < 0.f) {
    const float2 a = large_keys(m, s), b = large_keys(om, os), keys = make_float2(fmaxf(a.x, b.x), fmaxf(a.y, b.y));
    s = large_part(m, s, keys) + large_part(om, os, keys);
    m = large_whole(keys) ? keys.y : keys.x;
    if (large_whole(keys)) s = -s;
    return;
  }
  const float top = fmaxf(m, om);
  const float a = m == top ? s : s * ex2(m - top);
  const float b = om == top ? os : os * ex2(om - top);
  m = top;
  s = a + b;
}

// The same over the lanes of a warp: the largest top first, then one scaling and a plain sum.
__device__ __forceinline__ float warp_top(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ void warp_merge(float& m, float& s) {
  float top;
  const bool large = __any_sync(0xffffffffu, s < 0.f);
  bool whole = false;
  if (large) {
    float2 keys = large_keys(m, s);
    keys = make_float2(warp_top(keys.x), warp_top(keys.y));
    whole = large_whole(keys);
    s = large_part(m, s, keys);
    top = whole ? keys.y : keys.x;
  } else {
    top = warp_top(m);
    if (m != top) s *= ex2(m - top);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  m = top;
  if (whole) s = -s;
}

// Teacher entries of a chunk of a row in shared memory (gradient kernel).
struct Entries {
  float q[kDsMaxEntries];      // probability, 0 where there is no entry
  float s[kDsMaxEntries];      // the student's logit there (0 where the id is not in this chunk)
  int id[kDsMaxEntries];       // local id, -1 where there is no entry in this chunk
};
// Teacher statistics of a row (statistics kernel).
struct TeacherRow {
  float t[kDsMaxEntries];
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

// By one warp: the row's teacher statistics, and the student's logits at the ids that fall into this shard (0 at others).
template <typename T>
__device__ __forceinline__ void load_teacher(const DistillParams& p, const T* row_ptr, long long row, TeacherRow& e, int lane) {
  const float c = p.inv_tau * kLog2e;
  float tmax = -INFINITY;
  bool bad = false;            // fmaxf drops a NaN; it has to reach the loss
  for (int j = lane; j < p.K; j += 32) {
    const long long id = entry_id(p, row, j);
    const bool in = id >= 0 && id < p.vocab_total;
    const float t = in ? p.teacher[row * p.ld_t + j] : -INFINITY;
    const long long local = id - p.vocab_start;
    const bool here = in && t != -INFINITY && local >= 0 && local < p.V;
    e.t[j] = t;
    p.picked[row * p.K + j] = here ? Lane<T>::value(row_ptr + local) : 0.f;
    tmax = fmaxf(tmax, t);
    bad |= t != t;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) tmax = fmaxf(tmax, __shfl_xor_sync(0xffffffffu, tmax, o));
  if (__any_sync(0xffffffffu, bad)) tmax = __uint_as_float(0x7FC00000u);
  float tsum = 0.f;
  if (tmax != -INFINITY) {
    for (int j = lane; j < p.K; j += 32) tsum += ex2((e.t[j] - tmax) * c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) tsum += __shfl_xor_sync(0xffffffffu, tsum, o);
  }
  if (lane == 0) { e.tmax = tmax; e.tsum = tsum; }
}

// One term q (log2 q - log2 p) of the loss, times 2^-32, the difference of logarithms taken before the sum over the
// entries, so that a small divergence is not the difference of two large sums.
__device__ __forceinline__ float loss_term(float q, float log_q, float s, float c, const Exponent& e, float log_sum) {
  return q == 0.f ? 0.f : q * (log_q * kDown - (log_weight(s, c, e) - log_sum * kDown));
}
__device__ __forceinline__ float warp_total(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Gradient at the entries: written once more over the dense p, from the logit kept in shared memory, with the q of equal
// ids added in order.  The caller has a barrier between the dense writes and this.
template <typename TO>
__device__ __forceinline__ void write_entries(const DistillParams& p, const Entries& e, TO* grad_row, const Exponent& ex,
                                              float sum, float w) {
  const float g = w * p.inv_tau, inv = __fdiv_rn(1.f, sum);
  for (int j = threadIdx.x; j < p.K; j += blockDim.x) {
    const int id = e.id[j];
    if (id < 0) continue;
    bool first = true;
    float q = 0.f;
    for (int i = 0; i < p.K; ++i) {
      if (e.id[i] != id) continue;
      if (i < j) { first = false; break; }
      q += e.q[i];
    }
    if (first) Lane<TO>::store(grad_row + id, (ex2(fmaf(e.s[j], ex.c, -ex.top)) * inv - q) * g);
  }
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
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

// ------------------------------------------------------------------------------------------- whole rows, one pass
// One cluster of C CTAs is launched per row; a running cluster takes over the rows of clusters that have not started
// (clusterlaunchcontrol), so that its set-up is paid once and a cluster on less busy SMs does more rows (with fixed rows
// the first clusters were done after 385 us of 495).  Each CTA has a contiguous slice of the row's granules and makes two
// passes over it:
//
//   producer warp   bulk copies of 16 KB chunks into a ring that runs on from row to row.  The last chunks of a slice, as
//                   many as the ring holds, stay there for pass 2, which begins with them; the others are loaded again,
//                   from L2, where the first load asked for them to be kept
//   entries warps   two, for even and odd rows: the teacher's entries of a coming row, their statistics and the list of
//                   those that fall into this CTA's slice; behind pass 2 the loss and the gradient at the entries
//   compute warps   pass 1: (top, sum) of the slice.  Every warp sends its pair to all CTAs of the cluster (st.async onto
//                   their mbarriers) and merges all pairs when they are there.  Pass 2: the gradient, straight to global
//                   memory
//
// Loads, entries and the cluster's exchange thus run beside the arithmetic; nothing waits for the whole CTA.
//
// Without a gradient there is no pass 2, with given statistics no pass 1 and no exchange: a chunk is then released as soon
// as it has been read, and with enough rows one CTA takes a whole one (4096 x 151936 bf16: 198 us and 399 us, 6.3 and 6.2
// TB/s of 6.55 measured).
//
// Bound: DRAM for fp32 logits (2048 x 151936: 390 us, 6.4 TB/s).  For bf16 the exponentials (two per element, 16 a cycle
// and SM: 277 us of 4096 x 151936) and the issue slots are busy for 60 % of the time beside it: 457 us, 5.5 TB/s.  What a row
// costs a warp whatever its length (set-up, merging, exchange: half of the instructions with slices of 76 KB) asks for
// long slices; measured, same size, 1, 2, 4, 8 CTAs per row: 468, 457, 488, 699 us (fp32: 551, 456, 391, 409).  Loading
// nothing again (slices of 76 KB, all kept): 488.  4, 6, 10, 12 compute warps (at their best slice): 554, 588, 476, 458.
// Every fourth exponential by a polynomial instead of the special-function unit: 522 against 524 at the time.
constexpr int kU = 4;                            // granules per compute thread and chunk
constexpr int kRowWarps = 8;                     // compute warps
constexpr int kRowCompute = 32 * kRowWarps;
constexpr int kRowThreads = kRowCompute + 96;
constexpr int kChunk = kRowCompute * kU;         // granules: 16 KB
constexpr int kMaxChunks = 12;

struct RowPlan {
  int per;             // granules per CTA
  int chunks;          // per slice
  int ring;            // chunks in shared memory: two at least, and often fewer than a slice has
  int keep;            // last chunks of a slice that stay in the ring between the two passes; the others are loaded again
  int kpad;            // K rounded up to 4
};
struct RowBars {
  uint64_t full[kMaxChunks], empty[kMaxChunks];
  uint64_t e_full[2], e_empty[2];   // entries prepared; pass 2 of their row done
  uint64_t xchg[2];                 // the cluster's pairs
  uint64_t claim[4];                // answers to the requests for further rows
};
// Entries of a row, arrays of kpad: for the loss q, log2 q, s; of this CTA's slice q, s, the q of the gradient (summed
// over equal ids, -1: another entry carries it), id.
struct EntryHead {
  float tmax, tsum, weight;
  float top, sum;      // of the row, from the compute warps
};

__host__ __device__ constexpr int entry_bytes(int kpad) { return kpad * 28; }
// bitmap of a slice's elements: one bit each
__host__ __device__ constexpr int bitmap_bytes(int per, int n) { return ((per * n + 31) / 32 * 4 + 15) / 16 * 16; }

__device__ __forceinline__ void send_pair(float2* slot, uint64_t* bar, uint32_t rank, float a, float b) {
  uint32_t dst, rbar;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(dst) : "r"(smem_u32(slot)), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(rbar) : "r"(smem_u32(bar)), "r"(rank));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];"
               ::"r"(dst), "f"(a), "f"(b), "r"(rbar) : "memory");
}
// `how`: 0 as usual, 1 keep in L2 (it is read again soon), 2 drop from L2 (it was the last time)
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar, int how) {
  if (how == 0) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
    return;
  }
  uint64_t policy;
  if (how == 1) asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(policy));
  else asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy) : "memory");
}
__device__ __forceinline__ uint64_t ex2_2(uint64_t x) {
  float a, b;
  unpair(x, a, b);
  return pair(ex2(a), ex2(b));
}

// A granule as pairs, its largest value, and pairs back to an output granule.
template <typename T> struct Pairs;
template <> struct Pairs<__nv_bfloat16> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void widen(const uint4& u, uint64_t (&f)[4]) {
    f[0] = pair(bf16_lo(u.x), bf16_hi(u.x));
    f[1] = pair(bf16_lo(u.y), bf16_hi(u.y));
    f[2] = pair(bf16_lo(u.z), bf16_hi(u.z));
    f[3] = pair(bf16_lo(u.w), bf16_hi(u.w));
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t m;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
    return m;
  }
  static __device__ __forceinline__ float top(const uint4 (&v)[kU]) {      // a NaN is passed over; the sum shows it
    uint32_t m = max2(max2(v[0].x, v[0].y), max2(v[0].z, v[0].w));
#pragma unroll
    for (int u = 1; u < kU; ++u) m = max2(m, max2(max2(v[u].x, v[u].y), max2(v[u].z, v[u].w)));
    return fmaxf(bf16_lo(m), bf16_hi(m));
  }
};
template <> struct Pairs<float> {
  static constexpr int n = 2;
  static __device__ __forceinline__ void widen(const uint4& u, uint64_t (&f)[2]) {
    f[0] = pair(__uint_as_float(u.x), __uint_as_float(u.y));
    f[1] = pair(__uint_as_float(u.z), __uint_as_float(u.w));
  }
  static __device__ __forceinline__ float top(const uint4 (&v)[kU]) {
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < kU; ++u)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(v[u].x), __uint_as_float(v[u].y)),
                         fmaxf(__uint_as_float(v[u].z), __uint_as_float(v[u].w))));
    return m;
  }
};
template <typename TO, int NP>
__device__ __forceinline__ void store_pairs(TO* at, bool aligned, const uint64_t (&f)[NP]) {
  float v[2 * NP];
#pragma unroll
  for (int j = 0; j < NP; ++j) unpair(f[j], v[2 * j], v[2 * j + 1]);
  if (aligned) {
    if constexpr (sizeof(TO) == 4) {
      __stcs(reinterpret_cast<float4*>(at), make_float4(v[0], v[1], v[2], v[3]));
    } else if constexpr (NP == 4) {
      __stcs(reinterpret_cast<uint4*>(at), make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]),
                                                 pack_bf16(v[6], v[7])));
    } else {
      __stcs(reinterpret_cast<uint2*>(at), make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 2 * NP; ++j) Lane<TO>::store(at + j, v[j]);
  }
}

// Bounded waits of this kernel.  `soon`: due within a microsecond, polled without looking at the clock first, whose
// reading alone takes that long.  `idle`: the warps that run ahead sleep between polls; polling without a pause took
// a third of the issue slots from the compute warps.
__device__ __forceinline__ bool mbar_wait_soon(uint64_t* bar, uint32_t phase) {
  for (int i = 0; i < 1024; ++i)
    if (mbar_try_wait(bar, phase)) return true;
  return mbar_wait(bar, phase);
}
// The cluster's pairs: with them the other CTAs say that they have read the logits that this one may overwrite.
__device__ __forceinline__ bool mbar_wait_pairs(uint64_t* bar, uint32_t phase) {
  for (int i = 0; i < 1024; ++i)
    if (mbar_try_wait_cluster(bar, phase)) return true;
  return mbar_wait_cluster(bar, phase);
}
__device__ __forceinline__ bool mbar_wait_idle(uint64_t* bar, uint32_t phase, unsigned ns) {
  if (mbar_try_wait(bar, phase)) return true;
  const uint64_t t0 = global_timer_ns();
  for (uint32_t i = 1; i < kSpinLimit; ++i) {
    __nanosleep(ns);
    if (mbar_try_wait(bar, phase)) return true;
    if ((i & 255u) == 0 && global_timer_ns() - t0 > kWaitBudgetNs) return false;
  }
  return false;
}

// Request for the row of a cluster that has not started; the answer goes to every CTA of this cluster.
template <int C>
__device__ __forceinline__ void request_row(uint4* answer, uint64_t* bar) {
  if constexpr (C > 1)
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.multicast::cluster::all.b128 [%0], [%1];"
                 ::"r"(smem_u32(answer)), "r"(smem_u32(bar)) : "memory");
  else
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                 ::"r"(smem_u32(answer)), "r"(smem_u32(bar)) : "memory");
}
// First CTA of the cluster whose launch was cancelled, or -1: there was none left.
__device__ __forceinline__ int granted_cta(const uint4* answer) {
  uint32_t got, x;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
      : "=&r"(got), "=&r"(x) : "r"(smem_u32(answer)) : "memory");     // written before the address is read
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // read before the next answer may land here
  return got ? static_cast<int>(x) : -1;
}

// Where the granules of this CTA's slice of a row are: [gs, ge) are whole; the row's elements before its first and behind
// its last whole granule (fewer than n each) are `edge` elements, one for a thread of its own each.
template <typename T>
struct Slice {
  int g0, gs, ge, whole;
  __device__ __forceinline__ Slice(const Granules<T>& gr, int rank, int per, int V) {
    g0 = rank * per;
    whole = (gr.lead + V) / Lane<T>::n;
    gs = max(g0, gr.lead > 0 ? 1 : 0);
    ge = min(g0 + per, whole);
  }
  __device__ __forceinline__ int edge(const Granules<T>& gr, int rank, int per, int V, int thread) const {
    constexpr int n = Lane<T>::n;
    if (thread < 8) return rank == 0 && gr.lead > 0 && thread < min(n - gr.lead, V) ? thread : -1;
    if (thread >= 16) return -1;
    const int at = whole * n - gr.lead + thread - 8;
    return whole >= g0 && whole < g0 + per && (whole > 0 || gr.lead == 0) && at < V ? at : -1;
  }
};

template <typename T, typename TO, int C>
__global__ void __launch_bounds__(kRowThreads, 2)
distill_row_kernel(const DistillParams p, const RowPlan plan) {
  constexpr int n = Lane<T>::n;
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ RowBars bars;
  __shared__ float2 part[2][C * kRowWarps];
  __shared__ EntryHead head[2];
  __shared__ __align__(16) uint4 answer[4];
  __shared__ volatile int failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = C > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int first_row = blockIdx.x / C;
  uint8_t* entry_base = dyn + plan.ring * kChunk * 16;
  const float c = p.inv_tau * kLog2e;
  const bool both = p.grad != nullptr && p.given == nullptr;       // passes

  if (threadIdx.x == 0) {
    for (int i = 0; i < plan.ring; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], kRowWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.e_full[i], 1);
      mbar_init(&bars.e_empty[i], kRowWarps);
      mbar_init(&bars.xchg[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&bars.claim[i], 1);
    failed = 0;
    fence_barrier_init();
  }
  if (p.grad != nullptr) {
    uint32_t* bitmaps = reinterpret_cast<uint32_t*>(entry_base + 2 * entry_bytes(plan.kpad));
    for (int i = threadIdx.x; i < 2 * bitmap_bytes(plan.per, n) / 4; i += kRowThreads) bitmaps[i] = 0;
  }
  __syncthreads();
  if constexpr (C > 1) {                   // the other CTAs' barriers are initialised, too
    cluster_arrive();
    cluster_wait();
  }

  // The rows of this cluster: number 0 is its own; number i > 0 is requested after the exchange of row i - 2 (with given
  // statistics, and one CTA: when the entries of that row are prepared, which follows the end of row i - 4), when every
  // warp of every CTA has read the answers up to i - 4 at least, of which four are kept: number i in place (i - 1) % 4,
  // the (i - 1) / 4-th answer there.  No request follows a refused one.
  auto request = [&](int i) {              // by one thread of each CTA
    const int at = (i - 1) & 3;
    mbar_arrive_expect_tx(&bars.claim[at], 16);
    if (rank == 0) request_row<C>(&answer[at], &bars.claim[at]);
  };
  auto answered = [&](int i) { return mbar_wait_soon(&bars.claim[(i - 1) & 3], ((i - 1) >> 2) & 1); };
  auto granted = [&](int i) { return granted_cta(&answer[(i - 1) & 3]); };
  auto next_row = [&](int i, long long& row) {     // by whole warps; every role asks for every number
    const bool ok = warp < kRowWarps ? answered(i) : mbar_wait_idle(&bars.claim[(i - 1) & 3], ((i - 1) >> 2) & 1, 100);
    if (!__all_sync(0xffffffffu, ok)) {
      report_error(p.status, kErrProducerWait);
      failed = 1;
      return false;
    }
    const int cta = granted(i);
    row = cta / C;
    return cta >= 0 && row < p.T;
  };
  if (threadIdx.x == 0) request(1);

  if (warp == kRowWarps) {
    // ---------------------------------------------------------------- producer
    int slot = 0;
    uint32_t lap = 0;                      // parity of the ring's passes
    bool ok = true, more = true;
    long long row = first_row;
    for (int number = 1; ok && more; more = ok && next_row(number++, row)) {
      const T* src = static_cast<const T*>(p.logits) + row * p.ld;
      const Granules<T> gr(src, p.V);
      const Slice<T> sl(gr, rank, plan.per, p.V);
      const int again = both ? plan.chunks - plan.keep : 0;
      for (int i = 0; i < plan.chunks + again; ++i) {
        const int k = i < plan.chunks ? i : i - plan.chunks;
        ok = __all_sync(0xffffffffu, !failed && mbar_wait_idle(&bars.empty[slot], lap ^ 1, 100));
        if (!ok) { report_error(p.status, kErrProducerWait); failed = 1; break; }
        if (lane == 0) {
          const int k0 = sl.g0 + k * kChunk, a = max(k0, sl.gs), b = min(k0 + kChunk, sl.ge);
          if (b > a) {
            const uint32_t bytes = static_cast<uint32_t>(b - a) * 16;
            mbar_arrive_expect_tx(&bars.full[slot], bytes);
            bulk_load(dyn + (slot * kChunk + a - k0) * 16, src + (static_cast<long long>(a) * n - gr.lead), bytes,
                      &bars.full[slot], i < again ? 1 : again > 0 ? 2 : 0);
          } else {
            mbar_arrive(&bars.full[slot]);
          }
        }
        if (++slot == plan.ring) { slot = 0; lap ^= 1; }
      }
    }
  } else if (warp > kRowWarps) {
    // ---------------------------------------------------------------- entries of every second row
    const int b = warp - kRowWarps - 1;
    float* eq = reinterpret_cast<float*>(entry_base + b * entry_bytes(plan.kpad));
    float *elq = eq + plan.kpad, *es = elq + plan.kpad, *oq = es + plan.kpad, *os = oq + plan.kpad, *gq = os + plan.kpad;
    int* oid = reinterpret_cast<int*>(gq + plan.kpad);
    uint32_t* bitmap = reinterpret_cast<uint32_t*>(entry_base + 2 * entry_bytes(plan.kpad) + b * bitmap_bytes(plan.per, n));
    EntryHead& hd = head[b];
    uint32_t phase = 0;
    long long row = first_row;
    bool more = true;
    for (int number = 0; more; more = next_row(++number, row)) {
      if ((number & 1) != b) continue;
      const T* src = static_cast<const T*>(p.logits) + row * p.ld;
      const Granules<T> gr(src, p.V);
      const int e0 = rank * plan.per * n - gr.lead, e1 = e0 + plan.per * n;
      const float w = p.weight != nullptr ? p.weight[row] : 1.f;
      const float4 given = p.given != nullptr ? p.given[row] : make_float4(0.f, 0.f, 0.f, 0.f);
      float tmax = -INFINITY;
      bool bad = false;                    // fmaxf drops a NaN; it has to reach the loss
      int own = 0;
      for (int j0 = 0; j0 < p.K; j0 += 64) {
        long long id[2];
        float t[2], sv[2];
        bool here[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int j = j0 + 32 * u + lane;
          id[u] = j < p.K ? entry_id(p, row, j) : -1;
          t[u] = j < p.K ? p.teacher[row * p.ld_t + j] : -INFINITY;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const bool in = id[u] >= 0 && id[u] < p.V && t[u] != -INFINITY;
          if (!in) t[u] = -INFINITY;
          here[u] = in && id[u] >= e0 && id[u] < e1;
          sv[u] = in && (here[u] || rank == 0) ? Lane<T>::value(src + id[u]) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int j = j0 + 32 * u + lane;
          if (j < p.K) { elq[j] = t[u]; es[j] = sv[u]; }
          tmax = fmaxf(tmax, t[u]);
          bad |= t[u] != t[u];
          const uint32_t votes = __ballot_sync(0xffffffffu, here[u]);
          if (here[u]) {
            const int at = own + __popc(votes & ((1u << lane) - 1));
            oid[at] = static_cast<int>(id[u]);
            oq[at] = t[u];
            os[at] = sv[u];
          }
          own += __popc(votes);
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) tmax = fmaxf(tmax, __shfl_xor_sync(0xffffffffu, tmax, o));
      if (__any_sync(0xffffffffu, bad)) tmax = __uint_as_float(0x7FC00000u);
      const bool some = tmax != -INFINITY;
      float tsum = 0.f;
      if (p.given != nullptr) {
        tmax = given.z;
        tsum = given.w;
      } else {
        for (int j = lane; j < p.K; j += 32) {
          const float e = some ? ex2((elq[j] - tmax) * c) : 0.f;
          eq[j] = e;
          tsum += e;
        }
        tsum = warp_total(tsum);
      }
      // what the compute warps need, and the word that the logits at the entries have been read
      if (lane == 0) {
        hd.tmax = tmax;
        hd.tsum = tsum;
        hd.weight = w;
        if (p.given != nullptr) {
          hd.top = given.x;
          hd.sum = given.y;
        }
      }
      mbar_arrive_warp(&bars.e_full[b]);
      const float inv = some ? __fdiv_rn(1.f, tsum) : 0.f;
      if (p.loss != nullptr) {
        const float log_tsum = some ? log2f(tsum) : 0.f;
        for (int j = lane; j < p.K; j += 32) {
          eq[j] *= inv;
          elq[j] = (elq[j] - tmax) * c - log_tsum;
        }
      }
      if (p.grad == nullptr) own = 0;
      // the same id twice?  One bit per element of the slice tells, and only then are the equal ids looked for
      bool twice = false;
      for (int j = lane; j < own; j += 32) {
        const float q = entry_q(oq[j], tmax, inv, c);
        oq[j] = gq[j] = q;
        const int at = oid[j] - e0;
        twice |= (atomicOr(&bitmap[at >> 5], 1u << (at & 31)) >> (at & 31)) & 1u;
      }
      __syncwarp();
      for (int j = lane; j < own; j += 32) bitmap[(oid[j] - e0) >> 5] = 0;
      if (__any_sync(0xffffffffu, twice)) {
        // the first of equal ids takes the sum, in their order; the others are left out
        for (int j = lane; j < own; j += 32) {
          float q = 0.f;
          bool lead = true;
          for (int i = 0; i < own; ++i) {
            if (oid[i] != oid[j]) continue;
            lead = lead && i >= j;
            q += oq[i];
          }
          gq[j] = lead ? q : -1.f;
        }
      }
      // pass 2 has written the dense gradient: the loss, and the gradient at the entries over it
      bool ok = !failed && mbar_wait_idle(&bars.e_empty[b], phase, 300);
      if (!__all_sync(0xffffffffu, ok)) {
        report_error(p.status, kErrCorrectionWait);
        failed = 1;
        break;
      }
      float sum = hd.sum;
      const Exponent ex = exponent_of(hd.top, sum, c);
      if (rank == 0) {
        if (p.loss != nullptr) {
          const float log_sum = log2f(sum);
          float l = 0.f;
          for (int j = lane; j < p.K; j += 32)
            l += loss_term(eq[j], elq[j], es[j], c, ex, log_sum);
          l = warp_total(l) * kLn2;
          if (lane == 0) p.loss[row] = l / kDown;
        }
        if (p.stats != nullptr && lane == 0) p.stats[row] = make_float4(hd.top, hd.sum, tmax, tsum);
      }
      if (p.grad != nullptr && w != 0.f) {
        TO* dst = static_cast<TO*>(p.grad) + row * p.ldg;
        const float rs = __fdiv_rn(1.f, sum), gw = w * p.inv_tau;
        for (int j = lane; j < own; j += 32)
          if (!(gq[j] < 0.f)) Lane<TO>::store(dst + oid[j], (ex2(fmaf(os[j], ex.c, -ex.top)) * rs - gq[j]) * gw);
      }
      __syncwarp();
      phase ^= 1;
    }
  } else {
    // ---------------------------------------------------------------- compute
    constexpr int kP = Pairs<T>::n;
    constexpr uint32_t kNone = sizeof(T) == 2 ? 0xFF80FF80u : 0xFF800000u;    // -inf
    const uint64_t c2 = pair(c, c);
    // Chunks are awaited in the order of their loads, at ring position `slot` in its `lap`-th round, and released in the
    // same order: what stays between the passes is released by pass 2, which goes to it first, at position `slot2`.
    const int through = both ? plan.chunks - plan.keep : plan.chunks;
    int it = 0, slot = 0;
    uint32_t lap = 0;
    auto arrived = [&] { return __all_sync(0xffffffffu, mbar_wait_soon(&bars.full[slot], lap)); };
    auto advance = [&] {
      if (++slot == plan.ring) { slot = 0; lap ^= 1; }
    };
    long long row = first_row;
    for (bool more = true; more; more = next_row(++it, row)) {
      const int b = it & 1;
      const uint32_t phase = (it >> 1) & 1;
      const T* src = static_cast<const T*>(p.logits) + row * p.ld;
      const Granules<T> gr(src, p.V);
      const Slice<T> sl(gr, rank, plan.per, p.V);
      const int edge = sl.edge(gr, rank, plan.per, p.V, threadIdx.x);
      const float x_edge = edge >= 0 ? Lane<T>::value(src + edge) : -INFINITY;
      bool ok = true;
      // pass 1: a thread that has seen nothing but -inf adds exp2(-inf) = 0
      float top = -INFINITY;
      uint64_t acc[2] = {0, 0};                       // two pairs of sums
      auto leave = [&] {                              // by the whole warp, when a wait has run out
        report_error(p.status, kErrEpilogueWait);
        failed = 1;
      };
      auto raise = [&](float m) {
        if (m > top) {
          const float scale = ex2(top - m);
          acc[0] = mul2(acc[0], pair(scale, scale));
          acc[1] = mul2(acc[1], pair(scale, scale));
          top = m;
        }
        return top == -INFINITY ? 0.f : -top;
      };
      auto take = [&](const uint4 (&v)[kU]) {
        const float base = raise(Pairs<T>::top(v) * c);
        const uint64_t minus = pair(base, base);
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          uint64_t f[kP];
          Pairs<T>::widen(v[u], f);
#pragma unroll
          for (int j = 0; j < kP; ++j) acc[j & 1] = add2(acc[j & 1], ex2_2(fma2(f[j], c2, minus)));
        }
      };
      float sum = 0.f;
      if (p.given != nullptr) {
        ok = __all_sync(0xffffffffu, mbar_wait_soon(&bars.e_full[b], phase));
        if (!ok) { leave(); break; }
        top = head[b].top;
        sum = head[b].sum;
      } else {
        for (int k = 0; k < plan.chunks; ++k) {
          const int k0 = sl.g0 + k * kChunk;
          ok = arrived();
          if (!ok) break;
          const uint4* chunk = reinterpret_cast<const uint4*>(dyn) + slot * kChunk;
          const int lo = sl.gs - k0, hi = min(sl.ge - k0, kChunk);
          const int g = threadIdx.x;
          uint4 v[kU];
          if (lo <= 0 && hi == kChunk) {
#pragma unroll
            for (int u = 0; u < kU; ++u) v[u] = chunk[g + u * kRowCompute];
            take(v);
          } else if (g < hi) {
#pragma unroll
            for (int u = 0; u < kU; ++u) {
              const int i = g + u * kRowCompute;
              v[u] = i >= lo && i < hi ? chunk[i] : make_uint4(kNone, kNone, kNone, kNone);
            }
            take(v);
          }
          if (k < through) mbar_arrive_warp(&bars.empty[slot]);
          advance();
        }
        if (edge >= 0) {
          const float base = raise(x_edge * c);
          acc[0] = add2(acc[0], pair(ex2(fmaf(x_edge, c, base)), 0.f));
        }
        float sum1;
        unpair(add2(acc[0], acc[1]), sum, sum1);
        sum += sum1;
        if (!(fabsf(top) < kLarge)) {                 // once more, and nobody has written over the logits yet
          LargePart<T> again;
          for (int g = sl.g0 + static_cast<int>(threadIdx.x); g < sl.ge; g += kRowCompute)
            if (g >= sl.gs) again.add(load_granule<T>(src, g, gr.lead, p.V));
          again.add(x_edge);
          again.result(top, sum);
        }
        warp_merge(top, sum);
        // the logits at the entries have been read: only now may another CTA overwrite them
        ok = ok && mbar_wait_soon(&bars.e_full[b], phase);
        if (threadIdx.x == 0) mbar_arrive_expect_tx(&bars.xchg[b], C * kRowWarps * 8);
        __syncwarp();
        if (lane < C) send_pair(&part[b][rank * kRowWarps + warp], &bars.xchg[b], lane, top, sum);
        ok = ok && mbar_wait_pairs(&bars.xchg[b], phase);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) { leave(); break; }
        constexpr int kPairs = C * kRowWarps;
        top = lane < kPairs ? part[b][lane].x : -INFINITY;
        sum = lane < kPairs ? part[b][lane].y : 0.f;
#pragma unroll
        for (int i = 32; i < kPairs; i += 32)
          if (lane + i < kPairs) merge(top, sum, part[b][lane + i].x, part[b][lane + i].y);
        warp_merge(top, sum);
      }
      if (threadIdx.x == 0) {
        if (p.given == nullptr) {
          head[b].top = top;
          head[b].sum = sum;
        }
        if (answered(it + 1) && granted(it + 1) >= 0) request(it + 2);
      }
      if (p.grad != nullptr) {
        TO* dst = static_cast<TO*>(p.grad) + row * p.ldg;
        const bool aligned = granules_aligned<TO, n>(dst, gr.lead);
        const float w = head[b].weight;
        const Exponent ex = exponent_of(top, sum, c);
        // no entries, or a token that does not count: zero whatever the logits hold
        const bool zero = head[b].tsum == 0.f || w == 0.f;
        const float scale = w * p.inv_tau * __fdiv_rn(1.f, sum);
        const uint64_t scale2 = pair(scale, scale), minus = pair(-ex.top, -ex.top), cx = pair(ex.c, ex.c);
        TO* out = dst - gr.lead;
        if (zero) {
          const uint64_t none[kP] = {};
          for (int g = sl.gs + static_cast<int>(threadIdx.x); g < sl.ge; g += kRowCompute)
            store_pairs<TO, kP>(out + g * n, aligned, none);
        }
        auto give = [&](const uint4& v, int granule) {
          uint64_t f[kP];
          Pairs<T>::widen(v, f);
#pragma unroll
          for (int j = 0; j < kP; ++j) f[j] = mul2(ex2_2(fma2(f[j], cx, minus)), scale2);
          store_pairs<TO, kP>(out + granule * n, aligned, f);
        };
        auto finish = [&](int k, int at) {            // chunk k of the slice, at this place of the ring
          const int k0 = sl.g0 + k * kChunk;
          const uint4* chunk = reinterpret_cast<const uint4*>(dyn) + at * kChunk;
          const int lo = sl.gs - k0, hi = min(sl.ge - k0, kChunk);
          const int g = threadIdx.x;
          if (zero) {
          } else if (lo <= 0 && hi == kChunk) {
            uint4 v[kU];
#pragma unroll
            for (int u = 0; u < kU; ++u) v[u] = chunk[g + u * kRowCompute];
#pragma unroll
            for (int u = 0; u < kU; ++u) give(v[u], k0 + g + u * kRowCompute);
          } else {
#pragma unroll
            for (int u = 0; u < kU; ++u) {
              const int i = g + u * kRowCompute;
              if (i >= lo && i < hi) give(chunk[i], k0 + i);
            }
          }
          mbar_arrive_warp(&bars.empty[at]);
        };
        int kept = both ? plan.keep : 0;              // chunks that pass 1 has left in the ring, then those of another load
        int slot2 = slot - kept < 0 ? slot - kept + plan.ring : slot - kept;
        const int from = plan.chunks - kept;
        for (int i = 0; i < plan.chunks; ++i) {
          if (i < kept) {
            finish(from + i, slot2);
            if (++slot2 == plan.ring) slot2 = 0;
          } else {
            ok = arrived();
            if (!ok) break;
            finish(i - kept, slot);
            advance();
          }
        }
        if (!ok) { leave(); break; }
        if (edge >= 0) Lane<TO>::store(dst + edge, zero ? 0.f : ex2(fmaf(x_edge, ex.c, -ex.top)) * scale);
      }
      mbar_arrive_warp(&bars.e_empty[b]);
    }
  }
  __syncthreads();
  if (failed) drain_delay();
  if constexpr (C > 1) {                   // nobody sends to a CTA that has left
    cluster_arrive();
    cluster_wait();
  }
}

// ------------------------------------------------------------------------------------------- statistics, any row
constexpr int kDsStatsThreads = 512;

template <typename T>
__global__ void __launch_bounds__(kDsStatsThreads)
distill_stats_kernel(const DistillParams p) {
  constexpr int n = Lane<T>::n;
  __shared__ TeacherRow e;
  __shared__ float2 red[kDsStatsThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row = blockIdx.x;
  const T* src = static_cast<const T*>(p.logits) + row * p.ld;
  const Granules<T> gr(src, p.V);
  const float c = p.inv_tau * kLog2e;
  if (warp == 0) load_teacher<T>(p, src, row, e, lane);
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
  if (!(fabsf(top) < kLarge)) {
    LargePart<T> again;
    for (int g = threadIdx.x; g < gr.count; g += kDsStatsThreads) again.add(load_granule<T>(src, g, gr.lead, p.V));
    again.result(top, sum);
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
  float sum = st.y;
  const Exponent ex = exponent_of(st.x, sum, c);
  float l = 0.f;
  if (st.w != 0.f) {
    const float inv = __fdiv_rn(1.f, st.w), log_sum = log2f(sum), log_tsum = log2f(st.w);
    for (int j = lane; j < p.K; j += 32) {
      const long long id = entry_id(p, row, j);
      if (id < 0 || id >= p.vocab_total) continue;
      const float t = p.teacher[row * p.ld_t + j];
      l += loss_term(entry_q(t, st.z, inv, c), (t - st.z) * c - log_tsum, p.picked[row * p.K + j], c, ex, log_sum);
    }
  }
  l = warp_total(l) * kLn2;
  if (lane == 0) p.loss[row] = l / kDown;
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
  float sum = st.y;
  const Exponent ex = exponent_of(st.x, sum, c);
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
  const float g = w * p.inv_tau * __fdiv_rn(1.f, sum);
#pragma unroll
  for (int i = 0; i < kGradVec; ++i) {
    const int k = g0 + i * kDsThreads + threadIdx.x;
    if (k >= gr.count) continue;
    float f[n];
    if (!zero) Lane<T>::widen(v[i], f);
#pragma unroll
    for (int j = 0; j < n; ++j) f[j] = zero ? 0.f : ex2(fmaf(f[j], ex.c, -ex.top)) * g;
    store_granule<TO, n>(dst, k, gr.lead, p.V, aligned, f);
  }
  if (zero) return;
  __syncthreads();
  write_entries<TO>(p, e, dst, ex, sum, w);
}

// ------------------------------------------------------------------------------------------- fused head: total, scaling
// sum_t w_t loss_t in a fixed order, tokens of weight 0 left out whatever their loss; one CTA, a few microseconds for the
// tokens of a step.
__global__ void __launch_bounds__(1024)
distill_total_kernel(const float* __restrict__ loss, const float* __restrict__ w, int T, float* __restrict__ total) {
  __shared__ float red[32];
  float s = 0.f;
  for (int t = threadIdx.x; t < T; t += 1024) s += w[t] == 0.f ? 0.f : w[t] * loss[t];
  s = warp_total(s);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = warp_total(red[threadIdx.x]);
    if (threadIdx.x == 0) *total = s;
  }
}

// Hidden states for the weight gradient: the rows of tokens that count, zeros for the others, whose gradient is 0 but whose
// states may hold anything, and 0 * NaN would reach every weight.  One CTA per row; 4 bytes per element, beside the products
// of the block it belongs to (2048 x 2048: 3.5 us of 4 ms).
__global__ void __launch_bounds__(128)
distill_live_kernel(const DistillParams p, const uint4* __restrict__ h, long long ldh, uint4* __restrict__ out, int width) {
  const long long row = blockIdx.x;
  bool entry = false;
  if (p.weight[row] != 0.f)
    for (int j = threadIdx.x; j < p.K; j += 128) {
      const long long id = entry_id(p, row, j);
      entry |= id >= 0 && id < p.vocab_total && p.teacher[row * p.ld_t + j] != -INFINITY;
    }
  const bool counts = __syncthreads_or(entry);
  for (int i = threadIdx.x; i < width; i += 128) out[row * width + i] = counts ? h[row * ldh + i] : make_uint4(0, 0, 0, 0);
}

// bf16(x * *scale): the gradients that the forward pass left, times the incoming one.  6 bytes per element, DRAM bound.
__global__ void __launch_bounds__(256)
distill_scale_kernel(const float4* __restrict__ x, const float* __restrict__ scale, uint2* __restrict__ y, long long n4) {
  const float s = *scale;
  const long long step = static_cast<long long>(gridDim.x) * 256;
  long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  for (; i + 3 * step < n4; i += 4 * step) {
    float4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = __ldcs(x + i + u * step);
#pragma unroll
    for (int u = 0; u < 4; ++u) y[i + u * step] = make_uint2(pack_bf16(v[u].x * s, v[u].y * s), pack_bf16(v[u].z * s, v[u].w * s));
  }
  for (; i < n4; i += step) {
    const float4 v = x[i];
    y[i] = make_uint2(pack_bf16(v.x * s, v.y * s), pack_bf16(v.z * s, v.w * s));
  }
}

// ------------------------------------------------------------------------------------------- launchers
// Granules of a row whose start may lie anywhere in its first granule.
static long long max_granules(int V, int n) { return (static_cast<long long>(V) + 2 * (n - 1)) / n; }

constexpr int kRowSmem = 224 * 1024;               // dynamic shared memory of an SM that the row kernel counts on
constexpr int kRowSlice = 144 * 1024;              // largest slice: 1024 entries, bitmaps and barriers fit beside it

// Shared memory beside the ring, and the chunks of a ring with this many CTAs on an SM.
static int row_side(int K, int per, int n, bool gradient) {
  return 2 * (entry_bytes((K + 3) & ~3) + (gradient ? bitmap_bytes(per, n) : 0));
}
static int row_ring(int side, int ctas) {
  const int ring = (kRowSmem / ctas - 2048 - side) / (kChunk * 16);
  return ring < kMaxChunks ? ring : kMaxChunks;
}
// Whether one CTA can pass through a whole row and has room for its entries and bitmaps.
static bool one_cta_streams(int V, int K, int n) {
  return row_ring(row_side(K, static_cast<int>(max_granules(V, n)), n, true), 1) >= 2;
}

template <typename T, typename TO, int C>
static cudaError_t launch_row(const DistillParams& p, cudaStream_t stream) {
  constexpr int n = Lane<T>::n;
  RowPlan plan{};
  plan.per = static_cast<int>((max_granules(p.V, n) + C - 1) / C);
  plan.chunks = (plan.per + kChunk - 1) / kChunk;
  plan.kpad = (p.K + 3) & ~3;
  const int side = row_side(p.K, plan.per, n, p.grad != nullptr);
  // two CTAs per SM where that leaves each a ring of two chunks, so that one computes while the other waits; else one CTA
  plan.ring = row_ring(side, 2) >= 2 ? row_ring(side, 2) : row_ring(side, 1);
  if (plan.ring < 2) return cudaErrorInvalidValue;
  plan.keep = plan.chunks < plan.ring ? plan.chunks : plan.ring;
  const int smem = plan.ring * kChunk * 16 + side;
  auto kernel = distill_row_kernel<T, TO, C>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  // the shared-memory limit is raised once per device
  static std::atomic<unsigned long long> raised{0};
  if (dev >= 64 || !((raised.load() >> dev) & 1ull)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowSmem);
    if (e != cudaSuccess) return e;
    if (dev < 64) raised.fetch_or(1ull << dev);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.T) * C);
  cfg.blockDim = dim3(kRowThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p, plan);
}

// CTAs per row: the fewest whose slices are not much longer than a ring (96 KB with two CTAs per SM), so that most of a
// slice is not loaded again, more (up to 8) while the rows alone do not fill the SMs.
constexpr int kWidestSlice = 160 * 1024;

// Whether there are rows enough for one CTA each where a row is only passed through.
static bool many_rows(int T) { return T >= 2 * sm_count(); }

template <typename T, typename TO>
static cudaError_t run_row(const DistillParams& p, cudaStream_t stream) {
  if ((p.grad == nullptr && many_rows(p.T)) || p.given != nullptr) return launch_row<T, TO, 1>(p, stream);
  const long long bytes = max_granules(p.V, Lane<T>::n) * 16;
  int c = 1;
  while (c < 8 && bytes > static_cast<long long>(c) * kWidestSlice) c *= 2;
  while (c < 8 && static_cast<long long>(p.T) * c < sm_count() && bytes > static_cast<long long>(c) * 4096) c *= 2;
  switch (c) {
    case 1: return launch_row<T, TO, 1>(p, stream);
    case 2: return launch_row<T, TO, 2>(p, stream);
    case 4: return launch_row<T, TO, 4>(p, stream);
    default: return launch_row<T, TO, 8>(p, stream);
  }
}

}  // namespace stb

using namespace stb;

// Longest row that stb_distill_row takes, for 2- or 4-byte logits.
extern "C" int stb_distill_row_limit(int elem_bytes) {
  const int n = 16 / elem_bytes;
  return 8 * (kRowSlice / 16) * n - 2 * (n - 1);
}

static bool distill_args_ok(const DistillParams& p) {
  return p.T > 0 && p.T <= 0x0FFFFFFF && p.V > 0 && p.V <= (1 << 30) && p.K >= 0 && p.K <= kDsMaxEntries && p.inv_tau > 0.f;
}

// The gradient has the logits' type, or is bf16 for fp32 logits.
static bool distill_types_ok(int elem_bytes, int grad_bytes) {
  return (elem_bytes == 2 && grad_bytes == 2) || (elem_bytes == 4 && (grad_bytes == 4 || grad_bytes == 2));
}

// Loss, statistics and (grad != null) gradient of whole rows in one pass; grad may be the logits where the types are equal.
extern "C" int stb_distill_row(const void* logits, long long ld, void* grad, long long ldg, const void* ids, int ids64,
                               long long ld_ids, const float* teacher, long long ld_t, const float* weight, float* loss,
                               float* stats, int T, int V, int K, float inv_tau, int elem_bytes, int grad_bytes,
                               int* status, cudaStream_t stream) {
  if (T == 0) return 0;
  DistillParams p{};
  p.logits = logits; p.ld = ld; p.grad = grad; p.ldg = ldg; p.ids = ids; p.ids64 = ids64; p.ld_ids = ld_ids;
  p.teacher = teacher; p.ld_t = ld_t; p.weight = weight; p.loss = loss; p.stats = reinterpret_cast<float4*>(stats);
  p.T = T; p.V = V; p.K = K; p.vocab_start = 0; p.vocab_total = V; p.inv_tau = inv_tau; p.status = status;
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
                                float inv_tau, int elem_bytes, int grad_bytes, int* status, cudaStream_t stream) {
  if (T == 0) return 0;
  DistillParams p{};
  p.logits = logits; p.ld = ld; p.grad = grad; p.ldg = ldg; p.ids = ids; p.ids64 = ids64; p.ld_ids = ld_ids;
  p.teacher = teacher; p.ld_t = ld_t; p.weight = weight; p.stats = reinterpret_cast<float4*>(const_cast<float*>(stats));
  p.T = T; p.V = V; p.K = K; p.vocab_start = vocab_start; p.vocab_total = vocab_total; p.inv_tau = inv_tau;
  if (!distill_args_ok(p) || grad == nullptr || !distill_types_ok(elem_bytes, grad_bytes)) return -kErrBadArgument;
  if (logits != grad && vocab_start == 0 && vocab_total == V && many_rows(T) &&
      one_cta_streams(V, K, 16 / elem_bytes)) {
    p.given = p.stats;
    p.stats = nullptr;
    p.status = status;
    cudaError_t e;
    if (elem_bytes == 2) e = run_row<__nv_bfloat16, __nv_bfloat16>(p, stream);
    else if (grad_bytes == 4) e = run_row<float, float>(p, stream);
    else e = run_row<float, __nv_bfloat16>(p, stream);
    return -static_cast<int>(e);
  }
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

extern "C" int stb_distill_total(const float* loss, const float* weight, int T, float* total, cudaStream_t stream) {
  distill_total_kernel<<<1, 1024, 0, stream>>>(loss, weight, T, total);
  return -static_cast<int>(cudaGetLastError());
}

// out [T][H] = h [T][H] where the token's weight is not 0 and it has an entry, else 0; rows on 16-byte boundaries, H a
// multiple of 8, strides in elements.
extern "C" int stb_distill_live(const void* h, long long ldh, const void* ids, int ids64, long long ld_ids,
                                const float* teacher, long long ld_t, const float* weight, void* out, int T, int H, int K,
                                long long vocab_total, cudaStream_t stream) {
  if (T == 0 || H == 0) return 0;
  if (T < 0 || H < 0 || H % 8 || ldh % 8 || K < 0 || (reinterpret_cast<uintptr_t>(h) & 15) ||
      (reinterpret_cast<uintptr_t>(out) & 15))
    return -kErrBadArgument;
  DistillParams p{};
  p.ids = ids; p.ids64 = ids64; p.ld_ids = ld_ids; p.teacher = teacher; p.ld_t = ld_t; p.weight = weight; p.K = K; p.T = T;
  p.vocab_total = vocab_total;
  distill_live_kernel<<<T, 128, 0, stream>>>(p, static_cast<const uint4*>(h), ldh / 8, static_cast<uint4*>(out), H / 8);
  return -static_cast<int>(cudaGetLastError());
}

// y (bf16) = x (fp32) * *scale; count a multiple of 4, both 16-byte aligned.
extern "C" int stb_distill_scale(const float* x, const float* scale, void* y, long long count, cudaStream_t stream) {
  if (count == 0) return 0;
  if (count % 4 || (reinterpret_cast<uintptr_t>(x) & 15) || (reinterpret_cast<uintptr_t>(y) & 15)) return -kErrBadArgument;
  const long long blocks = (count / 4 + 1023) / 1024, most = static_cast<long long>(sm_count()) * 8;
  distill_scale_kernel<<<static_cast<unsigned>(blocks < most ? blocks : most), 256, 0, stream>>>(
      reinterpret_cast<const float4*>(x), scale, static_cast<uint2*>(y), count / 4);
  return -static_cast<int>(cudaGetLastError());
}
