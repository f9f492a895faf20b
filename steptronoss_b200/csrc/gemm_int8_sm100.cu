// 8-bit integer GEMM for sm_100a with one scale per token and one per output channel:
//
//     Y[m, n] = sx[m] * sw[n] * sum_k Xq[m, k] * Wq[n, k]          Xq [M, K], Wq [N, K] int8, sums in int32, Y bf16/fp32
//
// tcgen05.mma.kind::i8 accumulates in int32, so the product is exact and independent of the order of its sums; K is at
// most 131071 (2^31 / 128^2).  The sum is converted to fp32 once, multiplied by the two scales and rounded to Y's type.
//
// The weights are the A operand (128 channels of the tile are the 128 TMEM lanes) and the tokens the B operand (TMEM
// columns), whatever their number: a decode step of a few tokens then takes a 16-, 32- or 64-column tile instead of
// a mostly empty 128-row one, and a warp that reads one column writes 32 neighbouring channels of one token.
//
//   gemm_int8_pair_kernel   many tokens: persistent, 256 x 256 tiles on pairs of CTAs, accumulators double-buffered in TMEM
//   gemm_int8_split_kernel  few tokens: one tile per cluster, K cut over the CTAs of the cluster so that the weights
//                           stream through all SMs; partial sums meet in distributed shared memory
#include "common.cuh"

namespace stb {

constexpr int kI8BlockN = 128;      // channels per tile
constexpr int kI8BlockK = 128;      // one 128-byte swizzle span
constexpr int kI8WTile = kI8BlockN * kI8BlockK;
constexpr int kI8Threads = 192;     // producer, MMA issuer, four epilogue warps

struct Int8GemmParams {
  int M, N, K;
  long long ldy;
  const float* sx;
  const float* sw;
  void* Y;
  int* status;
  int tma_out;                      // bf16 output that a tensor map describes
};

// kind::i8: int32 accumulators (D format 2), signed 8-bit A and B (format 1), both K-major
__host__ __device__ constexpr uint32_t umma_idesc_s8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// 4 steps of K = 32 over one 128-byte swizzle span; `accumulate` applies to the first step only.
__device__ __forceinline__ void umma4_s8(uint32_t d, uint64_t a0, uint64_t b0, uint32_t idesc, uint32_t accumulate) {
  const uint64_t a1 = umma_desc_advance(a0, 32), a2 = umma_desc_advance(a0, 64), a3 = umma_desc_advance(a0, 96);
  const uint64_t b1 = umma_desc_advance(b0, 32), b2 = umma_desc_advance(b0, 64), b3 = umma_desc_advance(b0, 96);
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %10, 0;\n\t"
      "setp.eq.b32 q, 0, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %5, %9, p;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %2, %6, %9, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %3, %7, %9, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %4, %8, %9, q;\n\t}"
      ::"r"(d), "l"(a0), "l"(a1), "l"(a2), "l"(a3), "l"(b0), "l"(b1), "l"(b2), "l"(b3), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 lanes x 16 consecutive columns: thread t of the warp receives row (lane base + t).
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void cluster_sync_all() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ------------------------------------------------------------------------------------------------- many tokens
// CTA pairs (cta_group::2): a tile of 256 channels x 256 tokens on two SMs.  CTA r of the pair loads 128 channels and 128
// tokens, a third less than a 128 x 256 tile of its own would take, and the tensor cores of both read both halves of
// the tokens; the first CTA issues the products, each holds the sums of its own 128 channels (256 TMEM columns, two
// buffers) and writes them.  What bounds the single-CTA form is the traffic from L2 to the SMs: 48 KB per 512 cycles of
// products, of which about 58 bytes a cycle and SM arrive (128 x 256 tiles measured 2513 TOPS, 656 us for 8192 x 24576 x
// 4096); a pair needs 32 KB.
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* slot, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// Address of `p` in the shared memory of CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_smem(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
// A tile into this CTA's shared memory, counted on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* d, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(d)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
// Arrive on the barrier at this offset in both CTAs once the products issued so far are done.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(smem_u32(bar)), "h"(static_cast<uint16_t>(3)) : "memory");
}
__device__ __forceinline__ void mbar_arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Whether `ok` holds for all 128 threads that meet at named barrier `id`.
__device__ __forceinline__ bool group_and(int id, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %2, 0;\n\t"
      "bar.red.and.pred q, %1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r) : "r"(id), "r"(static_cast<uint32_t>(ok)) : "memory");
  return r != 0;
}
// The pair's products of one k block: M = 256 (128 rows of A in each CTA), N = 256 (128 rows of B in each).
__device__ __forceinline__ void umma4_s8_pair(uint32_t d, uint64_t a0, uint64_t b0, uint32_t idesc, uint32_t accumulate) {
  const uint64_t a1 = umma_desc_advance(a0, 32), a2 = umma_desc_advance(a0, 64), a3 = umma_desc_advance(a0, 96);
  const uint64_t b1 = umma_desc_advance(b0, 32), b2 = umma_desc_advance(b0, 64), b3 = umma_desc_advance(b0, 96);
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %10, 0;\n\t"
      "setp.eq.b32 q, 0, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %5, %9, p;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %2, %6, %9, q;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %3, %7, %9, q;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %4, %8, %9, q;\n\t}"
      ::"r"(d), "l"(a0), "l"(a1), "l"(a2), "l"(a3), "l"(b0), "l"(b1), "l"(b2), "l"(b3), "r"(idesc), "r"(accumulate)
      : "memory");
}

constexpr int kPairTile = 256;                                   // channels and tokens of a pair's tile
constexpr int kPairStages = 6;
constexpr int kPairStageBytes = kI8WTile + 128 * kI8BlockK;      // of one CTA
constexpr int kPairStoreBytes = 2 * 2 * 32 * 128 * 2;            // two groups of epilogue warps, two chunks each
constexpr int kPairThreads = 320;                                // producer, MMA issuer, eight epilogue warps
constexpr int kPairSmem = kPairStages * kPairStageBytes + kPairStoreBytes + 256 + 1024;

// Tiles are walked in bands of kBand channel tiles so that the pairs of a wave share weights and tokens in L2.
__device__ __forceinline__ void int8_tile(int tile, int num_n, int num_m, int& n_tile, int& m_tile) {
  constexpr int kBand = 8;
  const int band = tile / (kBand * num_m);
  const int first = band * kBand;
  const int rows = min(num_n - first, kBand);
  const int r = tile - band * kBand * num_m;
  n_tile = first + r % rows;
  m_tile = r / rows;
}

template <typename TY>
__device__ __forceinline__ void store_y(TY* p, float v);
template <> __device__ __forceinline__ void store_y<float>(float* p, float v) { *p = v; }
template <> __device__ __forceinline__ void store_y<__nv_bfloat16>(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename TY>
__global__ void __launch_bounds__(kPairThreads, 1)
gemm_int8_pair_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                      const __grid_constant__ CUtensorMap tmap_y, const Int8GemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  // the same offset in both CTAs: the dynamic segment starts at the same address in all CTAs of a cluster
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* store_stage = smem + kPairStages * kPairStageBytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(store_stage + kPairStoreBytes);   // used in the first CTA
  uint64_t* empty_bar = full_bar + kPairStages;                                      // one in each CTA
  uint64_t* tmem_full = empty_bar + kPairStages;                                     // one in each CTA
  uint64_t* tmem_empty = tmem_full + 2;                                              // used in the first CTA
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int num_n = (p.N + kPairTile - 1) / kPairTile;
  const int num_m = (p.M + kPairTile - 1) / kPairTile;
  const int num_tiles = num_n * num_m, pairs = gridDim.x / 2;
  const int k_blocks = (p.K + kI8BlockK - 1) / kI8BlockK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tmem_full[a], 1);
      mbar_init(&tmem_empty[a], 16);         // eight epilogue warps of each CTA
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 2 * kPairTile);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                        // the other CTA's barriers are initialised, too
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  wait_for_previous_kernel();
  let_next_kernel_start();

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      for (int tile = blockIdx.x / 2; tile < num_tiles && !*abort_flag; tile += pairs) {
        int n_tile, m_tile;
        int8_tile(tile, num_n, num_m, n_tile, m_tile);
        for (int kb = 0; kb < k_blocks; ++kb, ++it) {
          const int s = it % kPairStages;
          if (!mbar_wait_cluster(&empty_bar[s], ((it / kPairStages) & 1) ^ 1)) {
            report_error(p.status, kErrProducerWait);
            *abort_flag = 1;
            break;
          }
          uint8_t* sw = smem + s * kPairStageBytes;
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[s], 2 * kPairStageBytes);     // both CTAs' loads
          const uint32_t bar = peer_smem(&full_bar[s], 0);
          tma_load_2d_pair(sw, &tmap_w, bar, kb * kI8BlockK, n_tile * kPairTile + rank * 128);
          tma_load_2d_pair(sw + kI8WTile, &tmap_x, bar, kb * kI8BlockK, m_tile * kPairTile + rank * 128);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = umma_idesc_s8(256, 256);
      uint32_t it = 0, local = 0;
      bool ok = true;
      for (int tile = blockIdx.x / 2; tile < num_tiles && ok && !*abort_flag; tile += pairs, ++local) {
        const int acc = local & 1;
        ok = mbar_wait_cluster(&tmem_empty[acc], ((local >> 1) & 1) ^ 1);
        if (!ok) { report_error(p.status, kErrMmaWaitTmem); break; }
        tc_fence_after();
        for (int kb = 0; kb < k_blocks; ++kb, ++it) {
          const int s = it % kPairStages;
          ok = mbar_wait_cluster(&full_bar[s], (it / kPairStages) & 1);
          if (!ok) { report_error(p.status, kErrMmaWaitFull); break; }
          tc_fence_after();
          const uint32_t sw = smem_u32(smem + s * kPairStageBytes);
          umma4_s8_pair(tmem_base + acc * kPairTile, umma_smem_desc(sw, 16, 1024), umma_smem_desc(sw + kI8WTile, 16, 1024),
                        idesc, kb > 0 ? 1u : 0u);
          umma_commit_pair(&empty_bar[s]);
        }
        if (!ok) break;
        umma_commit_pair(&tmem_full[acc]);
      }
      if (!ok) *abort_flag = 1;
    }
  } else {
    // eight warps: two groups of four, which take the tile's chunks of 32 tokens in turn
    const int quarter = warp & 3, group = (warp - 2) >> 2;
    uint8_t* my_stage = store_stage + (warp - 2) * 4096;                  // two buffers of 32 tokens x 32 channels
    __nv_bfloat16* group_stage = reinterpret_cast<__nv_bfloat16*>(store_stage + group * 16384);   // two of 32 x 128
    uint32_t local = 0, stores = 0;
    for (int tile = blockIdx.x / 2; tile < num_tiles; tile += pairs, ++local) {
      int n_tile, m_tile;
      int8_tile(tile, num_n, num_m, n_tile, m_tile);
      const int acc = local & 1;
      const int cta_n0 = n_tile * kPairTile + rank * 128;
      const int n0 = cta_n0 + quarter * 32, n = n0 + lane, m0 = m_tile * kPairTile;
      const float sw = n < p.N ? p.sw[n] : 0.f;
      // the group goes on or leaves as one: its warps meet at barriers below
      const bool ok = group_and(1 + group, mbar_wait_cluster(&tmem_full[acc], (local >> 1) & 1));
      if (!ok) { report_error(p.status, kErrEpilogueWait); *abort_flag = 1; break; }
      tc_fence_after();
      const int cols = min(kPairTile, p.M - m0);
#pragma unroll 1
      for (int c = group * 32; c < cols; c += 64) {
        const float sx = c + lane < cols ? p.sx[m0 + c + lane] : 0.f;
        uint32_t v[32];
        tmem_ld_32x32(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * kPairTile + c, v);
        tmem_wait_ld();
        auto value = [&](int j) {
          return static_cast<float>(static_cast<int>(v[j])) * __shfl_sync(0xffffffffu, sx, j) * sw;
        };
        if constexpr (sizeof(TY) == 4) {
          TY* y = static_cast<TY*>(p.Y) + static_cast<long long>(m0 + c) * p.ldy + n;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float f = value(j);
            if (n < p.N && c + j < cols) store_y<TY>(y + j * p.ldy, f);
          }
        } else if (p.tma_out) {
          if (stores >= 2) {
            if (lane == 0) tma_store_wait_read<1>();
            __syncwarp();
          }
          uint8_t* buf = my_stage + (stores++ & 1) * 2048;
          __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(buf) + lane;
#pragma unroll
          for (int j = 0; j < 32; ++j) out[j * 32] = __float2bfloat16_rn(value(j));
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (n0 < p.N) tma_store_2d(&tmap_y, buf, n0, m0 + c);   // rows and channels past the end are clipped
            tma_store_commit();
          }
        } else {
          // rows on any address: the group's 128 channels of a token lie side by side in shared memory and leave as
          // 16-byte stores from the first 16-byte boundary on, what is before and behind them element by element.  (With
          // one 2-byte store per channel 1333 x 5001 x 2050 took 42 us instead of 27.)
          __nv_bfloat16* buf = group_stage + (stores++ & 1) * (32 * 128);
          __nv_bfloat16* out = buf + quarter * 32 + lane;
#pragma unroll
          for (int j = 0; j < 32; ++j) out[j * 128] = __float2bfloat16_rn(value(j));
          asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");
          const int l = lane & 15, width = min(128, p.N - cta_n0);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int t = quarter * 8 + i * 2 + (lane >> 4);
            if (c + t >= cols || width <= 0) continue;
            __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.Y) + static_cast<long long>(m0 + c + t) * p.ldy + cta_n0;
            const uint16_t* src = reinterpret_cast<const uint16_t*>(buf) + t * 128;
            const int head = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(dst) & 15)) & 15) / 2, width);
            const int vecs = (width - head) / 8;
            if (l < vecs) {
              const uint16_t* e = src + head + l * 8;
              uint32_t u[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) u[k] = e[2 * k] | (static_cast<uint32_t>(e[2 * k + 1]) << 16);
              *reinterpret_cast<uint4*>(dst + head + l * 8) = make_uint4(u[0], u[1], u[2], u[3]);
            }
            const int at = l < 8 ? l : head + vecs * 8 + l - 8;
            if (l < 8 ? l < head : at < width) reinterpret_cast<uint16_t*>(dst)[at] = src[at];
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_at(peer_smem(&tmem_empty[acc], 0));
    }
    if (lane == 0) tma_store_wait<0>();
  }

  __syncthreads();
  if (*abort_flag) drain_delay();
  cluster_sync_all();                        // nobody signals or reads a CTA that has left
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * kPairTile);
  }
}

// ------------------------------------------------------------------------------------------------- few tokens
template <int BM>
struct Int8SplitSmem {
  static constexpr int kXTile = BM * kI8BlockK;
  static constexpr int kStageBytes = kI8WTile + kXTile;
  // two CTAs per SM (about 110 KB each)
  static constexpr int kStages = BM == 16 ? 6 : BM == 32 ? 5 : BM == 64 ? 4 : 3;
  static constexpr int kPartBytes = kI8BlockN * BM * 4;       // [source CTA][column of this CTA][128 channels] int32
  static constexpr int kTotal = kStages * kStageBytes + 256 + 1024;
  static_assert(kPartBytes <= kStages * kStageBytes, "the partial sums reuse the operand ring");
};

// One output tile (128 channels, BM tokens) per cluster of S CTAs; CTA r takes every k block kb with kb % S == r.
// When all products of the cluster are done, column c of the tile belongs to CTA c % S: every CTA stores its partial sums
// of that column into that CTA's shared memory (over the operand ring, which nobody reads any more), and after one more
// cluster barrier each CTA adds, scales and writes its columns.
//
// Bound: the weights' bytes.  Two CTAs fit on an SM, so up to 296 stream at a time (48 x 24576 x 4096, 192 tiles: 33 us with
// one CTA per SM in two waves, 20.3 us).
template <int BM, int S, typename TY>
__global__ void __launch_bounds__(kI8Threads, 2)
gemm_int8_split_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                       const Int8GemmParams p) {
  using L = Int8SplitSmem<BM>;
  constexpr int kStages = L::kStages;
  constexpr int kTmemCols = BM < 32 ? 32 : BM;
  extern __shared__ uint8_t smem_raw[];
  // the same offset in every CTA of the cluster: the dynamic segment starts at the same address in all of them
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  int* part = reinterpret_cast<int*>(smem);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + kStages * L::kStageBytes);
  uint64_t* empty_bar = full_bar + kStages;
  uint64_t* done_bar = empty_bar + kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = S > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int num_n = (p.N + kI8BlockN - 1) / kI8BlockN;
  const int tile = blockIdx.x / S;
  const int n_tile = tile % num_n, m_tile = tile / num_n;
  const int m0 = m_tile * BM, cols = min(BM, p.M - m0);
  const int all_blocks = (p.K + kI8BlockK - 1) / kI8BlockK;
  const int k_blocks = (all_blocks - rank + S - 1) / S;     // one at least: S is at most half of all_blocks

  auto load = [&](int i) {
    const int s = i % kStages, kb = i * S + rank;
    uint8_t* sw = smem + s * L::kStageBytes;
    mbar_arrive_expect_tx(&full_bar[s], L::kStageBytes);
    tma_load_2d(sw, &tmap_w, &full_bar[s], kb * kI8BlockK, n_tile * kI8BlockN);
    tma_load_2d(sw + kI8WTile, &tmap_x, &full_bar[s], kb * kI8BlockK, m0);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    wait_for_previous_kernel();
    for (int i = 0; i < min(kStages, k_blocks); ++i) load(i);     // on their way while the rest is set up
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  wait_for_previous_kernel();
  let_next_kernel_start();
  // The scales are read by plain loads from here on: this kernel was running while the one before it wrote them, and the
  // read-only path asks for memory that nobody writes during a kernel's whole life.

  if (warp == 0) {
    if (lane == 0) {
      for (int i = kStages; i < k_blocks; ++i) {
        if (!mbar_wait(&empty_bar[i % kStages], ((i / kStages) & 1) ^ 1)) {
          report_error(p.status, kErrProducerWait);
          *abort_flag = 1;
          break;
        }
        load(i);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = umma_idesc_s8(kI8BlockN, BM);
      bool ok = true;
      for (int i = 0; i < k_blocks; ++i) {
        const int s = i % kStages;
        ok = mbar_wait(&full_bar[s], (i / kStages) & 1);
        if (!ok) { report_error(p.status, kErrMmaWaitFull); *abort_flag = 1; break; }
        tc_fence_after();
        const uint32_t sw = smem_u32(smem + s * L::kStageBytes);
        umma4_s8(tmem_base, umma_smem_desc(sw, 16, 1024), umma_smem_desc(sw + kI8WTile, 16, 1024), idesc, i > 0 ? 1u : 0u);
        umma_commit(&empty_bar[s]);
      }
      umma_commit(done_bar);
    }
    __syncwarp();
  }
  const int quarter = warp & 3;
  const int row = quarter * 32 + lane;
  const int n = n_tile * kI8BlockN + row;
  const float swn = warp >= 2 && n < p.N ? p.sw[n] : 0.f;
  bool ok = mbar_wait(done_bar, 0);           // every warp: the cluster barrier below says that this CTA's products are done
  ok = __all_sync(0xffffffffu, ok) && !*abort_flag;
  if (!ok) { report_error(p.status, kErrEpilogueWait); *abort_flag = 1; }
  tc_fence_after();
  if constexpr (S > 1) cluster_sync_all();
  // columns of the tile in groups of 16; with S > 1 each goes to the CTA that owns it
  if (warp >= 2 && ok) {
    for (int c = 0; c < cols; c += 16) {
      uint32_t v[16];
      float sx[16];                             // before the stores, which the compiler has to take for writes to them
      if constexpr (S == 1) {
#pragma unroll
        for (int j = 0; j < 16; ++j) sx[j] = c + j < cols ? p.sx[m0 + c + j] : 0.f;
      }
      tmem_ld_32x16(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + c, v);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (c + j >= cols) continue;
        if constexpr (S > 1) {
          const int owner = (c + j) % S, slot = (c + j) / S;
          uint32_t addr;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                       : "=r"(addr) : "r"(smem_u32(part + (rank * (BM / S) + slot) * kI8BlockN + row)), "r"(owner));
          asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v[j]) : "memory");
        } else if (n < p.N) {
          const float f = static_cast<float>(static_cast<int>(v[j])) * sx[j] * swn;
          store_y<TY>(static_cast<TY*>(p.Y) + static_cast<long long>(m0 + c + j) * p.ldy + n, f);
        }
      }
    }
  }
  if constexpr (S > 1) {
    cluster_sync_all();
    if (warp >= 2 && n < p.N) {
#pragma unroll 4
      for (int slot = 0; slot * S + rank < cols; ++slot) {
        int sum = 0;
#pragma unroll
        for (int r = 0; r < S; ++r) sum += part[(r * (BM / S) + slot) * kI8BlockN + row];
        const int m = m0 + slot * S + rank;
        store_y<TY>(static_cast<TY*>(p.Y) + static_cast<long long>(m) * p.ldy + n, static_cast<float>(sum) * p.sx[m] * swn);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) drain_delay();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

// ------------------------------------------------------------------------------------------------- launchers
// Shared-memory limit of a kernel, raised once per device.
template <typename Kernel>
static cudaError_t allow_smem(Kernel kernel, int bytes, unsigned long long& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && ((__atomic_load_n(&done, __ATOMIC_RELAXED) >> dev) & 1ull)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) __atomic_fetch_or(&done, 1ull << dev, __ATOMIC_RELAXED);
  return e;
}

static int maps_wx(CUtensorMap& tw, CUtensorMap& tx, const void* xq, const void* wq, const Int8GemmParams& p,
                   long long ldx, long long ldw, int bm) {
  int r = make_tmap_2d(&tw, wq, 1, p.K, p.N, static_cast<uint64_t>(ldw), kI8BlockK, kI8BlockN, 1);
  if (r) return r;
  return make_tmap_2d(&tx, xq, 1, p.K, p.M, static_cast<uint64_t>(ldx), kI8BlockK, bm, 1);
}

template <typename TY>
static int launch_pair(const void* xq, const void* wq, Int8GemmParams p, long long ldx, long long ldw, cudaStream_t stream) {
  CUtensorMap tw, tx, ty;
  int r = maps_wx(tw, tx, xq, wq, p, ldx, ldw, 128);
  if (r) return r;
  p.tma_out = sizeof(TY) == 2 && p.ldy % 8 == 0 && reinterpret_cast<uintptr_t>(p.Y) % 16 == 0;
  if (p.tma_out) {
    r = make_tmap_2d(&ty, p.Y, 2, p.N, p.M, static_cast<uint64_t>(p.ldy) * 2, 32, 32, 0);
    if (r) return r;
  } else {
    ty = tw;
  }
  static unsigned long long done = 0;
  cudaError_t e = allow_smem(gemm_int8_pair_kernel<TY>, kPairSmem, done);
  if (e != cudaSuccess) return -static_cast<int>(e);
  const long long tiles = static_cast<long long>((p.N + kPairTile - 1) / kPairTile) * ((p.M + kPairTile - 1) / kPairTile);
  if (tiles > 0x3FFFFFFFll) return -kErrBadArgument;
  const int most = sm_count() / 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * static_cast<unsigned>(tiles < most ? tiles : most));
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = kPairSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {overlap_launch()};
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return -static_cast<int>(cudaLaunchKernelEx(&cfg, gemm_int8_pair_kernel<TY>, tw, tx, ty, p));
}

template <int BM, int S, typename TY>
static int launch_split(const void* xq, const void* wq, const Int8GemmParams& p, long long ldx, long long ldw,
                        long long tiles, cudaStream_t stream) {
  CUtensorMap tw, tx;
  int r = maps_wx(tw, tx, xq, wq, p, ldx, ldw, BM);
  if (r) return r;
  static unsigned long long done = 0;
  cudaError_t e = allow_smem(gemm_int8_split_kernel<BM, S, TY>, Int8SplitSmem<BM>::kTotal, done);
  if (e != cudaSuccess) return -static_cast<int>(e);
  if (tiles * S > 0x7FFFFFFFll) return -kErrBadArgument;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * S));
  cfg.blockDim = dim3(kI8Threads);
  cfg.dynamicSmemBytes = Int8SplitSmem<BM>::kTotal;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {overlap_launch()};
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = S;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = S > 1 ? 2 : 1;
  return -static_cast<int>(cudaLaunchKernelEx(&cfg, gemm_int8_split_kernel<BM, S, TY>, tw, tx, p));
}

template <int BM, typename TY>
static int run_split(const void* xq, const void* wq, const Int8GemmParams& p, long long ldx, long long ldw, cudaStream_t stream) {
  const long long tiles = static_cast<long long>((p.N + kI8BlockN - 1) / kI8BlockN) * ((p.M + BM - 1) / BM);
  const int blocks = (p.K + kI8BlockK - 1) / kI8BlockK;
  int s = 1;   // as many CTAs as the SMs hold two of, each with two k blocks at least
  while (s < 8 && tiles * s * 2 <= 2 * sm_count() && blocks >= 4 * s) s *= 2;
  switch (s) {
    case 1: return launch_split<BM, 1, TY>(xq, wq, p, ldx, ldw, tiles, stream);
    case 2: return launch_split<BM, 2, TY>(xq, wq, p, ldx, ldw, tiles, stream);
    case 4: return launch_split<BM, 4, TY>(xq, wq, p, ldx, ldw, tiles, stream);
    default: return launch_split<BM, 8, TY>(xq, wq, p, ldx, ldw, tiles, stream);
  }
}

template <typename TY>
static int run_int8(const void* xq, const void* wq, const Int8GemmParams& p, long long ldx, long long ldw, cudaStream_t stream) {
  if (p.M <= 16) return run_split<16, TY>(xq, wq, p, ldx, ldw, stream);
  if (p.M <= 32) return run_split<32, TY>(xq, wq, p, ldx, ldw, stream);
  if (p.M <= 64) return run_split<64, TY>(xq, wq, p, ldx, ldw, stream);
  // 64-token tiles (K cut where they leave SMs idle) while all of them run at a time; else 128 tokens per CTA up to the
  // half of a pair's tile, and pairs above.  Measured, in us: 128 x 4096 x 4096 10.2 with 64-token tiles, 11.2 with 128, 15.2
  // on pairs; 512 x 4096 x 4096 16.5, 17.9, 16.7; 128 x 24576 x 4096 37.0, 27.8, 29.6; 1024 x 4096 x 4096 31.7, 23.4, 18.6
  const long long n_tiles = (p.N + kI8BlockN - 1) / kI8BlockN;
  if (n_tiles * ((p.M + 63) / 64) <= 2 * sm_count()) return run_split<64, TY>(xq, wq, p, ldx, ldw, stream);
  if (p.M <= 128) return launch_split<128, 1, TY>(xq, wq, p, ldx, ldw, n_tiles, stream);
  return launch_pair<TY>(xq, wq, p, ldx, ldw, stream);
}

}  // namespace stb

using namespace stb;

// xq [M][K], wq [N][K] int8 (row strides ldx, ldw bytes, multiples of 16; bases 16-byte aligned), sx [M], sw [N] fp32,
// Y [M][N] bf16 or fp32 (row stride ldy elements).
extern "C" int stb_gemm_int8(const void* xq, const float* sx, const void* wq, const float* sw, void* Y, int M, int N,
                             int K, long long ldx, long long ldw, long long ldy, int out_f32, int* status,
                             cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (M > (1 << 30) || N > (1 << 30) || K <= 0 || K > 131071 || (ldx & 15) || (ldw & 15) || ldx < K || ldw < K || ldy < N ||
      (reinterpret_cast<uintptr_t>(xq) & 15) || (reinterpret_cast<uintptr_t>(wq) & 15))
    return -kErrBadArgument;
  Int8GemmParams p{};
  p.M = M; p.N = N; p.K = K; p.ldy = ldy; p.sx = sx; p.sw = sw; p.Y = Y; p.status = status;
  return out_f32 ? run_int8<float>(xq, wq, p, ldx, ldw, stream) : run_int8<__nv_bfloat16>(xq, wq, p, ldx, ldw, stream);
}
