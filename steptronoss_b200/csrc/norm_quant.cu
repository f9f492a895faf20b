// Rows to 8 bits, with the residual add and the RMS norm in front of it, in one pass:
//
//     s = bf16(x + delta)            the residual stream, written back        (delta optional)
//     y = s * rsqrt(mean(s^2) + eps) * (w [+ 1])                              (norm optional: y = s)
//     int8,  one scale per row        : scale = max|y| / 127,  q = round(y / scale)
//     e4m3,  one scale per 128 columns: scale = max|y| / 448,  q = e4m3(y / scale)
//
// The int8 form feeds stb_gemm_int8, the e4m3 form stb_gemm_fp8_block_scaled.  y stays in fp32 between the norm and
// its single rounding to 8 bits.  A row (block) without a non-zero value gets scale 1; one that holds an infinity or
// a NaN gets scale NaN, so that it cannot turn into finite numbers downstream.
//
// Memory bound: 2 + 2 bytes read, 2 + 1 written per element.  A row lives in the registers of its threads (16 bytes
// per vector, packed bf16), so everything is read once; the statistics are one sum and one maximum over the row.
#include "common.cuh"

#include <cuda_fp8.h>

namespace stb {

constexpr int kNqMaxVec = 4;        // vectors of 8 columns per thread
constexpr int kNqMaxThreads = 1024; // 1024 * 4 * 8 = 32768 columns

struct NormQuantParams {
  const __nv_bfloat16* x;
  const __nv_bfloat16* delta;   // nullptr: no residual add
  const __nv_bfloat16* w;       // nullptr: no norm
  __nv_bfloat16* s;             // nullptr: the sum is not kept
  uint8_t* q;
  float* scale;
  long long rows, ldx, ldd, lds, ldq;
  int H;
  float eps;
  int zero_centered;
};

template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (TPR > 32) {
    const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
    if (l == 0) red[w] = v;
    __syncthreads();
    v = l < TPR / 32 ? red[l] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}
// The bits of non-negative floats, NaN included, are ordered like integers.
template <int TPR>
__device__ __forceinline__ float row_max(float top, uint32_t* red) {
  uint32_t v = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
  if constexpr (TPR > 32) {
    const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
    if (l == 0) red[w] = v;
    __syncthreads();
    v = __reduce_max_sync(0xffffffffu, l < TPR / 32 ? red[l] : 0u);
  }
  return __uint_as_float(v);
}

// Largest |y| of eight values; a NaN stays one (fmaxf would drop it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
// Whether max|y| gives a scale.  Below 6e-36 max / 448 leaves the range of normal numbers; such values count as zero.
__device__ __forceinline__ bool usable(float amax) { return amax >= 6e-36f && amax < INFINITY; }
__device__ __forceinline__ float scale_of(float amax, float quotient) {
  return usable(amax) ? quotient : amax < 6e-36f ? 1.f : __uint_as_float(0x7FC00000u);
}
// x / 448 by its reciprocal in two parts, off by 2^-48 before the rounding.  A seventh has a distance of a fourteenth of a
// unit in the last place at least from where the rounding turns: this is the rounded quotient.
__device__ __forceinline__ float over_448(float x) {
  constexpr float hi = static_cast<float>(1.0 / 448), lo = static_cast<float>(1.0 / 448 - static_cast<double>(hi));
  return fmaf(x, hi, x * lo);
}
// y / d, rounded once: the reciprocal in two parts, its rounded value and what that leaves, so that the quotient is off by
// 2^-46 of itself before its rounding (while d is below 2^100 and the second part a normal number).  The rounded reciprocal
// alone misses neighbours of a border between two 8-bit values, and bf16 rows hold many quotients that lie on one (63.5 steps
// at half of a largest value that is a power of two).  4 of about 100 instructions per eight columns, and registers that have
// to be held at 32 for whole occupancy: 16384 x 4096 to int8 71.1 us (70.3 with the reciprocal alone), to e4m3 72.1 (71.6),
// plain int8 rows 33.9 (34.1).
//
// int8 divides by the stored scale.  e4m3 divides two exact numbers: rsqrt is the same factor in y and max|y|, so that only
// its power of two is kept there (7/8 of it, since 448 is 7/8 of 2^9); s * w is a product of two bf16 numbers, t = 7/8 s w
// has 19 bits, and 448 y / max|y| is t over a 448-th of the largest t.  It lies on a border between two values exactly
// where it does in real numbers, and takes the even one.  (The weight 1 + w of a zero-centred norm has more bits: one
// rounding.)
struct Divisor {
  uint64_t high, low;                              // 1 / d in two parts; 0, 0: everything finite becomes 0
  __device__ __forceinline__ Divisor(bool some, float d) : high(0), low(0) {
    if (!some) return;
    const float r = __frcp_rn(d), rest = fmaf(-d, r, 1.f) * r;
    high = pair(r, r);
    low = pair(rest, rest);
  }
  __device__ __forceinline__ uint64_t divide(uint64_t y) const {
    uint64_t q;
    asm("{\n\t.reg .b64 t;\n\t"
        "mul.rn.f32x2 t, %1, %3;\n\t"
        "fma.rn.f32x2 %0, %1, %2, t;\n\t}"
        : "=l"(q) : "l"(y), "l"(high), "l"(low));
    return q;
  }
};
__device__ __forceinline__ void widen4x2(const uint4& u, uint64_t (&f)[4]) {
  f[0] = pair(bf16_lo(u.x), bf16_hi(u.x));
  f[1] = pair(bf16_lo(u.y), bf16_hi(u.y));
  f[2] = pair(bf16_lo(u.z), bf16_hi(u.z));
  f[3] = pair(bf16_lo(u.w), bf16_hi(u.w));
}
// bf16(a + b) of two pairs.  One rounding of the exact sum is what an fp32 addition followed by a rounding gives: the fp32
// sum of two bf16 numbers is inexact only where one of them is too small to move the other at all.
__device__ __forceinline__ uint32_t add_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 s = __hadd2_rn(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&s);
}

// How a thread's i-th eight columns lie and are accessed:
//   kVec    eight neighbouring columns in one access; every row starts on a 16-byte boundary, H is a multiple of 8
//   kPair   four pairs, neighbouring threads side by side in each, 4 bytes per access; rows start on 4-byte boundaries, H
//           is even
//   kSingle the same pairs, element by element
//   kBlock  eight neighbouring columns element by element (e4m3 blocks in rows on any address)
// (515 x 1990: 8.6 us with eight neighbouring columns element by element, 3.6 us with pairs.)
enum Access { kVec, kPair, kSingle, kBlock };

template <Access A, int TPR>
__device__ __forceinline__ int column(int tid, int i, int j) {     // of pair j
  return A == kVec || A == kBlock ? 8 * (tid + i * TPR) + 2 * j : 2 * (tid + (4 * i + j) * TPR);
}
// Whether the warp of this thread has columns in round i at all (16384 x 5120: 102 us, 109 when all warps go through both
// rounds).
template <Access A, int TPR>
__device__ __forceinline__ bool warp_has(int tid, int i, int H) { return column<A, TPR>(tid & ~31, i, 0) < H; }
// Columns from H on read as zero.
template <Access A, int TPR>
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* row, int tid, int i, int H) {
  if constexpr (A == kVec) {
    const int c = column<A, TPR>(tid, i, 0);
    return c < H ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
  } else {
    const uint16_t* r = reinterpret_cast<const uint16_t*>(row);
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = column<A, TPR>(tid, i, j);
      if constexpr (A == kPair) u[j] = c < H ? *reinterpret_cast<const uint32_t*>(r + c) : 0u;
      else u[j] = (c < H ? r[c] : 0u) | (c + 1 < H ? static_cast<uint32_t>(r[c + 1]) << 16 : 0u);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
}
template <Access A, int TPR>
__device__ __forceinline__ void store8(__nv_bfloat16* row, int tid, int i, int H, const uint4& v) {
  if constexpr (A == kVec) {
    const int c = column<A, TPR>(tid, i, 0);
    if (c < H) *reinterpret_cast<uint4*>(row + c) = v;
  } else {
    uint16_t* r = reinterpret_cast<uint16_t*>(row);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = column<A, TPR>(tid, i, j);
      if constexpr (A == kPair) {
        if (c < H) *reinterpret_cast<uint32_t*>(r + c) = u[j];
      } else {
        if (c < H) r[c] = static_cast<uint16_t>(u[j]);
        if (c + 1 < H) r[c + 1] = static_cast<uint16_t>(u[j] >> 16);
      }
    }
  }
}
template <Access A, int TPR>
__device__ __forceinline__ void store8_bytes(uint8_t* row, int tid, int i, int H, uint32_t lo, uint32_t hi) {
  if constexpr (A == kVec) {
    const int c = column<A, TPR>(tid, i, 0);
    if (c < H) *reinterpret_cast<uint2*>(row + c) = make_uint2(lo, hi);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = column<A, TPR>(tid, i, j);
      const uint32_t b = (j < 2 ? lo : hi) >> (16 * (j & 1));
      if constexpr (A == kPair) {
        if (c < H) *reinterpret_cast<uint16_t*>(row + c) = static_cast<uint16_t>(b);
      } else {
        if (c < H) row[c] = static_cast<uint8_t>(b);
        if (c + 1 < H) row[c + 1] = static_cast<uint8_t>(b >> 8);
      }
    }
  }
}

// TPR threads share a row (a whole CTA, or one of the CTA's four warps when TPR is 32); NV times 8 columns per thread.
template <int TPR, int NV, bool E4M3, Access A>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR, NV <= 2 && A == kVec ? 2048 / (TPR == 32 ? 128 : TPR) : 1)
norm_quant_kernel(const NormQuantParams p) {
  __shared__ float red_sum[32];
  __shared__ uint32_t red_max[32];
  const int tid = TPR == 32 ? (threadIdx.x & 31) : threadIdx.x;
  const long long row = TPR == 32 ? static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
  if (TPR == 32 && row >= p.rows) return;     // whole warps leave, and no block barrier follows
  const __nv_bfloat16* xr = p.x + row * p.ldx;
  const __nv_bfloat16* dr = p.delta != nullptr ? p.delta + row * p.ldd : nullptr;

  wait_for_previous_kernel();
  let_next_kernel_start();
  uint4 v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    v[i] = load8<A, TPR>(xr, tid, i, p.H);
  }
  if (dr != nullptr) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint4 d = load8<A, TPR>(dr, tid, i, p.H);
      v[i] = make_uint4(add_bf16x2(v[i].x, d.x), add_bf16x2(v[i].y, d.y), add_bf16x2(v[i].z, d.z), add_bf16x2(v[i].w, d.w));
    }
  }
  if (p.s != nullptr) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      store8<A, TPR>(p.s + row * p.lds, tid, i, p.H, v[i]);
    }
  }
  float rstd = 1.f;
  if (p.w != nullptr) {
    uint64_t ss2 = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      uint64_t f[4];
      widen4x2(v[i], f);
#pragma unroll
      for (int j = 0; j < 4; ++j) ss2 = fma2(f[j], f[j], ss2);
    }
    float a, b;
    unpair(ss2, a, b);
    rstd = __frsqrt_rn(__fdiv_rn(row_sum<TPR>(a + b, red_sum), static_cast<float>(p.H)) + p.eps);
  }

  // e4m3: the power of two of rsqrt goes into y, its mantissa into the scales (1 where there is none: 0, infinity)
  const float factor = E4M3 ? 0.875f * __uint_as_float(__float_as_uint(rstd) & 0x7F800000u) : rstd;
  const float mantissa = __uint_as_float((__float_as_uint(rstd) & 0x007FFFFFu) | 0x3F800000u);

  // y of eight columns, in fp32 (recomputed where it is needed twice and not kept: the registers hold the bf16 sum)
  auto normed = [&](int i, uint64_t (&f)[4]) {
    widen4x2(v[i], f);
    if (p.w == nullptr) return;
    uint64_t g[4];
    widen4x2(load8<A, TPR>(p.w, tid, i, p.H), g);
    if (p.zero_centered) {
#pragma unroll
      for (int j = 0; j < 4; ++j) g[j] = add2(g[j], pair(1.f, 1.f));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = mul2(mul2(f[j], pair(factor, factor)), g[j]);
  };
  auto top_of = [](const uint64_t (&f)[4]) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a, b;
      unpair(f[j], a, b);
      m = max_nan(m, max_nan(fabsf(a), fabsf(b)));
    }
    return m;
  };
  uint8_t* qr = p.q + row * p.ldq;
  if constexpr (E4M3) {
    // 128 columns are 16 neighbouring lanes
    const int kbs = p.H / 128;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i > 0 && !warp_has<A, TPR>(tid, i, p.H)) break;
      const int k = tid + i * TPR;
      uint64_t f[4];
      normed(i, f);
      float m = top_of(f);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (k * 8 >= p.H) continue;
      const float top = over_448(m), amax = top * 512.f * mantissa;
      const Divisor by(usable(amax), top);
      uint32_t out[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float a, b, c, d;
        unpair(by.divide(f[2 * h]), a, b);
        unpair(by.divide(f[2 * h + 1]), c, d);
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
        out[h] = lo | (hi << 16);
      }
      store8_bytes<A, TPR>(qr, tid, i, p.H, out[0], out[1]);
      if ((k & 15) == 0) p.scale[row * kbs + (k >> 4)] = scale_of(amax, over_448(amax));
    }
  } else {
    constexpr bool kKeep = NV <= 2;            // y stays in registers where it is small
    uint64_t y[kKeep ? NV : 1][4];
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      uint64_t (&f)[4] = y[kKeep ? i : 0];
      normed(i, f);
      m = max_nan(m, top_of(f));
    }
    m = row_max<TPR>(m, red_max);
    const float scale = scale_of(m, __fdiv_rn(m, 127.f));
    const Divisor by(usable(m), scale);
    if (tid == 0) p.scale[row] = scale;
    const bool some = usable(m);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i > 0 && !warp_has<A, TPR>(tid, i, p.H)) break;
      uint64_t (&f)[4] = y[kKeep ? i : 0];
      if constexpr (!kKeep) normed(i, f);
      uint32_t out[2] = {0u, 0u};
      if (some) {                              // rows without a scale become zeros, whatever they hold
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // y / scale + 1.5 * 2^23 leaves the nearest integer (ties to even) in the low bits; |y / scale| <= 127 up to rounding
          uint32_t r[4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float a, b;
            unpair(add2(by.divide(f[2 * h + j]), pair(12582912.f, 12582912.f)), a, b);
            r[2 * j] = __float_as_uint(a);
            r[2 * j + 1] = __float_as_uint(b);
          }
          out[h] = __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
        }
      }
      store8_bytes<A, TPR>(qr, tid, i, p.H, out[0], out[1]);
    }
  }
}

template <int TPR, bool E4M3, Access A>
static cudaError_t launch_norm_quant(const NormQuantParams& p, int nv, cudaStream_t stream) {
  const int threads = TPR == 32 ? 128 : TPR;
  const long long blocks = TPR == 32 ? (p.rows + 3) / 4 : p.rows;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr = overlap_launch();
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (nv <= 1) return cudaLaunchKernelEx(&cfg, norm_quant_kernel<TPR, 1, E4M3, A>, p);
  if (nv <= 2) return cudaLaunchKernelEx(&cfg, norm_quant_kernel<TPR, 2, E4M3, A>, p);
  return cudaLaunchKernelEx(&cfg, norm_quant_kernel<TPR, 4, E4M3, A>, p);
}

template <bool E4M3, Access A>
static cudaError_t dispatch_norm_quant(const NormQuantParams& p, cudaStream_t stream) {
  // Threads per row: two vectors per thread, so that a row's loads are in flight together and an SM holds many rows
  // (16384 x 4096 with 1, 2, 4, 8 vectors: 89, 85, 87, 100 us before the paired arithmetic).
  const int nvec = (p.H + 7) / 8;
  if (nvec <= 64) return launch_norm_quant<32, E4M3, A>(p, (nvec + 31) / 32, stream);
  if (nvec <= 128) return launch_norm_quant<64, E4M3, A>(p, 2, stream);
  if (nvec <= 256) return launch_norm_quant<128, E4M3, A>(p, 2, stream);
  if (nvec <= 512) return launch_norm_quant<256, E4M3, A>(p, 2, stream);
  if (nvec <= 1024) return launch_norm_quant<512, E4M3, A>(p, 2, stream);
  return launch_norm_quant<1024, E4M3, A>(p, (nvec + 1023) / 1024, stream);
}

}  // namespace stb

using namespace stb;

// fmt 0: int8 with scale [rows]; fmt 1: e4m3 with scale [rows][H / 128] (H a multiple of 128).  Strides in elements.
extern "C" int stb_norm_quant(const void* x, const void* delta, const void* w, void* s, void* q, float* scale,
                              long long rows, int H, long long ldx, long long ldd, long long lds, long long ldq,
                              float eps, int zero_centered, int fmt, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (H <= 0 || H > kNqMaxThreads * kNqMaxVec * 8 || rows > 0x7FFFFFFFll || (fmt == 1 && H % 128)) return -kErrBadArgument;
  NormQuantParams p{};
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.delta = static_cast<const __nv_bfloat16*>(delta);
  p.w = static_cast<const __nv_bfloat16*>(w);
  p.s = static_cast<__nv_bfloat16*>(s);
  p.q = static_cast<uint8_t*>(q);
  p.scale = scale;
  p.rows = rows; p.ldx = ldx; p.ldd = ldd; p.lds = lds; p.ldq = ldq;
  p.H = H; p.eps = eps; p.zero_centered = zero_centered;
  auto on16 = [](const void* t, long long ld) { return t == nullptr || (reinterpret_cast<uintptr_t>(t) % 16 == 0 && ld % 8 == 0); };
  const bool vec = H % 8 == 0 && on16(x, ldx) && on16(delta, ldd) && on16(s, lds) && on16(w, 0) &&
                   reinterpret_cast<uintptr_t>(q) % 8 == 0 && ldq % 8 == 0;
  cudaError_t e;
  auto on4 = [](const void* t, long long ld) { return t == nullptr || (reinterpret_cast<uintptr_t>(t) % 4 == 0 && ld % 2 == 0); };
  const bool pairs = H % 2 == 0 && on4(x, ldx) && on4(delta, ldd) && on4(s, lds) && on4(w, 0) &&
                     reinterpret_cast<uintptr_t>(q) % 2 == 0 && ldq % 2 == 0;
  if (fmt == 1) e = vec ? dispatch_norm_quant<true, kVec>(p, stream) : dispatch_norm_quant<true, kBlock>(p, stream);
  else if (vec) e = dispatch_norm_quant<false, kVec>(p, stream);
  else e = pairs ? dispatch_norm_quant<false, kPair>(p, stream) : dispatch_norm_quant<false, kSingle>(p, stream);
  return -static_cast<int>(e);
}
