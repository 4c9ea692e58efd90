// INT8 linear layer with a scale per token (row of x) and per output channel:
//
//   s_m  = max(max_k |x_mk| / 127, 2^-126)            (fp32, rounded once)
//   q_mk = x_mk / s_m rounded to the nearest integer  (ties to even)
//   y_mn = act(s_m t_n sum_k q_mk w_nk + b_n)         (w_nk, t_n: the weights'
//                                                      codes and scales, made
//                                                      by the same quantiser)
//
// the numerics that tocr_dwpw_block uses per pixel, for the recognizer's
// linear layers. The sum is exact in s32 (K up to 131072); the epilogue is
// fp32 and rounds once to the output type. A row that holds an infinity or a
// NaN gets the scale NaN, so its outputs are NaN instead of silently wrong.
//
// Quantiser: one pass over x from memory (a row's values stay in registers
// between its maximum and its codes); bound by HBM.
//
// Product: one persistent CTA per SM. Warp 0 loads 128 x 128-byte tiles of
// the token codes and BN x 128-byte tiles of the weight codes by TMA (128-byte
// swizzle) into a ring, one thread of warp 1 issues tcgen05.mma kind::i8
// (M 128, N = BN, K 32) into one of two TMEM accumulators, eight epilogue warps
// read the other, scale, add the bias, apply the activation and write the rows
// out through shared memory (a row piece of 128 bytes per store instruction,
// whatever the alignment of y's rows: the dictionary's 18385 columns leave
// every other row on an odd 2-byte boundary, where TMA cannot store). BN is
// 256, or 128 or 64 where larger tiles would leave SMs idle.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "tc_ptx.cuh"
#include "tma_map.cuh"
#include "tocr_common.cuh"

namespace tocr {
namespace {

using namespace ptx;

// --------------------------------------------------------------- quantiser --
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// x / s to the nearest integer, ties to even, of the exact quotient. q is the
// product with 1/s rounded by adding 1.5 * 2^23 (one fused step); the rounding
// of 1/s can only miss next to a border, so where the remainder r = x - q s
// reaches half a step it decides (it is exact there: x and q s are on grids no
// finer than s 2^-24). Returns the sum, whose low byte is the code.
constexpr float kMagic = 12582912.f;
__device__ __forceinline__ float code_sum(float x, float s, float inv, float &r) {
  const float t = fmaf(x, inv, kMagic);
  r = fmaf(kMagic - t, s, x);
  return t;
}
__device__ __noinline__ float code_exact(float x, float s, float inv) {
  float r;
  float q = code_sum(x, s, inv, r) - kMagic;
  const float h = 0.5f * s;
  const bool odd = (static_cast<int>(q) & 1) != 0;
  if (r > h || (r == h && odd)) q += 1.f;
  else if (r < -h || (r == -h && odd)) q -= 1.f;
  return q + kMagic;
}
// four codes, first in the low byte
__device__ __forceinline__ uint32_t codes4(const float (&x)[4], float s, float inv) {
  float t[4], r[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) t[k] = code_sum(x[k], s, inv, r[k]);
  const float far = fmaxf(fmaxf(fabsf(r[0]), fabsf(r[1])), fmaxf(fabsf(r[2]), fabsf(r[3])));
  if (far >= 0.5f * s) {
#pragma unroll
    for (int k = 0; k < 4; ++k) t[k] = code_exact(x[k], s, inv);
  }
  return __byte_perm(__byte_perm(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040),
                     __byte_perm(__float_as_uint(t[2]), __float_as_uint(t[3]), 0x0040), 0x5410);
}

// largest |x| of a 16-byte vector, as the bits of the type (monotonic; an
// infinity or a NaN beats every number)
template <typename T>
__device__ __forceinline__ uint32_t top_of(const uint4 &w, uint32_t top) {
  if constexpr (sizeof(T) == 4) {
    const uint32_t m = 0x7fffffffu;
    return max(max(max(w.x & m, w.y & m), max(w.z & m, w.w & m)), top);
  } else {
    const uint32_t m = 0x7fff7fffu;  // two at a time
    return __vmaxu2(__vmaxu2(__vmaxu2(w.x & m, w.y & m), __vmaxu2(w.z & m, w.w & m)), top);
  }
}
template <typename T>
__device__ __forceinline__ uint32_t bits_of(T v) {
  if constexpr (sizeof(T) == 4)
    return __float_as_uint(v) & 0x7fffffffu;
  else
    return *reinterpret_cast<const uint16_t *>(&v) & 0x7fffu;
}
template <typename T>
__device__ __forceinline__ float from_bits(uint32_t b) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(b);
  } else {
    const uint16_t h = (uint16_t)b;
    return to_f32(*reinterpret_cast<const T *>(&h));
  }
}

constexpr int kQuantThreads = 256;

// One team of TEAM threads per row. VEC: rows start on 16-byte boundaries, and
// a thread keeps KEEP vectors of its row between the two steps.
template <typename T, int TEAM, bool VEC, int KEEP>
__global__ void __launch_bounds__(kQuantThreads)
quant_rows_kernel(const T *__restrict__ x, long long rows, int K, int pitch,
                  int8_t *__restrict__ q, float *__restrict__ scale) {
  constexpr int E = 16 / sizeof(T);
  constexpr int TEAMS = kQuantThreads / TEAM;
  __shared__ uint32_t smax[kQuantThreads / 32];
  const int tid = threadIdx.x % TEAM;
  const long long row = (long long)blockIdx.x * TEAMS + threadIdx.x / TEAM;
  const bool live = row < rows;
  const T *xr = x + (live ? row : 0) * K;
  const uint4 *xv = reinterpret_cast<const uint4 *>(xr);
  uint32_t top = 0;
  uint4 keep[KEEP];
  const int nv = VEC && live ? K / E : 0;
  if (VEC) {
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      const int v = tid + i * TEAM;
      keep[i] = v < nv ? __ldg(xv + v) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < KEEP; ++i) top = top_of<T>(keep[i], top);
    for (int v = tid + KEEP * TEAM; v < nv; v += TEAM) top = top_of<T>(__ldg(xv + v), top);
    if (sizeof(T) == 2) top = max(top & 0xffffu, top >> 16);
  } else if (live) {
#pragma unroll 4
    for (int k = tid; k < K; k += TEAM) top = max(top, bits_of(xr[k]));
  }
  top = __reduce_max_sync(~0u, top);
  if (TEAM > 32) {
    if ((threadIdx.x & 31) == 0) smax[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TEAM / 32; ++i) top = max(top, smax[threadIdx.x / TEAM * (TEAM / 32) + i]);
  }
  if (!live) return;
  const float big = from_bits<T>(top);
  const bool finite = big < INFINITY;  // false for NaN too
  const float s = finite ? fmaxf(big / 127.f, 1.17549435e-38f) : __uint_as_float(0x7fc00000u);
  if (tid == 0) scale[row] = s;
  const float inv = 1.f / s;
  int8_t *qr = q + row * pitch;
  if (VEC) {
    auto put = [&](int v, const uint4 &w) {
      const T *e = reinterpret_cast<const T *>(&w);
      uint32_t p[E / 4];
#pragma unroll
      for (int k = 0; k < E; k += 4) {
        const float f[4] = {to_f32(e[k]), to_f32(e[k + 1]), to_f32(e[k + 2]), to_f32(e[k + 3])};
        p[k / 4] = finite ? codes4(f, s, inv) : 0u;
      }
      if constexpr (E == 8)
        reinterpret_cast<uint2 *>(qr)[v] = make_uint2(p[0], p[1]);
      else
        reinterpret_cast<uint32_t *>(qr)[v] = p[0];
    };
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      const int v = tid + i * TEAM;
      if (v < nv) put(v, keep[i]);
    }
    for (int v = tid + KEEP * TEAM; v < nv; v += TEAM) put(v, __ldg(xv + v));
    for (int k = K + tid; k < pitch; k += TEAM) qr[k] = 0;  // the pad behind K
  } else {
    for (int k = 4 * tid; k < pitch; k += 4 * TEAM) {
      float f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = k + j < K ? to_f32(xr[k + j]) : 0.f;
      *reinterpret_cast<uint32_t *>(qr + k) = finite ? codes4(f, s, inv) : 0u;
    }
  }
}

template <typename T>
int launch_quant(const void *x, long long rows, int K, int8_t *q, float *scale, cudaStream_t st) {
  const int pitch = (K + 15) / 16 * 16;
  const T *xt = static_cast<const T *>(x);
  const size_t bytes = (size_t)K * sizeof(T);
  const bool vec = aligned(x, 16) && bytes % 16 == 0;
  // a warp per row while its lanes can keep the row (16 vectors each: 8 KB),
  // else a CTA per row
  const unsigned warps = (unsigned)((rows + 7) / 8), ctas = (unsigned)rows;
  constexpr int B = kQuantThreads;
  if (vec && bytes <= 32 * 16 * 4)
    quant_rows_kernel<T, 32, true, 4><<<warps, B, 0, st>>>(xt, rows, K, pitch, q, scale);
  else if (vec && bytes <= 32 * 16 * 16 && rows >= 8 * sm_count())
    quant_rows_kernel<T, 32, true, 16><<<warps, B, 0, st>>>(xt, rows, K, pitch, q, scale);
  else if (vec)
    quant_rows_kernel<T, 256, true, 8><<<ctas, B, 0, st>>>(xt, rows, K, pitch, q, scale);
  else if (bytes <= 32 * 16 * 4)
    quant_rows_kernel<T, 32, false, 1><<<warps, B, 0, st>>>(xt, rows, K, pitch, q, scale);
  else
    quant_rows_kernel<T, 256, false, 1><<<ctas, B, 0, st>>>(xt, rows, K, pitch, q, scale);
  return check_launch("quant_rows_kernel");
}

int quant_rows(const void *x, int dtype, long long rows, int K, int8_t *q, float *scale,
               cudaStream_t st) {
  if (dtype == TOCR_DTYPE_F16) return launch_quant<__half>(x, rows, K, q, scale, st);
  if (dtype == TOCR_DTYPE_BF16) return launch_quant<__nv_bfloat16>(x, rows, K, q, scale, st);
  return launch_quant<float>(x, rows, K, q, scale, st);
}

// ----------------------------------------------------------------- product --
constexpr int kBM = 128;
constexpr int kEpiWarp0 = 2, kEpiWarps = 8;
constexpr int kThreads = 32 * (kEpiWarp0 + kEpiWarps);
constexpr int kPitchW = 36;  // words of a staged row piece: 32, and 4 against bank conflicts

template <int BN>
struct Cfg {
  static constexpr int STAGE_A = kBM * 128, STAGE_B = BN * 128;
  static constexpr int STAGE = STAGE_A + STAGE_B;
  static constexpr int STAGES = BN == 256 ? 3 : BN == 128 ? 5 : 7;
  static constexpr int OFF_BAR = STAGES * STAGE;
  static constexpr int OFF_MISC = OFF_BAR + (2 * STAGES + 4) * 8;
  static constexpr int OFF_STG = (OFF_MISC + 16 + 15) / 16 * 16;
  static constexpr int OFF_COL = OFF_STG + kEpiWarps * 32 * kPitchW * 4;
  static constexpr int SMEM = OFF_COL + kEpiWarps * 64 * 8 + 1024;
  static constexpr int TMEM = 2 * BN;
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct LinParams {
  const float *sx, *sw, *bias;
  void *y;
  long long rows;
  int N, ksteps, K;
  long long tiles_n, tiles;
  int act;
  bool vec;          // rows of y start on 16-byte boundaries
  int *err;
};

// One 32-row piece of y (32 words per row at most, PC columns from `col` on,
// clipped at N), staged by the calling warp at stg (row pitch kPitchW words),
// to global memory. vec: every row of y starts on a 16-byte boundary.
template <typename T, int PC>
__device__ __forceinline__ void write_piece(T *y, long long row0, long long rows, int N, int col,
                                            bool vec, const uint32_t *stg, int lane) {
  constexpr int PER = 4 / sizeof(T);      // elements per word
  constexpr int W = PC / PER;             // words of a row
  const int n = min(N - col, PC);         // elements of a row
  const int nr = (int)min((long long)32, rows - row0);
  T *o = y + row0 * N + col;
  if (vec && n == PC) {
    constexpr int LPR = W / 4, RPI = 32 / LPR;  // lanes per row, rows per instruction
    const int r = lane / LPR, w = lane % LPR * 4;
#pragma unroll 8
    for (int r0 = 0; r0 < 32; r0 += RPI)
      if (r0 + r < nr)
        *reinterpret_cast<uint4 *>(reinterpret_cast<uint32_t *>(o + (long long)(r0 + r) * N) + w) =
            *reinterpret_cast<const uint4 *>(stg + (r0 + r) * kPitchW + w);
  } else if constexpr (PER == 1) {
    if (lane < n)
#pragma unroll 8
      for (int r = 0; r < 32; ++r)
        if (r < nr) reinterpret_cast<uint32_t *>(o + (long long)r * N)[lane] = stg[r * kPitchW + lane];
  } else {
    // 4-byte stores on 4-byte boundaries: a row that starts between two takes
    // its words one element further on, and its first element on its own
#pragma unroll 8
    for (int r = 0; r < 32; ++r) {
      if (r >= nr) break;
      uint16_t *orow = reinterpret_cast<uint16_t *>(o + (long long)r * N);
      const uint32_t a = stg[r * kPitchW + lane], b = stg[r * kPitchW + lane + 1];
      const int odd = (int)(reinterpret_cast<uintptr_t>(orow) >> 1) & 1;
      const int e = 2 * lane + odd;
      if (e + 1 < n)
        *reinterpret_cast<uint32_t *>(orow + e) = odd ? __byte_perm(a, b, 0x5432) : a;
      else if (e < n)
        orow[e] = (uint16_t)(odd ? a >> 16 : a);
      if (odd && lane == 0) orow[0] = (uint16_t)a;
    }
  }
}

__device__ __forceinline__ float activate(float y, int act) {
  if (act == TOCR_ACT_RELU) return y < 0.f ? 0.f : y;  // keeps NaN
  if (act == TOCR_ACT_HARDSWISH) return y * (fminf(fmaxf(y + 3.f, 0.f), 6.f) * (1.f / 6.f));
  return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// SMALLK: |sum| < 2^22, so an s32 becomes fp32 by adding it to the bits of
// 1.5 * 2^23 (two full-rate instructions; the conversion instruction runs at an
// eighth of their rate and would bound layers of small K).
template <typename T, int BN, bool SMALLK>
__global__ void __launch_bounds__(kThreads, 1)
linear_i8_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
                 const LinParams p) {
  using C = Cfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::OFF_BAR);
  uint64_t *empty = full + C::STAGES;
  uint64_t *acc_full = empty + C::STAGES;  // [2]
  uint64_t *acc_empty = acc_full + 2;      // [2]
  uint32_t *s_tmem = reinterpret_cast<uint32_t *>(smem + C::OFF_MISC);
  volatile int *s_abort = reinterpret_cast<volatile int *>(smem + C::OFF_MISC + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], kEpiWarps);
    }
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(s_tmem, C::TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const int KS = p.ksteps;

  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&xmap);
      tma_prefetch_desc(&wmap);
      long long j = 0;
      bool ok = true;
      for (long long t = blockIdx.x; ok && t < p.tiles; t += gridDim.x) {
        const int m0 = (int)(t / p.tiles_n) * kBM, n0 = (int)(t % p.tiles_n) * BN;
        for (int k = 0; k < KS; ++k, ++j) {
          const int s = (int)(j % C::STAGES);
          const uint32_t u = (uint32_t)(j / C::STAGES);
          if (u > 0 && !mbar_wait_bounded(&empty[s], (u - 1) & 1, s_abort, p.err, 81)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[s], C::STAGE);
          tma_load_2d(smem + s * C::STAGE, &xmap, &full[s], 128 * k, m0);
          tma_load_2d(smem + s * C::STAGE + C::STAGE_A, &wmap, &full[s], 128 * k, n0);
        }
      }
      if (*s_abort) {  // leave no copy in flight
        for (long long i = j > C::STAGES ? j - C::STAGES : 0; i < j; ++i) {
          const long long t0 = clock64();
          while (!mbar_try_wait(&full[i % C::STAGES], (uint32_t)(i / C::STAGES) & 1))
            if (clock64() - t0 > (1ll << 30)) break;
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = idesc_i8(kBM, BN);
      long long j = 0;
      int i = 0;
      bool ok = true;
      for (long long t = blockIdx.x; ok && t < p.tiles; t += gridDim.x, ++i) {
        const int b = i & 1;
        if (i > 1 && !mbar_wait_bounded(&acc_empty[b], (uint32_t)((i >> 1) - 1) & 1, s_abort, p.err, 82))
          break;
        tc_fence_after();
        for (int k = 0; k < KS; ++k, ++j) {
          const int s = (int)(j % C::STAGES);
          if (!mbar_wait_bounded(&full[s], (uint32_t)(j / C::STAGES) & 1, s_abort, p.err, 83)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = smem_u32(smem + s * C::STAGE), w = a + C::STAGE_A;
#pragma unroll
          for (int q = 0; q < 4; ++q)
            mma_i8(tmem + (uint32_t)(b * BN), sw128_kmajor_desc(a + 32u * q),
                   sw128_kmajor_desc(w + 32u * q), idesc, k > 0 || q > 0 ? 1u : 0u);
          mma_commit(&empty[s]);
        }
        mma_commit(&acc_full[b]);
      }
    }
  } else {
    const int ew = warp - kEpiWarp0;
    const int half = ew >> 2;   // its columns of the tile
    const int quad = warp & 3;  // the TMEM lanes a warp may read
    uint32_t *stg = reinterpret_cast<uint32_t *>(smem + C::OFF_STG) + ew * 32 * kPitchW;
    float2 *cols = reinterpret_cast<float2 *>(smem + C::OFF_COL) + ew * 64;
    constexpr int HC = BN / 2;                 // columns of a warp
    constexpr int PC = 32 * (4 / sizeof(T)) < HC ? 32 * (4 / sizeof(T)) : HC;  // of a piece
    constexpr int PER = 4 / sizeof(T);
    T *y = static_cast<T *>(p.y);
    int i = 0;
    for (long long t = blockIdx.x; t < p.tiles; t += gridDim.x, ++i) {
      const int b = i & 1;
      const long long row0 = t / p.tiles_n * kBM + quad * 32;
      const int n0 = (int)(t % p.tiles_n) * BN + half * HC;
      const float sx = row0 + lane < p.rows ? __ldg(p.sx + row0 + lane) : 0.f;
      if (!mbar_wait_bounded(&acc_full[b], (uint32_t)(i >> 1) & 1, s_abort, p.err, 84)) break;
      tc_fence_after();
      const uint32_t ta = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(b * BN + half * HC);
#pragma unroll 1
      for (int c = 0; c < HC; c += PC) {
        if (n0 + c >= p.N) break;
        __syncwarp();
#pragma unroll
        for (int g = 0; g < PC; g += 32) {
          const int n = n0 + c + g + lane;
          cols[g + lane] = n < p.N ? make_float2(__ldg(p.sw + n), p.bias ? __ldg(p.bias + n) : 0.f)
                                   : make_float2(0.f, 0.f);
        }
        __syncwarp();
#pragma unroll
        for (int g = 0; g < PC; g += 32) {
          uint32_t v[32];
          tmem_ld32(ta + c + g, v);
          tmem_ld_wait(v);
          uint32_t o[32 / PER];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float4 cc = *reinterpret_cast<const float4 *>(&cols[g + e]);
            const float a0 = SMALLK ? __uint_as_float(v[e] + 0x4B400000u) - 12582912.f
                                    : (float)(int)v[e];
            const float a1 = SMALLK ? __uint_as_float(v[e + 1] + 0x4B400000u) - 12582912.f
                                    : (float)(int)v[e + 1];
            const float y0 = activate(fmaf(a0 * sx, cc.x, cc.y), p.act);
            const float y1 = activate(fmaf(a1 * sx, cc.z, cc.w), p.act);
            if constexpr (PER == 2) {
              o[e / 2] = pack2<T>(y0, y1);
            } else {
              o[e] = __float_as_uint(y0);
              o[e + 1] = __float_as_uint(y1);
            }
          }
          uint4 *so = reinterpret_cast<uint4 *>(stg + lane * kPitchW + g / PER);
#pragma unroll
          for (int e = 0; e < 8 / PER; ++e)
            so[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
        __syncwarp();
        if (row0 < p.rows) write_piece<T, PC>(y, row0, p.rows, p.N, n0 + c, p.vec, stg, lane);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[b]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM);
  }
}

template <typename T, int BN, bool SMALLK>
int launch_product(const void *xq, const void *wq, const LinParams &p, int pitch, cudaStream_t st) {
  using C = Cfg<BN>;
  CUtensorMap xm, wm;
  int rc = tma_map_rows(&xm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, xq, pitch, p.rows, pitch, kBM);
  if (rc) return rc;
  rc = tma_map_rows(&wm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, wq, pitch, p.N, pitch, BN);
  if (rc) return rc;
  cudaError_t e = cudaFuncSetAttribute(linear_i8_kernel<T, BN, SMALLK>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return set_error(TOCR_ERR_CUDA, "tocr_linear_i8: %s", cudaGetErrorString(e));
  const int grid = (int)(p.tiles < sm_count() ? p.tiles : sm_count());
  linear_i8_kernel<T, BN, SMALLK><<<grid, kThreads, C::SMEM, st>>>(xm, wm, p);
  return check_launch("linear_i8_kernel");
}

template <typename T, int BN>
int product_bn(const void *xq, const void *wq, LinParams p, int pitch, cudaStream_t st) {
  p.tiles_n = (p.N + BN - 1) / BN;
  p.tiles = (p.rows + kBM - 1) / kBM * p.tiles_n;
  // 127^2 K < 2^22
  return p.K <= 260 ? launch_product<T, BN, true>(xq, wq, p, pitch, st)
                    : launch_product<T, BN, false>(xq, wq, p, pitch, st);
}

template <typename T>
int product(const void *xq, const void *wq, const LinParams &p, int pitch, cudaStream_t st) {
  // the tile width whose waves of CTAs take least: a tile costs its columns and
  // a fixed part worth about 64 columns
  const long long tm = (p.rows + kBM - 1) / kBM, sms = sm_count();
  long long best = -1;
  int bn = 256;
  for (int b = 256; b >= 64; b /= 2) {
    const long long cost = (tm * ((p.N + b - 1) / b) + sms - 1) / sms * (b + 64);
    if (best < 0 || cost < best) {
      best = cost;
      bn = b;
    }
  }
  if (bn == 256) return product_bn<T, 256>(xq, wq, p, pitch, st);
  if (bn == 128) return product_bn<T, 128>(xq, wq, p, pitch, st);
  return product_bn<T, 64>(xq, wq, p, pitch, st);
}

constexpr long long kMaxRows = 1ll << 24;
constexpr int kMaxK = 1 << 17;  // 127^2 K stays inside s32
constexpr int kMaxN = 1 << 24;

bool is_dtype(int d) {
  return d == TOCR_DTYPE_F16 || d == TOCR_DTYPE_BF16 || d == TOCR_DTYPE_F32;
}

int check_linear(const char *fn, long long rows, int K, int N, int act, int out_dtype) {
  TOCR_REQUIRE(rows >= 0 && rows <= kMaxRows && K > 0 && K <= kMaxK && N > 0 && N <= kMaxN,
               "%s: bad sizes rows=%lld K=%d N=%d", fn, rows, K, N);
  TOCR_REQUIRE(act == TOCR_ACT_NONE || act == TOCR_ACT_RELU || act == TOCR_ACT_HARDSWISH,
               "%s: unknown activation %d", fn, act);
  TOCR_REQUIRE(is_dtype(out_dtype), "%s: unknown output type %d", fn, out_dtype);
  return TOCR_OK;
}

int run_product(const void *xq, const float *sx, long long rows, int K, const void *wq,
                const float *sw, const float *bias, int N, int act, int out_dtype, void *y,
                int *err, cudaStream_t st) {
  LinParams p{};
  p.sx = sx;
  p.sw = sw;
  p.bias = bias;
  p.y = y;
  p.rows = rows;
  p.N = N;
  p.K = K;
  p.ksteps = (K + 127) / 128;
  p.act = act;
  p.vec = aligned(y, 16) && (size_t)N * (out_dtype == TOCR_DTYPE_F32 ? 4 : 2) % 16 == 0;
  p.err = err;
  const int pitch = (K + 15) / 16 * 16;
  if (out_dtype == TOCR_DTYPE_F16) return product<__half>(xq, wq, p, pitch, st);
  if (out_dtype == TOCR_DTYPE_BF16) return product<__nv_bfloat16>(xq, wq, p, pitch, st);
  return product<float>(xq, wq, p, pitch, st);
}

size_t codes_bytes(long long rows, int K) {
  return ((size_t)rows * ((K + 15) / 16 * 16) + 255) / 256 * 256;
}

}  // namespace
}  // namespace tocr

using namespace tocr;

extern "C" {

TOCR_API int tocr_quant_rows_i8(const void *d_x, int x_dtype, long long rows, int K, void *d_codes,
                                float *d_scales, void *stream) {
  TOCR_ENTRY();
  TOCR_REQUIRE(rows >= 0 && rows <= kMaxRows && K > 0 && K <= kMaxK,
               "tocr_quant_rows_i8: bad sizes rows=%lld K=%d", rows, K);
  TOCR_REQUIRE(is_dtype(x_dtype), "tocr_quant_rows_i8: unknown type %d", x_dtype);
  if (rows == 0) return TOCR_OK;
  TOCR_REQUIRE(d_x && d_codes && d_scales, "tocr_quant_rows_i8: null pointer");
  TOCR_REQUIRE(aligned(d_codes, 16), "tocr_quant_rows_i8: the codes must be 16-byte aligned");
  return quant_rows(d_x, x_dtype, rows, K, static_cast<int8_t *>(d_codes), d_scales,
                    as_stream(stream));
}

TOCR_API int tocr_linear_i8_codes(const void *d_xq, const float *d_sx, long long rows, int K,
                                  const void *d_wq, const float *d_sw, const float *d_bias, int N,
                                  int act, int out_dtype, void *d_y, int *d_err, void *stream) {
  TOCR_ENTRY();
  int rc = check_linear("tocr_linear_i8_codes", rows, K, N, act, out_dtype);
  if (rc || rows == 0) return rc;
  TOCR_REQUIRE(d_xq && d_sx && d_wq && d_sw && d_y && d_err, "tocr_linear_i8_codes: null pointer");
  TOCR_REQUIRE(aligned(d_xq, 16) && aligned(d_wq, 16),
               "tocr_linear_i8_codes: the codes must be 16-byte aligned");
  return run_product(d_xq, d_sx, rows, K, d_wq, d_sw, d_bias, N, act, out_dtype, d_y, d_err,
                     as_stream(stream));
}

TOCR_API size_t tocr_linear_i8_workspace_bytes(long long rows, int K) {
  if (rows < 0 || rows > kMaxRows || K <= 0 || K > kMaxK) return 0;
  return codes_bytes(rows, K) + (size_t)rows * 4;
}

TOCR_API int tocr_linear_i8(const void *d_x, int x_dtype, long long rows, int K, const void *d_wq,
                            const float *d_sw, const float *d_bias, int N, int act, int out_dtype,
                            void *d_y, void *d_workspace, size_t workspace_bytes, int *d_err,
                            void *stream) {
  TOCR_ENTRY();
  int rc = check_linear("tocr_linear_i8", rows, K, N, act, out_dtype);
  if (rc) return rc;
  TOCR_REQUIRE(is_dtype(x_dtype), "tocr_linear_i8: unknown type %d", x_dtype);
  if (rows == 0) return TOCR_OK;
  TOCR_REQUIRE(d_x && d_wq && d_sw && d_y && d_workspace && d_err, "tocr_linear_i8: null pointer");
  TOCR_REQUIRE(aligned(d_wq, 16), "tocr_linear_i8: the codes must be 16-byte aligned");
  TOCR_REQUIRE(aligned(d_workspace, 256) && workspace_bytes >= codes_bytes(rows, K) + (size_t)rows * 4,
               "tocr_linear_i8: the workspace must be 256-byte aligned and hold %zu bytes",
               codes_bytes(rows, K) + (size_t)rows * 4);
  cudaStream_t st = as_stream(stream);
  int8_t *q = static_cast<int8_t *>(d_workspace);
  float *sx = reinterpret_cast<float *>(q + codes_bytes(rows, K));
  rc = quant_rows(d_x, x_dtype, rows, K, q, sx, st);
  if (rc) return rc;
  return run_product(q, sx, rows, K, d_wq, d_sw, d_bias, N, act, out_dtype, d_y, d_err, st);
}

}  // extern "C"
