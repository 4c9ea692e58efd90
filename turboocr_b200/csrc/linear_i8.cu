// INT8 linear layer with a scale per token (row of x) and per output channel:
//
//   s_m  = max(max_k |x_mk| * (1 / 127), 2^-126)      (1 / 127 and the product
//                                                      rounded to fp32)
//   q_mk = x_mk / s_m rounded to the nearest integer  (ties to even)
//   y_mn = act(s_m t_n sum_k q_mk w_nk + b_n)         (w_nk, t_n: the weights'
//                                                      codes and scales, made
//                                                      by the same quantiser)
//
// for the recognizer's linear layers: symmetric codes and the two kinds of scales
// as in tocr_dwpw_block, but not its bits. That block and its packer divide the
// maximum by 127, which differs in the last place from the product here in one
// row of 22, and the block's codes are products with 127 / max instead of exact
// quotients by the scale. The sum is exact in s32 (K up to
// 131072, with codes of -128 on both sides one less); the epilogue is
// fp32, the channel's scale first (weights are of ordinary size, so neither the
// largest nor the least activations leave fp32's range on the way), and rounds
// once to the output type. A row that holds an infinity or a
// NaN gets the scale NaN, so its outputs are NaN instead of silently wrong.
//
// Quantiser: one pass over x from memory (a row's values stay in registers
// between its maximum and its codes). 16384 x 4096 bf16: 44 us, 4.6 TB/s of
// 6.4; bound by the loads in flight that the registers leave room for.
//
// Product: the output channels are the rows of the MMA (M 128, the lanes of
// tensor memory) and the tokens its columns (N = BT, 16 to 256), so a thread of
// the epilogue keeps its channel's scale and bias in registers, and a warp
// stores 32 neighbouring channels of one token with one instruction straight
// from registers, whatever the alignment of y's rows (the dictionary's 18385
// columns leave most of them off every boundary; large outputs of that kind have
// their own kernel, linear_i8_rows.cu). One persistent CTA per SM:
// warp 0 loads 128 x 128-byte tiles of the weight codes and BT x 128-byte tiles
// of the token codes by TMA (128-byte swizzle) into a ring, one thread of warp 1
// issues tcgen05.mma kind::i8 into one of two TMEM accumulators, and sixteen
// warps run the epilogue of the other. 16384 x 4096 x 4096 bf16: 180 us, 3.05 POP/s
// (the tensor pipe is 77 % busy); with K 128 and 18384 channels the stores are
// the bound (366 us for 40960 tokens in fp16, 4.1 TB/s as a plain fill).
#include <cmath>

#include "linear_i8.cuh"

namespace tocr {
namespace {

using namespace ptx;
using namespace linear;

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
// N codes (a multiple of 4), first in the low byte: in pairs, and one test of the
// remainders for all (16384 x 4096 bf16: 45 us, four at a time by themselves 47).
template <int N>
__device__ __forceinline__ void codes_of(uint32_t (&out)[N / 4], const float (&x)[N], float s, float inv) {
  const uint64_t s2 = pk(s, s), inv2 = pk(inv, inv), magic2 = pk(kMagic, kMagic);
  const uint64_t minus2 = pk(-1.f, -1.f);
  float t[N], far = 0.f;
#pragma unroll
  for (int k = 0; k < N; k += 2) {
    const uint64_t x2 = pk(x[k], x[k + 1]);
    const uint64_t t2 = fma2(x2, inv2, magic2);
    float r0, r1;
    upk(fma2(fma2(t2, minus2, magic2), s2, x2), r0, r1);
    upk(t2, t[k], t[k + 1]);
    far = fmaxf(fmaxf(far, fabsf(r0)), fabsf(r1));
  }
  if (far >= 0.5f * s) {
#pragma unroll
    for (int k = 0; k < N; ++k) t[k] = code_exact(x[k], s, inv);
  }
#pragma unroll
  for (int k = 0; k < N; k += 4)
    out[k / 4] = __byte_perm(__byte_perm(__float_as_uint(t[k]), __float_as_uint(t[k + 1]), 0x0040),
                             __byte_perm(__float_as_uint(t[k + 2]), __float_as_uint(t[k + 3]), 0x0040),
                             0x5410);
}

// a row's scale, from its largest |x|
__device__ __forceinline__ float scale_of(float big) {
  return fmaxf(big * (1.f / 127.f), 1.17549435e-38f);
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

// Threads of a CTA (16384 x 4096 bf16: 44 us with 128, 45 with 256).
template <int TEAM>
constexpr int kQuantThreads = TEAM > 128 ? TEAM : 128;

// One team of TEAM threads per row. VEC: rows start on 16-byte boundaries, and
// a thread keeps KEEP vectors of its row between the two steps.
template <typename T, int TEAM, bool VEC, int KEEP>
__global__ void __launch_bounds__(kQuantThreads<TEAM>)
quant_rows_kernel(const T *__restrict__ x, long long rows, int K, int pitch,
                  int8_t *__restrict__ q, float *__restrict__ scale) {
  constexpr int E = 16 / sizeof(T);
  constexpr int TEAMS = kQuantThreads<TEAM> / TEAM;
  __shared__ uint32_t smax[kQuantThreads<TEAM> / 32];
  release_next();
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
  const float s = finite ? scale_of(big) : __uint_as_float(0x7fc00000u);
  if (tid == 0) scale[row] = s;
  const float inv = 1.f / s;
  int8_t *qr = q + row * pitch;
  if (VEC) {
    auto put = [&](int v, const uint4 &w) {
      const T *e = reinterpret_cast<const T *>(&w);
      uint32_t p[E / 4];
      float f[E];
#pragma unroll
      for (int k = 0; k < E; ++k) f[k] = to_f32(e[k]);
      codes_of<E>(p, f, s, inv);
      if (!finite) {
#pragma unroll
        for (int k = 0; k < E / 4; ++k) p[k] = 0u;
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
      uint32_t p[1];
      codes_of<4>(p, f, s, inv);
      *reinterpret_cast<uint32_t *>(qr + k) = finite ? p[0] : 0u;
    }
  }
}

template <typename T, int TEAM, bool VEC, int KEEP>
int launch_quant(const T *x, long long rows, int K, int8_t *q, float *scale, cudaStream_t st) {
  constexpr int B = kQuantThreads<TEAM>, TEAMS = B / TEAM;
  quant_rows_kernel<T, TEAM, VEC, KEEP><<<(unsigned)((rows + TEAMS - 1) / TEAMS), B, 0, st>>>(
      x, rows, K, (K + 15) / 16 * 16, q, scale);
  return check_launch("quant_rows_kernel");
}
template <typename T>
int launch_quant(const void *xv, long long rows, int K, int8_t *q, float *scale, cudaStream_t st) {
  const T *x = static_cast<const T *>(xv);
  const size_t bytes = (size_t)K * sizeof(T);
  const bool vec = aligned(x, 16) && bytes % 16 == 0;
  // a warp per row of up to 2 KB (its lanes keep 4 vectors each); two warps up to
  // 8 KB where there are rows for the whole GPU (8 vectors each; 16384 x 4096
  // bf16: 44 us, one warp that keeps 16 each 58); else a CTA per row, smaller where
  // single values are loaded (4099 x 1001 fp32: 13 us, 256 threads 15)
  if (vec && bytes <= 32 * 16 * 4) return launch_quant<T, 32, true, 4>(x, rows, K, q, scale, st);
  if (vec && bytes <= 64 * 16 * 8 && rows >= 8 * sm_count())
    return launch_quant<T, 64, true, 8>(x, rows, K, q, scale, st);
  if (vec) return launch_quant<T, 256, true, 8>(x, rows, K, q, scale, st);
  if (bytes <= 32 * 16 * 4) return launch_quant<T, 32, false, 1>(x, rows, K, q, scale, st);
  return launch_quant<T, 128, false, 1>(x, rows, K, q, scale, st);
}

int quant_rows(const void *x, int dtype, long long rows, int K, int8_t *q, float *scale,
               cudaStream_t st) {
  if (dtype == TOCR_DTYPE_F16) return launch_quant<__half>(x, rows, K, q, scale, st);
  if (dtype == TOCR_DTYPE_BF16) return launch_quant<__nv_bfloat16>(x, rows, K, q, scale, st);
  return launch_quant<float>(x, rows, K, q, scale, st);
}

// ----------------------------------------------------------------- product --
constexpr int kBM = 128;         // channels of a tile
constexpr int kMaxBT = 256;      // tokens of a tile, a multiple of 16
constexpr int kUnit = 16;        // tokens an epilogue warp takes at a time
constexpr int kMaxStages = 10;
constexpr int kEpiWarp0 = 2, kEpiWarps = 16;
constexpr int kThreads = 32 * (kEpiWarp0 + kEpiWarps);
constexpr int kStageA = kBM * 128;
constexpr int kOffSx = 0;                                 // [warps][2][64] token scales
constexpr int kOffBar = kOffSx + kEpiWarps * 2 * 64 * 4;
constexpr int kOffMisc = kOffBar + (2 * kMaxStages + 4) * 8;
constexpr int kOffRing = (kOffMisc + 16 + 1023) / 1024 * 1024;
constexpr int kSmem = 226 * 1024;
constexpr int kRingBytes = kSmem - 1024 - kOffRing;

// f[j] to token j's row: g, g + ld, ... for the first n of 16 tokens
template <typename T, bool FULL>
__device__ __forceinline__ void store_unit(T *g, long long ld, const float (&f)[kUnit], int n) {
  if constexpr (sizeof(T) == 2) {
    uint16_t *o = reinterpret_cast<uint16_t *>(g);
#pragma unroll
    for (int j = 0; j < kUnit; j += 2) {
      const uint32_t w = pack2<T>(f[j], f[j + 1]);
      if (FULL || j < n) o[0] = (uint16_t)w;
      if (FULL || j + 1 < n) o[ld] = (uint16_t)(w >> 16);
      o += 2 * ld;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kUnit; ++j) {
      if (FULL || j < n) *g = f[j];
      g += ld;
    }
  }
}

template <typename T, bool SMALLK>
__global__ void __launch_bounds__(kThreads, 1)
linear_i8_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
                 const LinParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + kOffBar);
  uint64_t *empty = full + kMaxStages;
  uint64_t *acc_full = empty + kMaxStages;  // [2]
  uint64_t *acc_empty = acc_full + 2;       // [2]
  uint32_t *s_tmem = reinterpret_cast<uint32_t *>(smem + kOffMisc);
  volatile int *s_abort = reinterpret_cast<volatile int *>(smem + kOffMisc + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) {
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
    tmem_alloc(s_tmem, 2 * kMaxBT);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  after_previous();
  const int KS = p.ksteps, stage = kStageA + p.bt * 128;
  uint8_t *ring = smem + kOffRing;

  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&xmap);
      tma_prefetch_desc(&wmap);
      int s = 0, used = 0;  // slot, slots ever filled
      uint32_t phase = 0;
      bool ok = true;
      for (TileWalk t(p); ok && !t.done(); t.next()) {
        const int m0 = t.mi * p.bt, n0 = t.ni * kBM;
        for (int k = 0; k < KS; ++k) {
          if (used == p.stages && !mbar_wait_bounded(&empty[s], phase ^ 1, s_abort, p.err, 81)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[s], stage);
          tma_load_2d(ring + s * stage, &wmap, &full[s], 128 * k, n0);
          tma_load_2d(ring + s * stage + kStageA, &xmap, &full[s], 128 * k, m0);
          if (used < p.stages) ++used;
          if (++s == p.stages) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      if (*s_abort) {  // leave no copy in flight
        for (int i = 0; i < used; ++i) {
          const long long t0 = clock64();
          while (!mbar_try_wait(&full[i], i < s ? phase : phase ^ 1))
            if (clock64() - t0 > (1ll << 30)) break;
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = idesc_i8(kBM, p.bt);
      const uint64_t desc0 = sw128_kmajor_desc(smem_u32(ring));
      int s = 0;
      uint32_t phase = 0;
      Ring<2> acc;
      bool ok = true;
      for (TileWalk t(p); ok && !t.done(); t.next()) {
        if (!acc.first && !mbar_wait_bounded(&acc_empty[acc.i], acc.phase ^ 1, s_abort, p.err, 82))
          break;
        tc_fence_after();
        const uint32_t d = tmem + acc.i * kMaxBT;
        for (int k = 0; k < KS; ++k) {
          if (!mbar_wait_bounded(&full[s], phase, s_abort, p.err, 83)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t a = desc0 + (uint64_t)((s * stage) >> 4);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            mma_i8(d, a + 2 * q, a + (kStageA >> 4) + 2 * q, idesc, k > 0 || q > 0 ? 1u : 0u);
          mma_commit(&empty[s]);
          if (++s == p.stages) {
            s = 0;
            phase ^= 1;
          }
        }
        mma_commit(&acc_full[acc.i]);
        acc.next();
      }
    }
  } else {
    const int ew = warp - kEpiWarp0;
    const int g = ew >> 2;      // takes units g, g + 4, ... of the tile's tokens
    const int quad = warp & 3;  // the TMEM lanes a warp may read
    const uint32_t tl = tmem + ((uint32_t)(quad * 32) << 16);
    float *slice = reinterpret_cast<float *>(smem + kOffSx) + ew * 128;
    T *y = static_cast<T *>(p.y);
    // a tile's channel scale and bias, and the scales of the warp's tokens,
    // loaded while the tile before is worked on
    float nsw = 0.f, nb = 0.f, ns0 = 0.f, ns1 = 0.f;
    auto prefetch = [&](const TileWalk &t) {
      const int n = t.ni * kBM + quad * 32 + lane;
      const long long m =
          (long long)t.mi * p.bt + (g + 4 * (lane / kUnit)) * kUnit + lane % kUnit;
      nsw = n < p.N ? __ldg(p.sw + n) : 0.f;
      nb = n < p.N && p.bias ? __ldg(p.bias + n) : 0.f;
      // not read-only loads: the quantiser may still write when this kernel begins
      ns0 = m < p.rows ? p.sx[m] : 0.f;
      ns1 = m + 8 * kUnit < p.rows ? p.sx[m + 8 * kUnit] : 0.f;
    };
    TileWalk ahead(p);
    if (!ahead.done()) prefetch(ahead);
    Ring<2> acc;
    for (TileWalk t(p); !t.done(); t.next(), acc.next()) {
      const int n = t.ni * kBM + quad * 32 + lane;
      const long long m0 = (long long)t.mi * p.bt;
      const uint64_t sw2 = pk(nsw, nsw), b2 = pk(nb, nb);
      float *sx = slice + acc.i * 64;
      sx[lane] = ns0;
      sx[32 + lane] = ns1;
      __syncwarp();
      ahead.next();
      if (!ahead.done()) prefetch(ahead);
      if (!mbar_wait_bounded(&acc_full[acc.i], acc.phase, s_abort, p.err, 84)) break;
      tc_fence_after();
      const uint32_t ta = tl + acc.i * kMaxBT;
      const int units = p.bt / kUnit;
#pragma unroll
      for (int k = 0; k < kMaxBT / kUnit / 4; ++k) {
        const int u = g + 4 * k;
        if (u >= units) break;
        uint32_t v[kUnit];
        tmem_ld16(ta + u * kUnit, v);
        tmem_ld_wait(v);
        float f[kUnit];
        const ulonglong2 *sq = reinterpret_cast<const ulonglong2 *>(sx + k * kUnit);
#pragma unroll
        for (int j = 0; j < kUnit; j += 4) {
          const ulonglong2 s4 = sq[j / 4];
#pragma unroll
          for (int h = 0; h < 4; h += 2) {
            const uint64_t a = sums2<SMALLK>(v[j + h], v[j + h + 1]);
            upk(fma2(mul2(a, sw2), h ? s4.y : s4.x, b2), f[j + h], f[j + h + 1]);
          }
        }
        if (p.act) {
#pragma unroll
          for (int j = 0; j < kUnit; ++j) f[j] = activate(f[j], p.act);
        }
        const long long m = m0 + u * kUnit;
        if (n < p.N && m < p.rows) {
          T *o = y + m * p.N + n;
          if (m + kUnit <= p.rows)
            store_unit<T, true>(o, p.N, f, kUnit);
          else
            store_unit<T, false>(o, p.N, f, (int)(p.rows - m));
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc.i]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * kMaxBT);
  }
}

template <typename T, bool SMALLK>
int launch_product(const void *xq, const void *wq, LinParams p, int K, int pitch, cudaStream_t st) {
  CUtensorMap xm, wm;
  int rc = tma_map_rows(&xm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, xq, K, p.rows, pitch, p.bt);
  if (rc) return rc;
  rc = tma_map_rows(&wm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, wq, K, p.N, pitch, kBM);
  if (rc) return rc;
  p.stages = kRingBytes / (kStageA + p.bt * 128);
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  auto *kernel = linear_i8_kernel<T, SMALLK>;
  rc = allow_dynamic_smem(reinterpret_cast<const void *>(kernel), kSmem, "linear_i8_kernel");
  if (rc) return rc;
  const int grid = (int)(p.tiles < sm_count() ? p.tiles : sm_count());
  if (p.behind_quant)
    return launch_overlapped("linear_i8_kernel", kernel, grid, kThreads, kSmem, st, xm, wm, p);
  kernel<<<grid, kThreads, kSmem, st>>>(xm, wm, p);
  return check_launch("linear_i8_kernel");
}

template <typename T>
int product(const void *xq, const void *wq, LinParams p, int K, int pitch, cudaStream_t st) {
  p.tiles_n = (p.N + kBM - 1) / kBM;
  // the tokens of a tile for which the waves of CTAs take least: a tile costs
  // its tokens and a fixed part worth about 64 tokens
  const long long sms = sm_count();
  long long best = -1;
  for (int bt = kMaxBT; bt >= kUnit; bt -= kUnit) {
    const long long cost = ((long long)p.tiles_n * ((p.rows + bt - 1) / bt) + sms - 1) / sms * (bt + 64);
    if (best < 0 || cost < best) {
      best = cost;
      p.bt = bt;
    }
  }
  p.tiles = p.tiles_n * ((p.rows + p.bt - 1) / p.bt);
  return K <= kSmallK ? launch_product<T, true>(xq, wq, p, K, pitch, st)
                      : launch_product<T, false>(xq, wq, p, K, pitch, st);
}

// ---------------------------------------------------------------- few tokens --
// The same product for few tokens, whose quantiser is part of it: every CTA
// makes the codes of all of them itself, in the layout of the MMA operand, while
// its first weights arrive: one launch and no scratch memory. That serves calls
// that the host paces; on the device the rows that a warp takes one after the
// other cost more than a second launch. us per call from Python, and replayed
// from a graph, with the two launches behind the stroke: 1 x 512 x 18385 fp16
// 11.4 / 16.1, 6.2 / 6.2; 80 x 128 x 384 11.3 / 15.8, 8.2 / 6.2; 128 x 256 x 1024
// 14.4 / 16.0, 14.3 / 7.7; 8 x 4096 x 4096, where the rows are longest for the
// limit, 18.5 / 16.0, 18.4 / 10.3.
constexpr int kFewTokens = 128, kFewElements = 32768, kFewCodes = 64 * 1024, kFewStages = 8;

bool is_few(long long rows, int K) {
  if (rows > kFewTokens || rows * K > kFewElements) return false;
  const int bt = (int)(rows + kUnit - 1) / kUnit * kUnit;
  return (K + 127) / 128 * bt * 128 <= kFewCodes;
}

constexpr int kFewOffSx = 0;                                      // [kFewTokens]
constexpr int kFewOffBar = kFewOffSx + kFewTokens * 4;
constexpr int kFewOffMisc = kFewOffBar + (2 * kFewStages + 5) * 8;
constexpr int kFewOffCodes = (kFewOffMisc + 16 + 1023) / 1024 * 1024;  // [ksteps][bt][128]
constexpr int few_smem(int ksteps, int bt, int stages) {
  return kFewOffCodes + ksteps * bt * 128 + stages * kStageA + 1024;
}

struct FewParams {
  LinParams lin;
  const void *x;
  int K;
  bool vec;  // four elements of a row at a time
};

template <typename X>
__device__ __forceinline__ void load4(float (&f)[4], const X *x, int k, int K, bool vec) {
  if (vec) {
    if constexpr (sizeof(X) == 4) {
      const float4 v = __ldg(reinterpret_cast<const float4 *>(x + k));
      f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
    } else {
      const uint2 v = __ldg(reinterpret_cast<const uint2 *>(x + k));
      const X *e = reinterpret_cast<const X *>(&v);
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = to_f32(e[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = k + j < K ? to_f32(x[k + j]) : 0.f;
  }
}

template <typename X, typename T>
__global__ void __launch_bounds__(kThreads, 1)
linear_i8_few_kernel(const __grid_constant__ CUtensorMap wmap, const FewParams q) {
  const LinParams &p = q.lin;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float *sx = reinterpret_cast<float *>(smem + kFewOffSx);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + kFewOffBar);
  uint64_t *empty = full + kFewStages;
  uint64_t *acc_full = empty + kFewStages;  // [2]
  uint64_t *acc_empty = acc_full + 2;       // [2]
  uint64_t *codes_ready = acc_empty + 2;
  uint32_t *s_tmem = reinterpret_cast<uint32_t *>(smem + kFewOffMisc);
  volatile int *s_abort = reinterpret_cast<volatile int *>(smem + kFewOffMisc + 4);
  const int KS = p.ksteps;
  uint8_t *codes = smem + kFewOffCodes, *ring = codes + KS * p.bt * 128;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kFewStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], kEpiWarps);
    }
    mbar_init(codes_ready, kEpiWarps);
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(s_tmem, 2 * kFewTokens);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;

  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&wmap);
      int s = 0, used = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (TileWalk t(p); ok && !t.done(); t.next()) {
        for (int k = 0; k < KS; ++k) {
          if (used == p.stages && !mbar_wait_bounded(&empty[s], phase ^ 1, s_abort, p.err, 85)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[s], kStageA);
          tma_load_2d(ring + s * kStageA, &wmap, &full[s], 128 * k, t.ni * kBM);
          if (used < p.stages) ++used;
          if (++s == p.stages) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      if (*s_abort) {  // leave no copy in flight
        for (int i = 0; i < used; ++i) {
          const long long t0 = clock64();
          while (!mbar_try_wait(&full[i], i < s ? phase : phase ^ 1))
            if (clock64() - t0 > (1ll << 30)) break;
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = idesc_i8(kBM, p.bt);
      const uint64_t wdesc = sw128_kmajor_desc(smem_u32(ring));
      const uint64_t xdesc = sw128_kmajor_desc(smem_u32(codes));
      int s = 0;
      uint32_t phase = 0;
      Ring<2> acc;
      bool ok = mbar_wait_bounded(codes_ready, 0, s_abort, p.err, 86);
      for (TileWalk t(p); ok && !t.done(); t.next()) {
        if (!acc.first && !mbar_wait_bounded(&acc_empty[acc.i], acc.phase ^ 1, s_abort, p.err, 87))
          break;
        tc_fence_after();
        const uint32_t d = tmem + acc.i * kFewTokens;
        for (int k = 0; k < KS; ++k) {
          if (!mbar_wait_bounded(&full[s], phase, s_abort, p.err, 88)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t a = wdesc + (uint64_t)(s * kStageA >> 4);
          const uint64_t b = xdesc + (uint64_t)(k * p.bt * 128 >> 4);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            mma_i8(d, a + 2 * i, b + 2 * i, idesc, k > 0 || i > 0 ? 1u : 0u);
          mma_commit(&empty[s]);
          if (++s == p.stages) {
            s = 0;
            phase ^= 1;
          }
        }
        mma_commit(&acc_full[acc.i]);
        acc.next();
      }
    }
  } else {
    const int ew = warp - kEpiWarp0;
    // codes: a warp per row; what lies behind K or behind the last row meets
    // weights of zero, or is not stored
    for (int r = ew; r < (int)p.rows; r += kEpiWarps) {
      const X *xr = static_cast<const X *>(q.x) + (size_t)r * q.K;
      uint32_t top = 0;
#pragma unroll 4
      for (int k = 4 * lane; k < q.K; k += 128) {
        float f[4];
        load4(f, xr, k, q.K, q.vec);
#pragma unroll
        for (int j = 0; j < 4; ++j) top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
      }
      const float big = __uint_as_float(__reduce_max_sync(~0u, top));
      const bool finite = big < INFINITY;
      const float s = finite ? scale_of(big) : __uint_as_float(0x7fc00000u);
      const float inv = 1.f / s;
      if (lane == 0) sx[r] = s;
#pragma unroll 4
      for (int k = 4 * lane; k < q.K; k += 128) {
        float f[4];
        load4(f, xr, k, q.K, q.vec);
        uint32_t c[1];
        codes_of<4>(c, f, s, inv);
        // 128-byte swizzle: 16-byte pieces of a row change places by row mod 8
        *reinterpret_cast<uint32_t *>(codes + (k >> 7) * p.bt * 128 + r * 128 +
                                      ((k & 127) ^ ((r & 7) << 4))) = finite ? c[0] : 0u;
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(codes_ready);
    // every warp needs every row's scale
    const bool ready = mbar_wait_bounded(codes_ready, 0, s_abort, p.err, 89);

    const int g = ew >> 2;      // takes units g, g + 4, ... of the tokens
    const int quad = warp & 3;  // the TMEM lanes a warp may read
    const uint32_t tl = tmem + ((uint32_t)(quad * 32) << 16);
    const int units = p.bt / kUnit;
    Ring<2> acc;
    for (TileWalk t(p); ready && !t.done(); t.next(), acc.next()) {
      const int n = t.ni * kBM + quad * 32 + lane;
      const float sw = n < p.N ? __ldg(p.sw + n) : 0.f;
      const float b = n < p.N && p.bias ? __ldg(p.bias + n) : 0.f;
      if (!mbar_wait_bounded(&acc_full[acc.i], acc.phase, s_abort, p.err, 90)) break;
      tc_fence_after();
      for (int u = g; u < units; u += 4) {
        uint32_t v[kUnit];
        tmem_ld16(tl + acc.i * kFewTokens + u * kUnit, v);
        tmem_ld_wait(v);
        float f[kUnit];
#pragma unroll
        for (int j = 0; j < kUnit; ++j) {
          f[j] = fmaf((float)(int)v[j] * sw, sx[u * kUnit + j], b);
          if (p.act) f[j] = activate(f[j], p.act);
        }
        if (n < p.N) {
          T *o = static_cast<T *>(p.y) + (long long)u * kUnit * p.N + n;
          store_unit<T, false>(o, p.N, f, (int)p.rows - u * kUnit);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc.i]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * kFewTokens);
  }
}

template <typename X, typename T>
int launch_few(FewParams q, const void *wq, int pitch, cudaStream_t st) {
  LinParams &p = q.lin;
  CUtensorMap wm;
  int rc = tma_map_rows(&wm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, wq, q.K, p.N, pitch, kBM);
  if (rc) return rc;
  q.vec = q.K % 4 == 0 && aligned(q.x, 4 * sizeof(X));
  p.bt = (int)(p.rows + kUnit - 1) / kUnit * kUnit;
  p.tiles_n = (p.N + kBM - 1) / kBM;
  p.tiles = p.tiles_n;
  const int grid = (int)(p.tiles < sm_count() ? p.tiles : sm_count());
  const long long steps = (p.tiles + grid - 1) / grid * p.ksteps;
  p.stages = steps < kFewStages ? (int)steps : kFewStages;
  auto *kernel = linear_i8_few_kernel<X, T>;
  constexpr int most = kFewOffCodes + kFewCodes + kFewStages * kStageA + 1024;
  static_assert(most <= 227 * 1024, "shared memory");
  rc = allow_dynamic_smem(reinterpret_cast<const void *>(kernel), most, "linear_i8_few_kernel");
  if (rc) return rc;
  kernel<<<grid, kThreads, few_smem(p.ksteps, p.bt, p.stages), st>>>(wm, q);
  return check_launch("linear_i8_few_kernel");
}

template <typename X>
int few(const FewParams &q, const void *wq, int pitch, int out_dtype, cudaStream_t st) {
  if (out_dtype == TOCR_DTYPE_F16) return launch_few<X, __half>(q, wq, pitch, st);
  if (out_dtype == TOCR_DTYPE_BF16) return launch_few<X, __nv_bfloat16>(q, wq, pitch, st);
  return launch_few<X, float>(q, wq, pitch, st);
}

constexpr long long kMaxRows = 1ll << 24;
// Sums stay inside s32: 127 * 128 K where one side's codes are the quantiser's
// (-127 to 127), 128^2 K where both are any codes.
constexpr int kMaxK = 1 << 17, kMaxCodesK = kMaxK - 1;
constexpr int kMaxN = 1 << 24;

bool is_dtype(int d) {
  return d == TOCR_DTYPE_F16 || d == TOCR_DTYPE_BF16 || d == TOCR_DTYPE_F32;
}

int check_linear(const char *fn, long long rows, int K, int most_k, int N, int act,
                 int out_dtype) {
  TOCR_REQUIRE(rows >= 0 && rows <= kMaxRows && K > 0 && K <= most_k && N > 0 && N <= kMaxN,
               "%s: bad sizes rows=%lld K=%d N=%d", fn, rows, K, N);
  TOCR_REQUIRE(act == TOCR_ACT_NONE || act == TOCR_ACT_RELU || act == TOCR_ACT_HARDSWISH,
               "%s: unknown activation %d", fn, act);
  TOCR_REQUIRE(is_dtype(out_dtype), "%s: unknown output type %d", fn, out_dtype);
  return TOCR_OK;
}

LinParams params(const float *sx, long long rows, int K, const float *sw, const float *bias, int N,
                 int act, void *y, int *err) {
  LinParams p{};
  p.sx = sx;
  p.sw = sw;
  p.bias = bias;
  p.y = y;
  p.rows = rows;
  p.N = N;
  p.ksteps = (K + 127) / 128;
  p.act = act;
  p.err = err;
  return p;
}

int run_product(const void *xq, const void *wq, const LinParams &p, int K, int out_dtype,
                cudaStream_t st) {
  const int pitch = (K + 15) / 16 * 16;
  if (wants_row_kernel(p.y, p.rows, p.N, out_dtype == TOCR_DTYPE_F32 ? 4 : 2))
    return launch_row_kernel(xq, wq, p, K, pitch, out_dtype, st);
  if (out_dtype == TOCR_DTYPE_F16) return product<__half>(xq, wq, p, K, pitch, st);
  if (out_dtype == TOCR_DTYPE_BF16) return product<__nv_bfloat16>(xq, wq, p, K, pitch, st);
  return product<float>(xq, wq, p, K, pitch, st);
}

// the codes of a call's tokens; its scales lie behind them
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
  TOCR_REQUIRE(aligned(d_x, x_dtype == TOCR_DTYPE_F32 ? 4 : 2),
               "tocr_quant_rows_i8: x must be aligned to its element");
  TOCR_REQUIRE(aligned(d_codes, 16) && aligned(d_scales, 4),
               "tocr_quant_rows_i8: the codes must be 16-byte, the scales 4-byte aligned");
  return quant_rows(d_x, x_dtype, rows, K, static_cast<int8_t *>(d_codes), d_scales,
                    as_stream(stream));
}

TOCR_API int tocr_linear_i8_codes(const void *d_xq, const float *d_sx, long long rows, int K,
                                  const void *d_wq, const float *d_sw, const float *d_bias, int N,
                                  int act, int out_dtype, void *d_y, int *d_err, void *stream) {
  TOCR_ENTRY();
  int rc = check_linear("tocr_linear_i8_codes", rows, K, kMaxCodesK, N, act, out_dtype);
  if (rc || rows == 0) return rc;
  TOCR_REQUIRE(d_xq && d_sx && d_wq && d_sw && d_y && d_err, "tocr_linear_i8_codes: null pointer");
  TOCR_REQUIRE(aligned(d_xq, 16) && aligned(d_wq, 16),
               "tocr_linear_i8_codes: the codes must be 16-byte aligned");
  TOCR_REQUIRE(aligned(d_y, out_dtype == TOCR_DTYPE_F32 ? 4 : 2),
               "tocr_linear_i8_codes: y must be aligned to its element");
  TOCR_REQUIRE(aligned(d_sx, 4) && aligned(d_sw, 4) && aligned(d_bias, 4) && aligned(d_err, 4),
               "tocr_linear_i8_codes: scales, bias and the error word must be 4-byte aligned");
  return run_product(d_xq, d_wq, params(d_sx, rows, K, d_sw, d_bias, N, act, d_y, d_err), K,
                     out_dtype, as_stream(stream));
}

TOCR_API size_t tocr_linear_i8_workspace_bytes(long long rows, int K) {
  if (rows < 0 || rows > kMaxRows || K <= 0 || K > kMaxK || is_few(rows, K)) return 0;
  return codes_bytes(rows, K) + (size_t)rows * 4;
}

TOCR_API int tocr_linear_i8(const void *d_x, int x_dtype, long long rows, int K, const void *d_wq,
                            const float *d_sw, const float *d_bias, int N, int act, int out_dtype,
                            void *d_y, void *d_workspace, size_t workspace_bytes, int *d_err,
                            void *stream) {
  TOCR_ENTRY();
  int rc = check_linear("tocr_linear_i8", rows, K, kMaxK, N, act, out_dtype);
  if (rc) return rc;
  TOCR_REQUIRE(is_dtype(x_dtype), "tocr_linear_i8: unknown type %d", x_dtype);
  if (rows == 0) return TOCR_OK;
  TOCR_REQUIRE(d_x && d_wq && d_sw && d_y && d_err, "tocr_linear_i8: null pointer");
  TOCR_REQUIRE(aligned(d_wq, 16), "tocr_linear_i8: the codes must be 16-byte aligned");
  TOCR_REQUIRE(aligned(d_x, x_dtype == TOCR_DTYPE_F32 ? 4 : 2) &&
                   aligned(d_y, out_dtype == TOCR_DTYPE_F32 ? 4 : 2),
               "tocr_linear_i8: x and y must be aligned to their elements");
  TOCR_REQUIRE(aligned(d_sw, 4) && aligned(d_bias, 4) && aligned(d_err, 4),
               "tocr_linear_i8: scales, bias and the error word must be 4-byte aligned");
  cudaStream_t st = as_stream(stream);
  LinParams p = params(nullptr, rows, K, d_sw, d_bias, N, act, d_y, d_err);
  if (is_few(rows, K)) {
    const FewParams q = {p, d_x, K, false};
    const int pitch = (K + 15) / 16 * 16;
    if (x_dtype == TOCR_DTYPE_F16) return few<__half>(q, d_wq, pitch, out_dtype, st);
    if (x_dtype == TOCR_DTYPE_BF16) return few<__nv_bfloat16>(q, d_wq, pitch, out_dtype, st);
    return few<float>(q, d_wq, pitch, out_dtype, st);
  }
  const size_t need = codes_bytes(rows, K) + (size_t)rows * 4;
  TOCR_REQUIRE(d_workspace && aligned(d_workspace, 256) && workspace_bytes >= need,
               "tocr_linear_i8: the workspace must be 256-byte aligned and hold %zu bytes", need);
  int8_t *q = static_cast<int8_t *>(d_workspace);
  float *sx = reinterpret_cast<float *>(q + codes_bytes(rows, K));
  rc = quant_rows(d_x, x_dtype, rows, K, q, sx, st);
  if (rc) return rc;
  p.sx = sx;
  p.behind_quant = true;
  return run_product(q, d_wq, p, K, out_dtype, st);
}

}  // extern "C"
