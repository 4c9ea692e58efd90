// Cross entropy of the recognizer's linear head, forward and backward, with
// the logits neither stored nor read.
//
//   l = F W^T + b                       [n][V], n the rows that have a target
//   lse_i = log sum_j exp(l_ij),  loss_i = lse_i - l_i,t(i)
//   G_ij  = g_i (exp(l_ij - lse_i) - [j = t(i)])
//   dF = G W,  dW = G^T F,  db_j = sum_i G_ij
//
// Rows whose target lies outside [0, V) are padding. They are left out before
// the products (the kept rows are numbered in order, deterministically), so
// they cost nothing and whatever they hold reaches no output.
//
// Both directions are products of a stationary tile of 128 rows with a
// streamed matrix: the tile's features sit in tensor memory as the A operand
// of S = A B^T, the streamed rows arrive by TMA in chunks of CN rows (128-byte
// swizzle), and the epilogue warps turn the fp32 accumulators S into what is
// wanted: the running maximum and sum of exp of each row (forward), or the
// 16-bit tile P of G, put back into tensor memory as the A operand of the
// second product D += P B over the same chunk in shared memory, read as an
// MN-major operand (backward). For dF the tile is 128 rows of F and W is
// streamed; for dW the tile is 128 rows of W and F is streamed, so one kernel
// does both, and nothing of size n x V touches memory. Keeping the stationary
// operand in tensor memory halves what the first product reads of shared
// memory: at 128 x 128 tiles both operands from shared memory would need all
// of its 128 bytes a clock.
//
// The (tile, chunk) steps of a call form one line that is cut into equal
// ranges, one per CTA, so that any shape fills the GPU; a tile cut by a range
// border is summed from fp32 partials in the order of the CTAs by a second
// kernel (no atomics: a call's results do not depend on timing).
//
// Numbers: S, the softmax statistics, D and db are fp32. P is rounded to the
// inputs' type for the second product (one rounding of each G_ij, relative
// 2^-11 in fp16 and 2^-8 in bf16); fp16 holds it scaled by 2^14, so that a
// probability of 2^-28 is still a normal number, and for dW the row weights
// enter divided by their largest, so that small weights do not underflow.
// The outputs are rounded once more to their type.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cmath>
#include <cstdint>

#include "tc_ptx.cuh"
#include "tma_map.cuh"
#include "tocr_common.cuh"

namespace tocr {
namespace {

using namespace ptx;

constexpr int kTile = 128;       // rows of a stationary tile (MMA M, TMEM lanes)
constexpr int kEpiWarp0 = 2;
constexpr int kEpiWarps = 16;    // two groups of eight; a group takes every other chunk
constexpr int kThreads = 32 * (kEpiWarp0 + kEpiWarps);
constexpr int kEpiThreads = 32 * kEpiWarps;
constexpr int kTmemCols = 512;
constexpr int kRowBlock = 256;   // rows per block of the numbering kernels
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxK = 256;
constexpr long long kMaxRows = 1ll << 24;
constexpr int kMaxGrid = 148;    // CTAs of a product kernel: one per SM
constexpr int kShift = 14;       // fp16: log2 of the scale of P

// ------------------------------------------------------------- workspace ----
struct Header {
  int n;        // rows with a target
  float gmax;   // largest |g| among them
};

__host__ __device__ constexpr size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

struct Workspace {
  Header *hdr;
  int *cnt;        // per block of rows
  float *gblk;
  int *rowidx;     // [rows_pad] the row of each kept row
  int *tgt;        // [rows_pad] its target (-1 behind the last)
  // forward
  float *lt;       // [rows_pad] target logit * log2(e)
  float2 *part;    // [tiles + grid][128] (max, sum) of a range's piece of a tile
  // backward
  uint8_t *xc;     // [rows_pad][K] the kept rows of F, zero behind the last
  float *nlse;     // [rows_pad] -lse * log2(e) (-inf behind the last)
  float *gc;       // [rows_pad] g
  float *gs;       // [rows_pad] g / gmax * 2^shift
  float *dpart;    // [2 * grid][128][KP]
  float *bpart;    // [2 * grid][128]
  size_t bytes;
};

// Layout of the caller's workspace for `rows` rows; base may be null (sizes).
inline Workspace carve(uint8_t *base, long long rows, int K, bool backward) {
  constexpr int grid = kMaxGrid;
  Workspace w{};
  size_t off = 0;
  auto take = [&](size_t bytes) {
    uint8_t *p = base + off;
    off += up256(bytes);
    return p;
  };
  const long long pad = (rows + kTile - 1) / kTile * kTile + kTile;
  const long long blocks = (rows + kRowBlock - 1) / kRowBlock + 1;
  const int KP = (K + 63) / 64 * 64;
  w.hdr = reinterpret_cast<Header *>(take(sizeof(Header)));
  w.cnt = reinterpret_cast<int *>(take(blocks * 4));
  w.gblk = reinterpret_cast<float *>(take(blocks * 4));
  w.rowidx = reinterpret_cast<int *>(take(pad * 4));
  w.tgt = reinterpret_cast<int *>(take(pad * 4));
  if (!backward) {
    w.lt = reinterpret_cast<float *>(take(pad * 4));
    w.part = reinterpret_cast<float2 *>(take((size_t)(pad / kTile + grid) * kTile * 8));
  } else {
    w.xc = take((size_t)pad * K * 2);
    w.nlse = reinterpret_cast<float *>(take(pad * 4));
    w.gc = reinterpret_cast<float *>(take(pad * 4));
    w.gs = reinterpret_cast<float *>(take(pad * 4));
    w.dpart = reinterpret_cast<float *>(take((size_t)2 * grid * kTile * KP * 4));
    w.bpart = reinterpret_cast<float *>(take((size_t)2 * grid * kTile * 4));
  }
  w.bytes = off;
  return w;
}

// ---------------------------------------------------------- kept rows -------
__device__ __forceinline__ int target_of(const void *t, bool wide, long long i, int V) {
  if (wide) {
    const long long v = static_cast<const long long *>(t)[i];
    return v >= 0 && v < V ? (int)v : -1;
  }
  const int v = static_cast<const int *>(t)[i];
  return v >= 0 && v < V ? v : -1;
}

// Kept rows and largest weight of every block of 256 rows.
__global__ void __launch_bounds__(kRowBlock)
ce_count_kernel(const void *targets, bool wide, int rows, int V, const float *g, int *cnt,
                float *gblk) {
  __shared__ float sm[kRowBlock / 32];
  const long long i = (long long)blockIdx.x * kRowBlock + threadIdx.x;
  const bool keep = i < rows && target_of(targets, wide, i, V) >= 0;
  const int n = __syncthreads_count(keep);
  float m = keep && g ? fabsf(g[i]) : 0.f;
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < kRowBlock / 32; ++k) m = fmaxf(m, sm[k]);
    cnt[blockIdx.x] = n;
    gblk[blockIdx.x] = m;
  }
}

struct PlaceParams {
  const void *targets;
  bool wide;
  int rows, V, K;
  float shift;       // 2^14 for fp16, 1 for bf16
  const int *cnt;
  const float *gblk;
  Header *hdr;
  int *rowidx, *tgt;
  // forward: outputs of the padding rows
  float *loss, *lse_out;
  // backward
  const uint8_t *feat;
  const float *lse, *g;
  uint8_t *xc, *dfeat;
  float *nlse, *gc, *gs;
};

// Numbers the kept rows in their order and writes what the products take of
// each (backward: a copy of its features); padding rows get their zero outputs.
template <bool BWD>
__global__ void __launch_bounds__(kRowBlock) ce_place_kernel(const PlaceParams p) {
  __shared__ int swarp[kRowBlock / 32];
  __shared__ int s_off, s_total;
  __shared__ float s_gmax;
  __shared__ int s_dst[kRowBlock];  // place of each row of the block, -1: padding
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // kept rows before this block, and the largest weight of all
  int before = 0;
  float gm = 0.f;
  for (int b = tid; b < (int)gridDim.x; b += kRowBlock) {
    if (b < (int)blockIdx.x) before += p.cnt[b];
    if (BWD) gm = fmaxf(gm, p.gblk[b]);
  }
  if (tid == 0) s_off = 0;
  __syncthreads();
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    before += __shfl_xor_sync(~0u, before, o);
    gm = fmaxf(gm, __shfl_xor_sync(~0u, gm, o));
  }
  __shared__ float sg[kRowBlock / 32];
  if (lane == 0) {
    atomicAdd(&s_off, before);  // integers: the order does not matter
    sg[warp] = gm;
  }
  const long long row0 = (long long)blockIdx.x * kRowBlock;
  const long long i = row0 + tid;
  const int t = i < p.rows ? target_of(p.targets, p.wide, i, p.V) : -1;
  const uint32_t bal = __ballot_sync(~0u, t >= 0);
  if (lane == 0) swarp[warp] = __popc(bal);
  __syncthreads();
  if (tid == 0) {
    float m = sg[0];
    for (int k = 1; k < kRowBlock / 32; ++k) m = fmaxf(m, sg[k]);
    s_gmax = m;
    int total = 0;
    for (int k = 0; k < kRowBlock / 32; ++k) total += swarp[k];
    s_total = total;
  }
  int rank = __popc(bal & ((1u << lane) - 1u));
  for (int k = 0; k < warp; ++k) rank += swarp[k];
  __syncthreads();
  const int off = s_off;
  const int dst = t >= 0 ? off + rank : -1;
  if (i < p.rows) {
    if (t >= 0) {
      p.rowidx[dst] = (int)i;
      p.tgt[dst] = t;
      if (BWD) {
        const float g = p.g[i];
        p.nlse[dst] = -p.lse[i] * kLog2e;
        p.gc[dst] = g;
        p.gs[dst] = s_gmax > 0.f ? g / s_gmax * p.shift : g * 0.f;
      }
    } else if (!BWD) {
      p.loss[i] = 0.f;
      p.lse_out[i] = 0.f;
    }
  }
  const bool last = blockIdx.x == gridDim.x - 1;
  const int n = off + s_total;  // all kept rows, in the last block
  if (last && tid == 0) {
    p.hdr->n = n;
    p.hdr->gmax = s_gmax;
  }
  // the unused rows up to the end of the last tile
  const int end = max(kTile, (n + kTile - 1) / kTile * kTile);
  if (last) {
    for (int j = n + tid; j < end; j += kRowBlock) {
      p.rowidx[j] = -1;
      p.tgt[j] = -1;
      if (BWD) {
        p.nlse[j] = -INFINITY;
        p.gc[j] = 0.f;
        p.gs[j] = 0.f;
      }
    }
  }
  if (BWD) {
    s_dst[tid] = dst;
    __syncthreads();
    const int q = p.K / 8;  // 16-byte pieces of a row
    const int here = (int)min((long long)kRowBlock, (long long)p.rows - row0);
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int e = tid; e < here * q; e += kRowBlock) {
      const int r = e / q, c = e - r * q;
      const int d = s_dst[r];
      if (d >= 0)
        reinterpret_cast<uint4 *>(p.xc)[(size_t)d * q + c] =
            __ldg(reinterpret_cast<const uint4 *>(p.feat) + (size_t)(row0 + r) * q + c);
      else if (p.dfeat)
        reinterpret_cast<uint4 *>(p.dfeat)[(size_t)(row0 + r) * q + c] = zero;
    }
    if (last)
      for (long long e = tid; e < (long long)(end - n) * q; e += kRowBlock)
        reinterpret_cast<uint4 *>(p.xc)[(size_t)n * q + e] = zero;
  }
}

// ------------------------------------------------------------ step line -----
// Steps [begin, end) of the line of CTA c out of G.
__host__ __device__ __forceinline__ long long cut(long long total, int c, int G) {
  return total / G * c + total % G * c / G;
}
// The CTA whose range holds step `it`.
__device__ __forceinline__ int owner(long long total, long long it, int G) {
  int c = (int)(it / (total / G + 1));
  while (c + 1 < G && cut(total, c + 1, G) <= it) ++c;
  return c;
}

// ------------------------------------------------------------ small parts ---
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two fp32 lanes of one 64-bit register
__device__ __forceinline__ uint64_t pk(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void upk(uint64_t v, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if (BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// One warp's share of a stationary tile into tensor memory: lane = row, the
// warp's quarter `w4` of the features (8 * KA columns of two features).
// src: this lane's row, or null for a zero row.
template <int KA>
__device__ __forceinline__ void load_tile_tmem(uint32_t tx, const uint8_t *src, int K, int w4) {
#pragma unroll
  for (int a = 0; a < KA; ++a) {
    const int col = (w4 * KA + a) * 8;  // 16 features
    uint4 v0 = make_uint4(0, 0, 0, 0), v1 = v0;
    if (src) {
      if (2 * col < K) v0 = __ldg(reinterpret_cast<const uint4 *>(src + 4 * col));
      if (2 * col + 8 < K) v1 = __ldg(reinterpret_cast<const uint4 *>(src + 4 * col + 16));
    }
    const uint32_t r[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
    tmem_st8(tx + col, r);
  }
}

// Waits (bounded) until the loads that the producer issued and nobody waited
// for have landed: a CTA that gives up leaves no copy in flight into its
// shared memory.
__device__ __forceinline__ void drain_loads(uint64_t *b_full, long long issued, int stages) {
  const long long first = issued > stages ? issued - stages : 0;
  for (long long n = first; n < issued; ++n) {
    const long long t0 = clock64();
    while (!mbar_try_wait(&b_full[n % stages], (uint32_t)(n / stages) & 1))
      if (clock64() - t0 > (1ll << 30)) break;
  }
}

// ------------------------------------------------------------- forward ------
template <int KA>
struct FwdCfg {
  static constexpr int KP = 64 * KA;
  static constexpr int CN = 128;                      // vocabulary rows of a chunk (MMA N)
  static constexpr int STAGE = KP * CN * 2;
  static constexpr int STAGES = KA == 1 ? 8 : KA == 2 ? 6 : KA == 3 ? 4 : 3;
  static constexpr int NBUF = 3;                      // S buffers
  static constexpr int TX = 0, TS = 128;              // TMEM columns: features, S buffers
  static constexpr int OFF_BAR = STAGES * STAGE;
  static constexpr int NBAR = 2 * STAGES + 2 * NBUF + 1;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int OFF_COMB = (OFF_MISC + 16 + 15) / 16 * 16;   // [2][4][2][128] floats
  static constexpr int OFF_COL = OFF_COMB + 2 * 4 * 2 * kTile * 4;  // [16][32] floats
  static constexpr int SMEM = OFF_COL + kEpiWarps * 32 * 4 + 1024;
};

struct FwdParams {
  const uint8_t *feat;
  const float *bias;
  const Header *hdr;
  const int *rowidx, *tgt;
  float *lt;
  float2 *part;
  int V, K, chunks;
  int *err;
};

template <int KA, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
ce_fwd_kernel(const __grid_constant__ CUtensorMap wmap, const FwdParams p) {
  using C = FwdCfg<KA>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *b_full = reinterpret_cast<uint64_t *>(smem + C::OFF_BAR);
  uint64_t *b_empty = b_full + C::STAGES;
  uint64_t *s_full = b_empty + C::STAGES;
  uint64_t *s_empty = s_full + C::NBUF;
  uint64_t *x_ready = s_empty + C::NBUF;
  uint32_t *s_tmem = reinterpret_cast<uint32_t *>(smem + C::OFF_MISC);
  volatile int *s_abort = reinterpret_cast<volatile int *>(smem + C::OFF_MISC + 4);
  float *comb = reinterpret_cast<float *>(smem + C::OFF_COMB);
  float *scol = reinterpret_cast<float *>(smem + C::OFF_COL);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&b_full[s], 1);
      mbar_init(&b_empty[s], 1);
    }
    for (int b = 0; b < C::NBUF; ++b) {
      mbar_init(&s_full[b], 1);
      mbar_init(&s_empty[b], kEpiWarps / 2);
    }
    mbar_init(x_ready, kEpiWarps);
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(s_tmem, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const int n = p.hdr->n;
  const int NC = p.chunks;
  const long long total = (long long)((n + kTile - 1) / kTile) * NC;
  const long long it0 = cut(total, blockIdx.x, gridDim.x);
  const long long it1 = cut(total, blockIdx.x + 1, gridDim.x);

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&wmap);
      long long j = 0;
      for (long long it = it0; it < it1; ++it, ++j) {
        const int s = (int)(j % C::STAGES);
        const uint32_t u = (uint32_t)(j / C::STAGES);
        if (u > 0 && !mbar_wait_bounded(&b_empty[s], (u - 1) & 1, s_abort, p.err, 61)) break;
        mbar_arrive_expect_tx(&b_full[s], C::STAGE);
        const int c = (int)(it % NC);
        for (int k = 0; k < KA; ++k)
          tma_load_2d(smem + s * C::STAGE + k * C::CN * 128, &wmap, &b_full[s], 64 * k, c * C::CN);
      }
      if (*s_abort) drain_loads(b_full, j, C::STAGES);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = BF16 ? idesc_bf16(kTile, C::CN) : idesc_f16(kTile, C::CN);
      long long j = 0;
      uint32_t seg = 0;
      bool ok = true;
      for (long long it = it0; ok && it < it1; ++it, ++j) {
        if (it == it0 || it % NC == 0) {
          ok = mbar_wait_bounded(x_ready, seg & 1, s_abort, p.err, 62);
          ++seg;
          if (!ok) break;
        }
        const int s = (int)(j % C::STAGES), b = (int)(j % C::NBUF);
        const uint32_t u = (uint32_t)(j / C::STAGES), ub = (uint32_t)(j / C::NBUF);
        if (!mbar_wait_bounded(&b_full[s], u & 1, s_abort, p.err, 63)) break;
        if (ub > 0 && !mbar_wait_bounded(&s_empty[b], (ub - 1) & 1, s_abort, p.err, 64)) break;
        tc_fence_after();
        const uint32_t baddr = smem_u32(smem + s * C::STAGE);
#pragma unroll
        for (int k = 0; k < 4 * KA; ++k)
          mma_f16_ts(tmem + C::TS + b * C::CN, tmem + C::TX + 8 * k,
                     sw128_kmajor_desc(baddr + (k >> 2) * (C::CN * 128) + 32u * (k & 3)), idesc,
                     k > 0 ? 1u : 0u);
        mma_commit(&b_empty[s]);
        mma_commit(&s_full[b]);
      }
    }
  } else {
    const int ew = warp - kEpiWarp0;
    const int grp = ew >> 3;             // chunk parity this warp takes
    const int half = (ew >> 2) & 1;      // its 64 columns of the chunk
    const int quad = warp & 3;           // the TMEM lanes a warp may read
    const int r = quad * 32 + lane;
    const uint32_t tl = tmem + ((uint32_t)(quad * 32) << 16);
    float *col = scol + ew * 32;
    const uint64_t l2e2 = pk(kLog2e, kLog2e);
    long long j = 0;
    int seg = 0;
    bool ok = true;
    for (long long it = it0; it < it1; ++seg) {
      const int tile = (int)(it / NC), c0 = (int)(it % NC);
      const int cnt = (int)min((long long)(NC - c0), it1 - it);
      const int row = tile * kTile + r;  // kept rows are numbered from 0
      const int src = row < n ? p.rowidx[row] : -1;
      const int tg = row < n ? p.tgt[row] : -1;
      load_tile_tmem<KA>(tl + C::TX, src >= 0 ? p.feat + (size_t)src * p.K * 2 : nullptr, p.K,
                         ew >> 2);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(x_ready);
      // running maximum of y = l * log2(e), and the sum of exp2(y - base)
      float my = -INFINITY, sum = 0.f, base = 0.f;
      for (int i = 0; i < cnt; ++i, ++j) {
        if ((int)(j & 1) != grp) continue;
        const int b = (int)(j % C::NBUF);
        const uint32_t ub = (uint32_t)(j / C::NBUF);
        const int v0 = (c0 + i) * C::CN + half * 64;
        float bl[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const int v = v0 + 32 * g + lane;
          bl[g] = v < p.V ? (p.bias ? __ldg(p.bias + v) * kLog2e : 0.f) : -INFINITY;
        }
        ok = ok && mbar_wait_bounded(&s_full[b], ub & 1, s_abort, p.err, 65);
        if (!ok) break;
        tc_fence_after();
        const uint32_t ts = tl + C::TS + b * C::CN + half * 64;
        uint32_t va[32], vb[32];
        tmem_ld32(ts, va);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          uint32_t(&v)[32] = g ? vb : va;
          const int cb = v0 + 32 * g;
          __syncwarp();
          col[lane] = bl[g];
          __syncwarp();
          tmem_ld_wait(v);
          if (g == 0) tmem_ld32(ts + 32, vb);
          if (g == 1) {  // all of this warp's columns are in registers
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_empty[b]);
          }
          if (cb >= p.V) continue;
          uint64_t y[16];
          const ulonglong2 *cq = reinterpret_cast<const ulonglong2 *>(col);
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const ulonglong2 bb = cq[q];
            y[2 * q] = fma2(pk(__uint_as_float(v[4 * q]), __uint_as_float(v[4 * q + 1])), l2e2,
                            bb.x);
            y[2 * q + 1] = fma2(pk(__uint_as_float(v[4 * q + 2]), __uint_as_float(v[4 * q + 3])),
                                l2e2, bb.y);
          }
          float f[32];
#pragma unroll
          for (int q = 0; q < 16; ++q) upk(y[q], f[2 * q], f[2 * q + 1]);
          const bool hit = tg >= cb && tg < cb + 32;
          if (__any_sync(~0u, hit)) {
            float l = 0.f;
#pragma unroll
            for (int q = 0; q < 32; ++q)
              if (tg == cb + q) l = f[q];
            if (hit) p.lt[row] = l;
          }
          float m[11];
#pragma unroll
          for (int q = 0; q < 10; ++q) m[q] = fmaxf(fmaxf(f[3 * q], f[3 * q + 1]), f[3 * q + 2]);
          m[10] = fmaxf(f[30], f[31]);
          const float m0 = fmaxf(fmaxf(m[0], m[1]), m[2]), m1 = fmaxf(fmaxf(m[3], m[4]), m[5]);
          const float m2 = fmaxf(fmaxf(m[6], m[7]), m[8]), m3 = fmaxf(m[9], m[10]);
          const float gm = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
          if (gm > my) {
            my = gm;
            // base stays 0 while the maximum is within 2^64 of it
            if (my > base + 64.f || my < base - 64.f) {
              sum = sum > 0.f ? sum * ex2(base - my) : 0.f;
              base = my;
            }
          }
          uint64_t s4[4] = {0, 0, 0, 0};
          if (__any_sync(~0u, base != 0.f)) {
            const uint64_t nb = pk(-base, -base);
#pragma unroll
            for (int q = 0; q < 16; ++q) {
              float a0, a1;
              upk(add2(y[q], nb), a0, a1);
              s4[q & 3] = add2(s4[q & 3], pk(ex2(a0), ex2(a1)));
            }
          } else {
#pragma unroll
            for (int q = 0; q < 16; ++q)
              s4[q & 3] = add2(s4[q & 3], pk(ex2(f[2 * q]), ex2(f[2 * q + 1])));
          }
          float a0, a1;
          upk(add2(add2(s4[0], s4[1]), add2(s4[2], s4[3])), a0, a1);
          sum += a0 + a1;
        }
      }
      // the four column shares of a row into one (max, sum relative to it).
      // A NaN logit does not show in the maximum but makes the sum NaN.
      const float rel = my == -INFINITY ? sum : sum * ex2(base - my);
      float *cp = comb + (seg & 1) * 8 * kTile;
      cp[(ew >> 2) * 2 * kTile + r] = my;
      cp[(ew >> 2) * 2 * kTile + kTile + r] = rel;
      ok = named_bar_and(1, kEpiThreads, ok);
      if (!ok) break;
      if ((ew >> 2) == 0) {
        float M = my;
#pragma unroll
        for (int q = 1; q < 4; ++q) M = fmaxf(M, cp[q * 2 * kTile + r]);
        float S = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float mq = cp[q * 2 * kTile + r], sq = cp[q * 2 * kTile + kTile + r];
          S += mq == -INFINITY ? sq : sq * ex2(mq - M);
        }
        p.part[(size_t)(tile + blockIdx.x) * kTile + r] = make_float2(M, S);
      }
      it += cnt;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the pieces of every kept row, in the order of the vocabulary.
__global__ void __launch_bounds__(128)
ce_loss_kernel(const Header *hdr, const int *rowidx, const float *lt, const float2 *part,
               int chunks, int G, float *loss, float *lse) {
  const int n = hdr->n;
  const int tile = blockIdx.x, r = threadIdx.x;
  const int row = tile * kTile + r;
  if (row >= n) return;
  const long long total = (long long)((n + kTile - 1) / kTile) * chunks;
  const int ca = owner(total, (long long)tile * chunks, G);
  const int cb = owner(total, (long long)(tile + 1) * chunks - 1, G);
  float M = -INFINITY, S = 0.f;
  for (int c = ca; c <= cb; ++c) {
    if (cut(total, c, G) == cut(total, c + 1, G)) continue;
    const float2 v = part[(size_t)(tile + c) * kTile + r];
    const float m = fmaxf(M, v.x);
    S = (M == -INFINITY ? S : S * exp2f(M - m)) + (v.x == -INFINITY ? v.y : v.y * exp2f(v.x - m));
    M = m;
  }
  const float ls = logf(S);
  const int i = rowidx[row];
  lse[i] = fmaf(M, kLn2, ls);
  loss[i] = fmaf(M - lt[row], kLn2, ls);
}

// ------------------------------------------------------------- backward -----
template <int KA>
struct BwdCfg {
  static constexpr int KP = 64 * KA;
  static constexpr int CN = KA <= 2 ? 128 : 64;       // streamed rows of a chunk
  static constexpr int HC = CN / 2;                   // columns of S per epilogue warp
  static constexpr int STAGE = KP * CN * 2;
  static constexpr int STAGES = KA == 1 ? 8 : KA == 2 ? 5 : KA == 3 ? 7 : 5;
  static constexpr int TD = 0, TX = KP, TS = KP + KP / 2;  // TMEM columns: D, tile, two S
  static constexpr int OFF_BAR = STAGES * STAGE;
  static constexpr int NBAR = 2 * STAGES + 6;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int OFF_BSUM = (OFF_MISC + 16 + 15) / 16 * 16;   // [2][4][128] floats
  static constexpr int OFF_COL = OFF_BSUM + 2 * 4 * kTile * 4;      // [16][3][32] words
  static constexpr int SMEM = OFF_COL + kEpiWarps * 96 * 4 + 1024;
  static_assert(TS + 2 * CN <= kTmemCols, "tensor memory");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct BwdParams {
  const uint8_t *w, *xc;
  const float *bias;
  const Header *hdr;
  const int *rowidx, *tgt;
  const float *nlse, *gc, *gs;
  uint8_t *dfeat, *dw;
  float *dbias;
  float *dpart, *bpart;
  int V, K, chunks_v;
  int tiles_w;       // 0: no gradient of the weights or bias wanted
  int want_x;        // 0: no gradient of the features wanted
  float shift;       // log2 of the scale of P for dF
  float unscale;     // 2^-shift
  int *err;
};

// The line of steps of a backward call: first the tiles of F (dF), then the
// tiles of W (dW, db).
struct BwdLine {
  int n, chunks_v, chunks_r, tiles_x, tiles_w;
  long long its_x, total;
  __device__ BwdLine(const Header *h, int cn, int cv, int want_x, int tw) {
    n = h->n;
    chunks_v = cv;
    chunks_r = max(1, (n + cn - 1) / cn);  // no rows: one chunk of zeros, so that dW is written
    tiles_x = want_x ? (n + kTile - 1) / kTile : 0;
    tiles_w = tw;
    its_x = (long long)tiles_x * chunks_v;
    total = its_x + (long long)tiles_w * chunks_r;
  }
  // the tile and chunk of a step, and the chunks of that tile
  __device__ void at(long long it, bool &dw, int &tile, int &chunk, int &chunks) const {
    dw = it >= its_x;
    if (dw) it -= its_x;
    chunks = dw ? chunks_r : chunks_v;
    tile = (int)(it / chunks);
    chunk = (int)(it % chunks);
  }
};

template <int KA, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
ce_bwd_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
              const BwdParams p) {
  using C = BwdCfg<KA>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *b_full = reinterpret_cast<uint64_t *>(smem + C::OFF_BAR);
  uint64_t *b_empty = b_full + C::STAGES;
  uint64_t *s_full = b_empty + C::STAGES;   // [2]
  uint64_t *p_full = s_full + 2;            // [2]
  uint64_t *x_ready = p_full + 2;
  uint64_t *d_full = x_ready + 1;
  uint32_t *s_tmem = reinterpret_cast<uint32_t *>(smem + C::OFF_MISC);
  volatile int *s_abort = reinterpret_cast<volatile int *>(smem + C::OFF_MISC + 4);
  float *bsum = reinterpret_cast<float *>(smem + C::OFF_BSUM);
  float *scol = reinterpret_cast<float *>(smem + C::OFF_COL);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&b_full[s], 1);
      mbar_init(&b_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&s_full[b], 1);
      mbar_init(&p_full[b], kEpiWarps / 2);
    }
    mbar_init(x_ready, kEpiWarps);
    mbar_init(d_full, 1);
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(s_tmem, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const BwdLine line(p.hdr, C::CN, p.chunks_v, p.want_x, p.tiles_w);
  const long long it0 = cut(line.total, blockIdx.x, gridDim.x);
  const long long it1 = cut(line.total, blockIdx.x + 1, gridDim.x);

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&wmap);
      tma_prefetch_desc(&xmap);
      long long j = 0;
      for (long long it = it0; it < it1; ++it, ++j) {
        const int s = (int)(j % C::STAGES);
        const uint32_t u = (uint32_t)(j / C::STAGES);
        if (u > 0 && !mbar_wait_bounded(&b_empty[s], (u - 1) & 1, s_abort, p.err, 71)) break;
        mbar_arrive_expect_tx(&b_full[s], C::STAGE);
        bool dw;
        int tile, c, nc;
        line.at(it, dw, tile, c, nc);
        for (int k = 0; k < KA; ++k)
          tma_load_2d(smem + s * C::STAGE + k * C::CN * 128, dw ? &xmap : &wmap, &b_full[s], 64 * k,
                      c * C::CN);
      }
      if (*s_abort) drain_loads(b_full, j, C::STAGES);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t id1 = BF16 ? idesc_bf16(kTile, C::CN) : idesc_f16(kTile, C::CN);
      constexpr uint32_t id2 =
          (BF16 ? idesc_bf16(kTile, C::KP) : idesc_f16(kTile, C::KP)) | kIdescBMnMajor;
      long long j = 0;  // chunk of this CTA
      uint32_t seg = 0;
      bool ok = true;
      // S = tile x chunk^T of chunk jj into its buffer
      auto first = [&](long long jj) {
        const int s = (int)(jj % C::STAGES);
        const uint32_t u = (uint32_t)(jj / C::STAGES);
        if (!mbar_wait_bounded(&b_full[s], u & 1, s_abort, p.err, 72)) return false;
        tc_fence_after();
        const uint32_t baddr = smem_u32(smem + s * C::STAGE);
#pragma unroll
        for (int k = 0; k < 4 * KA; ++k)
          mma_f16_ts(tmem + C::TS + (uint32_t)(jj & 1) * C::CN, tmem + C::TX + 8 * k,
                     sw128_kmajor_desc(baddr + (k >> 2) * (C::CN * 128) + 32u * (k & 3)), id1,
                     k > 0 ? 1u : 0u);
        mma_commit(&s_full[jj & 1]);
        return true;
      };
      for (long long it = it0; ok && it < it1; ++seg) {
        bool dw;
        int tile, c0, nc;
        line.at(it, dw, tile, c0, nc);
        const int cnt = (int)min((long long)(nc - c0), it1 - it);
        ok = mbar_wait_bounded(x_ready, seg & 1, s_abort, p.err, 73);
        if (!ok) break;
        tc_fence_after();
        ok = first(j) && (cnt < 2 || first(j + 1));
        for (int i = 0; ok && i < cnt; ++i, ++j) {
          const int s = (int)(j % C::STAGES), b = (int)(j & 1);
          ok = mbar_wait_bounded(&p_full[b], (uint32_t)(j >> 1) & 1, s_abort, p.err, 74);
          if (!ok) break;
          tc_fence_after();
          const uint32_t baddr = smem_u32(smem + s * C::STAGE);
#pragma unroll
          for (int k = 0; k < C::CN / 16; ++k) {
            // P of each half of the chunk lies at the head of that half's S columns
            const uint32_t pc = (16 * k / C::HC) * C::HC + (16 * k % C::HC) / 2;
            mma_f16_ts(tmem + C::TD, tmem + C::TS + (uint32_t)b * C::CN + pc,
                       sw128_mnmajor_desc(baddr + 2048u * k, C::CN * 128), id2,
                       i > 0 || k > 0 ? 1u : 0u);
          }
          mma_commit(&b_empty[s]);
          if (i + 1 == cnt) mma_commit(d_full);
          // the next S into this buffer: issued after the product that reads P
          // there, and the tensor pipe keeps that order
          if (i + 2 < cnt) ok = first(j + 2);
        }
        it += cnt;
      }
    }
  } else {
    const int ew = warp - kEpiWarp0;
    const int grp = ew >> 3;
    const int half = (ew >> 2) & 1;
    const int w4 = ew >> 2;
    const int quad = warp & 3;
    const int r = quad * 32 + lane;
    const uint32_t tl = tmem + ((uint32_t)(quad * 32) << 16);
    float *ccol = scol + ew * 96;      // additive term of y per column
    float *csc = ccol + 32;            // dW: scale per column
    int *ctg = reinterpret_cast<int *>(ccol + 64);  // dW: target per column
    const uint64_t l2e2 = pk(kLog2e, kLog2e);
    long long j = 0;
    int seg = 0;
    bool ok = true;
    for (long long it = it0; it < it1; ++seg) {
      bool dw;
      int tile, c0, nc;
      line.at(it, dw, tile, c0, nc);
      const int cnt = (int)min((long long)(nc - c0), it1 - it);
      const int row = tile * kTile + r;                // kept row, or class
      const bool real = row < (dw ? p.V : line.n);
      load_tile_tmem<KA>(tl + C::TX,
                         real ? (dw ? p.w : p.xc) + (size_t)row * p.K * 2 : nullptr, p.K, w4);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(x_ready);
      // y = S * log2(e) + column term + row term; P = exp2(y) (* column scale)
      const int tg = !dw && real ? p.tgt[row] : -1;
      float rterm = -INFINITY;
      if (real) rterm = dw ? (p.bias ? p.bias[row] * kLog2e : 0.f) : p.nlse[row] + p.shift;
      const uint64_t rt2 = pk(rterm, rterm);
      const float one = exp2f(p.shift);
      uint64_t acc2 = 0;
      for (int i = 0; i < cnt; ++i, ++j) {
        const int b = (int)(j & 1);
        if (b != grp) continue;
        const int v0 = (c0 + i) * C::CN + half * C::HC;
        float ct[C::HC / 32], cs[C::HC / 32];
        int cg[C::HC / 32];
#pragma unroll
        for (int g = 0; g < C::HC / 32; ++g) {
          const int v = v0 + 32 * g + lane;
          if (dw) {  // the arrays reach to the end of the last tile
            ct[g] = __ldg(p.nlse + v);
            cs[g] = __ldg(p.gs + v);
            cg[g] = __ldg(p.tgt + v);
          } else {
            ct[g] = v < p.V ? (p.bias ? __ldg(p.bias + v) * kLog2e : 0.f) : -INFINITY;
          }
        }
        ok = ok && mbar_wait_bounded(&s_full[b], (uint32_t)(j >> 1) & 1, s_abort, p.err, 75);
        if (!ok) break;
        tc_fence_after();
        const uint32_t ts = tl + C::TS + b * C::CN + half * C::HC;
#pragma unroll
        for (int g = 0; g < C::HC / 32; ++g) {
          uint32_t v[32];
          tmem_ld32(ts + 32 * g, v);
          const int cb = v0 + 32 * g;
          __syncwarp();
          ccol[lane] = ct[g];
          if (dw) {
            csc[lane] = cs[g];
            ctg[lane] = cg[g];
          }
          __syncwarp();
          tmem_ld_wait(v);
          float f[32];
          const ulonglong2 *cq = reinterpret_cast<const ulonglong2 *>(ccol);
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const ulonglong2 bb = cq[q];
            upk(add2(fma2(pk(__uint_as_float(v[4 * q]), __uint_as_float(v[4 * q + 1])), l2e2, bb.x),
                     rt2),
                f[4 * q], f[4 * q + 1]);
            upk(add2(fma2(pk(__uint_as_float(v[4 * q + 2]), __uint_as_float(v[4 * q + 3])), l2e2,
                          bb.y),
                     rt2),
                f[4 * q + 2], f[4 * q + 3]);
          }
#pragma unroll
          for (int q = 0; q < 32; ++q) f[q] = ex2(f[q]);
          if (dw) {
            // columns whose target is among this warp's 32 classes
            const int v32 = tile * kTile + quad * 32;
            const bool any = __any_sync(~0u, cg[g] >= v32 && cg[g] < v32 + 32);
            if (any) {
#pragma unroll
              for (int q = 0; q < 32; ++q)
                if (ctg[q] == row) f[q] -= 1.f;
            }
            const ulonglong2 *sq = reinterpret_cast<const ulonglong2 *>(csc);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const ulonglong2 ss = sq[q];
              const uint64_t a = mul2(pk(f[4 * q], f[4 * q + 1]), ss.x);
              const uint64_t c = mul2(pk(f[4 * q + 2], f[4 * q + 3]), ss.y);
              acc2 = add2(acc2, add2(a, c));
              upk(a, f[4 * q], f[4 * q + 1]);
              upk(c, f[4 * q + 2], f[4 * q + 3]);
            }
          } else {
            if (__any_sync(~0u, tg >= cb && tg < cb + 32)) {
#pragma unroll
              for (int q = 0; q < 32; ++q)
                if (tg == cb + q) f[q] -= one;
            }
          }
          uint32_t h[16];
#pragma unroll
          for (int q = 0; q < 16; ++q) h[q] = pack16<BF16>(f[2 * q], f[2 * q + 1]);
          tmem_st16(ts + 16 * g, h);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[b]);
      }
      float a0, a1;
      upk(acc2, a0, a1);
      float *bs = bsum + (seg & 1) * 4 * kTile;
      if (dw) bs[w4 * kTile + r] = a0 + a1;
      ok = ok && mbar_wait_bounded(d_full, seg & 1, s_abort, p.err, 76);
      ok = named_bar_and(1, kEpiThreads, ok);
      if (!ok) break;
      tc_fence_after();
      const bool whole = cnt == nc;
      const int slot = 2 * blockIdx.x + (c0 == 0 ? 1 : 0);
      float scale = 1.f;
      uint8_t *out = nullptr;
      if (whole && real) {
        if (dw) {
          scale = p.hdr->gmax * p.unscale;
          if (p.dw) out = p.dw + (size_t)row * p.K * 2;
        } else {
          scale = p.gc[row] * p.unscale;
          out = p.dfeat + (size_t)p.rowidx[row] * p.K * 2;
        }
      }
      if (dw && real && w4 == 0) {
        const float s = (bs[r] + bs[kTile + r]) + (bs[2 * kTile + r] + bs[3 * kTile + r]);
        if (!whole)
          p.bpart[(size_t)slot * kTile + r] = s;
        else if (p.dbias)
          p.dbias[row] = s * scale;
      }
#pragma unroll
      for (int a = 0; a < KA; ++a) {
        const int col = (w4 * KA + a) * 16;
        uint32_t v[16];
        tmem_ld16(tl + C::TD + col, v);
        tmem_ld_wait(v);
        if (!real) continue;
        if (whole) {
          if (out) {
            uint32_t h[8];
#pragma unroll
            for (int q = 0; q < 8; ++q)
              h[q] = pack16<BF16>(__uint_as_float(v[2 * q]) * scale,
                                  __uint_as_float(v[2 * q + 1]) * scale);
            uint4 *o = reinterpret_cast<uint4 *>(out + 2 * col);
            if (col < p.K) o[0] = make_uint4(h[0], h[1], h[2], h[3]);
            if (col + 8 < p.K) o[1] = make_uint4(h[4], h[5], h[6], h[7]);
          }
        } else {
          uint4 *o = reinterpret_cast<uint4 *>(p.dpart + ((size_t)slot * kTile + r) * C::KP + col);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            o[q] = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        }
      }
      tc_fence_before();  // D and the tile are read before the next x_ready
      it += cnt;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Sums the pieces of the tiles that a range border cut, in the order of the
// CTAs, and rounds them as the main kernel rounds a whole tile. blockIdx.x:
// border (CTA c > 0), y: a slice of the tile.
template <bool BF16>
__global__ void __launch_bounds__(256)
ce_join_kernel(const BwdParams p, int cn, int KP, int G) {
  const BwdLine line(p.hdr, cn, p.chunks_v, p.want_x, p.tiles_w);
  // the first border inside a tile handles that tile (with few steps some
  // CTAs have an empty range)
  const int c = blockIdx.x + 1;
  const long long at = cut(line.total, c, G);
  if (at == 0 || at == cut(line.total, c + 1, G)) return;
  bool dw;
  int tile, chunk, nc;
  line.at(at, dw, tile, chunk, nc);
  if (chunk == 0) return;
  const long long t0 = at - chunk;  // first step of the tile
  const int head = owner(line.total, at - 1, G);
  if (cut(line.total, head, G) > t0) return;
  int last = c;
  while (last + 1 < G && cut(line.total, last + 1, G) < t0 + nc) ++last;
  const int lim = min(kTile, (dw ? p.V : line.n) - tile * kTile);
  const int q4 = KP / 4;
  const float gmax = p.hdr->gmax;
  const int step = gridDim.y * blockDim.x;
  for (int e = blockIdx.y * blockDim.x + threadIdx.x; e < lim * q4; e += step) {
    const int r = e / q4, k = (e - r * q4) * 4;
    if (k >= p.K || (dw && !p.dw)) continue;
    const size_t o = (size_t)r * KP + k;
    const float *src = p.dpart + o;
    const size_t ps = (size_t)kTile * KP;
    float4 s = *reinterpret_cast<const float4 *>(src + (2 * head + 1) * ps);
    for (int d = c; d <= last; ++d) {
      if (cut(line.total, d, G) == cut(line.total, d + 1, G)) continue;
      const float4 v = *reinterpret_cast<const float4 *>(src + 2 * d * ps);
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
    const int row = tile * kTile + r;
    const float sc = (dw ? gmax : p.gc[row]) * p.unscale;
    const uint2 h = make_uint2(pack16<BF16>(s.x * sc, s.y * sc), pack16<BF16>(s.z * sc, s.w * sc));
    uint8_t *out = dw ? p.dw + (size_t)row * p.K * 2 : p.dfeat + (size_t)p.rowidx[row] * p.K * 2;
    *reinterpret_cast<uint2 *>(out + 2 * k) = h;
  }
  if (dw && p.dbias && blockIdx.y == 0)
    for (int r = threadIdx.x; r < lim; r += blockDim.x) {
      float s = p.bpart[(size_t)(2 * head + 1) * kTile + r];
      for (int d = c; d <= last; ++d)
        if (cut(line.total, d, G) != cut(line.total, d + 1, G))
          s += p.bpart[(size_t)2 * d * kTile + r];
      p.dbias[tile * kTile + r] = s * (gmax * p.unscale);
    }
}

// ----------------------------------------------------------------- host -----
template <typename F>
int allow_smem(F *kernel, int bytes, const char *what) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  return e == cudaSuccess ? TOCR_OK
                          : set_error(TOCR_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

int grid_for(long long steps, int least) {
  const long long g = (steps + least - 1) / least;
  const int most = sm_count() < kMaxGrid ? sm_count() : kMaxGrid;
  return (int)(g < 1 ? 1 : g < most ? g : most);
}

template <int KA, bool BF16>
int launch_fwd(const FwdParams &p, const void *w, int grid, cudaStream_t st) {
  using C = FwdCfg<KA>;
  CUtensorMap wm;
  int rc = tma_map_rows(&wm, BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                        2, w, p.K, p.V, 2ll * p.K, C::CN);
  if (rc) return rc;
  rc = allow_smem(ce_fwd_kernel<KA, BF16>, C::SMEM, "tocr_rec_head_ce");
  if (rc) return rc;
  ce_fwd_kernel<KA, BF16><<<grid, kThreads, C::SMEM, st>>>(wm, p);
  return check_launch("ce_fwd_kernel");
}

template <int KA, bool BF16>
int launch_bwd(const BwdParams &p, int rows_pad, int grid, cudaStream_t st) {
  using C = BwdCfg<KA>;
  CUtensorMap wm, xm;
  const CUtensorMapDataType ty =
      BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  int rc = tma_map_rows(&wm, ty, 2, p.w, p.K, p.V, 2ll * p.K, C::CN);
  if (rc) return rc;
  rc = tma_map_rows(&xm, ty, 2, p.xc, p.K, rows_pad, 2ll * p.K, C::CN);
  if (rc) return rc;
  rc = allow_smem(ce_bwd_kernel<KA, BF16>, C::SMEM, "tocr_rec_head_ce_backward");
  if (rc) return rc;
  ce_bwd_kernel<KA, BF16><<<grid, kThreads, C::SMEM, st>>>(wm, xm, p);
  rc = check_launch("ce_bwd_kernel");
  if (rc || grid == 1) return rc;
  ce_join_kernel<BF16><<<dim3(grid - 1, 8), 256, 0, st>>>(p, C::CN, C::KP, grid);
  return check_launch("ce_join_kernel");
}

template <bool BWD>
int launch_place(const Workspace &ws, const void *targets, bool wide, int rows, int V, int K,
                 int dtype, const void *feat, const float *lse, const float *g, void *dfeat,
                 float *loss, float *lse_out, cudaStream_t st) {
  const int blocks = rows > kRowBlock ? (rows + kRowBlock - 1) / kRowBlock : 1;
  ce_count_kernel<<<blocks, kRowBlock, 0, st>>>(targets, wide, rows, V, g, ws.cnt, ws.gblk);
  int rc = check_launch("ce_count_kernel");
  if (rc) return rc;
  PlaceParams p{};
  p.targets = targets;
  p.wide = wide;
  p.rows = rows;
  p.V = V;
  p.K = K;
  p.shift = dtype == TOCR_DTYPE_F16 ? (float)(1 << kShift) : 1.f;
  p.cnt = ws.cnt;
  p.gblk = ws.gblk;
  p.hdr = ws.hdr;
  p.rowidx = ws.rowidx;
  p.tgt = ws.tgt;
  p.loss = loss;
  p.lse_out = lse_out;
  p.feat = static_cast<const uint8_t *>(feat);
  p.lse = lse;
  p.g = g;
  p.xc = ws.xc;
  p.dfeat = static_cast<uint8_t *>(dfeat);
  p.nlse = ws.nlse;
  p.gc = ws.gc;
  p.gs = ws.gs;
  ce_place_kernel<BWD><<<blocks, kRowBlock, 0, st>>>(p);
  return check_launch("ce_place_kernel");
}

int check_sizes(const char *fn, long long rows, int K, int V, int dtype) {
  TOCR_REQUIRE(rows >= 0 && rows <= kMaxRows && V > 0 && V <= (1 << 24),
               "%s: bad sizes rows=%lld classes=%d", fn, rows, V);
  TOCR_REQUIRE(K >= 8 && K <= kMaxK && K % 8 == 0,
               "%s: K must be a multiple of 8 up to 256 (got %d)", fn, K);
  TOCR_REQUIRE(dtype == TOCR_DTYPE_F16 || dtype == TOCR_DTYPE_BF16,
               "%s: features and weights must be fp16 or bf16", fn);
  return TOCR_OK;
}

}  // namespace
}  // namespace tocr

using namespace tocr;

extern "C" {

TOCR_API size_t tocr_rec_head_ce_workspace_bytes(long long rows, int K, int num_classes,
                                                 int backward) {
  if (rows < 0 || rows > kMaxRows || K < 8 || K > kMaxK || K % 8 || num_classes <= 0) return 0;
  return carve(nullptr, rows, K, backward != 0).bytes;
}

TOCR_API int tocr_rec_head_ce(const void *d_feat, const void *d_w, const float *d_bias,
                              const void *d_targets, int targets_i64, long long rows, int K,
                              int num_classes, int dtype, float *d_loss, float *d_lse,
                              void *d_workspace, size_t workspace_bytes, int *d_err,
                              void *stream) {
  TOCR_ENTRY();
  int rc = check_sizes("tocr_rec_head_ce", rows, K, num_classes, dtype);
  if (rc || rows == 0) return rc;
  TOCR_REQUIRE(d_feat && d_w && d_targets && d_loss && d_lse && d_workspace && d_err,
               "tocr_rec_head_ce: null pointer");
  TOCR_REQUIRE(aligned(d_feat, 16) && aligned(d_w, 16),
               "tocr_rec_head_ce: features and weights must be 16-byte aligned");
  TOCR_REQUIRE(aligned(d_workspace, 256) &&
                   workspace_bytes >= carve(nullptr, rows, K, false).bytes,
               "tocr_rec_head_ce: the workspace must be 256-byte aligned and hold %zu bytes",
               carve(nullptr, rows, K, false).bytes);
  cudaStream_t st = as_stream(stream);
  const Workspace ws = carve(static_cast<uint8_t *>(d_workspace), rows, K, false);
  rc = launch_place<false>(ws, d_targets, targets_i64 != 0, (int)rows, num_classes, K, dtype,
                           nullptr, nullptr, nullptr, nullptr, d_loss, d_lse, st);
  if (rc) return rc;
  FwdParams p{};
  p.feat = static_cast<const uint8_t *>(d_feat);
  p.bias = d_bias;
  p.hdr = ws.hdr;
  p.rowidx = ws.rowidx;
  p.tgt = ws.tgt;
  p.lt = ws.lt;
  p.part = ws.part;
  p.V = num_classes;
  p.K = K;
  p.chunks = (num_classes + FwdCfg<1>::CN - 1) / FwdCfg<1>::CN;
  p.err = d_err;
  const int tiles = (int)((rows + kTile - 1) / kTile);
  const int grid = grid_for((long long)tiles * p.chunks, 1);
  const bool bf = dtype == TOCR_DTYPE_BF16;
  switch ((K + 63) / 64) {
    case 1: rc = bf ? launch_fwd<1, true>(p, d_w, grid, st) : launch_fwd<1, false>(p, d_w, grid, st); break;
    case 2: rc = bf ? launch_fwd<2, true>(p, d_w, grid, st) : launch_fwd<2, false>(p, d_w, grid, st); break;
    case 3: rc = bf ? launch_fwd<3, true>(p, d_w, grid, st) : launch_fwd<3, false>(p, d_w, grid, st); break;
    default: rc = bf ? launch_fwd<4, true>(p, d_w, grid, st) : launch_fwd<4, false>(p, d_w, grid, st);
  }
  if (rc) return rc;
  ce_loss_kernel<<<tiles, kTile, 0, st>>>(ws.hdr, ws.rowidx, ws.lt, ws.part, p.chunks, grid, d_loss,
                                          d_lse);
  return check_launch("ce_loss_kernel");
}

TOCR_API int tocr_rec_head_ce_backward(const void *d_feat, const void *d_w, const float *d_bias,
                                       const void *d_targets, int targets_i64, long long rows,
                                       int K, int num_classes, int dtype, const float *d_lse,
                                       const float *d_grad_loss, void *d_dfeat, void *d_dw,
                                       float *d_dbias, void *d_workspace, size_t workspace_bytes,
                                       int *d_err, void *stream) {
  TOCR_ENTRY();
  int rc = check_sizes("tocr_rec_head_ce_backward", rows, K, num_classes, dtype);
  if (rc) return rc;
  if (!d_dfeat && !d_dw && !d_dbias) return TOCR_OK;
  if (rows == 0 && !d_dw && !d_dbias) return TOCR_OK;
  TOCR_REQUIRE(d_w && d_workspace && d_err &&
                   (rows == 0 || (d_feat && d_targets && d_lse && d_grad_loss)),
               "tocr_rec_head_ce_backward: null pointer");
  TOCR_REQUIRE(aligned(d_feat, 16) && aligned(d_w, 16) && aligned(d_dfeat, 16) && aligned(d_dw, 16),
               "tocr_rec_head_ce_backward: features, weights and their gradients must be 16-byte "
               "aligned");
  TOCR_REQUIRE(aligned(d_workspace, 256) && workspace_bytes >= carve(nullptr, rows, K, true).bytes,
               "tocr_rec_head_ce_backward: the workspace must be 256-byte aligned and hold %zu bytes",
               carve(nullptr, rows, K, true).bytes);
  cudaStream_t st = as_stream(stream);
  const Workspace ws = carve(static_cast<uint8_t *>(d_workspace), rows, K, true);
  rc = launch_place<true>(ws, d_targets, targets_i64 != 0, (int)rows, num_classes, K, dtype, d_feat,
                          d_lse, d_grad_loss, d_dfeat, nullptr, nullptr, st);
  if (rc) return rc;
  const int KA = (K + 63) / 64;
  const int cn = KA <= 2 ? 128 : 64;
  BwdParams p{};
  p.w = static_cast<const uint8_t *>(d_w);
  p.xc = ws.xc;
  p.bias = d_bias;
  p.hdr = ws.hdr;
  p.rowidx = ws.rowidx;
  p.tgt = ws.tgt;
  p.nlse = ws.nlse;
  p.gc = ws.gc;
  p.gs = ws.gs;
  p.dfeat = static_cast<uint8_t *>(d_dfeat);
  p.dw = static_cast<uint8_t *>(d_dw);
  p.dbias = d_dbias;
  p.dpart = ws.dpart;
  p.bpart = ws.bpart;
  p.V = num_classes;
  p.K = K;
  p.chunks_v = (num_classes + cn - 1) / cn;
  p.tiles_w = d_dw || d_dbias ? (num_classes + kTile - 1) / kTile : 0;
  p.want_x = d_dfeat && rows > 0;
  p.shift = dtype == TOCR_DTYPE_F16 ? (float)kShift : 0.f;
  p.unscale = dtype == TOCR_DTYPE_F16 ? 1.f / (1 << kShift) : 1.f;
  p.err = d_err;
  const long long tiles_x = p.want_x ? (rows + kTile - 1) / kTile : 0;
  const long long chunks_r = rows > cn ? (rows + cn - 1) / cn : 1;
  const int grid = grid_for(tiles_x * p.chunks_v + p.tiles_w * chunks_r, 1);
  const int rows_pad = (int)((rows + kTile - 1) / kTile * kTile + kTile);
  const bool bf = dtype == TOCR_DTYPE_BF16;
  switch (KA) {
    case 1: return bf ? launch_bwd<1, true>(p, rows_pad, grid, st) : launch_bwd<1, false>(p, rows_pad, grid, st);
    case 2: return bf ? launch_bwd<2, true>(p, rows_pad, grid, st) : launch_bwd<2, false>(p, rows_pad, grid, st);
    case 3: return bf ? launch_bwd<3, true>(p, rows_pad, grid, st) : launch_bwd<3, false>(p, rows_pad, grid, st);
    default: return bf ? launch_bwd<4, true>(p, rows_pad, grid, st) : launch_bwd<4, false>(p, rows_pad, grid, st);
  }
}

}  // extern "C"
