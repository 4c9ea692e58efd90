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
// 2^-11 in fp16 and 2^-8 in bf16), or, for up to 512 rows, to the sum of two such
// numbers. The one rounding shows in dW, most of whose rows have few G_ij of
// weight, at any number of rows: its error against 64 bits (2-norm) is 1.3 times
// what the rounding of the output alone leaves, 2.7e-4 instead of 2.1e-4 at 10240
// x 128 x 18385 fp16, 2.1e-3 instead of 1.6e-3 at 16384 x 256 x 18385 bf16 (dF
// 1.03 times). The second number costs its product: nothing at 175 x 64 x 5000
// (18.5 us of backward pass), 5 % at 512 x 128 x 18385 (45 -> 47), 13 % at 2560
// rows, 23 % at 10240 (209 -> 256, 16384 x 256 x 18385 bf16 538 -> 669). So few
// rows, which are a matter of latency, have it, and more rows do not. fp16 holds P
// scaled by 2^14, so that a probability of 2^-28 is still a normal number, and for
// dW the row weights enter divided by their largest, so that small weights do not
// underflow.
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
constexpr int kEpiWarps = 16;    // forward: two groups of eight that take every other chunk
constexpr int kThreads = 32 * (kEpiWarp0 + kEpiWarps);
constexpr int kEpiThreads = 32 * kEpiWarps;
constexpr int kTmemCols = 512;
constexpr int kPolyPairs = 2;    // of 16 pairs of exponentials, those not left to the special-function unit
constexpr int kColSlots = 8;     // ring of the streamed rows' per-row terms
constexpr int kRowBlock = 256;   // rows per block of the numbering kernels
constexpr int kJoinThreads = 256;
constexpr int kDirect = 4;       // blocks whose rows the placing kernel counts itself
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxK = 256;
constexpr long long kMaxRows = 1ll << 24;
constexpr int kMaxClasses = 1 << 24;
constexpr int kMaxGrid = 148;    // CTAs of a product kernel: one per SM
constexpr int kShift = 14;       // fp16: log2 of the scale of P
constexpr int kSplitRows = 512;  // rows up to which P is the sum of two numbers (see "Numbers")

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
  float *bias2;    // [V to 128] bias * log2(e) (backward: + log2 of P's scale), -inf behind the last
  // forward
  float *lt;       // [rows_pad] the target's logit
  float2 *part;    // [tiles + grid][128] (base, sum) of a range's piece of a tile
  // backward
  uint8_t *xc;     // [rows_pad][K] the kept rows of F; behind the last, copies of one
  float *nlse;     // [rows_pad] -lse (-inf behind the last)
  float *gc;       // [rows_pad] g
  float *gs;       // [rows_pad] g / gmax * 2^shift
  float *dpart;    // [2 * grid][128][KP]
  float *bpart;    // [2 * grid][128]
  size_t bytes;
};

// Layout of the caller's workspace for `rows` rows; base may be null (sizes).
inline Workspace carve(uint8_t *base, long long rows, int K, int V, bool backward) {
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
  w.bias2 = reinterpret_cast<float *>(take(((size_t)V + 127) / 128 * 128 * 4));
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

// Kept rows and largest weight of every block of 256 rows (calls of more than
// kDirect blocks; below that the placing kernel counts for itself, which saves
// a launch).
__global__ void __launch_bounds__(kRowBlock)
ce_count_kernel(const void *targets, bool wide, int rows, int V, const float *g, int *cnt,
                float *gblk) {
  __shared__ float sm[kRowBlock / 32];
  release_next();
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
  float shift;       // scale of P: 2^14 for fp16, 1 for bf16
  float shift2;      // its log2
  bool direct;       // no cnt, gblk: count here
  const int *cnt;
  const float *gblk;
  Header *hdr;
  int *rowidx, *tgt;
  const float *bias;
  float *bias2;
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
// The bias goes to the log2 domain, padded to whole chunks.
// blockIdx.x: 256 rows; y: a share of the copying (share 0 writes the rest).
template <bool BWD>
__global__ void __launch_bounds__(kRowBlock) ce_place_kernel(const PlaceParams p) {
  __shared__ int swarp[kRowBlock / 32];
  __shared__ int s_off, s_total;
  __shared__ float s_gmax;
  __shared__ int s_seen, s_src;     // last kept row (direct) or block with one before this block; a kept row
  __shared__ int s_dst[kRowBlock];  // place of each row of the block, -1: padding
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  release_next();
  if (!p.direct) after_previous();
  // kept rows before this block, and the largest weight of all
  int before = 0, seen = -1;
  float gm = 0.f;
  if (p.direct) {
    const int mine = blockIdx.x * kRowBlock, upto = BWD ? p.rows : mine;
#pragma unroll 4
    for (int k = tid; k < upto; k += kRowBlock) {
      if (target_of(p.targets, p.wide, k, p.V) < 0) continue;
      if (k < mine) {
        ++before;
        seen = k;
      }
      if (BWD) gm = fmaxf(gm, fabsf(p.g[k]));
    }
  } else {
    for (int b = tid; b < (int)gridDim.x; b += kRowBlock) {
      if (b < (int)blockIdx.x && p.cnt[b]) {
        before += p.cnt[b];
        seen = b;
      }
      if (BWD) gm = fmaxf(gm, p.gblk[b]);
    }
  }
  if (tid == 0) {
    s_off = 0;
    s_seen = s_src = -1;
  }
  __syncthreads();
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    before += __shfl_xor_sync(~0u, before, o);
    gm = fmaxf(gm, __shfl_xor_sync(~0u, gm, o));
    if (BWD) seen = max(seen, __shfl_xor_sync(~0u, seen, o));
  }
  __shared__ float sg[kRowBlock / 32];
  if (lane == 0) {
    atomicAdd(&s_off, before);  // integers: the order does not matter
    if (BWD) atomicMax(&s_seen, seen);
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
  const bool share0 = blockIdx.y == 0;
  for (int v = (blockIdx.y * gridDim.x + blockIdx.x) * kRowBlock + tid; v < (p.V + 127) / 128 * 128;
       v += gridDim.x * gridDim.y * kRowBlock)
    p.bias2[v] = v < p.V ? (p.bias ? p.bias[v] * kLog2e : 0.f) + (BWD ? p.shift2 : 0.f) : -INFINITY;
  if (share0 && i < p.rows) {
    if (t >= 0) {
      p.rowidx[dst] = (int)i;
      p.tgt[dst] = t;
      if (BWD) {
        const float g = p.g[i];
        p.nlse[dst] = -p.lse[i];
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
  if (last && share0 && tid == 0) {
    p.hdr->n = n;
    p.hdr->gmax = s_gmax;
  }
  // the unused rows up to the end of the last tile
  const int end = max(kTile, (n + kTile - 1) / kTile * kTile);
  if (last && share0) {
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
    if (last) {  // some kept row: the last one
      if (t >= 0 && dst == n - 1) s_src = (int)i;
      if (s_total == 0 && s_seen >= 0) {
        const int r = p.direct ? s_seen : s_seen * kRowBlock + tid;
        if (target_of(p.targets, p.wide, r, p.V) >= 0) atomicMax(&s_src, r);
      }
    }
    __syncthreads();
    const int q = p.K / 8;  // 16-byte pieces of a row
    const int here = (int)min((long long)kRowBlock, (long long)p.rows - row0);
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const int from = blockIdx.y * kRowBlock + tid, step = gridDim.y * kRowBlock;
    // Behind the last row, copies of a kept one: their P is exp(-inf) = 0, which
    // rows of zeros would not be sure of (0 times an infinite weight is a NaN).
    // Without a kept row, zeros, whose products are not used.
    const int pad = last ? end - n : 0;
    for (int e = from; e < (here + pad) * q; e += step) {
      const int r = e / q, c = e - r * q;
      const int d = r < here ? s_dst[r] : n + r - here;
      const long long src = r < here ? row0 + r : s_src;
      if (d >= 0)
        reinterpret_cast<uint4 *>(p.xc)[(size_t)d * q + c] =
            src >= 0 ? __ldg(reinterpret_cast<const uint4 *>(p.feat) + (size_t)src * q + c) : zero;
      else if (p.dfeat)
        reinterpret_cast<uint4 *>(p.dfeat)[(size_t)src * q + c] = zero;
    }
  }
}

// ------------------------------------------------------------ step line -----
// The line of `total` steps in G ranges of equal length (to one step). G is
// the grid, or the steps where they are fewer, so that no range is empty.
struct Cuts {
  long long total, q, r;
  int G;
  __device__ Cuts(long long steps, int grid) {
    total = steps;
    G = (int)min((long long)grid, steps);
    q = G ? total / G : 0;
    r = G ? total - q * G : 0;
  }
  // first step of range c
  __device__ long long at(int c) const { return c >= G ? total : q * c + r * c / G; }
  // the range that holds step `it`: at(c) = floor(total c / G) <= it
  __device__ int owner(long long it) const { return (int)(((it + 1) * G - 1) / total); }
};

// ------------------------------------------------------------ small parts ---
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

template <bool BF16>
__device__ __forceinline__ float2 unpack16(uint32_t v) {
  if (BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&v));
  return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}

// y = S * log2(e) + terms of 32 columns, in pairs
__device__ __forceinline__ void logits32(uint64_t (&y)[16], const uint32_t (&v)[32],
                                         const float *terms) {
  const uint64_t l2e2 = pk(kLog2e, kLog2e);
  const ulonglong2 *cq = reinterpret_cast<const ulonglong2 *>(terms);
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const ulonglong2 c = cq[q];
    y[2 * q] = fma2(pk(__uint_as_float(v[4 * q]), __uint_as_float(v[4 * q + 1])), l2e2, c.x);
    y[2 * q + 1] =
        fma2(pk(__uint_as_float(v[4 * q + 2]), __uint_as_float(v[4 * q + 3])), l2e2, c.y);
  }
}
// takes column `at` out of 32 (leaves -inf there)
__device__ __forceinline__ void take_out(uint32_t (&v)[32], int at, float &taken) {
#pragma unroll
  for (int q = 0; q < 32; ++q)
    if (at == q) {
      taken = __uint_as_float(v[q]);
      v[q] = 0xff800000u;
    }
}
// x within [-126, 128]; NaN for NaN
__device__ __forceinline__ float ex2_range(float x) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;\n min.NaN.f32 %0, %0, %3;" : "=&f"(y) : "f"(x), "f"(-126.f), "f"(128.f));
  return y;
}
// exp2 of a pair without the special-function unit: y = n + f, |f| <= 1/2, by
// adding and taking off 1.5 * 2^23; exp2(f) by its Taylor polynomial in f ln 2
// up to f^6 (the next term is 1.2e-7 at |f| = 1/2; 2.2e-7 of the result at most
// with the roundings, ex2.approx has 2.4e-7); 2^n from the bits of its exponent. y
// below -126 counts as -126 (2^-126 instead of less). From 127.5 on n is 128, whose
// bits are those of an infinity, and y above 128 counts as 128: what is about to
// pass fp32 is an infinity here, so that the sums show it. A NaN stays one: the
// bounds keep it, and 2^n is a factor, not a sum with the bits of exp2(f).
__device__ __forceinline__ uint64_t ex2_poly(uint64_t y) {
  float a, b;
  upk(y, a, b);
  y = pk(ex2_range(a), ex2_range(b));
  const uint64_t t = add2(y, pk(12582912.f, 12582912.f));
  const uint64_t n = add2(t, pk(-12582912.f, -12582912.f));
  const uint64_t f = fma2(n, pk(-1.f, -1.f), y);
  uint64_t r = pk(1.5403530e-4f, 1.5403530e-4f);
  r = fma2(r, f, pk(1.3333558e-3f, 1.3333558e-3f));
  r = fma2(r, f, pk(9.6181291e-3f, 9.6181291e-3f));
  r = fma2(r, f, pk(5.5504109e-2f, 5.5504109e-2f));
  r = fma2(r, f, pk(2.4022651e-1f, 2.4022651e-1f));
  r = fma2(r, f, pk(6.9314718e-1f, 6.9314718e-1f));
  r = fma2(r, f, pk(1.f, 1.f));
  float t0, t1;
  upk(t, t0, t1);
  return mul2(r, pk(__uint_as_float((__float_as_uint(t0) << 23) + 0x3f800000u),
                    __uint_as_float((__float_as_uint(t1) << 23) + 0x3f800000u)));
}
// adds exp2(y) (exp2(y - base), nb = -base twice) of 32 columns to four sums
template <bool BASE>
__device__ __forceinline__ void add_exp(uint64_t (&s)[4], const uint64_t (&y)[16], uint64_t nb) {
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    const uint64_t z = BASE ? add2(y[q], nb) : y[q];
    if (q < kPolyPairs) {
      s[q & 3] = add2(s[q & 3], ex2_poly(z));
    } else {
      float a, b;
      upk(z, a, b);
      s[q & 3] = add2(s[q & 3], pk(ex2(a), ex2(b)));
    }
  }
}
__device__ __forceinline__ float sum4(const uint64_t (&s)[4]) {
  float a, b;
  upk(add2(add2(s[0], s[1]), add2(s[2], s[3])), a, b);
  return a + b;
}

// One warp's share of a stationary tile into tensor memory: lane = row, the
// warp's quarter `w4` of the features (8 * KA columns of two features).
// src: this lane's row, or null for a zero row. Not read-only loads: the rows may
// be those that the kernel before, which may still run when this one begins, writes.
template <int KA>
__device__ __forceinline__ void load_tile_tmem(uint32_t tx, const uint8_t *src, int K, int w4) {
  uint4 v[KA][2];  // all loads first: they do not pass the stores
#pragma unroll
  for (int a = 0; a < KA; ++a) {
    const int col = (w4 * KA + a) * 8;  // 16 features
    v[a][0] = v[a][1] = make_uint4(0, 0, 0, 0);
    if (src) {
      if (2 * col < K) v[a][0] = *reinterpret_cast<const uint4 *>(src + 4 * col);
      if (2 * col + 8 < K) v[a][1] = *reinterpret_cast<const uint4 *>(src + 4 * col + 16);
    }
  }
#pragma unroll
  for (int a = 0; a < KA; ++a) {
    const uint4 &v0 = v[a][0], &v1 = v[a][1];
    const uint32_t r[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
    tmem_st8(tx + (w4 * KA + a) * 8, r);
  }
}

// Waits (bounded) until every load that was issued into a ring has landed, `at`
// being the slot after the last one: a CTA that gives up leaves no copy in
// flight into its shared memory.
template <int N>
__device__ __forceinline__ void drain_loads(uint64_t *full, const Ring<N> &at) {
  for (int s = 0; s < N; ++s) {
    const bool wrapped = s >= at.i;  // last filled one round ago, if at all
    if (wrapped && at.first) continue;
    const uint32_t parity = wrapped ? at.phase ^ 1 : at.phase;
    const long long t0 = clock64();
    while (!mbar_try_wait(&full[s], parity))
      if (clock64() - t0 > (1ll << 30)) break;
  }
}

// ------------------------------------------------------------- forward ------
// 40960 x 128 x 18385 fp16: 292 us, 660 TFLOP/s. One exponential per logit sets the
// floor (167 us at the special-function unit's rate; it is 53 % busy); what else
// keeps the warps is shared memory, whose port carries the streamed rows in, the
// MMA's reads of them and the bias terms that each warp reads (231 us without the
// exponentials, 188 without the terms as well, 159 for the product alone). Two
// groups of eight warps take every other chunk and three S buffers keep the MMA
// ahead of them; 64-row chunks, 24 warps and other splits measured the same or
// slower.
template <int KA>
struct FwdCfg {
  static constexpr int KP = 64 * KA;
  static constexpr int CN = 128;                      // vocabulary rows of a chunk (MMA N)
  static constexpr int STAGE = KP * CN * 2;
  static constexpr int STAGES = KA == 1 ? 8 : KA == 2 ? 6 : KA == 3 ? 4 : 3;
  static constexpr int NBUF = 3;                      // S buffers
  static constexpr int TX = 0, TS = 128;              // TMEM columns: features, S buffers
  static constexpr int OFF_COL = STAGES * STAGE;                    // [kColSlots][CN] floats
  static constexpr int OFF_COMB = OFF_COL + kColSlots * CN * 4;     // [2][4][2][128] floats
  static constexpr int OFF_BAR = OFF_COMB + 2 * 4 * 2 * kTile * 4;
  static constexpr int NBAR = 2 * STAGES + 2 * NBUF + 2 * kColSlots + 1;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int SMEM = OFF_MISC + 16 + 1024;
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct FwdParams {
  const uint8_t *feat;
  const float *bias, *bias2;
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
  uint64_t *c_full = s_empty + C::NBUF;
  uint64_t *c_empty = c_full + kColSlots;
  uint64_t *x_ready = c_empty + kColSlots;
  uint32_t *s_tmem = reinterpret_cast<uint32_t *>(smem + C::OFF_MISC);
  volatile int *s_abort = reinterpret_cast<volatile int *>(smem + C::OFF_MISC + 4);
  float *comb = reinterpret_cast<float *>(smem + C::OFF_COMB);
  const float *scol = reinterpret_cast<const float *>(smem + C::OFF_COL);

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
    for (int b = 0; b < kColSlots; ++b) {
      mbar_init(&c_full[b], 1);
      mbar_init(&c_empty[b], kEpiWarps / 2);
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
  after_previous();
  const int n = p.hdr->n;
  const int NC = p.chunks;
  const long long total = (long long)((n + kTile - 1) / kTile) * NC;
  const Cuts cuts(total, gridDim.x);
  const long long it0 = cuts.at(blockIdx.x), it1 = cuts.at(blockIdx.x + 1);

  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&wmap);
      Ring<C::STAGES> bs;
      Ring<kColSlots> cr;
      int c = (int)(it0 % NC);
      for (int left = (int)(it1 - it0); left > 0; --left) {
        if (!bs.first && !mbar_wait_bounded(&b_empty[bs.i], bs.phase ^ 1, s_abort, p.err, 61)) break;
        mbar_arrive_expect_tx(&b_full[bs.i], C::STAGE);
        uint8_t *dst = smem + bs.i * C::STAGE;
#pragma unroll
        for (int k = 0; k < KA; ++k)
          tma_load_2d(dst + k * C::CN * 128, &wmap, &b_full[bs.i], 64 * k, c * C::CN);
        bs.next();
        if (!cr.first && !mbar_wait_bounded(&c_empty[cr.i], cr.phase ^ 1, s_abort, p.err, 66)) break;
        mbar_arrive_expect_tx(&c_full[cr.i], C::CN * 4);
        bulk_load(smem + C::OFF_COL + cr.i * C::CN * 4, p.bias2 + (size_t)c * C::CN, C::CN * 4,
                  &c_full[cr.i]);
        cr.next();
        if (++c == NC) c = 0;
      }
      if (*s_abort) {
        drain_loads(b_full, bs);
        drain_loads(c_full, cr);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = BF16 ? idesc_bf16(kTile, C::CN) : idesc_f16(kTile, C::CN);
      Ring<C::STAGES> bs;
      Ring<C::NBUF> sr;
      const uint64_t bdesc = sw128_kmajor_desc(smem_u32(smem));
      uint32_t seg = 0;
      int left_tile = NC - (int)(it0 % NC);  // chunks left of the tile
      bool fresh = true;
      for (int left = (int)(it1 - it0); left > 0; --left) {
        if (fresh) {
          if (!mbar_wait_bounded(x_ready, seg & 1, s_abort, p.err, 62)) break;
          ++seg;
        }
        if (!mbar_wait_bounded(&b_full[bs.i], bs.phase, s_abort, p.err, 63)) break;
        if (!sr.first && !mbar_wait_bounded(&s_empty[sr.i], sr.phase ^ 1, s_abort, p.err, 64)) break;
        tc_fence_after();
        const uint64_t bd = bdesc + (uint64_t)(bs.i * (C::STAGE >> 4));
        const uint32_t d = tmem + C::TS + sr.i * C::CN;
#pragma unroll
        for (int k = 0; k < 4 * KA; ++k)
          mma_f16_ts(d, tmem + C::TX + 8 * k, bd + (((k >> 2) * (C::CN * 128) + 32 * (k & 3)) >> 4),
                     idesc, k > 0 ? 1u : 0u);
        mma_commit(&b_empty[bs.i]);
        mma_commit(&s_full[sr.i]);
        bs.next();
        sr.next();
        fresh = --left_tile == 0;
        if (fresh) left_tile = NC;
      }
    }
  } else {
    const int ew = warp - kEpiWarp0;
    const int grp = ew >> 3;             // chunk parity this warp takes
    const int half = (ew >> 2) & 1;      // its 64 columns of the chunk
    const int quad = warp & 3;           // the TMEM lanes a warp may read
    const int r = quad * 32 + lane;
    const uint32_t tl = tmem + ((uint32_t)(quad * 32) << 16);
    Ring<C::NBUF> sr;
    Ring<kColSlots> cr;
    int seg = 0, odd = 0;  // odd: parity of the chunk
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
      // sum of exp2(y - base), y = l * log2(e), over the classes but the target
      // (whose logit is kept aside, so that a well recognised row has an exact
      // lse). The base is 0 if the first logits that the thread sees have their
      // maximum within 2^64 of it, else that maximum: the sum cannot vanish. It
      // grows with 64 logits whose sum passes 2^100, so it cannot overflow either,
      // and no maximum is taken of the others.
      float sum = 0.f, base = 0.f;
      bool seen = false;               // this lane has its base
      bool fresh = true, based = false;  // some lane of the warp has none; one other than 0
      for (int i = 0; i < cnt; ++i, odd ^= 1, sr.next(), cr.next()) {
        if (odd != grp) continue;
        const int b = sr.i, cs = cr.i;
        ok = ok && mbar_wait_bounded(&s_full[b], sr.phase, s_abort, p.err, 65) &&
             mbar_wait_bounded(&c_full[cs], cr.phase, s_abort, p.err, 67);
        if (!ok) break;
        tc_fence_after();
        const uint32_t ts = tl + C::TS + b * C::CN + half * 64;
        const float *terms = scol + cs * C::CN + half * 64;
        const int at = tg - ((c0 + i) * C::CN + half * 64);
        const bool hit = __any_sync(~0u, at >= 0 && at < 64);
        float add = 0.f, st = 0.f;  // st: S of the target
        bool slow = fresh;
        const uint64_t nb = pk(-base, -base);
        if (!slow && !hit) {
          uint64_t s4[4] = {0, 0, 0, 0}, y[16];
          uint32_t v[32], w[32];
          tmem_ld32(ts, v);
          tmem_ld_wait(v);
          tmem_ld32(ts + 32, w);
          logits32(y, v, terms);
          if (based)
            add_exp<true>(s4, y, nb);
          else
            add_exp<false>(s4, y, nb);
          tmem_ld_wait(w);
          logits32(y, w, terms + 32);
          if (based)
            add_exp<true>(s4, y, nb);
          else
            add_exp<false>(s4, y, nb);
          add = sum4(s4);
        } else if (!slow) {  // one chunk in nine (18385 classes): without the targets
          uint64_t s4[4] = {0, 0, 0, 0};
#pragma unroll 1
          for (int g = 0; g < 2; ++g) {
            uint32_t v[32];
            uint64_t y[16];
            tmem_ld32(ts + 32 * g, v);
            tmem_ld_wait(v);
            take_out(v, at - 32 * g, st);
            logits32(y, v, terms + 32 * g);
            add_exp<true>(s4, y, nb);
          }
          add = sum4(s4);
        }
        slow = slow || __any_sync(~0u, !(add < 0x1p100f));
        if (slow) {  // a first or a larger base
          float gm = -INFINITY;
#pragma unroll 1
          for (int g = 0; g < 2; ++g) {
            uint32_t v[32];
            uint64_t y[16];
            tmem_ld32(ts + 32 * g, v);
            tmem_ld_wait(v);
            take_out(v, at - 32 * g, st);
            logits32(y, v, terms + 32 * g);
#pragma unroll
            for (int q = 0; q < 16; ++q) {
              float f0, f1;
              upk(y[q], f0, f1);
              gm = fmaxf(fmaxf(gm, f0), f1);
            }
          }
          if (!seen && gm != -INFINITY) {
            seen = true;
            base = fabsf(gm) > 64.f && fabsf(gm) < INFINITY ? gm : 0.f;
          } else if (gm > base + 64.f && gm < INFINITY) {
            sum *= ex2(base - gm);
            base = gm;
          }
          fresh = __any_sync(~0u, !seen);
          based = __any_sync(~0u, base != 0.f);
          const uint64_t nb2 = pk(-base, -base);
          uint64_t s4[4] = {0, 0, 0, 0};
#pragma unroll 1
          for (int g = 0; g < 2; ++g) {
            uint32_t v[32];
            uint64_t y[16];
            tmem_ld32(ts + 32 * g, v);
            tmem_ld_wait(v);
            take_out(v, at - 32 * g, st);
            logits32(y, v, terms + 32 * g);
            add_exp<true>(s4, y, nb2);
          }
          add = sum4(s4);
        }
        if (at >= 0 && at < 64) p.lt[row] = st + (p.bias ? p.bias[tg] : 0.f);
        sum += add;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&s_empty[b]);
          mbar_arrive(&c_empty[cs]);
        }
      }
      const float top = seen ? base : -INFINITY;
      // the four column shares of a row into one (base, sum relative to it)
      float *cp = comb + (seg & 1) * 8 * kTile;
      cp[(ew >> 2) * 2 * kTile + r] = top;
      cp[(ew >> 2) * 2 * kTile + kTile + r] = sum;
      ok = named_bar_and(1, kEpiThreads, ok);
      if (!ok) break;
      tc_fence_after();  // the products that both groups waited for are done with the tile
      if ((ew >> 2) == 0) {
        float M = top;
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
  release_next();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the pieces of every kept row, a warp per row: lane c takes pieces c, c +
// 32, ... (a fixed order). With r = log sum exp of the other classes and l the
// target's logit, lse = max(r, l) + log(1 + exp(-|r - l|)): exactly l where the
// others do not count, so that the loss is exactly 0 and the backward pass finds
// a probability of exactly 1.
__global__ void __launch_bounds__(256)
ce_loss_kernel(const FwdParams p, int grid, float *loss, float *lse) {
  __shared__ int s_first, s_last;
  after_previous();
  const int n = p.hdr->n;
  const int lane = threadIdx.x & 31, row = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int tile = blockIdx.x * 8 / kTile;
  if ((int)blockIdx.x * 8 >= n) return;
  if (threadIdx.x == 0) {
    const Cuts cuts((long long)((n + kTile - 1) / kTile) * p.chunks, grid);
    s_first = cuts.owner((long long)tile * p.chunks);
    s_last = cuts.owner((long long)(tile + 1) * p.chunks - 1);
  }
  __syncthreads();
  if (row >= n) return;
  const int pieces = s_last - s_first + 1;
  const float2 *src = p.part + (size_t)(tile + s_first) * kTile + row % kTile;
  float M = -INFINITY, S = 0.f;  // a NaN shows in the sums only
#pragma unroll 4
  for (int c = lane; c < pieces; c += 32) {
    const float2 v = src[(size_t)c * kTile];
    const float m = fmaxf(M, v.x);
    S = (M == -INFINITY ? S : S * exp2f(M - m)) + (v.x == -INFINITY ? v.y : v.y * exp2f(v.x - m));
    M = m;
  }
  float top = M;
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  if (M != -INFINITY) S *= exp2f(M - top);
#pragma unroll
  for (int o = 16; o; o >>= 1) S += __shfl_xor_sync(~0u, S, o);
  if (lane > 0) return;
  const int i = p.rowidx[row];
  const float l = p.lt[row], rest = fmaf(top, kLn2, logf(S));  // -inf without other classes
  const float a = rest - l, z = (a > 0.f ? rest : l) + log1pf(expf(-fabsf(a)));
  loss[i] = z - l;
  lse[i] = z;
}

// ------------------------------------------------------------- backward -----
// 10240 x 128 x 18385 fp16, half of the rows padding: 115 us, 840 TFLOP/s; 16384 x
// 256 x 65537 bf16: 1390 us, 1.43 PFLOP/s of the four products, near what the GPU
// sustains under its power cap. Every chunk is a chain S -> P -> D through all
// sixteen warps; two S buffers let the MMA work on one while the warps have the
// other (tensor pipe 52 % busy at K 128, 62 % at K 256). Chunks of 128 rows where
// tensor memory has room (K up to 128), of 64 else; smaller chunks with more
// buffers and two groups of warps measured slower (130 and 154 us).
template <int KA>
struct BwdCfg {
  static constexpr int KP = 64 * KA;
  static constexpr int CN = KA <= 2 ? 128 : 64;       // streamed rows of a chunk
  static constexpr int QC = CN / 4;                   // columns of S per epilogue warp
  static constexpr int STAGE = KP * CN * 2;
  static constexpr int STAGES = KA == 1 ? 8 : KA == 2 ? 5 : KA == 3 ? 7 : 5;
  static constexpr int TD = 0, TX = KP, TS = KP + KP / 2;  // TMEM columns: D, tile, two S
  static constexpr int COL = 3 * CN * 4;              // addend, scale and target of each row
  static constexpr int OFF_COL = STAGES * STAGE;
  static constexpr int OFF_BSUM = OFF_COL + kColSlots * COL;        // [2][4][128] floats
  static constexpr int OFF_BAR = OFF_BSUM + 2 * 4 * kTile * 4;
  static constexpr int NBAR = 2 * STAGES + 2 * kColSlots + 6;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int SMEM = OFF_MISC + 16 + 1024;
  static_assert(TS + 2 * CN <= kTmemCols, "tensor memory");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct BwdParams {
  const uint8_t *w, *xc;
  const float *bias, *bias2;
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
    chunks_r = max(1, (n + cn - 1) / cn);  // no rows: one chunk, so that zeros are written
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

// SPLIT: P as the sum of two 16-bit numbers
template <int KA, bool BF16, bool SPLIT>
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
  uint64_t *c_full = d_full + 1;
  uint64_t *c_empty = c_full + kColSlots;
  uint32_t *s_tmem = reinterpret_cast<uint32_t *>(smem + C::OFF_MISC);
  volatile int *s_abort = reinterpret_cast<volatile int *>(smem + C::OFF_MISC + 4);
  float *bsum = reinterpret_cast<float *>(smem + C::OFF_BSUM);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&b_full[s], 1);
      mbar_init(&b_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&s_full[b], 1);
      mbar_init(&p_full[b], kEpiWarps);
    }
    for (int b = 0; b < kColSlots; ++b) {
      mbar_init(&c_full[b], 1);
      mbar_init(&c_empty[b], kEpiWarps);
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
  after_previous();
  const BwdLine line(p.hdr, C::CN, p.chunks_v, p.want_x, p.tiles_w);
  const Cuts cuts(line.total, gridDim.x);
  const long long it0 = cuts.at(blockIdx.x), it1 = cuts.at(blockIdx.x + 1);

  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&wmap);
      tma_prefetch_desc(&xmap);
      Ring<C::STAGES> bs;
      Ring<kColSlots> cr;
      bool ok = true;
      for (long long it = it0; ok && it < it1;) {
        bool dw;
        int tile, c0, nc;
        line.at(it, dw, tile, c0, nc);
        const int cnt = (int)min((long long)(nc - c0), it1 - it);
        it += cnt;
        const CUtensorMap *map = dw ? &xmap : &wmap;
        for (int c = c0; c < c0 + cnt; ++c) {
          ok = bs.first || mbar_wait_bounded(&b_empty[bs.i], bs.phase ^ 1, s_abort, p.err, 71);
          if (!ok) break;
          mbar_arrive_expect_tx(&b_full[bs.i], C::STAGE);
          uint8_t *dst = smem + bs.i * C::STAGE;
#pragma unroll
          for (int k = 0; k < KA; ++k)
            tma_load_2d(dst + k * C::CN * 128, map, &b_full[bs.i], 64 * k, c * C::CN);
          bs.next();
          ok = cr.first || mbar_wait_bounded(&c_empty[cr.i], cr.phase ^ 1, s_abort, p.err, 77);
          if (!ok) break;
          uint8_t *col = smem + C::OFF_COL + cr.i * C::COL;
          const size_t at = (size_t)c * C::CN;
          mbar_arrive_expect_tx(&c_full[cr.i], dw ? C::COL : C::CN * 4);
          if (dw) {
            bulk_load(col, p.nlse + at, C::CN * 4, &c_full[cr.i]);
            bulk_load(col + C::CN * 4, p.gs + at, C::CN * 4, &c_full[cr.i]);
            bulk_load(col + 2 * C::CN * 4, p.tgt + at, C::CN * 4, &c_full[cr.i]);
          } else {
            bulk_load(col, p.bias2 + at, C::CN * 4, &c_full[cr.i]);
          }
          cr.next();
        }
      }
      if (*s_abort) {
        drain_loads(b_full, bs);
        drain_loads(c_full, cr);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t id1 = BF16 ? idesc_bf16(kTile, C::CN) : idesc_f16(kTile, C::CN);
      // neither product takes more than 8 features of padding: steps of 16 in the
      // first, columns of D in the second (8191 x 200 x 18385 bf16: 235 us, 255 with
      // 256 features; the forward pass, bound elsewhere, gains nothing by it)
      const int kn = (p.K + 15) / 16 * 16;
      const uint32_t id2 = (BF16 ? idesc_bf16(kTile, kn) : idesc_f16(kTile, kn)) | kIdescBMnMajor;
      const uint64_t kdesc = sw128_kmajor_desc(smem_u32(smem));
      const uint64_t mdesc = sw128_mnmajor_desc(smem_u32(smem), C::CN * 128);
      Ring<C::STAGES> b1, b2;  // chunks of the first and of the second product
      Ring<2> s1, s2;
      uint32_t seg = 0;
      bool ok = true;
      // S = tile x chunk^T of the next chunk into its buffer
      auto first = [&]() {
        if (!mbar_wait_bounded(&b_full[b1.i], b1.phase, s_abort, p.err, 72)) return false;
        tc_fence_after();
        const uint64_t bd = kdesc + (uint64_t)(b1.i * (C::STAGE >> 4));
        const uint32_t d = tmem + C::TS + s1.i * C::CN;
#pragma unroll
        for (int k = 0; k < 4 * KA; ++k)
          if (k <= 4 * KA - 4 || 16 * k < p.K)
            mma_f16_ts(d, tmem + C::TX + 8 * k,
                       bd + (((k >> 2) * (C::CN * 128) + 32 * (k & 3)) >> 4), id1, k > 0 ? 1u : 0u);
        mma_commit(&s_full[s1.i]);
        b1.next();
        s1.next();
        return true;
      };
      for (long long it = it0; ok && it < it1; ++seg) {
        bool dw;
        int tile, c0, nc;
        line.at(it, dw, tile, c0, nc);
        const int cnt = (int)min((long long)(nc - c0), it1 - it);
        it += cnt;
        ok = mbar_wait_bounded(x_ready, seg & 1, s_abort, p.err, 73);
        if (!ok) break;
        tc_fence_after();
        ok = first() && (cnt < 2 || first());
        for (int i = 0; ok && i < cnt; ++i) {
          ok = mbar_wait_bounded(&p_full[s2.i], s2.phase, s_abort, p.err, 74);
          if (!ok) break;
          tc_fence_after();
          const uint64_t bd = mdesc + (uint64_t)(b2.i * (C::STAGE >> 4));
          const uint32_t pa = tmem + C::TS + s2.i * C::CN;
#pragma unroll
          for (int k = 0; k < C::CN / 16; ++k) {
            // P of each quarter of the chunk lies at the head of that quarter's S columns
            const uint32_t pc = (16 * k / C::QC) * C::QC + (16 * k % C::QC) / 2;
            mma_f16_ts(tmem + C::TD, pa + pc, bd + ((2048 * k) >> 4), id2, i > 0 || k > 0 ? 1u : 0u);
          }
          if (SPLIT) {  // and the second part of P behind the first
#pragma unroll
            for (int k = 0; k < C::CN / 16; ++k) {
              const uint32_t pc = (16 * k / C::QC) * C::QC + (16 * k % C::QC) / 2 + C::QC / 2;
              mma_f16_ts(tmem + C::TD, pa + pc, bd + ((2048 * k) >> 4), id2, 1u);
            }
          }
          mma_commit(&b_empty[b2.i]);
          b2.next();
          s2.next();
          // the next S into this buffer: issued after the product that reads P
          // there, and the tensor pipe keeps that order
          if (i + 2 < cnt) ok = first();
          if (i + 1 == cnt) mma_commit(d_full);
        }
      }
    }
  } else {
    const int ew = warp - kEpiWarp0;
    const int w4 = ew >> 2;              // its quarter of the columns
    const int quad = warp & 3;
    const int r = quad * 32 + lane;
    const uint32_t tl = tmem + ((uint32_t)(quad * 32) << 16);
    const uint64_t l2e2 = pk(kLog2e, kLog2e);
    constexpr int QC = C::QC;
    Ring<2> sr;
    Ring<kColSlots> cr;
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
      // y = (S - lse) log2(e) + bias log2(e), P = exp2(y) (* column scale). The
      // target's y is ((S + bias) - lse) log2(e), rounded as the forward pass
      // rounds its logit: exactly 0 where the target alone counts.
      const int tg = !dw && real ? p.tgt[row] : -1;
      const float bt = !p.bias ? 0.f : dw ? (real ? p.bias[row] : 0.f) : tg >= 0 ? p.bias[tg] : 0.f;
      float rterm = -INFINITY;  // dF: -lse, dW: bias * log2(e)
      if (real) rterm = dw ? bt * kLog2e : p.nlse[row];
      const uint64_t rt2 = pk(rterm, rterm), bt2 = pk(bt, bt);
      const float one = exp2f(p.shift);
      uint64_t acc2 = 0;
      for (int i = 0; i < cnt; ++i, sr.next(), cr.next()) {
        const int b = sr.i, cs = cr.i;
        ok = ok && mbar_wait_bounded(&c_full[cs], cr.phase, s_abort, p.err, 78) &&
             mbar_wait_bounded(&s_full[b], sr.phase, s_abort, p.err, 75);
        if (!ok) break;
        tc_fence_after();
        const uint32_t ts = tl + C::TS + b * C::CN + w4 * QC;
        const float *col = reinterpret_cast<const float *>(smem + C::OFF_COL + cs * C::COL) + w4 * QC;
        uint32_t v[QC];
        if constexpr (QC == 32)
          tmem_ld32(ts, v);
        else
          tmem_ld16(ts, v);
        tmem_ld_wait(v);
        float f[QC];
        const ulonglong2 *cq = reinterpret_cast<const ulonglong2 *>(col);
        auto pair = [&](int q) {
          return pk(__uint_as_float(v[2 * q]), __uint_as_float(v[2 * q + 1]));
        };
        if (dw) {
          // column terms: -lse; targets among this warp's 32 classes?
          const int *ctg = reinterpret_cast<const int *>(col + 2 * C::CN);
          const int off = ctg[lane % QC] - (tile * kTile + quad * 32);
          const bool any = __any_sync(~0u, off >= 0 && off < 32);
          if (any) {
#pragma unroll
            for (int q = 0; q < QC / 2; q += 2) {
              const ulonglong2 c = cq[q / 2];
              upk(mul2(add2(add2(pair(q), bt2), c.x), l2e2), f[2 * q], f[2 * q + 1]);
              upk(mul2(add2(add2(pair(q + 1), bt2), c.y), l2e2), f[2 * q + 2], f[2 * q + 3]);
            }
          } else {
#pragma unroll
            for (int q = 0; q < QC / 2; q += 2) {
              const ulonglong2 c = cq[q / 2];
              upk(fma2(add2(pair(q), c.x), l2e2, rt2), f[2 * q], f[2 * q + 1]);
              upk(fma2(add2(pair(q + 1), c.y), l2e2, rt2), f[2 * q + 2], f[2 * q + 3]);
            }
          }
#pragma unroll
          for (int q = 0; q < QC; ++q) f[q] = ex2(f[q]);
          if (any) {
#pragma unroll
            for (int q = 0; q < QC; ++q)
              if (ctg[q] == row) f[q] -= 1.f;
          }
          const ulonglong2 *sq = reinterpret_cast<const ulonglong2 *>(col + C::CN);
#pragma unroll
          for (int q = 0; q < QC / 4; ++q) {
            const ulonglong2 ss = sq[q];
            const uint64_t a = mul2(pk(f[4 * q], f[4 * q + 1]), ss.x);
            const uint64_t c = mul2(pk(f[4 * q + 2], f[4 * q + 3]), ss.y);
            acc2 = add2(acc2, add2(a, c));
            upk(a, f[4 * q], f[4 * q + 1]);
            upk(c, f[4 * q + 2], f[4 * q + 3]);
          }
        } else {
          // column terms: bias * log2(e) + log2 of P's scale
          const int at = tg - ((c0 + i) * C::CN + w4 * QC);
          const bool any = __any_sync(~0u, at >= 0 && at < QC);
          float pt = 0.f;
          if (any) {
#pragma unroll
            for (int q = 0; q < QC; ++q)
              if (at == q) pt = __uint_as_float(v[q]);
            pt = ex2(fmaf((pt + bt) + rterm, kLog2e, p.shift)) - one;
          }
#pragma unroll
          for (int q = 0; q < QC / 2; q += 2) {
            const ulonglong2 c = cq[q / 2];
            upk(fma2(add2(pair(q), rt2), l2e2, c.x), f[2 * q], f[2 * q + 1]);
            upk(fma2(add2(pair(q + 1), rt2), l2e2, c.y), f[2 * q + 2], f[2 * q + 3]);
          }
#pragma unroll
          for (int q = 0; q < QC; ++q) f[q] = ex2(f[q]);
          if (any) {
#pragma unroll
            for (int q = 0; q < QC; ++q)
              if (at == q) f[q] = pt;
          }
        }
        uint32_t h[QC / 2];
#pragma unroll
        for (int q = 0; q < QC / 2; ++q) h[q] = pack16<BF16>(f[2 * q], f[2 * q + 1]);
        if constexpr (QC == 32)
          tmem_st16(ts, h);
        else
          tmem_st8(ts, h);
        if (SPLIT) {
#pragma unroll
          for (int q = 0; q < QC / 2; ++q) {
            const float2 r = unpack16<BF16>(h[q]);
            h[q] = pack16<BF16>(f[2 * q] - r.x, f[2 * q + 1] - r.y);
          }
          if constexpr (QC == 32)
            tmem_st16(ts + QC / 2, h);
          else
            tmem_st8(ts + QC / 2, h);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&p_full[b]);
          mbar_arrive(&c_empty[cs]);
        }
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
        const float s =
            line.n ? (bs[r] + bs[kTile + r]) + (bs[2 * kTile + r] + bs[3 * kTile + r]) : 0.f;
        if (!whole)
          p.bpart[(size_t)slot * kTile + r] = s;
        else if (p.dbias)
          p.dbias[row] = s * p.unscale * p.hdr->gmax;
      }
#pragma unroll
      for (int a = 0; a < KA; ++a) {
        const int col = (w4 * KA + a) * 16;
        if (col >= p.K) break;  // no such columns of D
        uint32_t v[16];
        tmem_ld16(tl + C::TD + col, v);
        tmem_ld_wait(v);
        if (!real) continue;
        if (line.n == 0) {
#pragma unroll
          for (int q = 0; q < 16; ++q) v[q] = 0;
        }
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
  release_next();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Sums the pieces of the tiles that range borders cut, in a fixed order, and
// rounds them as the main kernel rounds a whole tile. blockIdx.x: border (CTA b >
// 0). The blocks of all borders inside a tile share its elements, and where that
// leaves a block fewer than its threads, groups of threads share the pieces: few
// rows cut the one tile of dF into many pieces (80 x 128 x 18385: 73, the
// backward pass takes 27 us; 62 where one border's blocks sum a tile, a thread
// per element).
template <bool BF16>
__global__ void __launch_bounds__(kJoinThreads)
ce_join_kernel(const BwdParams p, int cn, int KP, int grid) {
  __shared__ int s_tile, s_dw, s_first, s_last;
  __shared__ float4 s_sum[kJoinThreads];
  after_previous();
  const int tid = threadIdx.x;
  if (tid == 0) {
    s_tile = -1;
    const BwdLine line(p.hdr, cn, p.chunks_v, p.want_x, p.tiles_w);
    const Cuts cuts(line.total, grid);
    const int c = blockIdx.x + 1;
    if (c < cuts.G) {
      const long long at = cuts.at(c);
      bool dw;
      int tile, chunk, nc;
      line.at(at, dw, tile, chunk, nc);
      if (chunk > 0) {  // inside a tile
        const long long t0 = at - chunk;  // first step of the tile
        s_tile = tile;
        s_dw = dw;
        s_first = cuts.owner(t0) + 1;
        s_last = cuts.owner(t0 + nc - 1);
      }
    }
  }
  __syncthreads();
  const int tile = s_tile;
  if (tile < 0) return;
  const bool dw = s_dw;
  const int c = s_first, borders = s_last - c + 1;
  // pieces: the tail of CTA c - 1, then c .. last
  const int pieces = borders + 1;
  auto slot = [&](int j) { return 2 * (c + j - 1) + (j == 0 ? 1 : 0); };
  const int slices = borders * gridDim.y;
  const int slice = (blockIdx.x + 1 - c) * gridDim.y + blockIdx.y;
  const int lim = min(kTile, (dw ? p.V : p.hdr->n) - tile * kTile);
  const int q4 = KP / 4, total = lim * q4;  // elements: four columns of a row
  const float gmax = p.hdr->gmax;
  if (!dw || p.dw) {
    int groups = 1;
    while (groups < 32 && 2 * groups <= pieces &&
           slices * (kJoinThreads / (2 * groups)) >= total)
      groups *= 2;
    const int width = kJoinThreads / groups, group = tid / width, el = tid % width;
    for (int e0 = slice * width; e0 < total; e0 += slices * width) {
      const int e = e0 + el;
      const int r = e / q4, k = (e - r * q4) * 4;
      const bool mine = e < total && k < p.K;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      if (mine) {
        const float *src = p.dpart + (size_t)r * KP + k;
#pragma unroll 8
        for (int j = group; j < pieces; j += groups) {
          const float4 v = *reinterpret_cast<const float4 *>(src + (size_t)slot(j) * kTile * KP);
          s.x += v.x;
          s.y += v.y;
          s.z += v.z;
          s.w += v.w;
        }
      }
      if (groups > 1) {
        __syncthreads();
        s_sum[tid] = s;
        __syncthreads();
        if (group == 0)
          for (int g = 1; g < groups; ++g) {
            const float4 v = s_sum[g * width + el];
            s.x += v.x;
            s.y += v.y;
            s.z += v.z;
            s.w += v.w;
          }
      }
      if (!mine || group) continue;
      const int row = tile * kTile + r;
      const float sc = (dw ? gmax : p.gc[row]) * p.unscale;
      uint8_t *out = dw ? p.dw + (size_t)row * p.K * 2 : p.dfeat + (size_t)p.rowidx[row] * p.K * 2;
      *reinterpret_cast<uint2 *>(out + 2 * k) =
          make_uint2(pack16<BF16>(s.x * sc, s.y * sc), pack16<BF16>(s.z * sc, s.w * sc));
    }
  }
  if (dw && p.dbias)  // a warp per class
    for (int r = slice * (kJoinThreads / 32) + tid / 32; r < lim; r += slices * (kJoinThreads / 32)) {
      float s = 0.f;
      for (int j = tid % 32; j < pieces; j += 32) s += p.bpart[(size_t)slot(j) * kTile + r];
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
      if (tid % 32 == 0) p.dbias[tile * kTile + r] = s * p.unscale * gmax;
    }
}

// ----------------------------------------------------------------- host -----
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
  rc = allow_dynamic_smem(reinterpret_cast<const void *>(ce_fwd_kernel<KA, BF16>), C::SMEM,
                          "ce_fwd_kernel");
  if (rc) return rc;
  return launch_overlapped("ce_fwd_kernel", ce_fwd_kernel<KA, BF16>, grid, kThreads, C::SMEM, st, wm,
                           p);
}

template <int KA, bool BF16, bool SPLIT>
int launch_bwd(const BwdParams &p, int rows_pad, int grid, cudaStream_t st) {
  using C = BwdCfg<KA>;
  CUtensorMap wm, xm;
  const CUtensorMapDataType ty =
      BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  int rc = tma_map_rows(&wm, ty, 2, p.w, p.K, p.V, 2ll * p.K, C::CN);
  if (rc) return rc;
  rc = tma_map_rows(&xm, ty, 2, p.xc, p.K, rows_pad, 2ll * p.K, C::CN);
  if (rc) return rc;
  rc = allow_dynamic_smem(reinterpret_cast<const void *>(ce_bwd_kernel<KA, BF16, SPLIT>), C::SMEM,
                          "ce_bwd_kernel");
  if (rc) return rc;
  rc = launch_overlapped("ce_bwd_kernel", ce_bwd_kernel<KA, BF16, SPLIT>, grid, kThreads, C::SMEM, st, wm,
                         xm, p);
  if (rc || grid == 1) return rc;
  return launch_overlapped("ce_join_kernel", ce_join_kernel<BF16>, dim3(grid - 1, 4), kJoinThreads, 0, st, p,
                           C::CN, C::KP, grid);
}

template <int KA>
int launch_bwd_ka(const BwdParams &p, bool bf, bool split, int rows_pad, int grid,
                  cudaStream_t st) {
  if (bf)
    return split ? launch_bwd<KA, true, true>(p, rows_pad, grid, st)
                 : launch_bwd<KA, true, false>(p, rows_pad, grid, st);
  return split ? launch_bwd<KA, false, true>(p, rows_pad, grid, st)
               : launch_bwd<KA, false, false>(p, rows_pad, grid, st);
}

template <bool BWD>
int launch_place(const Workspace &ws, const void *targets, bool wide, int rows, int V, int K,
                 int dtype, const float *bias, const void *feat, const float *lse,
                 const float *g, void *dfeat, float *loss, float *lse_out, cudaStream_t st) {
  const int blocks = rows > kRowBlock ? (rows + kRowBlock - 1) / kRowBlock : 1;
  const bool direct = blocks <= kDirect;
  if (!direct) {
    ce_count_kernel<<<blocks, kRowBlock, 0, st>>>(targets, wide, rows, V, g, ws.cnt, ws.gblk);
    const int rc = check_launch("ce_count_kernel");
    if (rc) return rc;
  }
  PlaceParams p{};
  p.direct = direct;
  p.targets = targets;
  p.wide = wide;
  p.rows = rows;
  p.V = V;
  p.K = K;
  p.shift = dtype == TOCR_DTYPE_F16 ? (float)(1 << kShift) : 1.f;
  p.shift2 = dtype == TOCR_DTYPE_F16 ? (float)kShift : 0.f;
  p.bias = bias;
  p.bias2 = ws.bias2;
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
  // shares enough for one or two passes over the bias, 8 for the copies
  const int per = (V + blocks * kRowBlock - 1) / (blocks * kRowBlock);
  const dim3 shares(blocks, per < 8 ? 8 : per < 64 ? per : 64);
  if (!direct)
    return launch_overlapped("ce_place_kernel", ce_place_kernel<BWD>, shares, kRowBlock, 0, st, p);
  ce_place_kernel<BWD><<<shares, kRowBlock, 0, st>>>(p);
  return check_launch("ce_place_kernel");
}

int check_sizes(const char *fn, long long rows, int K, int V, int dtype) {
  TOCR_REQUIRE(rows >= 0 && rows <= kMaxRows && V > 0 && V <= kMaxClasses,
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
  if (rows < 0 || rows > kMaxRows || K < 8 || K > kMaxK || K % 8 || num_classes <= 0 ||
      num_classes > kMaxClasses)
    return 0;
  return carve(nullptr, rows, K, num_classes, backward != 0).bytes;
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
  TOCR_REQUIRE(aligned(d_targets, targets_i64 ? 8 : 4) && aligned(d_bias, 4) && aligned(d_loss, 4) &&
                   aligned(d_lse, 4) && aligned(d_err, 4),
               "tocr_rec_head_ce: a pointer is not aligned to its element");
  TOCR_REQUIRE(aligned(d_workspace, 256) &&
                   workspace_bytes >= carve(nullptr, rows, K, num_classes, false).bytes,
               "tocr_rec_head_ce: the workspace must be 256-byte aligned and hold %zu bytes",
               carve(nullptr, rows, K, num_classes, false).bytes);
  cudaStream_t st = as_stream(stream);
  const Workspace ws = carve(static_cast<uint8_t *>(d_workspace), rows, K, num_classes, false);
  rc = launch_place<false>(ws, d_targets, targets_i64 != 0, (int)rows, num_classes, K, dtype,
                           d_bias, nullptr, nullptr, nullptr, nullptr, d_loss, d_lse, st);
  if (rc) return rc;
  FwdParams p{};
  p.feat = static_cast<const uint8_t *>(d_feat);
  p.bias = d_bias;
  p.bias2 = ws.bias2;
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
  return launch_overlapped("ce_loss_kernel", ce_loss_kernel, tiles * (kTile / 8), 256, 0, st, p, grid,
                           d_loss, d_lse);
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
  TOCR_REQUIRE(aligned(d_targets, targets_i64 ? 8 : 4) && aligned(d_bias, 4) && aligned(d_lse, 4) &&
                   aligned(d_grad_loss, 4) && aligned(d_dbias, 4) && aligned(d_err, 4),
               "tocr_rec_head_ce_backward: a pointer is not aligned to its element");
  TOCR_REQUIRE(aligned(d_workspace, 256) &&
                   workspace_bytes >= carve(nullptr, rows, K, num_classes, true).bytes,
               "tocr_rec_head_ce_backward: the workspace must be 256-byte aligned and hold %zu bytes",
               carve(nullptr, rows, K, num_classes, true).bytes);
  cudaStream_t st = as_stream(stream);
  const Workspace ws = carve(static_cast<uint8_t *>(d_workspace), rows, K, num_classes, true);
  rc = launch_place<true>(ws, d_targets, targets_i64 != 0, (int)rows, num_classes, K, dtype, d_bias,
                          d_feat, d_lse, d_grad_loss, d_dfeat, nullptr, nullptr, st);
  if (rc) return rc;
  const int KA = (K + 63) / 64;
  const int cn = KA <= 2 ? 128 : 64;
  BwdParams p{};
  p.w = static_cast<const uint8_t *>(d_w);
  p.xc = ws.xc;
  p.bias = d_bias;
  p.bias2 = ws.bias2;
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
  // two steps at least: fewer pieces to join (175 x 64 x 5000: 80 CTAs and not 148)
  const int grid = grid_for(tiles_x * p.chunks_v + p.tiles_w * chunks_r, 2);
  const int rows_pad = (int)((rows + kTile - 1) / kTile * kTile + kTile);
  const bool bf = dtype == TOCR_DTYPE_BF16, split = rows <= kSplitRows;
  switch (KA) {
    case 1: return launch_bwd_ka<1>(p, bf, split, rows_pad, grid, st);
    case 2: return launch_bwd_ka<2>(p, bf, split, rows_pad, grid, st);
    case 3: return launch_bwd_ka<3>(p, bf, split, rows_pad, grid, st);
    default: return launch_bwd_ka<4>(p, bf, split, rows_pad, grid, st);
  }
}

}  // extern "C"
