// The INT8 linear layer's product for outputs whose rows lie off the 32-byte
// sectors and that are larger than L2 holds: the logits of a batch of lines, the
// dictionary having 18385 classes.
//
// Stores that fill a sector in part take the memory more than twice as long: the
// kernel of linear_i8.cu, which stores 64 bytes of a row straight from
// registers, needs 366 us for 40960 x 128 x 18384 in fp16 (a plain fill of as
// many bytes takes 385 us) but 833 us for 18385 channels, 861 us in a row of
// calls. Here the columns that a warp works on overlap by 16: whatever a row's
// offset, the warp has all channels of the whole sectors that it writes, and only
// the ends of y's rows are written in part. 587 us, in a row of calls too. Bound
// by the load/store pipe, which the staging through shared memory and the stores
// share (418 us with the stores alone, about 320 without them); sector-aligned
// and small outputs stay with the other kernel (580 us here for 18384).
//
// The tokens are the rows of the MMA (M 128) and the channels its columns, so
// that a row's channels are all in one warp's lanes. The warps read the
// accumulator in the layout of 8 x 8 matrices, in which a thread has four tokens
// of every channel that it has (a row of tensor memory per thread would read
// every scale and bias from shared memory for one product each), put the rows of
// their part into shared memory, and store them from there in 16-byte pieces
// shifted to the row's offset.
#include "linear_i8.cuh"

namespace tocr {
namespace {

using namespace ptx;
using namespace linear;

constexpr int kBM = 128;         // tokens of a tile
constexpr int kOverlap = 16;     // channels that two parts share (a sector of 16-bit elements)
constexpr int kMaxStages = 10;
constexpr int kEpiWarp0 = 2, kEpiWarps = 8;  // four TMEM lane quadrants, two parts of the channels
constexpr int kThreads = 32 * (kEpiWarp0 + kEpiWarps);
constexpr int kStageA = kBM * 128;
// channels of a tile: a row of a part is staged in 256 bytes and the overlap
template <int E>
constexpr int kMaxBN = 512 / E;
template <int E>
constexpr int kPart = kMaxBN<E> / 2 + kOverlap;
// bytes from row to row of a staged part: matrix rows (16 bytes) and pairs of
// fp32 then fall on different banks
template <int E>
constexpr int kSlot = E == 2 ? 304 : 352;
static_assert(kSlot<2> >= kPart<2> * 2 + 16 && kSlot<4> >= kPart<4> * 4 + 16);
constexpr int kOffBar = 0;
constexpr int kOffMisc = kOffBar + (2 * kMaxStages + 4) * 8;
constexpr int kOffCols = (kOffMisc + 16 + 15) / 16 * 16;  // [warps][kPart] scales and biases
template <int E>
constexpr int kOffStg = (kOffCols + kEpiWarps * kPart<E> * 8 + 15) / 16 * 16;
template <int E>
constexpr int kOffRing = (kOffStg<E> + kEpiWarps * 32 * kSlot<E> + 1023) / 1024 * 1024;
constexpr int kSmem = 227 * 1024;
template <int E>
constexpr int kRingBytes = kSmem - 1024 - kOffRing<E>;

// 16 bytes from byte `at` (a multiple of the element) of a staged part on; its
// rows begin on 16 bytes
template <int E>
__device__ __forceinline__ uint4 shifted(const uint8_t *stg, int at) {
  const uint4 *p = reinterpret_cast<const uint4 *>(stg + (at & ~15));
  const uint4 a = p[0], b = p[1];
  const bool by2 = at & 8, by1 = at & 4;
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t u[6], v[5];
#pragma unroll
  for (int i = 0; i < 6; ++i) u[i] = by2 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) v[i] = by1 ? u[i + 1] : u[i];
  if constexpr (E == 4) return make_uint4(v[0], v[1], v[2], v[3]);
  const uint32_t sel = at & 2 ? 0x5432 : 0x3210;
  return make_uint4(__byte_perm(v[0], v[1], sel), __byte_perm(v[1], v[2], sel),
                    __byte_perm(v[2], v[3], sel), __byte_perm(v[3], v[4], sel));
}

// A warp's staged part to y: rows [0, n), row r at g + r * ldb (the address of
// the part's first column), columns [kOverlap, to). A border that is not an end
// of y's rows (begin, end) moves down to its sector's begin: the part before and
// the part behind do the same.
template <typename T>
__device__ __forceinline__ void store_part(uint8_t *g, long long ldb, const uint8_t *stg, int n,
                                           int to, bool begin, bool end, int lane) {
  constexpr int E = sizeof(T), SLOT = kSlot<E>, FROM = kOverlap * E;
  const int k = lane % 16 * 16, half = lane / 16;  // 16 lanes per row, two rows at a time
  g += half * ldb;
  stg += half * SLOT;
  const long long step = 2 * ldb;
  if (!begin && !end) {
    const int bytes = to * E - FROM;  // whole sectors
#pragma unroll 4
    for (int r = half; r < 32; r += 2) {
      const int a = (int)(reinterpret_cast<uintptr_t>(g) & 31);
      const int b = ((FROM + a) & ~31) - a + k;
      if (r < n && k < bytes) *reinterpret_cast<uint4 *>(g + b) = shifted<E>(stg, b);
      g += step;
      stg += 2 * SLOT;
    }
    return;
  }
  for (int r = half; r < n; r += 2) {
    const int a = (int)(reinterpret_cast<uintptr_t>(g) & 31);
    const int lo = begin ? FROM : ((FROM + a) & ~31) - a;
    const int hi = end ? to * E : ((to * E + a) & ~31) - a;
    for (int b = ((lo + a) & ~15) - a + k; b < hi; b += 256) {
      if (b >= lo && b + 16 <= hi) {
        *reinterpret_cast<uint4 *>(g + b) = shifted<E>(stg, b);
      } else {
        for (int e = max(b, lo); e < min(b + 16, hi); e += E)
          *reinterpret_cast<T *>(g + e) = *reinterpret_cast<const T *>(stg + e);
      }
    }
    g += step;
    stg += 2 * SLOT;
  }
}

template <typename T, bool SMALLK>
__global__ void __launch_bounds__(kThreads, 1)
linear_i8_rows_kernel(const __grid_constant__ CUtensorMap xmap,
                      const __grid_constant__ CUtensorMap wmap,
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
    tmem_alloc(s_tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  after_previous();
  const int KS = p.ksteps, stage = kStageA + p.bt * 128;
  uint8_t *ring = smem + kOffRing<sizeof(T)>;
  const int own = p.bt - kOverlap;  // channels that a tile adds

  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&xmap);
      tma_prefetch_desc(&wmap);
      int s = 0, used = 0;  // slot, slots ever filled
      uint32_t phase = 0;
      bool ok = true;
      for (TileWalk t(p); ok && !t.done(); t.next()) {
        const int m0 = t.mi * kBM, n0 = t.ni * own - kOverlap;  // below 0 TMA reads zeros
        for (int k = 0; k < KS; ++k) {
          if (used == p.stages && !mbar_wait_bounded(&empty[s], phase ^ 1, s_abort, p.err, 81)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[s], stage);
          tma_load_2d(ring + s * stage, &xmap, &full[s], 128 * k, m0);
          tma_load_2d(ring + s * stage + kStageA, &wmap, &full[s], 128 * k, n0);
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
        const uint32_t d = tmem + acc.i * 256;
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
    const int half = ew >> 2;   // which part of the tile's channels
    const int quad = warp & 3;  // the TMEM lanes a warp may read
    constexpr int E = sizeof(T), SLOT = kSlot<E>;
    // the part: columns [begin, begin + cols) of the tile, the first kOverlap of
    // them shared with the part before
    const int split = p.bt / 2;
    const int begin = half ? split - kOverlap : 0, cols = half ? p.bt - begin : split;
    const uint32_t tl = tmem + ((uint32_t)(quad * 32) << 16) + begin;
    float *cs = reinterpret_cast<float *>(smem + kOffCols) + ew * kPart<E> * 2;
    uint8_t *stg = smem + kOffStg<E> + ew * 32 * SLOT;
    const long long ldb = (long long)p.N * E;
    // where this thread's elements of 16 rows x 16 columns go: 16 bits, the row of
    // the 8 x 8 matrix that it names; 32 bits, its first pair
    const uint32_t put = smem_u32(stg) + (E == 2 ? (lane & 15) * SLOT + (lane >> 4) * 16
                                                 : (lane >> 2) * SLOT + (lane & 3) * 8);
    // a tile's column scales and biases and its rows' scales (rows 8 i + lane / 4),
    // loaded while the tile before is worked on
    constexpr int CL = (kPart<E> + 31) / 32;
    float nsw[CL], nb[CL], nsx[4];
    auto prefetch = [&](const TileWalk &t) {
#pragma unroll
      for (int i = 0; i < CL; ++i) {
        const int n = t.ni * own - kOverlap + begin + 32 * i + lane;
        const bool real = n >= 0 && n < p.N;
        nsw[i] = real ? __ldg(p.sw + n) : 0.f;
        nb[i] = real && p.bias ? __ldg(p.bias + n) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long m = (long long)t.mi * kBM + quad * 32 + 8 * i + (lane >> 2);
        nsx[i] = m < p.rows ? p.sx[m] : 0.f;  // see linear_i8.cu: no read-only load
      }
    };
    TileWalk ahead(p);
    if (!ahead.done()) prefetch(ahead);
    Ring<2> acc;
    for (TileWalk t(p); !t.done(); t.next(), acc.next()) {
      const int n0 = t.ni * own - kOverlap + begin;  // the part's first channel
      const long long m0 = (long long)t.mi * kBM + quad * 32;
      uint64_t sx2[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) sx2[i] = pk(nsx[i], nsx[i]);
      __syncwarp();  // the part before is stored, its scales are read
#pragma unroll
      for (int i = 0; i < CL; ++i) {  // by pairs of columns: s0 s1 b0 b1
        const int c = 32 * i + lane;
        if (c < cols) {
          cs[c / 2 * 4 + (c & 1)] = nsw[i];
          cs[c / 2 * 4 + (c & 1) + 2] = nb[i];
        }
      }
      __syncwarp();
      ahead.next();
      if (!ahead.done()) prefetch(ahead);
      if (!mbar_wait_bounded(&acc_full[acc.i], acc.phase, s_abort, p.err, 84)) break;
      tc_fence_after();
      const uint32_t ta = tl + acc.i * 256;
      uint32_t v[2][2][8];  // two steps; rows 0-15, 16-31
      tmem_ld_16x256b_x2(ta, v[0][0]);
      tmem_ld_16x256b_x2(ta + (16u << 16), v[0][1]);
#pragma unroll
      for (int c = 0; c < kPart<E>; c += 16) {
        if (c >= cols) break;
        uint32_t(&w)[2][8] = v[c / 16 & 1];
        tmem_ld_wait(w[0], w[1]);
        if (c + 16 < cols) {
          uint32_t(&x)[2][8] = v[(c / 16 + 1) & 1];
          tmem_ld_16x256b_x2(ta + c + 16, x[0]);
          tmem_ld_16x256b_x2(ta + (16u << 16) + c + 16, x[1]);
        }
        ulonglong2 sb[2];  // scales and biases of the thread's two pairs of columns
#pragma unroll
        for (int h = 0; h < 2; ++h)
          sb[h] = *reinterpret_cast<const ulonglong2 *>(cs + 2 * (c + 8 * h + 2 * (lane & 3)));
        float f[4][2][2];  // [row 8 i][columns 8 h][column]
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t *q = &w[i >> 1][4 * h + 2 * (i & 1)];
            const uint64_t a = sums2<SMALLK>(q[0], q[1]);
            upk(fma2(mul2(a, sb[h].x), sx2[i], sb[h].y), f[i][h][0], f[i][h][1]);
          }
        if (p.act) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              f[i][h][0] = activate(f[i][h][0], p.act);
              f[i][h][1] = activate(f[i][h][1], p.act);
            }
        }
        if constexpr (E == 2) {
#pragma unroll
          for (int i = 0; i < 4; i += 2)  // rows 8 i and 8 (i + 1), columns 0-7 and 8-15
            stmatrix_x4(put + 8 * i * SLOT + c * 2, pack2<T>(f[i][0][0], f[i][0][1]),
                        pack2<T>(f[i + 1][0][0], f[i + 1][0][1]),
                        pack2<T>(f[i][1][0], f[i][1][1]),
                        pack2<T>(f[i + 1][1][0], f[i + 1][1][1]));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(put + 8 * i * SLOT +
                                                                     (c + 8 * h) * 4),
                           "f"(f[i][h][0]), "f"(f[i][h][1])
                           : "memory");
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc.i]);
      const int to = min(cols, p.N - n0);
      if (to > kOverlap && m0 < p.rows)
        store_part<T>(static_cast<uint8_t *>(p.y) + m0 * ldb + (long long)n0 * E, ldb, stg,
                      (int)min((long long)32, p.rows - m0), to, t.ni == 0 && half == 0,
                      n0 + cols >= p.N, lane);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, bool SMALLK>
int launch_product(const void *xq, const void *wq, const LinParams &p, int K, int pitch, cudaStream_t st) {
  CUtensorMap xm, wm;
  int rc = tma_map_rows(&xm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, xq, K, p.rows, pitch, kBM);
  if (rc) return rc;
  rc = tma_map_rows(&wm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, wq, K, p.N, pitch, p.bt);
  if (rc) return rc;
  auto *kernel = linear_i8_rows_kernel<T, SMALLK>;
  rc = allow_dynamic_smem(reinterpret_cast<const void *>(kernel), kSmem, "linear_i8_rows_kernel");
  if (rc) return rc;
  const int grid = (int)(p.tiles < sm_count() ? p.tiles : sm_count());
  if (p.behind_quant)
    return launch_overlapped("linear_i8_rows_kernel", kernel, grid, kThreads, kSmem, st, xm, wm, p);
  kernel<<<grid, kThreads, kSmem, st>>>(xm, wm, p);
  return check_launch("linear_i8_rows_kernel");
}

template <typename T>
int product(const void *xq, const void *wq, LinParams p, int K, int pitch, cudaStream_t st) {
  constexpr int E = sizeof(T);
  // the channels of a tile for which the waves of CTAs take least: a tile costs
  // its channels and a fixed part worth about 64; three slots of the ring where
  // there is more than one step of K
  const long long tm = (p.rows + kBM - 1) / kBM, sms = sm_count();
  long long best = -1;
  for (int bn = kMaxBN<E>; bn >= 64; bn -= 32) {
    const int own = bn - kOverlap, stages = kRingBytes<E> / (kStageA + bn * 128);
    if (stages < 3 && p.ksteps > 1) continue;
    const long long cost = (tm * ((p.N + own - 1) / own) + sms - 1) / sms * (bn + 64);
    if (best < 0 || cost < best) {
      best = cost;
      p.bt = bn;
      p.stages = stages < kMaxStages ? stages : kMaxStages;
    }
  }
  p.tiles_n = (p.N + p.bt - kOverlap - 1) / (p.bt - kOverlap);
  p.tiles = tm * p.tiles_n;
  return K <= kSmallK ? launch_product<T, true>(xq, wq, p, K, pitch, st)
                      : launch_product<T, false>(xq, wq, p, K, pitch, st);
}

}  // namespace

int linear::launch_row_kernel(const void *xq, const void *wq, const LinParams &p, int K, int pitch,
                              int out_dtype, cudaStream_t st) {
  if (out_dtype == TOCR_DTYPE_F16) return product<__half>(xq, wq, p, K, pitch, st);
  if (out_dtype == TOCR_DTYPE_BF16) return product<__nv_bfloat16>(xq, wq, p, K, pitch, st);
  return product<float>(xq, wq, p, K, pitch, st);
}

}  // namespace tocr
