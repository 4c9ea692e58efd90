// What the two kernels of the INT8 linear layer's product share.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "tc_ptx.cuh"
#include "tma_map.cuh"
#include "tocr_common.cuh"

namespace tocr::linear {

struct LinParams {
  const float *sx, *sw, *bias;
  void *y;
  long long rows;
  int N, ksteps;
  int bt, stages;                // tokens (channels) that are a tile's MMA columns; ring slots
  int tiles_n;                   // tiles along the channels
  long long tiles;
  int act;
  bool behind_quant;             // launched behind the quantiser of the same call
  int *err;
};

// y's rows are not sector-aligned and y is so large that its sectors leave L2
// before the neighbours have completed them: 40960 x 128 x 18385 (1.5 GB of bf16)
// 585 us with the row kernel, 833 with the other. The rule is a bound on that
// effect and looks at no other cost. At 134 MB, about what L2 holds, the other
// kernel would be the faster one in a row of calls, 45 against 67 us at 16384 x
// 128 x 4095 and 213 against 260 at 16384 x 4096 x 4095.
inline bool wants_row_kernel(const void *y, long long rows, int N, int elem) {
  const size_t row = (size_t)N * elem;
  return (row % 32 || !aligned(y, 32)) && row * (size_t)rows > (64u << 20);
}
// The product for such an output (linear_i8_rows.cu).
int launch_row_kernel(const void *xq, const void *wq, const LinParams &p, int K, int pitch,
                      int out_dtype, cudaStream_t st);

__device__ __forceinline__ float activate(float y, int act) {
  if (act == TOCR_ACT_RELU) return y < 0.f ? 0.f : y;  // keeps NaN
  return y * (fminf(fmaxf(y + 3.f, 0.f), 6.f) * (1.f / 6.f));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same_v<T, __half>)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Tiles blockIdx.x, blockIdx.x + gridDim.x, ...: channels fastest, so that the
// CTAs share few operand tiles at a time, and no division from tile to tile.
struct TileWalk {
  int ni, mi, dn, dm, tiles_n;
  long long left;
  __device__ __forceinline__ explicit TileWalk(const LinParams &p) {
    tiles_n = p.tiles_n;
    ni = blockIdx.x % tiles_n;
    mi = blockIdx.x / tiles_n;
    dn = gridDim.x % tiles_n;
    dm = gridDim.x / tiles_n;
    left = (p.tiles - blockIdx.x + gridDim.x - 1) / gridDim.x;  // the grid has no idle CTA
  }
  __device__ __forceinline__ bool done() const { return left <= 0; }
  __device__ __forceinline__ void next() {
    --left;
    ni += dn;
    mi += dm;
    if (ni >= tiles_n) {
      ni -= tiles_n;
      ++mi;
    }
  }
};

// An s32 pair as fp32. SMALL: |sum| <= 2^22, so adding it to the bits of
// 1.5 * 2^23 converts it (full-rate instructions; the conversion instruction runs
// at an eighth of their rate and would bound layers of small K).
template <bool SMALL>
__device__ __forceinline__ uint64_t sums2(uint32_t a, uint32_t b) {
  if (SMALL)
    return ptx::add2(ptx::pk(__uint_as_float(a + 0x4B400000u), __uint_as_float(b + 0x4B400000u)),
                     ptx::pk(-12582912.f, -12582912.f));
  return ptx::pk((float)(int)a, (float)(int)b);
}
constexpr int kSmallK = 256;  // 128^2 K <= 2^22: any codes

}  // namespace tocr::linear
