// Shared plumbing of the C-ABI entry points: status codes, the per-thread
// last-error message, host-side fault injection and launch checks.
#pragma once

#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <cstdint>
#include <cstdio>
#include <climits>

#include "tocr_capi.h"

namespace tocr {

// Records `msg` as this thread's last error and returns `status`.
int set_error(int status, const char *fmt, ...);
// Clears the thread's last error (called on entry of every compute call).
void clear_error();
// Returns a pending injected status (and consumes one injection), or TOCR_OK.
int take_injected();

inline cudaStream_t as_stream(void *s) { return reinterpret_cast<cudaStream_t>(s); }

// Checks the launch that was just enqueued.
inline int check_launch(const char *what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    return set_error(TOCR_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return TOCR_OK;
}

inline bool aligned(const void *p, size_t a) {
  return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0;
}

// SM count of the current device, cached per device.
int sm_count();

// Launches a kernel that may begin while the kernel before it in the stream
// still runs, and that waits for it itself (after_previous()) before it touches
// memory: its set-up overlaps the other's end. For kernels inside one call only,
// behind a first one that is launched as usual.
template <typename... P, typename... A>
int launch_overlapped(const char *what, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem,
                      cudaStream_t st, A &&...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  return e == cudaSuccess ? TOCR_OK
                          : set_error(TOCR_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}
#ifdef __CUDACC__
__device__ __forceinline__ void after_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
// lets the next kernel's set-up begin once every block of this one got here
__device__ __forceinline__ void release_next() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
#endif

// Allows `kernel` `bytes` of dynamic shared memory on the current device (asked
// of the driver once per kernel and device).
int allow_dynamic_smem(const void *kernel, int bytes, const char *what);

}  // namespace tocr

// Common prologue for a compute entry: clear error, honour injection.
#define TOCR_ENTRY()                               \
  do {                                             \
    ::tocr::clear_error();                         \
    int _inj = ::tocr::take_injected();            \
    if (_inj != TOCR_OK)                           \
      return ::tocr::set_error(_inj, "injected");  \
  } while (0)

#define TOCR_REQUIRE(cond, ...)                                 \
  do {                                                          \
    if (!(cond)) return ::tocr::set_error(TOCR_ERR_INVALID, __VA_ARGS__); \
  } while (0)
