// Per-kernel shared-memory bookkeeping behind ssb_kernel_smem (the reference's SHARED_BYTES), and the process-wide
// bound of the cooperative kernels' grid-barrier waits (ssb_set_wait_limit_ns).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

void ssb_note_smem_bytes(const char* name, int bytes);
uint64_t ssb_barrier_wait_ns();

// SMs of the current device (asked once per device).
int ssb_sm_count();

// One-time setup of a kernel on each device: its dynamic shared memory limit and its entry in the table above. `done` is a
// static of the caller, one bit per device; a device past the 64th is set up at every call.
template <typename K>
static inline int ssb_setup_kernel(std::atomic<uint64_t>& done, const char* name, K kern, size_t dyn) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (e == cudaSuccess && (done.load(std::memory_order_acquire) & bit)) return 0;
  cudaFuncAttributes a;
  if (e == cudaSuccess) e = cudaFuncSetAttribute((const void*)kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)dyn);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, (const void*)kern);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return (int)e;
  }
  ssb_note_smem_bytes(name, (int)(a.sharedSizeBytes + dyn));
  done.fetch_or(bit, std::memory_order_release);
  return 0;
}

template <typename K>
static inline void ssb_note_smem(const char* name, K kern, size_t dyn) {
  cudaFuncAttributes a;
  if (cudaFuncGetAttributes(&a, (const void*)kern) == cudaSuccess)
    ssb_note_smem_bytes(name, (int)(a.sharedSizeBytes + dyn));
  else
    (void)cudaGetLastError();
}
