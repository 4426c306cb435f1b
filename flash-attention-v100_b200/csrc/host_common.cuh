// What the launch layers (fmha_api.cu, paged_api.cu) share on the host: the driver's entry point for tensor maps,
// device queries, launches with a raised shared-memory limit, checks of pointers and strides.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "../../include/fmha_b200.h"

namespace {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn get_encode_fn() {
  // resolved once; the pointer is process-wide and immutable afterwards
  static EncodeTiledFn fn = []() -> EncodeTiledFn {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres) !=
            cudaSuccess ||
        qres != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<EncodeTiledFn>(ptr);
  }();
  return fn;
}

constexpr int kMaxDevices = 64;

int current_device() {
  int dev = -1;
  return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < kMaxDevices ? dev : -1;
}

// SMs of a device, asked once per device (the query costs as much host time as a tensor map)
int sm_count(int dev) {
  static std::atomic<int> cached[kMaxDevices];
  if (dev < 0) return 148;
  int n = cached[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
    cached[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Launches a kernel whose dynamic shared memory needs its limit raised, which is done once per kernel and
// device, and again where a launch is refused: the limit goes with the context when the host resets
// the device.
template <auto kKernel, typename... Args>
bool launch_with_smem(int dev, unsigned grid, unsigned threads, int bytes, cudaStream_t stream, const Args&... args) {
  static std::atomic<bool> raised[kMaxDevices];
  for (int attempt = 0; attempt < 2; ++attempt) {
    if (attempt > 0 || dev < 0 || !raised[dev].load(std::memory_order_acquire)) {
      if (cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
        return false;
      if (dev >= 0) raised[dev].store(true, std::memory_order_release);
    }
    kKernel<<<grid, threads, bytes, stream>>>(args...);
    if (cudaGetLastError() == cudaSuccess) return true;
  }
  return false;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_strides(const FmhaStrides& s, int N, int H, int Z) {
  if ((N > 1 && (s.row % 8 != 0 || s.row <= 0)) || (H > 1 && (s.head % 8 != 0 || s.head <= 0)) ||
      (Z > 1 && (s.batch % 8 != 0 || s.batch <= 0)))
    return FMHA_ERR_BAD_STRIDE;
  return FMHA_OK;
}

}  // namespace
