// Host-side helpers shared by the library's translation units: device
// properties and launching a kernel with programmatic stream serialisation.
// Everything is in an unnamed namespace: each translation unit has its own
// (small) caches.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <cstdlib>
#include <mutex>
#include <utility>

#include "../../include/b200_gemm.h"

namespace b200 {
namespace {

constexpr int kMaxDevices = 64;

struct DeviceInfo {
  bool ready = false;
  bool sm100 = false;
  int sm_count = 0;
  int64_t l2_bytes = 0;
};

std::mutex g_dev_mu;
DeviceInfo g_dev[kMaxDevices];

int current_device_info(DeviceInfo& out) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return B200_ERR_CUDA;
  std::lock_guard<std::mutex> lk(g_dev_mu);
  DeviceInfo& d = g_dev[dev];
  if (!d.ready) {
    int major = 0, sms = 0, l2 = 0;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&l2, cudaDevAttrL2CacheSize, dev) != cudaSuccess)
      return B200_ERR_CUDA;
    d.sm100 = (major == 10);
    d.sm_count = sms;
    d.l2_bytes = l2;
    d.ready = true;
  }
  out = d;
  return B200_OK;
}

// cudaFuncSetAttribute once per (kernel instantiation, device); `done` is
// the calling launch template's own flag array (all kernels share one
// function-pointer type, so the flags cannot live here).
template <typename Kern>
int ensure_smem_attr(Kern kern, int smem_bytes, std::atomic<uint8_t>* done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return B200_ERR_CUDA;
  if (dev >= 0 && dev < kMaxDevices && done[dev].load(std::memory_order_acquire)) return B200_OK;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes) != cudaSuccess)
    return B200_ERR_CUDA;
  if (dev >= 0 && dev < kMaxDevices) done[dev].store(1, std::memory_order_release);
  return B200_OK;
}

// GEMM kernels go out with programmatic stream serialisation (PDL): a kernel
// may be scheduled while the previous one on the stream drains, runs its
// setup (barriers, TMEM, tensor-map prefetch), and waits in griddep_wait()
// before its first global access.  B200_GEMM_PDL=0 turns it off.
bool pdl_enabled() {
  static const bool on = [] {
    const char* e = std::getenv("B200_GEMM_PDL");
    return !(e && e[0] == '0');
  }();
  return on;
}

template <typename... KArgs, typename... Args>
cudaError_t launch_gemm(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                        Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Every pointer on a multiple of `bytes` (NULL: fine).
template <typename... P>
bool aligned_to(uintptr_t bytes, const P*... p) {
  return ((reinterpret_cast<uintptr_t>(p) | ... | 0) & (bytes - 1)) == 0;
}

bool pitch_ok(const void* p, int64_t ld) { return aligned16(p) && (ld % 8) == 0; }

int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

}  // namespace
}  // namespace b200
