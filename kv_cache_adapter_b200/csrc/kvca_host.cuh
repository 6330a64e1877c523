// Launch helpers that the kernel files share.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <utility>

#include "kvca.h"

namespace kvca {
namespace {

// Launch as a programmatic dependent of the kernel before it on the stream
// (the kernel must wait for it with griddepcontrol.wait).
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, unsigned block, size_t smem,
                             cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
  return e != cudaSuccess ? e : cudaGetLastError();
}

int device_sm_count() { return kvca_device_sm_count(); }

// Function attributes (the dynamic shared-memory limit, the carve-out)
// belong to the current device's context, so a launcher sets them once per
// device: `done` records the ordinals done (devices past the table are set
// up on every call).
constexpr int kTrackedDevices = 64;
using DeviceFlags = std::atomic<bool>[kTrackedDevices];

bool needs_setup(const DeviceFlags& done, int* dev) {
  *dev = -1;
  if (cudaGetDevice(dev) != cudaSuccess) return true;
  return *dev < 0 || *dev >= kTrackedDevices || !done[*dev].load(std::memory_order_acquire);
}

void mark_setup(DeviceFlags& done, int dev) {
  if (dev >= 0 && dev < kTrackedDevices) done[dev].store(true, std::memory_order_release);
}

}  // namespace
}  // namespace kvca
