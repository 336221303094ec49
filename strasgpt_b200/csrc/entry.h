// Host side shared by the kernel-level entry points that refuse a call with
// -1 and a message instead of ending the process (rope.cu, lora.cu,
// attn_tree.cu, sample.cu).
#pragma once

#include <atomic>
#include <mutex>

#include "common.cuh"

namespace sg {

// Prints why `entry` refuses the call; the caller returns the -1.
inline int refuse(const char* entry, const char* why) {
  fprintf(stderr, "[StrasGPT] Error: %s: %s\n", entry, why);
  return -1;
}

inline int refuse_cuda(const char* entry, const char* what, cudaError_t e) {
  char m[256];
  snprintf(m, sizeof(m), "%s: %s", what, cudaGetErrorString(e));
  return refuse(entry, m);
}

// Why `p` cannot be a buffer of a kernel on the current device `dev`, or
// NULL. Host memory and another GPU's memory would fault inside the kernel.
inline const char* not_on_device(const void* p, int dev) {
  cudaPointerAttributes a;
  if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
    cudaGetLastError();  // the query's own error is not the next call's
    return "a buffer is not device memory";
  }
  if (a.type == cudaMemoryTypeManaged) return nullptr;
  if (a.type != cudaMemoryTypeDevice) return "a buffer is not device memory";
  if (a.device != dev) return "a buffer is on another device than the current one";
  return nullptr;
}

inline bool aligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

// Whether `bytes` from p and `bytes` from q on share any.
inline bool overlap(const void* p, const void* q, size_t bytes) {
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
  return a < b ? b - a < bytes : a - b < bytes;
}

// Device index below this bound: per-device set-up is remembered by index.
constexpr int kDevices = 64;

// The current device and its number of SMs (asked once per device). Returns
// NULL, or why there is none.
inline const char* current_device(int* dev, int* sms) {
  static std::atomic<int> known[kDevices];
  if (cudaGetDevice(dev) != cudaSuccess) {
    cudaGetLastError();
    return "no CUDA device";
  }
  if (*dev < 0 || *dev >= kDevices) return "device index above 63";
  int n = known[*dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *dev) != cudaSuccess || n < 1) {
      cudaGetLastError();
      return "no CUDA device";
    }
    known[*dev].store(n, std::memory_order_relaxed);
  }
  *sms = n;
  return nullptr;
}

// Raises `kernel`'s dynamic shared memory limit to `bytes`, and never lowers it
// (`done` belongs to the kernel: the limit on each device). Callers may ask
// for different sizes from several threads: reading the limit, setting it and
// noting it are one step under the lock.
inline std::mutex smem_lock;

template <typename K>
inline cudaError_t allow_smem(K kernel, size_t bytes, int dev, std::atomic<size_t>* done) {
  if (done[dev].load(std::memory_order_acquire) >= bytes) return cudaSuccess;
  const std::lock_guard<std::mutex> hold(smem_lock);
  if (done[dev].load(std::memory_order_relaxed) >= bytes) return cudaSuccess;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) done[dev].store(bytes, std::memory_order_release);
  return e;
}

// Launch with programmatic dependent launch (as sg::launch) and, for
// cluster > 1, a cluster along x; the error is the caller's to report.
template <typename... KArgs, typename... Args>
inline cudaError_t try_launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
                              int cluster, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    n++;
  }
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    n++;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, ((KArgs)args)...);
  if (e != cudaSuccess) cudaGetLastError();
  return e;
}

}  // namespace sg
