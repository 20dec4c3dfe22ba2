// Host helpers shared by the library's translation units: the last error's
// text, device attributes, argument checks and the tensor-map encoder.
#pragma once

#include <cudaTypedefs.h>

#include <cstring>
#include <mutex>
#include <string>
#include <type_traits>

#include "common.cuh"

namespace pcb {

inline thread_local std::string g_last_error;

inline int fail(int status, const char* what) {
  g_last_error = what;
  return status;
}

inline int check_launch(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    g_last_error = std::string(what) + ": " + cudaGetErrorString(e);
    return PCB_ERR_LAUNCH;
  }
  return PCB_OK;
}

struct DeviceInfo {
  int sm_count = 0;
  int major = 0;
};

inline DeviceInfo device_info() {
  static std::mutex mu;
  static DeviceInfo cache[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) dev = 0;
  std::lock_guard<std::mutex> lock(mu);
  if (cache[dev].sm_count == 0) {
    cudaDeviceGetAttribute(&cache[dev].sm_count, cudaDevAttrMultiProcessorCount, dev);
    cudaDeviceGetAttribute(&cache[dev].major, cudaDevAttrComputeCapabilityMajor, dev);
  }
  return cache[dev];
}

inline bool aligned(const void* p, int64_t a) { return (reinterpret_cast<uintptr_t>(p) % (uintptr_t)a) == 0; }

template <typename K>
void ensure_smem_attr(K kernel, int bytes) {
  // cudaFuncSetAttribute is per function and device; calling it again is cheap
  // and keeps this stateless across devices and threads.
  cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}


inline int elem_size(int dt) {
  switch (dt) {
    case PCB_DTYPE_F32: return 4;
    case PCB_DTYPE_F16:
    case PCB_DTYPE_BF16: return 2;
    case PCB_DTYPE_E4M3:
    case PCB_DTYPE_E5M2: return 1;
    default: return 0;
  }
}

inline bool is_float_in(int dt) { return dt == PCB_DTYPE_F32 || dt == PCB_DTYPE_F16 || dt == PCB_DTYPE_BF16; }
inline bool is_fp8(int dt) { return dt == PCB_DTYPE_E4M3 || dt == PCB_DTYPE_E5M2; }

// Dispatch a functor over (input dtype, fp8 output dtype) as compile-time ints.
template <typename F>
int dispatch_xy(int xt, int yt, F&& f) {
  auto with_y = [&](auto xc) -> int {
    if (yt == PCB_DTYPE_E4M3) return f(xc, std::integral_constant<int, PCB_DTYPE_E4M3>{});
    if (yt == PCB_DTYPE_E5M2) return f(xc, std::integral_constant<int, PCB_DTYPE_E5M2>{});
    return fail(PCB_ERR_INVALID, "output dtype must be E4M3 or E5M2");
  };
  if (xt == PCB_DTYPE_F32) return with_y(std::integral_constant<int, PCB_DTYPE_F32>{});
  if (xt == PCB_DTYPE_F16) return with_y(std::integral_constant<int, PCB_DTYPE_F16>{});
  if (xt == PCB_DTYPE_BF16) return with_y(std::integral_constant<int, PCB_DTYPE_BF16>{});
  return fail(PCB_ERR_INVALID, "input dtype must be F32, F16 or BF16");
}

// ---------------------------------------------------------------------------
// TMA descriptors (driver entry point fetched through the runtime, so the
// library does not link libcuda directly).
// ---------------------------------------------------------------------------
inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  // The encoder wants a context.  A thread that has only allocated from a
  // cache so far (autograd's worker, say) may have none bound yet.
  static thread_local bool bound = false;
  if (!bound) {
    int dev = 0;
    bound = cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
  }
  return fn;
}

}  // namespace pcb
