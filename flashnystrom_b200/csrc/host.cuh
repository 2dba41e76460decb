// Host-side helpers shared by the translation units of the library: error text, the optional per-kernel profiler, function
// attributes, device selection, launches with programmatic stream serialization.
#pragma once
#include "../../include/flashnystrom_b200.h"

#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <mutex>
#include <string>
#include <utility>
#include <vector>

namespace fnb {

inline thread_local char g_err[512] = "";
inline int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

#define FNB_CUDA(expr)                                                                     \
  do {                                                                                     \
    cudaError_t e_ = (expr);                                                               \
    if (e_ != cudaSuccess)                                                                 \
      return fail(FNB_ERR_CUDA, "%s failed: %s (%s:%d)", #expr, cudaGetErrorString(e_),    \
                  __FILE__, __LINE__);                                                     \
  } while (0)

// ---- optional per-kernel profiler -----------------------------------------------------------
// Off by default.  FNB_PROFILE=1 in the environment at load, or fnb_set_profiling(1), brackets
// every kernel with a pair of CUDA events on the caller's stream (no host synchronisation in the
// call itself); fnb_last_profile() waits for the last event and reads the times back.
inline int g_profile = [] {
  const char* e = getenv("FNB_PROFILE");
  return (e && e[0] == '1') ? 1 : 0;
}();
struct ProfState {
  int device = -1;
  std::vector<cudaEvent_t> pool;      // reused across calls on this thread
  std::vector<std::string> names;     // kernels of the most recent call
  size_t used = 0;
  cudaEvent_t get(int dev) {
    if (dev != device) {
      for (cudaEvent_t e : pool) cudaEventDestroy(e);
      pool.clear();
      device = dev;
      used = 0;
    }
    if (used == pool.size()) {
      cudaEvent_t e = nullptr;
      cudaEventCreate(&e);
      pool.push_back(e);
    }
    return pool[used++];
  }
};
inline thread_local ProfState g_prof;

struct Launcher {
  cudaStream_t stream;
  int device;
  bool prof;
  int status = 0;
  Launcher(cudaStream_t s, int dev) : stream(s), device(dev), prof(g_profile != 0) {
    if (prof) {
      g_prof.names.clear();
      g_prof.used = 0;
    }
  }
  void begin() {
    if (prof) cudaEventRecord(g_prof.get(device), stream);
  }
  int end(const char* name) {
    cudaError_t e = cudaPeekAtLastError();
    if (e != cudaSuccess) {
      cudaGetLastError();
      return status = fail(FNB_ERR_CUDA, "launch of %s failed: %s", name, cudaGetErrorString(e));
    }
    if (prof) {
      cudaEventRecord(g_prof.get(device), stream);
      g_prof.names.push_back(name);
    }
    return 0;
  }
};

// The two function attributes below are per kernel and device and stay until the context ends:
// they are set once (again only if a later call needs more), not on every launch.
inline std::mutex g_smem_mutex;
inline std::map<std::pair<const void*, int>, size_t> g_smem_set;

// Raises a kernel's opt-in dynamic shared memory size to `bytes` (never lowers it: the largest size asked
// for so far is remembered per kernel and device, and launches that need less skip the call).
inline cudaError_t raise_smem(const void* kernel, size_t bytes) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) device = -1;
  const std::pair<const void*, int> key(kernel, device);
  if (device >= 0) {
    std::lock_guard<std::mutex> lock(g_smem_mutex);
    auto it = g_smem_set.find(key);
    if (it != g_smem_set.end() && it->second >= bytes) return cudaSuccess;
  }
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  // ask for the largest shared-memory carveout so that co-residency is limited by the kernel's
  // own footprint, not by the driver's default split between L1 and shared memory
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess && device >= 0) {
    std::lock_guard<std::mutex> lock(g_smem_mutex);
    size_t& cur = g_smem_set[key];
    if (cur < bytes) cur = bytes;
  }
  return e;
}

template <class K>
inline int set_smem(K kernel, size_t bytes, int max_optin, const char* name) {
  if ((long long)bytes > (long long)max_optin)
    return fail(FNB_ERR_SMEM, "insufficient smem for %s: needs %zu bytes, device allows %d", name,
                bytes, max_optin);
  cudaError_t e = raise_smem(reinterpret_cast<const void*>(kernel), bytes);
  if (e != cudaSuccess)
    return fail(FNB_ERR_CUDA, "cudaFuncSetAttribute(%s, %zu) failed: %s", name, bytes,
                cudaGetErrorString(e));
  return 0;
}

struct DeviceGuard {
  int prev = -1;
  bool ok = true;
  explicit DeviceGuard(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) { ok = false; return; }
    // Always (re)select: besides switching devices this binds the device's primary context to
    // the calling thread, which the driver-level tensor-map encoder needs (an autograd worker
    // thread may not have touched the runtime yet).
    if (cudaSetDevice(dev) != cudaSuccess) ok = false;
  }
  ~DeviceGuard() {
    int cur = -1;
    if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
  }
};

inline int device_limits(int device, int* max_smem, int* cc_major, int* sm_count) {
  // attribute queries are cheap and keep the call free of cached, thread-affine state
  FNB_CUDA(cudaDeviceGetAttribute(max_smem, cudaDevAttrMaxSharedMemoryPerBlockOptin, device));
  FNB_CUDA(cudaDeviceGetAttribute(cc_major, cudaDevAttrComputeCapabilityMajor, device));
  FNB_CUDA(cudaDeviceGetAttribute(sm_count, cudaDevAttrMultiProcessorCount, device));
  if (*cc_major != 10)
    return fail(FNB_ERR_UNSUPPORTED_DEVICE,
                "device %d has compute capability %d.x; this library is built for sm_100a only",
                device, *cc_major);
  return 0;
}

// The limit of the bounded waits is a device variable of each translation unit with kernels that wait: that of fnb_operators.cu.
cudaError_t set_operators_wait_limit(unsigned long long ns);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Launch with programmatic stream serialization: the kernel may be scheduled while its
// predecessor in the stream is still running (every kernel launched this way calls pdl_wait()
// before it touches global memory that other kernels of the stream produce or consume).
template <class... KArgs, class... Args>
inline cudaError_t launch_pdl(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                              Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

}  // namespace fnb
