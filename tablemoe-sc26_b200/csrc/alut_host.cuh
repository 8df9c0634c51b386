// Host-side helpers shared by the translation units of the library: the thread's last error,
// launch checks, device properties and the programmatic-dependent launch.
#pragma once

#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <mutex>

#include "alut.h"

namespace alut {

inline thread_local char g_err[512] = "no error";

inline int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

inline int check_launch(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(ALUT_ECUDA, "%s: %s", what, cudaGetErrorString(e));
  return ALUT_OK;
}

inline int dtype_size(int d) { return d == ALUT_F32 ? 4 : 2; }
inline bool dtype_ok(int d) { return d == ALUT_F32 || d == ALUT_BF16 || d == ALUT_F16; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline int num_sms() {
  static int cache[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return 148;
  if (dev < 64 && cache[dev]) return cache[dev];
  int n = 148;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) n = 148;
  if (dev < 64) cache[dev] = n;
  return n;
}

// Raise a kernel's dynamic shared memory limit once per (kernel, device).
inline int allow_smem(const void* kernel, size_t bytes) {
  if (bytes <= 48 * 1024) return ALUT_OK;
  struct Entry { const void* k; int dev; int bytes; };
  static Entry table[256];
  static int used = 0;
  static std::mutex mu;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  for (int i = 0; i < used; ++i)
    if (table[i].k == kernel && table[i].dev == dev && table[i].bytes >= static_cast<int>(bytes))
      return ALUT_OK;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(bytes));
  if (e != cudaSuccess) return fail(ALUT_ECUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  if (used < 256) table[used++] = Entry{kernel, dev, static_cast<int>(bytes)};
  return ALUT_OK;
}

// Launch as a programmatic dependent of the previous kernel in the stream (it may start
// early and waits in griddepcontrol.wait for the predecessor's results).
template <typename... KArgs, typename... Args>
inline cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
                              cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace alut
