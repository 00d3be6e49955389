// Host-side helpers shared by the library's translation units: errors, tensor-map encoding, device
// properties, process-wide launch options and the kernel launcher.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <exception>
#include <string>
#include <utility>

#include "../../include/laya_b200.h"

namespace laya {

// ---------------------------------------------------------------------------------------------
// Errors
// ---------------------------------------------------------------------------------------------
inline thread_local std::string g_create_error;

struct Failure {
  int code;
  std::string msg;
};

[[noreturn]] inline void fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  throw Failure{code, buf};
}

#define CK(call)                                                                                    \
  do {                                                                                              \
    cudaError_t e_ = (call);                                                                        \
    if (e_ != cudaSuccess) fail(LAYA_ERR_CUDA, "%s failed: %s", #call, cudaGetErrorString(e_));     \
  } while (0)

// ---------------------------------------------------------------------------------------------
// Driver entry point for tensor-map encoding (no link-time dependency on libcuda).
// ---------------------------------------------------------------------------------------------
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static std::atomic<EncodeTiledFn> cached{nullptr};
  EncodeTiledFn fn = cached.load(std::memory_order_acquire);
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    CK(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q));
    if (!p || q != cudaDriverEntryPointSuccess) fail(LAYA_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
    fn = reinterpret_cast<EncodeTiledFn>(p);
    cached.store(fn, std::memory_order_release);
  }
  return fn;
}

// Streaming multiprocessors of `device`, read once (callers on several host threads included).
inline int sm_count(int device) {
  static std::atomic<int> cache[64];
  const bool cached = device >= 0 && device < 64;
  int n = cached ? cache[device].load(std::memory_order_relaxed) : 0;
  if (n) return n;
  CK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device));
  if (cached) cache[device].store(n, std::memory_order_relaxed);
  return n;
}

// Process-wide launch options (laya_set_launch_options): programmatic dependent launch on every
// kernel (on by default), and the wait limit every pipelined kernel's bounded waits use
// (0: the kernels' default of 2 s).  Passes captured into CUDA graphs keep the options in effect
// at capture.
inline std::atomic<bool> g_pdl{true};
inline std::atomic<unsigned long long> g_wait_ns{0};
inline bool pdl_enabled() { return g_pdl.load(std::memory_order_relaxed); }
inline unsigned long long wait_ns() { return g_wait_ns.load(std::memory_order_relaxed); }

template <typename... KArgs, typename... Args>
void launch_k(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  CK(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...));
}

// ---------------------------------------------------------------------------------------------
// Entry points of operators: exceptions end in status codes, with the message in laya_last_error(NULL).
// ---------------------------------------------------------------------------------------------
#define OP_API_BEGIN try {
#define OP_API_END                                     \
  }                                                    \
  catch (const Failure& f) {                           \
    g_create_error = f.msg;                            \
    return f.code;                                     \
  }                                                    \
  catch (const std::exception& x) {                    \
    g_create_error = x.what();                         \
    return LAYA_ERR_CUDA;                              \
  }                                                    \
  return LAYA_OK;

inline size_t dtype_size(int dtype) {
  switch (dtype) {
    case LAYA_DTYPE_F32: return 4;
    case LAYA_DTYPE_F16:
    case LAYA_DTYPE_BF16: return 2;
    default: fail(LAYA_ERR_INVALID, "dtype %d is not F32, F16 or BF16", dtype);
  }
}

// Calls f with a null pointer of the element type that `dtype` names.
template <typename F>
void with_type(int dtype, F f) {
  switch (dtype) {
    case LAYA_DTYPE_F32: return f((float*)nullptr);
    case LAYA_DTYPE_F16: return f((__half*)nullptr);
    case LAYA_DTYPE_BF16: return f((__nv_bfloat16*)nullptr);
    default: fail(LAYA_ERR_INVALID, "dtype %d is not F32, F16 or BF16", dtype);
  }
}

// The current device, checked to be `stream`'s.  A stream under capture cannot be asked.
inline int current_device(cudaStream_t stream) {
  int dev = 0;
  CK(cudaGetDevice(&dev));
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (stream) CK(cudaStreamIsCapturing(stream, &capture));
  if (stream && capture == cudaStreamCaptureStatusNone) {
    int of = -1;
    CK(cudaStreamGetDevice(stream, &of));
    if (of != dev) fail(LAYA_ERR_INVALID, "stream belongs to device %d, the current device is %d", of, dev);
  }
  return dev;
}

// Raises the kernel's dynamic shared memory limit once per device (`done`: one bit per device).
template <typename K>
void allow_smem(K kern, int bytes, int dev, std::atomic<uint64_t>& done) {
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return;
  CK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done.fetch_or(bit, std::memory_order_relaxed);
}

}  // namespace laya
