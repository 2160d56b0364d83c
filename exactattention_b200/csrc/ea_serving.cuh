// Shared by the serving-step operators (ea_plan.cu, ea_rope.cu, ea_tree.cu, ea_logits.cu): error
// text, element conversions, unsigned division by a launch constant.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/exactattn_serving.h"

namespace ea {
namespace serving {

// Stores the message for ea_serving_last_error and returns `code`.
int fail(int code, const char* msg);
// 0, or -4 with the CUDA error's text.
int cuda_rc(cudaError_t e);
// wait_debug of ea_set_test_hooks (ea_api.cu).
int wait_debug_hook();
// SMs of the current device (looked up once per device).
int sm_count();

__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(float x) { return x; }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }

// Launches a kernel that may start while the one before it on the stream still runs (programmatic dependent launch), which
// hides the launch's latency. Every block of every kernel here first calls begin(), which waits for all earlier work; only
// the second kernel of a call may read the call's inputs before it.
template <typename... P, typename... A>
cudaError_t launch_early(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  return e == cudaSuccess ? cudaGetLastError() : e;
}
// Waits for all earlier work on the stream, then lets the next kernel start.
__device__ __forceinline__ void begin() {
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
}

// n / d for n < 2^31 by one multiply: with s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1,
// n / d = (umulhi(n, m) + n) >> s (the sum stays below 2^32 for n < 2^31).
struct FastDiv {
  uint32_t d, m, s;
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return {d, (uint32_t)((((1ull << s) - d) << 32) / d + 1), s};
}
__device__ __forceinline__ uint32_t div_by(uint32_t n, FastDiv f) { return (__umulhi(n, f.m) + n) >> f.s; }

}  // namespace serving
}  // namespace ea
