// Host-side helpers shared by the entry-point files (esa_capi.cu,
// esa_capi_layer.cu): error text, argument checks, dtype dispatch, the
// device error word.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "esa_b200.h"

namespace esa {
namespace host {

// Records the message esa_last_error() returns and returns `code`.
__attribute__((visibility("hidden"))) int fail(int code, const char* fmt, ...);

// ESA_OK, or ESA_ERR_CUDA with the pending launch error of `what`.
__attribute__((visibility("hidden"))) int check_launch(const char* what);

// Base pointer and strides (in bytes) of an attention operand: non-null, 16-byte multiples.
__attribute__((visibility("hidden"))) int check_tensor(const char* name, const esa_tensor_t& t,
                                                       int esize);

// Address of the current device's error word (ESA_DEVERR_* bits).
__attribute__((visibility("hidden"))) int device_error_word(int** out);

inline int elem_size(int dtype) { return dtype == ESA_DTYPE_F32 ? 4 : 2; }

inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Row operands: known dtype, dim * element size a multiple of 16 bytes.
__attribute__((visibility("hidden"))) int check_rows_op(const char* what, int32_t dtype,
                                                        int64_t n_rows, int32_t dim);

// Launches `kernel` so that its CTAs may be placed while the kernel before it
// in the stream still runs (programmatic dependent launch).  The kernel calls
// cudaGridDependencySynchronize() before it touches memory, which waits for
// that kernel's end; what is saved is the launch latency between the two.
template <typename... P, typename... A>
int launch_after(const char* what, void (*kernel)(P...), dim3 grid, dim3 block, cudaStream_t s,
                 A... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = block;
  c.stream = s;
  cudaLaunchAttribute a[1];
  a[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a[0].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = a;
  c.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&c, kernel, P(args)...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(ESA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  }
  return ESA_OK;
}

template <typename F>
int by_dtype(int32_t dtype, F&& f) {
  switch (dtype) {
    case ESA_DTYPE_F32: return f(float{});
    case ESA_DTYPE_BF16: return f(__nv_bfloat16{});
    default: return f(__half{});
  }
}

}  // namespace host
}  // namespace esa
