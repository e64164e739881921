// What the translation units of the standalone operators share: the core's services (glypr_cuda.cu),
// error reporting, argument helpers.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <exception>
#include <string>

#include "glypr_cuda.h"

namespace glp {
// the calling thread's glp_last_error() message
void set_last_error(const std::string& msg);
// device address of the kernel-level status word that glp_kernel_status reads (current device dev)
int kernel_status_word(int dev, int** out);
// the driver's cuTensorMapEncodeTiled, or NULL
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn tensor_map_encoder();

namespace op {

inline int fail(int code, const char* msg) {
  set_last_error(msg);
  return code;
}

inline int launched(cudaError_t e) {
  if (e == cudaSuccess) return GLP_OK;
  cudaGetLastError();  // reported here and not once more by the next call that asks for it
  set_last_error(std::string("kernel launch: ") + cudaGetErrorString(e));
  return e == cudaErrorMemoryAllocation ? GLP_ERR_OOM : GLP_ERR_CUDA;
}

// One launch, as a programmatic dependent launch: the kernel may start while the one before it in the
// stream still runs, and waits for that one's end (griddep_wait) before it touches global memory.
template <class... Params, class... Args>
int launch(void (*kernel)(Params...), unsigned grid, unsigned block, size_t smem, int cluster, cudaStream_t st,
           const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return launched(cudaLaunchKernelEx(&cfg, kernel, args...));
}

inline int dtype_size(int dtype) {
  return dtype == GLP_DTYPE_F32 ? 4 : (dtype == GLP_DTYPE_F16 || dtype == GLP_DTYPE_BF16) ? 2 : 1;
}
inline bool wide_dtype(int dtype) { return dtype == GLP_DTYPE_F32 || dtype == GLP_DTYPE_F16 || dtype == GLP_DTYPE_BF16; }
inline bool code_dtype(int dtype) { return dtype == GLP_DTYPE_I8 || dtype == GLP_DTYPE_E4M3; }
inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// a row pitch in elements: 0 = packed; false when shorter than the row
inline bool pitch(int64_t* ld, int64_t cols) {
  if (*ld == 0) *ld = cols;
  return *ld >= cols;
}

// no C++ exception leaves a C entry (an error message is the only allocation)
template <class F>
int guarded(F&& f) {
  try {
    return f();
  } catch (const std::exception&) {
    return GLP_ERR_OOM;
  }
}

}  // namespace op
}  // namespace glp
