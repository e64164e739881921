// What operators.cu takes from the library's core (glypr_cuda.cu).
#pragma once
#include <cuda.h>

#include <string>

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
}  // namespace glp
