// What operators.cu takes from the library's core (glypr_cuda.cu).
#pragma once
#include <string>

namespace glp {
// the calling thread's glp_last_error() message
void set_last_error(const std::string& msg);
// device address of the kernel-level status word that glp_kernel_status reads (current device dev)
int kernel_status_word(int dev, int** out);
}  // namespace glp
