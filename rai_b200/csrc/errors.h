// Error reporting shared by the translation units behind the C ABI.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

namespace rai {

// Records the calling thread's last error (rai_gpu_last_error) and returns code.
int set_error(int code, const std::string& msg);
// The current device's status word of the kernel-level calls
// (rai_gpu_kernel_status).
int kernel_status_word(uint32_t** out);

}  // namespace rai
