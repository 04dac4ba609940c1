// The calling thread's last error message (pesti_last_error), shared by the
// library's translation units.
#pragma once
#include <cuda_runtime.h>

// Stores the message and returns `code`.  Both are defined beside pesti_last_error.
__attribute__((visibility("hidden"))) int pesti_set_error(int code, const char* msg);
__attribute__((visibility("hidden"))) int pesti_set_cuda_error(cudaError_t e, const char* what);
