// What the files of the C boundary share: the error message of the calling thread.
#pragma once

#include "../../include/chitu_b200.h"

#include <cuda_runtime.h>

namespace chitu {

// Store the message and return `code`.
int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);

}  // namespace chitu
