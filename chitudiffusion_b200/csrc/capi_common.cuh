// What the files of the C boundary share: the error message of the calling thread, the driver's tensor-map encoder.
#pragma once

#include "../../include/chitu_b200.h"

#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

namespace chitu {

// Store the message and return `code`.
int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);
// nullptr where the driver has none
PFN_cuTensorMapEncodeTiled_v12000 get_encode_fn();

}  // namespace chitu
