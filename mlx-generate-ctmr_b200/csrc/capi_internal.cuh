// What the files of the extern "C" boundary share (defined in capi.cu).
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

namespace ctmr {

// Record the reason of a failed call for ctmr_last_error and return its status.
int api_fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

// cuTensorMapEncodeTiled, or null where the driver does not offer it.
PFN_cuTensorMapEncodeTiled_v12000 api_tensor_map_encoder();

}  // namespace ctmr
