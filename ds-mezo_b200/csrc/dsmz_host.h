// Host helpers shared by the library's translation units (defined in dsmz_api.cu): the
// calling thread's error message and the driver's tensor-map encoder.
#pragma once

#include <cuda_runtime.h>
#include <cudaTypedefs.h>
#include <string>

namespace dsmz {

// Keep `msg` as the calling thread's dsmz_last_error() and return `code`.
int fail(int code, const std::string& msg);
int cuda_fail(const char* what, cudaError_t e);
// cuTensorMapEncodeTiled from the driver, looked up once per process (NULL: no driver).
PFN_cuTensorMapEncodeTiled_v12000 encode_fn();

}  // namespace dsmz

#define DSMZ_LAUNCHED(what)                                  \
  do {                                                        \
    cudaError_t e_ = cudaGetLastError();                      \
    if (e_ != cudaSuccess) return cuda_fail((what), e_);      \
  } while (0)
