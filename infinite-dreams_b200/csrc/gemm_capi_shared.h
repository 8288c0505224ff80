// Host-side helpers of gemm_capi.cu that the other C ABI sources share.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

namespace idb {

// Records the message gemm_last_error() returns and passes the status on.
int capi_fail(int status, const std::string& msg);
int capi_fail_cuda(cudaError_t e, const char* what);
void capi_clear_error();

// The current device: its SM count and the address of its error word.
// Fails on a device that is not sm_100.
int capi_device(int* sms, int** err_word);

// Tensor map of a 16-bit tensor: `rank` (2 to 4) extents, innermost first;
// strides[i] is the element stride of dimension i + 1.
int capi_encode(CUtensorMap* map, const void* base, int rank, const int64_t* extents, const int64_t* strides,
                const int* box, bool swizzled, const char* what);

}  // namespace idb
