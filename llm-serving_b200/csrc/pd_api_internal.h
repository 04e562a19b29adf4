// pd_api_internal.h -- what the entry-point files share: error text, the launch count, the current
// device (defined in pd_api.cu).
#pragma once

#include <cuda_runtime.h>

namespace pd {

// Records a failed CUDA call for pd_last_error_string and returns PD_ERR_CUDA.
int api_cuda_fail(cudaError_t e, const char* where);
// Records a text for pd_last_error_string and returns `status`.
int api_message(int status, const char* text);
void api_count_launch();
unsigned long long api_wait_limit_ns();
// The current device's multiprocessor count and error word; PD_ERR_CUDA without a device.
int api_device(int* sms, unsigned** err);

}  // namespace pd
