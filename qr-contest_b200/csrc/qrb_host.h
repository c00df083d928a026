// qrb200 -- host-side bookkeeping shared by the library's translation units (qrb_api.cu owns it).
#pragma once
#include <cuda_runtime.h>

namespace qrb {

// Adds to the count qrb200_launch_count reports.
void count_launches(int n);

// Remembers a failed runtime call for qrb200_last_cuda_error; returns its argument.
cudaError_t note(cudaError_t e);

}  // namespace qrb
