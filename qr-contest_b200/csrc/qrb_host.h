// qrb200 -- host-side bookkeeping shared by the library's translation units (qrb_api.cu owns it).
#pragma once
#include <cuda_runtime.h>

namespace qrb {

// Adds to the count qrb200_launch_count reports.
void count_launches(int n);

// Remembers a failed runtime call for qrb200_last_cuda_error; returns its argument.
cudaError_t note(cudaError_t e);

// The current device (below 128) and the identity of its context, made current when there is none:
// what is kept per device is kept for a context, and goes with it in cudaDeviceReset.
cudaError_t current_ctx(int* dev_out, unsigned long long* id_out);

}  // namespace qrb
