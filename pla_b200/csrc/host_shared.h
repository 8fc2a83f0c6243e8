// What the library's translation units share on the host side.
#pragma once

#include <cuda_runtime.h>

namespace pla {

// Records a CUDA error as the thread's last one (pla_last_cuda_error) and
// gives PLA_ERR_CUDA.  Defined in pla_capi.cu.
int record_cuda_error(cudaError_t e, const char* where);
// PLA_OK and the number of SMs if the current device is one the library runs on.
int current_sm100(int* sms);

// Reads (out != nullptr) or clears the sequence kernels' fault word.  Defined in pla_sequence.cu.
cudaError_t sequence_faults(unsigned int* out, bool clear);

}  // namespace pla
