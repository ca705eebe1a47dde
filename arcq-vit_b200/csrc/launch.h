// What the translation units of the library share on the host side: error text, device status word, launch options.
// Defined in arcq_b200.cu.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace arcq_host {

#pragma GCC visibility push(hidden)
int fail(int code, const char* text);              // keeps the text for arcq_last_error_string
int cuda_fail(cudaError_t e, const char* what);
int* status_ptr();                                 // the status word on the current device
int sm_count();                                    // of the current device
bool dependent_launches();                         // ARCQ_PDL
uint32_t poll_limit();                             // ARCQ_POLL_LIMIT
int launch_regs();                                 // ARCQ_LAUNCH_REGS
#pragma GCC visibility pop

}  // namespace arcq_host
