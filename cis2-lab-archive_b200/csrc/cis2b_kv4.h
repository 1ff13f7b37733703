// cis2b_kv4.h -- host helpers that the entry points of the 4-bit key/value
// cache share.
#pragma once

#include "../../include/cis2b.h"
#include "cis2b_kernels.h"

#include <cuda_runtime.h>

#include <atomic>

namespace cis2b {

int kv4_fail(int code, const char *msg) noexcept;                     // sets cis2b_last_error(), returns code
int kv4_cuda(cudaError_t e) noexcept;                                 // CIS2B_OK or CIS2B_ERR_CUDA
int kv4_check_cache(const cis2b_kv4_cache *c, bool pool) noexcept;    // argument checks of a cache
int kv4_sm_count(int device, int *sms) noexcept;
int kv4_page_shift(int page_size) noexcept;                            // its logarithm, -1 if no page has that size

}  // namespace cis2b
