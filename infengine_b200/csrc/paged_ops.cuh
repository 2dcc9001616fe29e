// Internal interface of the paged-cache kernels and the sampler.
#pragma once

namespace ie {

// Device status words: IE_ERR_INVALID_ARG for a token whose position, page or
// rotation row lies outside what the call was given, IE_ERR_TIMEOUT when a
// bounded wait for a copy or an MMA gave up.
int read_paged_norm_status(bool clear);
int read_paged_attn_status(bool clear);
int read_paged_tc_status(bool clear);
// Sets this device's limit of the kernels' bounded waits (current device).
cudaError_t set_paged_attn_wait_ns(unsigned long long ns);
cudaError_t set_paged_tc_wait_ns(unsigned long long ns);

}  // namespace ie
