// Launch interface of the key/value cache kernels (kv_kernels.cu).
#ifndef TORPOR_KV_KERNELS_HPP_
#define TORPOR_KV_KERNELS_HPP_

#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/torpor_swap.h"

namespace tsw {

// Arguments have been checked by the host entry points (kv_cache.cpp); device_sms is the SM count.
cudaError_t launch_kv_append(const tsw_kv_append_args& a, int device_sms, cudaStream_t stream);
cudaError_t launch_prefix_attention_rows(const tsw_prefix_attention_args& a, cudaStream_t stream);
cudaError_t kv_status_symbol(uint32_t** word);   // address on the current device
cudaError_t launch_kv_status_clear(uint32_t* word, uint32_t bits, cudaStream_t stream);

}  // namespace tsw
#endif
