// Device helpers that the key/value cache kernels share.
#ifndef TORPOR_KV_DEVICE_CUH_
#define TORPOR_KV_DEVICE_CUH_

#include <algorithm>
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "kv_dealing.hpp"

namespace tsw {

__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, o));
    return x;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    return x;
}

// The sequence whose rows contain `tok`, or -1 (kv_dealing.hpp).  All lanes of a warp call it.
__device__ __forceinline__ int find_sequence(const int* cu_q, uint32_t batch, uint32_t tok) {
    Search s(batch);
#pragma unroll 1
    while (s.open()) s.take(__ballot_sync(~0u, s.vote(cu_q, (int)tok, threadIdx.x & 31)));
    return s.sequence(batch);
}

}  // namespace tsw
#endif
