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

// The sequence whose rows contain `tok`, or -1: the last b with cu_q[b] <= tok, if tok < cu_q[b + 1].
// All lanes of a warp call it; each step narrows the range 32-fold.
__device__ __forceinline__ int find_sequence(const int* cu_q, uint32_t batch, uint32_t tok) {
    const int lane = threadIdx.x & 31;
    uint32_t lo = 0, hi = batch + 1;              // entries [0, lo) are <= tok (lo >= 1 once any is), [hi, ..) are > tok
#pragma unroll 1
    while (lo < hi) {
        const uint32_t span = hi - lo, step = (span + 31) / 32;
        const uint32_t at = lo + lane * step;     // first entry of this lane's piece
        const bool below = at < hi && cu_q[at] <= (int)tok;
        const unsigned votes = __ballot_sync(~0u, below);
        const int k = __popc(votes);              // pieces whose first entry is <= tok: a prefix when cu_q does not decrease
        if (k == 0) break;
        const uint32_t next_lo = lo + (k - 1) * step + 1;
        hi = min(hi, lo + k * step);
        lo = next_lo;
    }
    const int b = (int)lo - 1;
    if (b < 0 || b >= (int)batch) return -1;
    return b;
}

}  // namespace tsw
#endif
