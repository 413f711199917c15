// Device helpers that the key/value cache kernels share.
#ifndef TORPOR_KV_DEVICE_CUH_
#define TORPOR_KV_DEVICE_CUH_

#include <algorithm>
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/torpor_swap.h"

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

// Rows and length of one sequence, made safe: whatever the tables hold, 0 <= first, first + n <= tokens,
// n <= max_q and 0 <= len <= what the page table covers.  What had to be changed is recorded.
struct SeqRows { int first, n, len; };
__device__ __forceinline__ void read_rows(const tsw_kv_batch& t, int b, uint32_t max_q, uint32_t page_size, uint32_t* status, SeqRows& r) {
    const int* cu = (const int*)t.cu_q;
    const int lo = cu[b], hi = cu[b + 1];
    int len = ((const int*)t.seq_lens)[b];
    uint32_t bad = 0;
    r.first = lo;
    r.n = hi - lo;
    if (lo < 0 || hi < lo || hi > (int)t.tokens || (uint32_t)(hi - lo) > max_q) { bad |= TSW_KV_BAD_ROWS; r.first = 0; r.n = 0; }
    const uint64_t room = t.page_table ? (uint64_t)t.table_width * page_size : 0;
    if (len < 0) { bad |= TSW_KV_BAD_LENGTH; len = 0; }
    if ((uint64_t)len > room) { bad |= TSW_KV_BAD_LENGTH; len = (int)room; }
    r.len = len;
    if (bad) atomicOr(status, bad);
}

}  // namespace tsw
#endif
