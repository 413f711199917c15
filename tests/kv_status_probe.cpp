// tsw_kv_status between reports from elsewhere, without a GPU: the runtime calls it makes are replaced here, and another stream's
// kernel reports something in front of each of them.  Nothing that is reported may be lost: it is in an answer, or
// still in the word.  Linked with the library's host sources (tests/test_kv_guards.py).
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include <cuda_runtime.h>

#include "../include/torpor_swap.h"
#include "../torpor_b200/csrc/kernels.hpp"
#include "../torpor_b200/csrc/kv_attention.hpp"
#include "../torpor_b200/csrc/kv_kernels.hpp"

static uint32_t g_word, g_made, g_reports[8];
static int g_calls;
static void meanwhile() {
    const uint32_t bits = g_calls < 8 ? g_reports[g_calls] : 0;
    ++g_calls;
    g_word |= bits;
    g_made |= bits;
}

namespace tsw {
cudaError_t launch_place(const PlaceArgs&, int, cudaStream_t, int) { return cudaErrorNotSupported; }
cudaError_t launch_publish_rows(const PlaceArgs&, uint32_t, uint32_t, cudaStream_t) { return cudaErrorNotSupported; }
cudaError_t launch_checksum(const SumDesc*, uint32_t, uint32_t, uint32_t, unsigned long long*, int, cudaStream_t) { return cudaErrorNotSupported; }
int default_grid_ctas(int) { return 1; }
int default_grid_ctas_host(int) { return 1; }
cudaError_t launch_kv_append(const tsw_kv_append_args&, int, cudaStream_t) { return cudaErrorNotSupported; }
cudaError_t launch_prefix_attention_rows(const tsw_prefix_attention_args&, cudaStream_t) { return cudaErrorNotSupported; }
cudaError_t launch_prefix_attention_tiles(int, const tsw_prefix_attention_args&, const AttentionLayout&, uint32_t*, cudaStream_t) { return cudaErrorNotSupported; }
cudaError_t kv_status_symbol(uint32_t** word) {
    *word = &g_word;
    return cudaSuccess;
}
cudaError_t launch_kv_status_clear(uint32_t* word, uint32_t bits, cudaStream_t) {
    meanwhile();
    *word &= ~bits;
    return cudaSuccess;
}
}  // namespace tsw
extern "C" {
int tsw_place_segments_static(int, const tsw_segment*, int, uint32_t, uint32_t, uint32_t, const tsw_publish*, void*) { return TSW_ERR_NO_DEVICE; }
cudaError_t cudaGetDevice(int* d) { return *d = 0, cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int) { return *v = 148, cudaSuccess; }
cudaError_t cudaMemcpyAsync(void* dst, const void* src, size_t n, cudaMemcpyKind, cudaStream_t) {
    meanwhile();
    memcpy(dst, src, n);
    return cudaSuccess;
}
cudaError_t cudaMemsetAsync(void* p, int v, size_t n, cudaStream_t) {
    meanwhile();
    memset(p, v, n);
    return cudaSuccess;
}
cudaError_t cudaStreamSynchronize(cudaStream_t) {
    meanwhile();
    return cudaSuccess;
}
}

int main() {
    int n = 0;
    for (int seed = 0; seed < 4096; ++seed, ++n)
        for (int clear = 0; clear < 2; ++clear) {
            g_word = g_made = seed & 1 ? TSW_KV_BAD_PAGE : 0;
            g_calls = 0;
            for (int i = 0; i < 8; ++i) g_reports[i] = i < 4 ? seed >> (1 + 2 * i) & 3u << 1 : 0;      // lengths and rows
            uint32_t got = 0;
            if (tsw_kv_status(0, nullptr, &got, clear) != TSW_OK) return printf("refused: %s\n", tsw_last_error()), 1;
            if ((got | g_word) != g_made) return printf("seed %d: %u made, %u told, %u left\n", seed, g_made, got, g_word), 1;
            if (!clear && g_word != g_made) return printf("seed %d: cleared without being asked\n", seed), 1;
            if (clear && (got & g_word & TSW_KV_BAD_PAGE)) return printf("seed %d: told and not cleared\n", seed), 1;
        }
    printf("ok %d\n", n);
    return 0;
}
