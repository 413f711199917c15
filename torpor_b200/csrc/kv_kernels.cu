// Key/value cache kernels: append with rotation, and the general attention kernel.
//
// Both read the batch's tables on the device and never follow them out of bounds: a page number
// outside the cache, a length beyond the table or rows out of order are recorded in g_kv_status
// and the access is left out.

#include "kv_kernels.hpp"
#include "kv_device.cuh"

namespace tsw {

__device__ uint32_t g_kv_status;

cudaError_t kv_status_symbol(uint32_t** word) { return cudaGetSymbolAddress((void**)word, g_kv_status); }

namespace {

// ---------------------------------------------------------------------------------------------
// Append.
//
// A row is one head of one token of q, k or v.  It is cut into units of VEC pairs: two vectors of VEC
// elements whose elements i form a rotation pair (half style: half a rotary width apart;
// interleaved: the two vectors are neighbours and the pairs lie inside them).  Elements that are not
// rotated, and values, are cut the same way and copied.  A unit reads its two vectors and
// writes the same two places, so q_out may be q.
//
// Every byte is read once and written once, so the bound is HBM for many tokens and latency for few.
// The chain a CTA waits for is: its token's sequence (cu_q), the length, the page entry; the loads
// of q, k and v do not depend on it and are issued first.  One token: 5 us on the device.
constexpr int kAppendThreads = 256;
constexpr int kAppendUnroll = 3;
constexpr uint64_t kFarBytes = 64ull << 20;      // half of the L2

template <typename V> struct Two { V a, b; };

// Inputs are read once.  What is written is read next by the attention, so it stays in the L2 unless the call writes
// more than that holds (`far`): then it only drives out what is still to be read.  16384 tokens of 96 heads of
// 128: 165 us without the hints, 137 to 146 with them (144 to 146 in most calls), 123 at the copy rate.
template <typename V> __device__ __forceinline__ V load_once(uint64_t p) {
    V x;
    if constexpr (sizeof(V) == 16) *(uint4*)&x = __ldcs((const uint4*)p);
    else x = *(const V*)p;
    return x;
}
template <typename V> __device__ __forceinline__ void store(uint64_t p, const V& x, bool far) {
    if constexpr (sizeof(V) == 16) {
        if (far) __stcs((uint4*)p, *(const uint4*)&x);
        else *(uint4*)p = *(const uint4*)&x;
    } else *(V*)p = x;
}

template <typename T, int VEC> struct alignas(VEC * sizeof(T)) Vec { T e[VEC]; };

template <typename T, int VEC>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const __grid_constant__ tsw_kv_append_args a,
                                                                   uint32_t rows_per_cta, bool far) {
    extern __shared__ float2 s_turn[];            // cos, sin of the token's position for each pair
    __shared__ int s_found[3];                    // own token number, page, place; page < 0: nothing is cached
    const uint32_t tok = blockIdx.x;
    const uint32_t units = a.head_dim / (2 * VEC);             // per row
    const uint32_t rot_units = a.rotary_dim / (2 * VEC);
    const uint32_t q_rows = a.q ? a.q_heads : 0;
    const uint32_t rows = q_rows + 2 * a.kv_heads;
    const uint32_t row0 = blockIdx.y * rows_per_cta;
    const uint32_t n = (min(rows, row0 + rows_per_cta) - row0) * units;
    const uint32_t half = a.rotary_dim / 2, rest_half = (a.head_dim - a.rotary_dim) / 2;
    using V = Vec<T, VEC>;

    // Row, offsets of the two vectors and first pair (-1: copied) of unit i.
    struct Unit { uint32_t head, oa, ob; int pair, kind; };        // kind: 0 query, 1 key, 2 value
    auto cut = [&](uint32_t i) {
        const uint32_t row = row0 + i / units, u = i % units;
        Unit c;
        c.kind = row < q_rows ? 0 : row < q_rows + a.kv_heads ? 1 : 2;
        c.head = c.kind == 0 ? row : c.kind == 1 ? row - q_rows : row - q_rows - a.kv_heads;
        if (c.kind == 2) { c.oa = u * VEC; c.ob = a.head_dim / 2 + u * VEC; c.pair = -1; }
        else if (u >= rot_units) {
            c.oa = a.rotary_dim + (u - rot_units) * VEC;
            c.ob = c.oa + rest_half;
            c.pair = -1;
        } else if (a.interleaved) { c.oa = 2 * u * VEC; c.ob = c.oa + VEC; c.pair = u * VEC; }
        else { c.oa = u * VEC; c.ob = c.oa + half; c.pair = u * VEC; }
        return c;
    };
    auto load = [&](const Unit& c, Two<V>& x) {
        const uint64_t base = c.kind == 0 ? a.q + tok * a.q_token_stride + c.head * a.q_head_stride
                              : c.kind == 1 ? a.k + tok * a.k_token_stride + c.head * a.k_head_stride
                                            : a.v + tok * a.v_token_stride + c.head * a.v_head_stride;
        x.a = load_once<V>(base + c.oa * sizeof(T));
        x.b = load_once<V>(base + c.ob * sizeof(T));
    };
    auto finish = [&](const Unit& c, Two<V>& x) {
        uint64_t base;
        if (c.kind == 0) base = a.q_out + tok * a.q_out_token_stride + c.head * a.q_out_head_stride;
        else if (s_found[1] < 0) return;
        else if (c.kind == 1) base = a.cache.k + (uint64_t)s_found[1] * a.cache.k_page_stride +
                                     (uint64_t)s_found[2] * a.cache.k_token_stride + c.head * a.cache.k_head_stride;
        else base = a.cache.v + (uint64_t)s_found[1] * a.cache.v_page_stride +
                    (uint64_t)s_found[2] * a.cache.v_token_stride + c.head * a.cache.v_head_stride;
        if (c.pair >= 0) {
            if (a.interleaved) {
                if constexpr (VEC == 1) {
                    const float2 t = s_turn[c.pair];
                    const float f = to_float(x.a.e[0]), g = to_float(x.b.e[0]);
                    x.a.e[0] = from_float<T>(f * t.x - g * t.y);
                    x.b.e[0] = from_float<T>(f * t.y + g * t.x);
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; i += 2) {
                        const float2 t = s_turn[c.pair + i / 2], w = s_turn[c.pair + (VEC + i) / 2];
                        const float f = to_float(x.a.e[i]), g = to_float(x.a.e[i + 1]);
                        const float f2 = to_float(x.b.e[i]), g2 = to_float(x.b.e[i + 1]);
                        x.a.e[i] = from_float<T>(f * t.x - g * t.y);
                        x.a.e[i + 1] = from_float<T>(f * t.y + g * t.x);
                        x.b.e[i] = from_float<T>(f2 * w.x - g2 * w.y);
                        x.b.e[i + 1] = from_float<T>(f2 * w.y + g2 * w.x);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float2 t = s_turn[c.pair + i];
                    const float f = to_float(x.a.e[i]), g = to_float(x.b.e[i]);
                    x.a.e[i] = from_float<T>(f * t.x - g * t.y);
                    x.b.e[i] = from_float<T>(f * t.y + g * t.x);
                }
            }
        }
        store(base + c.oa * sizeof(T), x.a, far);
        store(base + c.ob * sizeof(T), x.b, far);
    };

    Two<V> x[kAppendUnroll];
#pragma unroll
    for (int u = 0; u < kAppendUnroll; ++u) {
        const uint32_t i = threadIdx.x + u * kAppendThreads;
        if (i < n) load(cut(i), x[u]);
    }
    // The token's sequence: one warp narrows the range 32-fold a step.
    if (threadIdx.x < 32) {
        const int b = find_sequence((const int*)a.batch.cu_q, a.batch.batch, tok);
        if (threadIdx.x == 0) {
            int j = -1, page = -1, at = 0;
            if (b >= 0) {
                SeqRows r;
                const uint32_t wrong = read_rows(a.batch, b, a.batch.tokens, a.cache.page_size, r);
                if (wrong) atomicOr(&g_kv_status, wrong);
                // a length that had to be changed says nothing about where a row goes: another token lies there
                j = (int)tok < r.first + r.n && !(wrong & TSW_KV_BAD_LENGTH) ? r.len - r.n + ((int)tok - r.first) : -1;
                if (j >= 0) {
                    page = ((const int*)a.batch.page_table)[(uint64_t)b * a.batch.table_stride + j / (int)a.cache.page_size];
                    at = j % (int)a.cache.page_size;
                    if ((uint32_t)page >= a.cache.pages) { atomicOr(&g_kv_status, TSW_KV_BAD_PAGE); page = -1; }
                }
            }
            s_found[0] = j; s_found[1] = page; s_found[2] = at;
        }
    }
    __syncthreads();
    const int own = s_found[0];
    if (own < 0) return;                           // nobody's row, or one that the length does not cover
    // Angles: position times frequency in 64 bits, taken to turns and reduced there, so that far positions
    // lose nothing; the sine and cosine of what remains are formed in 32 bits.
    for (uint32_t c = threadIdx.x; c < half; c += kAppendThreads) {
        double turns = (double)(a.position_offset + (uint64_t)own) * ((const double*)a.inv_freq)[c] * 0.15915494309189533577;
        turns -= rint(turns);
        float s, co;
        sincospif((float)(2.0 * turns), &s, &co);
        s_turn[c] = make_float2(co, s);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kAppendUnroll; ++u) {
        const uint32_t i = threadIdx.x + u * kAppendThreads;
        if (i < n) finish(cut(i), x[u]);
    }
    for (uint32_t i = threadIdx.x + kAppendUnroll * kAppendThreads; i < n; i += kAppendThreads) {
        const Unit c = cut(i);
        load(c, x[0]);
        finish(c, x[0]);
    }
}

// ---------------------------------------------------------------------------------------------
// The general attention kernel: any head width up to 512, any stride or page size, any scale: what the tile kernel
// does not take (kv_dealing.hpp says what that is: 16-byte alignment, heads of at most 128, pages of a
// power of two).  One warp holds one row (a token and a query head) and walks its keys 32 at a time: lane i forms
// the product with key i, then the warp takes maximum and sum over the 32 and each lane adds up its share of the
// output elements.  Bound by the L1: every row reads all its keys itself.  32 sequences behind 2048 tokens: 2250 us,
// against 71 us of the tile kernel; with heads of 256, 3500 us.
constexpr int kRowWarps = 4;
constexpr int kRowMaxDim = 512;
constexpr int kRowFold = 1024;

template <typename T>
__global__ void __launch_bounds__(32 * kRowWarps) attention_rows_kernel(const __grid_constant__ tsw_prefix_attention_args a) {
    __shared__ float s_q[kRowWarps][kRowMaxDim];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t row = (uint64_t)blockIdx.x * kRowWarps + warp;
    if (row >= (uint64_t)a.batch.tokens * a.q_heads) return;
    const uint32_t tok = (uint32_t)(row / a.q_heads), head = (uint32_t)(row % a.q_heads);
    const uint32_t kvh = head / (a.q_heads / a.kv_heads), dim = a.head_dim;
    const int b = find_sequence((const int*)a.batch.cu_q, a.batch.batch, tok);
    if (b < 0) return;
    SeqRows r;
    const uint32_t wrong = read_rows(a.batch, b, a.max_q, a.cache.page_size, r);
    if (wrong) atomicOr(&g_kv_status, wrong);
    if ((int)tok >= r.first + r.n) return;
    const int own_end = a.causal ? max(0, r.len - r.n + ((int)tok - r.first) + 1) : r.len;

    const T* q = (const T*)(a.q + tok * a.q_token_stride + head * a.q_head_stride);
    for (uint32_t d = lane; d < dim; d += 32) s_q[warp][d] = to_float(q[d]);
    __syncwarp();
    float acc[kRowMaxDim / 32];
#pragma unroll
    for (int i = 0; i < kRowMaxDim / 32; ++i) acc[i] = 0.f;
    // A sum of 2^24 equal weights takes up no more of them in 32 bits.  So the sums go over kRowFold rounds at a time, and those over
    // the rest of the keys: 2^15 additions and 2^16.
    float all[kRowMaxDim / 32], all_total = 0.f;
#pragma unroll
    for (int i = 0; i < kRowMaxDim / 32; ++i) all[i] = 0.f;
    int rounds = 0;
    float top = -INFINITY, total = 0.f;
    for (int part = 0; part < 2; ++part) {
        const tsw_kv_pages& pg = part ? a.cache : a.prefix;
        const int* table = part ? (const int*)a.batch.page_table + (uint64_t)b * a.batch.table_stride : (const int*)a.prefix_table;
        const int end = part ? own_end : (int)a.prefix_len;
        for (int k0 = 0; k0 < end; k0 += 32) {
            const int key = k0 + lane;
            int page = -1;
            uint32_t at = 0;
            if (key < end) {
                page = table[key / (int)pg.page_size];
                at = key % (int)pg.page_size;
                if ((uint32_t)page >= pg.pages) { atomicOr(&g_kv_status, TSW_KV_BAD_PAGE); page = -1; }
            }
            float s = -INFINITY;
            if (page >= 0) {
                const T* k = (const T*)(pg.k + (uint64_t)page * pg.k_page_stride + (uint64_t)at * pg.k_token_stride + kvh * pg.k_head_stride);
                s = 0.f;
                for (uint32_t d = 0; d < dim; ++d) s = fmaf(s_q[warp][d], to_float(k[d]), s);
                s *= a.scale;
            }
            const float new_top = fmaxf(top, warp_max(s));
            const float base = new_top == -INFINITY ? 0.f : new_top;
            const float keep = expf(top - base);
            const float e = expf(s - base);
            total = total * keep + warp_sum(e);
            all_total *= keep;
            top = new_top;
#pragma unroll
            for (int i = 0; i < kRowMaxDim / 32; ++i) {
                acc[i] *= keep;
                all[i] *= keep;
            }
            if (++rounds == kRowFold) {
                rounds = 0;
                all_total += total;
                total = 0.f;
#pragma unroll
                for (int i = 0; i < kRowMaxDim / 32; ++i) {
                    all[i] += acc[i];
                    acc[i] = 0.f;
                }
            }
            const int m = min(32, end - k0);
            for (int i = 0; i < m; ++i) {
                const float w = __shfl_sync(~0u, e, i);
                const int pi = __shfl_sync(~0u, page, i);
                const uint32_t ai = __shfl_sync(~0u, at, i);
                if (pi < 0) continue;
                const T* v = (const T*)(pg.v + (uint64_t)pi * pg.v_page_stride + (uint64_t)ai * pg.v_token_stride + kvh * pg.v_head_stride);
#pragma unroll
                for (int d = 0; d < kRowMaxDim / 32; ++d)
                    if (lane + 32 * d < dim) acc[d] = fmaf(w, to_float(v[lane + 32 * d]), acc[d]);
            }
        }
    }
    total += all_total;
    const float inv = total > 0.f ? 1.f / total : total == 0.f ? 0.f : total;   // a row that saw nothing: zeros; NaN stays
    T* out = (T*)(a.out + tok * a.out_token_stride + head * a.out_head_stride);
#pragma unroll
    for (int i = 0; i < kRowMaxDim / 32; ++i)
        if (lane + 32 * i < dim) out[lane + 32 * i] = from_float<T>((acc[i] + all[i]) * inv);
    if (a.lse && lane == 0) ((float*)a.lse)[row] = total == 0.f ? -INFINITY : top + logf(total);
}

__global__ void status_clear_kernel(uint32_t* word, uint32_t bits) { atomicAnd(word, ~bits); }

// Launch with an error of its own: the runtime's last error may be another call's.
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T, int VEC>
cudaError_t launch_append(const tsw_kv_append_args& a, dim3 grid, uint32_t rows_per_cta, bool far, cudaStream_t stream) {
    return launch(kv_append_kernel<T, VEC>, grid, kAppendThreads, sizeof(float2) * (a.rotary_dim / 2), stream, a, rows_per_cta, far);
}

template <typename T>
cudaError_t launch_append_vec(const tsw_kv_append_args& a, int vec, dim3 grid, uint32_t rows_per_cta, bool far, cudaStream_t stream) {
    switch (vec) {
        case 8: return launch_append<T, 8>(a, grid, rows_per_cta, far, stream);
        case 4: return launch_append<T, 4>(a, grid, rows_per_cta, far, stream);
        case 2: return launch_append<T, 2>(a, grid, rows_per_cta, far, stream);
        default: return launch_append<T, 1>(a, grid, rows_per_cta, far, stream);
    }
}

}  // namespace

cudaError_t launch_kv_status_clear(uint32_t* word, uint32_t bits, cudaStream_t stream) {
    return launch(status_clear_kernel, 1, 1, 0, stream, word, bits);
}

cudaError_t launch_kv_append(const tsw_kv_append_args& a, int device_sms, cudaStream_t stream) {
    // The widest vector that every address, stride and pair distance is a multiple of.
    uint64_t bits = a.k | a.v | a.k_token_stride | a.k_head_stride | a.v_token_stride | a.v_head_stride | a.cache.k | a.cache.v |
                    a.cache.k_page_stride | a.cache.k_token_stride | a.cache.k_head_stride | a.cache.v_page_stride |
                    a.cache.v_token_stride | a.cache.v_head_stride;
    if (a.q) bits |= a.q | a.q_out | a.q_token_stride | a.q_head_stride | a.q_out_token_stride | a.q_out_head_stride;
    bits |= (uint64_t)(a.rotary_dim / 2 | (a.head_dim - a.rotary_dim) / 2 | a.head_dim / 2) * 2;   // elements -> bytes
    int vec = 8;
    while (vec > 1 && (bits & (uint64_t)(2 * vec - 1))) vec >>= 1;
    // A CTA takes some rows of one token.  All rows of a token in one CTA is best for many tokens (its angles
    // are formed once); few tokens are spread over more CTAs, down to 8 rows each.
    const uint32_t rows = (a.q ? a.q_heads : 0) + 2 * a.kv_heads;
    const uint32_t groups = std::max(1u, std::min((rows + 7) / 8, (uint32_t)(2 * device_sms) / std::max(1u, a.batch.tokens)));
    const uint32_t rows_per_cta = (rows + groups - 1) / groups;
    const dim3 grid(a.batch.tokens, (rows + rows_per_cta - 1) / rows_per_cta);
    const bool far = 2ull * rows * a.batch.tokens * a.head_dim > kFarBytes;
    return a.dtype == TSW_F16 ? launch_append_vec<__half>(a, vec, grid, rows_per_cta, far, stream)
                              : launch_append_vec<__nv_bfloat16>(a, vec, grid, rows_per_cta, far, stream);
}

cudaError_t launch_prefix_attention_rows(const tsw_prefix_attention_args& a, cudaStream_t stream) {
    const uint64_t rows = (uint64_t)a.batch.tokens * a.q_heads;
    const unsigned grid = (unsigned)((rows + kRowWarps - 1) / kRowWarps);
    return a.dtype == TSW_F16 ? launch(attention_rows_kernel<__half>, grid, 32 * kRowWarps, 0, stream, a)
                              : launch(attention_rows_kernel<__nv_bfloat16>, grid, 32 * kRowWarps, 0, stream, a);
}

}  // namespace tsw
