// Attention behind a shared prefix on the fifth-generation tensor cores.
//
// For one key head the rows of a tile are (token, query head of the group) pairs, up to 128 of them, and a step takes 128
// keys: S = Q K^T and O += P V are one tcgen05.mma chain each (M = 128; accumulators in tensor memory,
// P goes back into tensor memory over S and is the A operand of the second product).  One thread holds
// one row of S: maximum, exponentials and sum need no exchange between threads.  The maximum that
// exponentials are taken against moves only when it grows by more than 2^8, so the running
// output is rarely rescaled; the quotient at the end makes the result independent of it.
//
// The work is two lists of (item, key tile) pairs: the prefix with the rows of ALL sequences (this is what makes it
// "computed once for all": a 128-row tile reads each prefix key once for 128 rows), and every sequence's own
// keys with its own rows.  Each list is cut into equal contiguous ranges of tiles, one per stream of
// the grid, wherever the cuts fall: long key axes are split, short ones batched, and no length
// needs to be known on the host.  What a range holds of an item is a partial result (output, maximum,
// sum); combine_kernel joins them.
//
// One CTA per SM runs two streams, a warpgroup of 128 rows each, so that one stream's products and loads
// run under the other's exponentials.  The streams take different items (few rows: bound by HBM), or two row tiles
// of one item that share every key tile ("pair": many rows, where the load of a key tile per 128 rows would bound).

#include "kv_kernels.hpp"
#include "kv_device.cuh"
#include "kv_attention.hpp"
#include "kv_dealing.hpp"

#include <atomic>
#include <cstring>

#include <cuda.h>

namespace tsw {

namespace {

constexpr int kThreads = 384;                 // two warpgroups of rows; warps for K, V, the products, Q
constexpr unsigned long long kWaitNs = 2000000000ull;
constexpr float kGrow = 8.f;                  // log2 of the growth of the maximum that is let pass

template <int DP> struct Shape {
    static constexpr int kTileBytes = kTile * DP * 2;
    static constexpr int kK = DP == 128 ? 2 : 5;      // stages of keys and of values: a value tile waits for its
    static constexpr int kV = DP == 128 ? 3 : 6;      // exponentials, so values get one more
    static constexpr int kSmem = (2 + kK + kV) * kTileBytes + 1024;
};

struct alignas(64) Params {
    CUtensorMap q_prefix, q_own, k_prefix, v_prefix, k_own, v_own;
    tsw_prefix_attention_args a;
    Deal d;
    uint32_t* status;
};

// ------------------------------------------------------------------ small PTX wrappers

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ unsigned long long now() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// Every wait ends: after two seconds, or when another warp of the CTA has given up, it answers false, and the
// caller leaves its loop.
__device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t parity, volatile uint32_t* gave_up) {
    const unsigned long long t0 = now();
    while (!mbar_try(bar, parity)) {
        if (*gave_up) return false;
        if (now() - t0 > kWaitNs) {
            *gave_up = 1;
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile uint32_t* gave_up) {     // a whole warp, one answer
    if (__all_sync(~0u, mbar_try(bar, parity))) return true;
    return __all_sync(~0u, wait_slow(bar, parity, gave_up));
}

__device__ __forceinline__ void load_box4(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar) : "memory");
}
__device__ __forceinline__ void load_box3(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define TSW_R8(r, o) "=r"((r)[o]), "=r"((r)[o + 1]), "=r"((r)[o + 2]), "=r"((r)[o + 3]), "=r"((r)[o + 4]), "=r"((r)[o + 5]), "=r"((r)[o + 6]), "=r"((r)[o + 7])
#define TSW_I8(r, o) "r"((r)[o]), "r"((r)[o + 1]), "r"((r)[o + 2]), "r"((r)[o + 3]), "r"((r)[o + 4]), "r"((r)[o + 5]), "r"((r)[o + 6]), "r"((r)[o + 7])
__device__ __forceinline__ void tmem_ld32(uint32_t* r, uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
                 "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : TSW_R8(r, 0), TSW_R8(r, 8), TSW_R8(r, 16), TSW_R8(r, 24) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
                 "%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(addr), TSW_I8(r, 0), TSW_I8(r, 8), TSW_I8(r, 16), TSW_I8(r, 24) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(addr), TSW_I8(r, 0), TSW_I8(r, 8) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Shared memory descriptors of the products' operands, 128-byte swizzle.  Tiles are [rows][64 elements] halves of 128 x 128
// bytes.  Q and K run along the head (the summed axis) in a row: eight-row groups lie 1024 bytes apart.
// V's summed axis is its rows (keys): groups of eight keys lie 1024 bytes apart, and the next 64 head elements
// a half (16 KB) further.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead_bytes) {
    return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)((lead_bytes >> 4) & 0x3fff) << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

struct Bars {                // mbarriers, byte addresses in shared memory
    uint32_t k_full, k_empty, v_full, v_empty, q_full, q_empty, s_full, p_full, o_full;
};

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1) attention_tiles_kernel(const __grid_constant__ Params p) {
    using S = Shape<DP>;
    constexpr int kHalves = DP / 64;
    constexpr uint32_t kHalfBytes = kTile * 128;
    extern __shared__ uint8_t s_raw[];
    __shared__ __align__(8) uint64_t s_bars[2 * (S::kK + S::kV) + 10];
    __shared__ Prologue s_pro;
    __shared__ uint32_t s_tmem, s_scan[kThreads / 32];
    __shared__ uint32_t s_gave_up;
    volatile uint32_t* gave_up = &s_gave_up;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const tsw_prefix_attention_args& a = p.a;
    const Deal& d = p.d;
    const AttentionLayout& w = d.w;
    const int group = w.group, tile_tokens = w.tile_tokens;
    uint8_t* ws = (uint8_t*)a.workspace;

    const uint32_t tiles = (smem_addr(s_raw) + 1023) & ~1023u;
    const uint32_t q_at = tiles, k_at = q_at + 2 * S::kTileBytes, v_at = k_at + S::kK * S::kTileBytes;
    Bars bar;
    {
        const uint32_t b = smem_addr(s_bars);
        bar.k_full = b;
        bar.k_empty = bar.k_full + 8 * S::kK;
        bar.v_full = bar.k_empty + 8 * S::kK;
        bar.v_empty = bar.v_full + 8 * S::kV;
        bar.q_full = bar.v_empty + 8 * S::kV;
        bar.q_empty = bar.q_full + 16;
        bar.s_full = bar.q_empty + 16;
        bar.p_full = bar.s_full + 16;
        bar.o_full = bar.p_full + 16;
    }
    if (tid == 0) {
        for (int i = 0; i < 2 * S::kK + 2 * S::kV + 6; ++i) mbar_init(bar.k_full + 8 * i, 1);
        mbar_init(bar.p_full, 4);
        mbar_init(bar.p_full + 8, 4);
        mbar_init(bar.o_full, 1);
        mbar_init(bar.o_full + 8, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        s_gave_up = 0;
        s_pro.own[0].left = s_pro.own[1].left = 0;
    }
    if (warp == 10) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }

    // ---- where this CTA's ranges begin: every CTA sums the tiles of all sequences
    const uint32_t batch = a.batch.batch, each = (batch + kThreads - 1) / kThreads;
    const uint32_t b_lo = min(batch, tid * each), b_hi = min(batch, b_lo + each);
    SeqRows r;
    uint32_t mine = 0, wrong = 0;
    for (uint32_t b = b_lo; b < b_hi; ++b) {
        wrong |= read_rows(a.batch, b, a.max_q, a.cache.page_size, r);
        mine += sequence_tiles(d, r);
    }
    if (wrong && blockIdx.x == 0) atomicOr(p.status, wrong);
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(~0u, incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    uint32_t before = incl - mine, total = 0;
    for (int i = 0; i < kThreads / 32; ++i) {
        if (i < warp) before += s_scan[i];
        total += s_scan[i];
    }
    int tok0, tok1;
    const uint32_t rts = prefix_rows(d, tok0, tok1);
    const uint32_t prefix_total = a.kv_heads * rts * w.prefix_tiles;
    if (tid < 2) s_pro.prefix[tid] = range_at(d, w.prefix_pair, prefix_total, blockIdx.x, tid);
    if (tid == 0) {
        s_pro.prefix_rt = max(1u, rts);
        s_pro.tok0 = tok0;
        s_pro.tok1 = tok1;
    }
    if (blockIdx.x == 0) {                        // for the joining kernel
        uint32_t* base = (uint32_t*)(ws + w.own_base);
        uint32_t at = before;
        for (uint32_t b = b_lo; b < b_hi; ++b) {
            base[b] = at;
            read_rows(a.batch, b, a.max_q, a.cache.page_size, r);
            at += sequence_tiles(d, r);
        }
        if (tid == 0) {
            base[batch] = total;
            base[batch + 1] = prefix_total;
        }
    }
    for (int s = 0; s < 2; ++s) {
        const Range g = range_at(d, w.own_pair, total, blockIdx.x, s);
        if (g.end > g.x && g.x >= before && g.x < before + mine) find_start(d, b_lo, b_hi, g.x - before, g.end - g.x, s_pro.own[s]);
    }
    fence_before();
    __syncthreads();
    fence_after();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = s_tmem;

    if (warp == 8 || warp == 9) {
        // ---------------------------------------------------------------- keys (8) and values (9)
        const bool is_v = warp == 9;
        const int stages = is_v ? S::kV : S::kK;
        const uint32_t at = is_v ? v_at : k_at, full = is_v ? bar.v_full : bar.k_full, empty = is_v ? bar.v_empty : bar.k_empty;
        const CUtensorMap* maps[2] = {is_v ? &p.v_prefix : &p.k_prefix, is_v ? &p.v_own : &p.k_own};
        Walk walk(d, s_pro);
        Job j;
        int tile, slot = 0;
        uint32_t phase = 0, issued = 0;
        bool u0, u1;
        while (walk.next(d, s_pro, j, tile, u0, u1)) {
            const tsw_kv_pages& pg = j.own ? a.cache : a.prefix;
            const int* table = j.own ? (const int*)a.batch.page_table + (uint64_t)j.b * a.batch.table_stride : (const int*)a.prefix_table;
            const int ps = pg.page_size, key0 = tile * kTile, n = min(kTile, j.keys - key0);
            const int box = min(ps, kTile), boxes = (n + box - 1) / box, first = key0 / ps, in_page = key0 - first * ps;
            int page = lane < boxes ? table[first + lane] : 0;        // before the wait: its latency passes under it
            if (!wait(empty + 8 * slot, phase ^ 1, gave_up)) break;
            if (lane == 0) mbar_expect(full + 8 * slot, boxes * box * 128 * kHalves);
            __syncwarp();
            for (int i = lane; i < boxes; i += 32) {
                if (i >= 32) page = table[first + i];
                // a number outside the cache is recorded; the copy unit fills such a box with zeros
                if ((uint32_t)page >= pg.pages) { atomicOr(p.status, TSW_KV_BAD_PAGE); page = pg.pages; }
                const uint32_t dst = at + slot * S::kTileBytes + i * box * 128;
#pragma unroll
                for (int h = 0; h < kHalves; ++h)
                    load_box4(dst + h * kHalfBytes, maps[j.own], h * 64, in_page, j.head, page, full + 8 * slot);
            }
            ++issued;
            if (++slot == stages) { slot = 0; phase ^= 1; }
        }
        if (*gave_up)        // copies in flight land before the CTA ends
            for (int i = 0; i < stages && i < (int)issued; ++i) {
                const unsigned long long t0 = now();
                const uint32_t last = (i < slot) ? phase : phase ^ 1;
                while (!mbar_try(full + 8 * i, last) && now() - t0 < kWaitNs / 8) {}
            }
    } else if (warp == 11) {
        // ---------------------------------------------------------------- queries
        Walk walk(d, s_pro);
        Job j;
        int tile;
        uint32_t count[2] = {0, 0};
        bool use[2];
        while (walk.next(d, s_pro, j, tile, use[0], use[1])) {
            if (tile != j.kt0) continue;
            bool ok = true;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (!use[s] || !ok) continue;
                ok = wait(bar.q_empty + 8 * s, (count[s] & 1) ^ 1, gave_up);
                if (!ok) break;
                ++count[s];
                if (lane == 0) {
                    const uint32_t box = j.own ? w.own_box_tokens : w.tile_tokens;
                    const int tok = j.tok + (walk.pair && s ? tile_tokens : 0);
                    mbar_expect(bar.q_full + 8 * s, box * group * 128 * kHalves);
#pragma unroll
                    for (int h = 0; h < kHalves; ++h)
                        load_box3(q_at + s * S::kTileBytes + h * kHalfBytes, j.own ? &p.q_own : &p.q_prefix, h * 64, j.head * group, tok,
                                  bar.q_full + 8 * s);
                }
            }
            if (!ok) break;
        }
        if (*gave_up)
            for (int s = 0; s < 2; ++s)
                if (count[s]) {
                    const unsigned long long t0 = now();
                    while (!mbar_try(bar.q_full + 8 * s, (count[s] - 1) & 1) && now() - t0 < kWaitNs / 8) {}
                }
    } else if (warp == 10) {
        // ---------------------------------------------------------------- products
        // Order: S of a tile, then the O product of the tile before it, whose exponentials ran meanwhile.
        constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : 1u << 7 | 1u << 10;
        constexpr uint32_t kDescS = 1u << 4 | kType | (kTile / 8) << 17 | (kTile / 16) << 24;
        constexpr uint32_t kDescO = 1u << 4 | kType | 1u << 16 | (DP / 8) << 17 | (kTile / 16) << 24;
        Walk walk(d, s_pro);
        Job j;
        int tile, k_slot = 0, v_slot = 0;
        uint32_t k_phase = 0, v_phase = 0, n_q[2] = {0, 0}, n_p[2] = {0, 0};
        struct Pending { bool any = false, first, load, release; int s, slot, keys; uint32_t phase; } pend;
        bool use[2], ok = true;

        auto product_o = [&]() {
            const Pending& u = pend;
            if (u.load) ok = wait(bar.v_full + 8 * u.slot, u.phase, gave_up);
            const uint32_t v = v_at + u.slot * S::kTileBytes;
            const int steps = (u.keys + 15) / 16;
            if (u.load && ok && (u.keys & 15)) {
                // Rows behind the last key hold whatever their page holds, and a weight of zero does not
                // silence an infinity: clear what the last step would read.
                const int rows = steps * 16 - u.keys;
                for (int i = lane; i < rows * 8 * kHalves; i += 32) {
                    const uint32_t at = v + (i / (rows * 8)) * kHalfBytes + (u.keys + (i / 8) % rows) * 128 + (i % 8) * 16;
                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            ok = ok && wait(bar.p_full + 8 * u.s, n_p[u.s]++ & 1, gave_up);
            if (!ok) return;
            fence_after();
            if (lane == 0) {
                const uint32_t base = tmem + u.s * 256;
                for (int k = 0; k < steps; ++k)
                    mma_ts(base + 128, base + k * 8, smem_desc(v + k * 2048, kHalfBytes), kDescO, !(u.first && k == 0));
                mma_commit(bar.o_full + 8 * u.s);
                if (u.release) mma_commit(bar.v_empty + 8 * u.slot);
            }
            __syncwarp();
            pend.any = false;
        };

        while (ok && walk.next(d, s_pro, j, tile, use[0], use[1])) {
            ok = wait(bar.k_full + 8 * k_slot, k_phase, gave_up);
            bool load = true;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (!use[s] || !ok) continue;
                if (pend.any && pend.s == s) product_o();
                if (!ok) break;
                const bool first = tile == j.kt0, ends = tile + 1 == min(j.kt1, seen_by(j, walk.pair, s));
                const bool release = s == 1 || !use[1];
                if (first) ok = wait(bar.q_full + 8 * s, n_q[s]++ & 1, gave_up);
                if (!ok) break;
                fence_after();
                if (lane == 0) {
                    const uint32_t q = q_at + s * S::kTileBytes, k = k_at + k_slot * S::kTileBytes;
#pragma unroll
                    for (int i = 0; i < DP / 16; ++i) {
                        const uint32_t off = (i / 4) * kHalfBytes + (i % 4) * 32;
                        mma_ss(tmem + s * 256, smem_desc(q + off, 16), smem_desc(k + off, 16), kDescS, i > 0);
                    }
                    mma_commit(bar.s_full + 8 * s);
                    if (release) mma_commit(bar.k_empty + 8 * k_slot);
                    if (ends) mma_commit(bar.q_empty + 8 * s);
                }
                __syncwarp();
                if (pend.any) product_o();
                if (!ok) break;
                pend.any = true;
                pend.first = first;
                pend.load = load;
                pend.release = release;
                pend.s = s;
                pend.slot = v_slot;
                pend.phase = v_phase;
                pend.keys = min(kTile, j.keys - tile * kTile);
                load = false;
            }
            if (++k_slot == S::kK) { k_slot = 0; k_phase ^= 1; }
            if (++v_slot == S::kV) { v_slot = 0; v_phase ^= 1; }
        }
        if (ok && pend.any) product_o();
    } else {
        // ---------------------------------------------------------------- rows: one thread each
        const int s = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;                 // this warp's quarter of the tensor memory's lanes
        const uint32_t t_s = tmem + lanes + s * 256, t_o = t_s + 128;
        const float c = a.scale * 1.4426950408889634f;
        const int tok_in_tile = row / group, head_in_group = row - tok_in_tile * group;
        uint32_t count = 0;
        bool ok = true;
        for (int own = 0; own < 2 && ok; ++own) {
            const bool pair = own ? w.own_pair : w.prefix_pair;
            Cursor cur(s_pro, pair ? 0 : s);
            Job j;
            while (ok && cur.next(d, s_pro, own, j)) {
                const int seen = seen_by(j, pair, s), end = min(j.kt1, seen);
                const int tokens = pair && s ? j.n_b : j.n_a, tok = j.tok + (pair && s ? tile_tokens : 0) + tok_in_tile;
                const bool mine = tok_in_tile < tokens;
                const bool warp_on = (warp & 3) * 32 < tokens * group;
                const int visible = min(j.keys, max(0, j.limit + tok + 1));     // keys this row sees, from the segment's start
                float top = -INFINITY, sum = 0.f;
                for (int tile = j.kt0; tile < end; ++tile, ++count) {
                    ok = wait(bar.s_full + 8 * s, count & 1, gave_up);
                    if (!ok) break;
                    fence_after();
                    if (warp_on) {
                        const int left = visible - tile * kTile;                // of this tile
                        const int chunks = (min(kTile, j.keys - tile * kTile) + 31) / 32;
                        float x[kTile];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (i < chunks) tmem_ld32((uint32_t*)x + 32 * i, t_s + 32 * i);
                        tmem_wait_ld();
                        if (__any_sync(~0u, left < chunks * 32)) {
#pragma unroll
                            for (int i = 0; i < kTile; ++i)
                                if (i >= left) x[i] = -INFINITY;
                        }
                        float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (i < chunks) {
#pragma unroll
                                for (int e = 0; e < 32; e += 4) {
                                    m0 = fmaxf(m0, x[32 * i + e]);
                                    m1 = fmaxf(m1, x[32 * i + e + 1]);
                                    m2 = fmaxf(m2, x[32 * i + e + 2]);
                                    m3 = fmaxf(m3, x[32 * i + e + 3]);
                                }
                            }
                        const float here = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
                        if (tile == j.kt0) {
                            top = here;
                        } else {
                            const bool grow = (here - top) * c > kGrow;          // also from -inf; never between two of them
                            if (__any_sync(~0u, grow)) {
                                const float f = grow ? exp2_fast((top - here) * c) : 1.f;
                                if (grow) top = here;
                                sum *= f;
                                ok = wait(bar.o_full + 8 * s, (count - 1) & 1, gave_up);
                                if (!ok) break;
                                fence_after();
#pragma unroll
                                for (int i = 0; i < DP / 32; ++i) {
                                    float o[32];
                                    tmem_ld32((uint32_t*)o, t_o + 32 * i);
                                    tmem_wait_ld();
#pragma unroll
                                    for (int e = 0; e < 32; ++e) o[e] *= f;
                                    tmem_st32(t_o + 32 * i, (uint32_t*)o);
                                }
                            }
                        }
                        const float base = top == -INFINITY ? 0.f : top * c;
                        float p0 = 0.f, p1 = 0.f, p2 = 0.f, p3 = 0.f;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (i < chunks) {
                                uint32_t packed[16];
#pragma unroll
                                for (int e = 0; e < 32; e += 4) {
                                    const float e0 = exp2_fast(fmaf(x[32 * i + e], c, -base)), e1 = exp2_fast(fmaf(x[32 * i + e + 1], c, -base));
                                    const float e2 = exp2_fast(fmaf(x[32 * i + e + 2], c, -base)), e3 = exp2_fast(fmaf(x[32 * i + e + 3], c, -base));
                                    p0 += e0; p1 += e1; p2 += e2; p3 += e3;
                                    packed[e / 2] = pack2<T>(e0, e1);
                                    packed[e / 2 + 1] = pack2<T>(e2, e3);
                                }
                                tmem_st16(t_s + 16 * i, packed);
                            }
                        sum += (p0 + p1) + (p2 + p3);
                        tmem_wait_st();
                    }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar.p_full + 8 * s);
                }
                if (!ok || j.kt0 >= end) continue;
                // ---- the range's result: into the output when it is all there is, else by row (an item's first
                // range) or by stream (one that continues)
                ok = wait(bar.o_full + 8 * s, (count - 1) & 1, gave_up);
                if (!ok) break;
                fence_after();
                if (!warp_on) continue;
                const bool direct = a.prefix_len == 0 && j.kt0 == 0 && end == seen;
                const uint32_t head = j.head * group + head_in_group;
                float* dst = nullptr;
                float2* ml = nullptr;
                uint8_t* out = nullptr;
                float inv = 0.f;
                if (mine) {
                    const uint64_t row_at = (uint64_t)tok * a.q_heads + head;
                    if (direct) {
                        out = (uint8_t*)(a.out + (uint64_t)tok * a.out_token_stride + (uint64_t)head * a.out_head_stride);
                        inv = sum == 0.f ? 0.f : 1.f / sum;
                        if (a.lse) ((float*)a.lse)[row_at] = sum == 0.f ? -INFINITY : (top * c + log2f(sum)) * 0.6931471805599453f;
                    } else if (j.kt0 == 0) {
                        const uint64_t at = home_index(d, own, row_at, a.q_heads);
                        dst = (float*)(ws + w.home_o) + at * a.head_dim;
                        ml = (float2*)(ws + w.home_ml) + at;
                    } else {
                        const uint64_t at = part_index(d, own, part_place(pair, range_index(d, pair, blockIdx.x, s), s), row);
                        dst = (float*)(ws + w.part_o) + at * a.head_dim;
                        ml = (float2*)(ws + w.part_ml) + at;
                    }
                    if (ml) *ml = make_float2(top == -INFINITY ? -INFINITY : top * c, sum);
                }
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) {
                    float o[32];
                    tmem_ld32((uint32_t*)o, t_o + 32 * i);
                    tmem_wait_ld();
                    if (out) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8)
                            if (32 * i + e < (int)a.head_dim)
                                *(uint4*)(out + 2 * (32 * i + e)) =
                                    make_uint4(pack2<T>(o[e] * inv, o[e + 1] * inv), pack2<T>(o[e + 2] * inv, o[e + 3] * inv),
                                               pack2<T>(o[e + 4] * inv, o[e + 5] * inv), pack2<T>(o[e + 6] * inv, o[e + 7] * inv));
                    } else if (dst) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            if (32 * i + e < (int)a.head_dim) *(float4*)(dst + 32 * i + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    }
                }
                fence_before();
            }
        }
    }
    fence_before();
    __syncthreads();
    if (tid == 0 && *gave_up) atomicOr(p.status, TSW_KV_WAIT_GAVE_UP);
    if (warp == 10) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// ---------------------------------------------------------------------------------------------
// Joining the partial results of a row: one warp per row, four elements of the head to a lane.  The
// ranges are visited in order, so the result does not depend on which finished first.
constexpr int kJoinWarps = 4;
template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps) combine_kernel(const __grid_constant__ tsw_prefix_attention_args a, const __grid_constant__ Deal d) {
    const int lane = threadIdx.x & 31;
    const uint64_t row = (uint64_t)blockIdx.x * kJoinWarps + (threadIdx.x >> 5);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (row >= (uint64_t)a.batch.tokens * a.q_heads) return;
    const AttentionLayout& w = d.w;
    const int tok = (int)(row / a.q_heads), head = (int)(row % a.q_heads), kv_head = head / w.group;
    const int b = find_sequence((const int*)a.batch.cu_q, a.batch.batch, tok);
    if (b < 0) return;
    SeqRows r;
    read_rows(a.batch, b, a.max_q, a.cache.page_size, r);
    if (tok >= r.first + r.n) return;
    const uint8_t* ws = (const uint8_t*)a.workspace;
    const uint32_t* base = (const uint32_t*)(ws + w.own_base);
    uint32_t before = 0;
    for (int rt = (tok - r.first) / own_item_tokens(d), i = lane; i < rt; i += 32) {
        const Cut c = cut_own(d, r, i);
        before += max(c.kt_a, c.kt_b);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) before += __shfl_xor_sync(~0u, before, o);
    const Parts parts[2] = {prefix_parts(d, tok, kv_head, base[a.batch.batch + 1]),
                            own_parts(d, r, tok, kv_head, base[b], before, base[a.batch.batch])};
    if (!a.prefix_len && parts[1].has && parts[1].first == parts[1].last) return;      // the tile kernel has written this row itself
    float top = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool on = 4 * lane < (int)a.head_dim;
    auto take = [&](const float2 ml, const float* o) {
        if (ml.x == -INFINITY && ml.y == 0.f) return;
        const float next = fmaxf(top, ml.x), base_ = next == -INFINITY ? 0.f : next;
        const float keep = exp2f(top - base_), f = exp2f(ml.x - base_);
        top = next;
        sum = sum * keep + ml.y * f;
        const float4 v = on ? *(const float4*)(o + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
        acc.x = acc.x * keep + v.x * f;
        acc.y = acc.y * keep + v.y * f;
        acc.z = acc.z * keep + v.z * f;
        acc.w = acc.w * keep + v.w * f;
    };
#pragma unroll
    for (int l = 0; l < 2; ++l) {
        const Parts& q = parts[l];
        if (!q.has) continue;
        const uint64_t home = home_index(d, l, row, a.q_heads);
        take(((const float2*)(ws + w.home_ml))[home], (const float*)(ws + w.home_o) + home * a.head_dim);
        const bool pair = l ? w.own_pair : w.prefix_pair;
        for (uint32_t i = q.first + 1; i <= q.last; ++i) {
            const uint64_t at = part_index(d, l, part_place(pair, i, q.half), q.place * w.group + head % w.group);
            take(((const float2*)(ws + w.part_ml))[at], (const float*)(ws + w.part_o) + at * a.head_dim);
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (on) {
        const uint2 v = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
        *(uint2*)(a.out + (uint64_t)tok * a.out_token_stride + (uint64_t)head * a.out_head_stride + 8 * lane) = v;
    }
    if (a.lse && lane == 0) ((float*)a.lse)[row] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

// ------------------------------------------------------------------------------------- host

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static std::atomic<EncodeTiled> known{nullptr};
    EncodeTiled f = known.load(std::memory_order_acquire);
    if (!f) {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &sym, 12000, cudaEnableDefault, &found) == cudaSuccess &&
            found == cudaDriverEntryPointSuccess)
            f = (EncodeTiled)sym;
        known.store(f, std::memory_order_release);
    }
    return f;
}

// A dimension of one entry may come with any stride: the map wants a legal one.
uint64_t legal(uint64_t stride, uint64_t count) { return count > 1 ? stride : 1 << 16; }

cudaError_t encode(CUtensorMap* map, uint32_t dtype, uint64_t addr, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    EncodeTiled f = encode_tiled();
    if (!f) return cudaErrorNotSupported;
    const CUresult rc = f(map, dtype == TSW_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, (void*)addr, dims, strides, box,
                          ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t encode_pages(CUtensorMap* map, const tsw_prefix_attention_args& a, const tsw_kv_pages& pg, bool v) {
    const cuuint64_t dims[4] = {a.head_dim, pg.page_size, a.kv_heads, pg.pages};
    const cuuint64_t strides[3] = {legal(v ? pg.v_token_stride : pg.k_token_stride, pg.page_size), legal(v ? pg.v_head_stride : pg.k_head_stride, a.kv_heads),
                                   legal(v ? pg.v_page_stride : pg.k_page_stride, pg.pages)};
    const cuuint32_t box[4] = {64, std::min<uint32_t>(pg.page_size, kTile), 1, 1};
    return encode(map, a.dtype, v ? pg.v : pg.k, 4, dims, strides, box);
}

cudaError_t encode_queries(CUtensorMap* map, const tsw_prefix_attention_args& a, uint32_t group, uint32_t box_tokens) {
    const cuuint64_t dims[3] = {a.head_dim, a.q_heads, a.batch.tokens};
    const cuuint64_t strides[2] = {legal(a.q_head_stride, a.q_heads), legal(a.q_token_stride, a.batch.tokens)};
    const cuuint32_t box[3] = {64, group, box_tokens};
    return encode(map, a.dtype, a.q, 3, dims, strides, box);
}

template <typename T, int DP>
cudaError_t launch_tiles(const Params& p, cudaStream_t stream) {
    cudaError_t err = cudaFuncSetAttribute(attention_tiles_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<DP>::kSmem);
    if (err != cudaSuccess) return err;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.d.w.ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Shape<DP>::kSmem;
    cfg.stream = stream;
    err = cudaLaunchKernelEx(&cfg, attention_tiles_kernel<T, DP>, p);
    if (err != cudaSuccess) return err;
    cudaLaunchAttribute early;           // its launch passes under the tile kernel; it waits there for the results
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3((unsigned)(((uint64_t)p.a.batch.tokens * p.a.q_heads + kJoinWarps - 1) / kJoinWarps));
    cfg.blockDim = dim3(32 * kJoinWarps);
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, combine_kernel<T>, p.a, p.d);
}

}  // namespace

cudaError_t launch_prefix_attention_tiles(const tsw_prefix_attention_args& a, const AttentionLayout& w, uint32_t* status, cudaStream_t stream) {
    Params p;
    p.a = a;
    p.d = Deal{a.batch, a.max_q, a.cache.page_size, a.kv_heads, a.prefix_len, a.causal, w};
    p.status = status;
    cudaError_t err = encode_pages(&p.k_own, a, a.cache, false);
    if (err == cudaSuccess) err = encode_pages(&p.v_own, a, a.cache, true);
    if (err == cudaSuccess) err = encode_queries(&p.q_own, a, w.group, w.own_box_tokens);
    if (err != cudaSuccess) return err;
    p.k_prefix = p.k_own;
    p.v_prefix = p.v_own;
    if (a.prefix_len && memcmp(&a.cache, &a.prefix, sizeof(a.cache)) != 0) {
        err = encode_pages(&p.k_prefix, a, a.prefix, false);
        if (err == cudaSuccess) err = encode_pages(&p.v_prefix, a, a.prefix, true);
        if (err != cudaSuccess) return err;
    }
    p.q_prefix = p.q_own;
    if (w.own_box_tokens != w.tile_tokens) err = encode_queries(&p.q_prefix, a, w.group, w.tile_tokens);
    if (err != cudaSuccess) return err;
    if (a.head_dim <= 64) return a.dtype == TSW_F16 ? launch_tiles<__half, 64>(p, stream) : launch_tiles<__nv_bfloat16, 64>(p, stream);
    return a.dtype == TSW_F16 ? launch_tiles<__half, 128>(p, stream) : launch_tiles<__nv_bfloat16, 128>(p, stream);
}

}  // namespace tsw
