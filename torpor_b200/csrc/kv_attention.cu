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
    int own_shift, prefix_shift;      // log2 of the page sizes
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
// caller leaves its loop.  A whole warp waits and gets one answer.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile uint32_t* gave_up) {
    if (__all_sync(~0u, mbar_try(bar, parity))) return true;
    const unsigned long long t0 = now();
    bool ok;
#pragma unroll 1
    do {
        ok = mbar_try(bar, parity);
        if (!ok && now() - t0 > kWaitNs) *gave_up = 1;
    } while (!__all_sync(~0u, ok) && !__any_sync(~0u, *gave_up));
    return __all_sync(~0u, ok);
}

// One lane of a converged warp, chosen in a way that leaves the code under it uniform: operands of the tensor and
// copy units are uniform registers.
__device__ __forceinline__ bool elect() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(~0u, x, 0); }

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
__device__ __forceinline__ void tmem_ld16(uint32_t* r, uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : TSW_R8(r, 0), TSW_R8(r, 8) : "r"(addr) : "memory");
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
// The low word holds the address and the lead (units of 16 bytes): steps along a tile are added to it.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lead_bytes) { return addr >> 4 | lead_bytes >> 4 << 16; }
__device__ __forceinline__ uint64_t desc(uint32_t lo) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(1024u >> 4 | 1u << 14 | 2u << 29));
    return r;
}

constexpr int kUnits = 16;                    // units on their way from the scheduling warp to the others
constexpr int kJobs = 4;                      // rows' jobs on their way, per stream

// mbarriers: byte offsets into the array in shared memory
template <int kK, int kV> struct Bars {
    static constexpr int k_full = 0, k_empty = k_full + 8 * kK, v_full = k_empty + 8 * kK, v_empty = v_full + 8 * kV, q_full = v_empty + 8 * kV,
                         s_full = q_full + 16, o_full = s_full + 16, unit_full = o_full + 16, job_full = unit_full + 8 * kUnits,
                         ones = (job_full + 16 * kJobs) / 8,                          // up to here one arrival completes a phase
                         unit_empty = 8 * ones, p_full = unit_empty + 8 * kUnits, job_empty = p_full + 16, bytes = job_empty + 16 * kJobs;
};

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1) attention_tiles_kernel(const __grid_constant__ Params p) {
    using S = Shape<DP>;
    using B = Bars<S::kK, S::kV>;
    constexpr int kHalves = DP / 64;
    constexpr uint32_t kHalfBytes = kTile * 128;
    extern __shared__ uint8_t s_raw[];
    __shared__ __align__(8) uint64_t s_bars[B::bytes / 8];
    __shared__ Unit s_units[kUnits];
    __shared__ RowJob s_jobs[2][kJobs];
    __shared__ Prologue s_pro;
    __shared__ uint32_t s_tmem, s_scan[kThreads / 32];
    __shared__ uint32_t s_gave_up;
    volatile uint32_t* gave_up = &s_gave_up;
    const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
    const tsw_prefix_attention_args& a = p.a;
    const Deal& d = p.d;
    const AttentionLayout& w = d.w;
    const uint32_t bar = smem_addr(s_bars);
    const uint32_t q_at = (smem_addr(s_raw) + 1023) & ~1023u, k_at = q_at + 2 * S::kTileBytes, v_at = k_at + S::kK * S::kTileBytes;

    // ---- where this CTA's ranges begin: every CTA sums the tiles of all sequences
    const uint32_t batch = a.batch.batch, each = (batch + kThreads - 1) / kThreads;
    const uint32_t b_lo = min(batch, tid * each), b_hi = min(batch, b_lo + each);
    uint32_t mine = 0, wrong = 0;
#pragma unroll 1
    for (uint32_t b = b_lo; b < b_hi; ++b) {
        SeqRows r;
        wrong |= read_rows(a.batch, b, a.max_q, a.cache.page_size, r);
        mine += sequence_tiles(d, r);
    }
    if (warp == 10) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (warp == 9) {
        for (int i = lane; i < B::bytes / 8; i += 32)
            mbar_init(bar + 8 * i, i < B::ones ? 1 : i < B::p_full / 8 ? 3 : 4);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8 && lane < 6) {
        const CUtensorMap* map = &p.q_prefix + lane;
        asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
    }
    if (tid == 0) {
        s_gave_up = 0;
        s_pro.own[0].left = s_pro.own[1].left = 0;
    }
    if (wrong && blockIdx.x == 0) atomicOr(p.status, wrong);
    uint32_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(~0u, before, o);
        if (lane >= o) before += up;
    }
    if (lane == 31) s_scan[warp] = before;
    before -= mine;
    __syncthreads();
    uint32_t total = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) {
        if (i == warp) before += total;
        total += s_scan[i];
    }
    if (warp == 11) {
        int tok0, tok1;
        const uint32_t rts = prefix_rows(d, tok0, tok1), prefix_total = a.kv_heads * rts * w.prefix_tiles;
        if (lane < 2) s_pro.prefix[lane] = range_at(d, w.prefix_pair, prefix_total, blockIdx.x, lane);
        if (lane == 0) {
            s_pro.prefix_rt = max(1u, rts);
            s_pro.tok0 = tok0;
            s_pro.tok1 = tok1;
            if (blockIdx.x == 0) {                    // for the joining kernel
                uint32_t* base = (uint32_t*)((uint8_t*)a.workspace + w.own_base);
                base[batch] = total;
                base[batch + 1] = prefix_total;
            }
        }
    }
    if (blockIdx.x == 0) {
        uint32_t* base = (uint32_t*)((uint8_t*)a.workspace + w.own_base);
        uint32_t at = before;
#pragma unroll 1
        for (uint32_t b = b_lo; b < b_hi; ++b) {
            base[b] = at;
            SeqRows r;
            read_rows(a.batch, b, a.max_q, a.cache.page_size, r);
            at += sequence_tiles(d, r);
        }
    }
#pragma unroll 1
    for (int s = 0; s < 2; ++s) {
        const Range g = range_at(d, w.own_pair, total, blockIdx.x, s);
        if (g.end > g.x && g.x >= before && g.x < before + mine) find_start(d, b_lo, b_hi, g.x - before, g.end - g.x, s_pro.own[s]);
    }
    fence_before();
    __syncthreads();
    fence_after();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = uniform(s_tmem);

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        if (warp == 11) {
            // ------------------------------------------------------------ scheduling
            Walk walk(d, s_pro);
            Job j;
            int tile;
            uint32_t n = 0, jobs[2] = {0, 0};
            bool use[2], ok = true;
#pragma unroll 1
            while (ok) {
                const bool more = walk.next(d, s_pro, j, tile, use[0], use[1]);
                if (!more) use[0] = use[1] = true;
#pragma unroll 1
                for (int s = 0; s < 2 && ok; ++s) {
                    if (s ? !use[1] : !use[0]) continue;
                    if (!more || tile == j.kt0) {                     // also tells both streams' rows of the end
                        const uint32_t i = s ? jobs[1]++ : jobs[0]++, at = s * kJobs + i % kJobs;
                        ok = wait(bar + B::job_empty + 8 * at, (i / kJobs & 1) ^ 1, gave_up);
                        if (!ok) break;
                        if (lane == 0) {
                            RowJob r = {};
                            if (more) r = make_row_job(d, j, walk.pair, s, blockIdx.x);
                            s_jobs[s][i % kJobs] = r;
                            mbar_arrive(bar + B::job_full + 8 * at);
                        }
                        if (!more && s == 0) continue;
                    }
                    ok = wait(bar + B::unit_empty + 8 * (n % kUnits), (n / kUnits & 1) ^ 1, gave_up);
                    if (!ok) break;
                    if (lane == 0) {
                        s_units[n % kUnits] = more ? make_unit(j, tile, s, use[0], use[1]) : Unit{kUnitEnd, 0, 0, 0};
                        mbar_arrive(bar + B::unit_full + 8 * (n % kUnits));
                    }
                    ++n;
                }
                if (!more) break;
            }
        } else if (warp < 10) {
            // ------------------------------------------------------------ keys (8) and values (9)
            const bool is_v = warp == 9;
            const int stages = is_v ? S::kV : S::kK;
            const uint32_t at = is_v ? v_at : k_at, full = bar + (is_v ? B::v_full : B::k_full), empty = bar + (is_v ? B::v_empty : B::k_empty);
            int slot = 0;
            uint32_t phase = 0, issued = 0;
#pragma unroll 1
            for (uint32_t n = 0;; ++n) {
                if (!wait(bar + B::unit_full + 8 * (n % kUnits), n / kUnits & 1, gave_up)) break;
                const Unit u = s_units[n % kUnits];
                __syncwarp();
                if (lane == 0) mbar_arrive(bar + B::unit_empty + 8 * (n % kUnits));
                if (u.flags & kUnitEnd) break;
                if (!(u.flags & kUnitLoad)) continue;
                const bool own = u.flags & kUnitOwn;
                const tsw_kv_pages& pg = own ? a.cache : a.prefix;
                const CUtensorMap* map = own ? (is_v ? &p.v_own : &p.k_own) : (is_v ? &p.v_prefix : &p.k_prefix);
                const int shift = own ? p.own_shift : p.prefix_shift, box = min(1 << shift, kTile);
                const int boxes = (unit_keys(u.flags) + box - 1) / box, first = u.tile * kTile >> shift, in_page = u.tile * kTile & ((1 << shift) - 1);
                const int* table = (own ? (const int*)a.batch.page_table + (uint64_t)u.b * a.batch.table_stride : (const int*)a.prefix_table) + first;
                int page = lane < boxes ? table[lane] : 0;                // before the wait: its latency passes under it
                if (!wait(empty + 8 * slot, phase ^ 1, gave_up)) break;
                if (lane == 0) mbar_expect(full + 8 * slot, boxes * box * 128 * kHalves);
                __syncwarp();
#pragma unroll 1
                for (int i = lane; i < boxes; i += 32) {
                    if (i >= 32) page = table[i];
                    // a number outside the cache is recorded; the copy unit fills such a box with zeros
                    if ((uint32_t)page >= pg.pages) { atomicOr(p.status, TSW_KV_BAD_PAGE); page = pg.pages; }
                    const uint32_t dst = at + slot * S::kTileBytes + i * box * 128;
#pragma unroll
                    for (int h = 0; h < kHalves; ++h)
                        load_box4(dst + h * kHalfBytes, map, h * 64, in_page, unit_head(u.flags), page, full + 8 * slot);
                }
                ++issued;
                if (++slot == stages) { slot = 0; phase ^= 1; }
            }
            if (*gave_up)        // copies in flight land before the CTA ends
                for (int i = 0; i < stages && i < (int)issued; ++i) {
                    const unsigned long long t0 = now();
                    while (!mbar_try(full + 8 * i, i < slot ? phase : phase ^ 1) && now() - t0 < kWaitNs / 8) {}
                }
        } else {
            // ------------------------------------------------------------ products
            // Order: S of a unit, then the O product of the unit before it, whose exponentials ran meanwhile.  When both
            // are one stream's, O goes first: S would overwrite the weights.
            constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : 1u << 7 | 1u << 10;
            constexpr uint32_t kDescS = 1u << 4 | kType | (kTile / 8) << 17 | (kTile / 16) << 24;
            constexpr uint32_t kDescO = 1u << 4 | kType | 1u << 16 | (DP / 8) << 17 | (kTile / 16) << 24;
            uint32_t n_q = 0, n_p = 0;                    // phases of both streams, bit s
            int k_slot = 0, v_slot = 0, old_v_slot = 0;
            uint32_t k_phase = 0, v_phase = 0, old_v_phase = 0, old = kUnitEnd;
            bool ok = true;
#pragma unroll 1
            for (uint32_t n = 0; ok; ++n) {
                ok = wait(bar + B::unit_full + 8 * (n % kUnits), n / kUnits & 1, gave_up);
                if (!ok) break;
                const uint32_t flags = uniform(s_units[n % kUnits].flags);
                if (elect()) mbar_arrive(bar + B::unit_empty + 8 * (n % kUnits));
                const bool same = !((flags ^ old) & kUnitStream);
#pragma unroll 1
                for (int step = 0; step < 2 && ok; ++step) {
                    if ((step == 0) == same) {
                        if (old & kUnitEnd) continue;
                        const int s = old & kUnitStream, keys = unit_keys(old), steps = (keys + 15) / 16;
                        const uint32_t v = v_at + old_v_slot * S::kTileBytes;
                        if (old & kUnitLoad) {
                            ok = wait(bar + B::v_full + 8 * old_v_slot, old_v_phase, gave_up);
                            if (ok && (keys & 15)) {
                                // Rows behind the last key hold whatever their page holds, and a weight of zero
                                // does not silence an infinity: clear what the last step would read.
                                const int rows = steps * 16 - keys;
#pragma unroll 1
                                for (int i = lane; i < rows * 8 * kHalves; i += 32) {
                                    const uint32_t to = v + (i / (rows * 8)) * kHalfBytes + (keys + (i / 8) % rows) * 128 + (i % 8) * 16;
                                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(to), "r"(0) : "memory");
                                }
                                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                                __syncwarp();
                            }
                        }
                        ok = ok && wait(bar + B::p_full + 8 * s, n_p >> s & 1, gave_up);
                        if (!ok) break;
                        n_p ^= 1u << s;
                        fence_after();
                        const uint32_t base = tmem + s * 256, v_lo = desc_lo(v, kHalfBytes);
                        const bool more = !(old & kUnitFirst);
                        if (elect()) {
                            if (keys == kTile) {
#pragma unroll
                                for (int k = 0; k < kTile / 16; ++k) mma_ts(base + 128, base + k * 8, desc(v_lo + (k * 2048 >> 4)), kDescO, k > 0 || more);
                            } else {
#pragma unroll 1
                                for (int k = 0; k < steps; ++k) mma_ts(base + 128, base + k * 8, desc(v_lo + (k * 2048 >> 4)), kDescO, k > 0 || more);
                            }
                            mma_commit(bar + B::o_full + 8 * s);
                            if (old & kUnitRelease) mma_commit(bar + B::v_empty + 8 * old_v_slot);
                        }
                        __syncwarp();
                    } else {
                        if (flags & kUnitEnd) continue;
                        const int s = flags & kUnitStream;
                        if (flags & kUnitLoad) ok = wait(bar + B::k_full + 8 * k_slot, k_phase, gave_up);
                        if (ok && (flags & kUnitFirst)) {
                            ok = wait(bar + B::q_full + 8 * s, n_q >> s & 1, gave_up);
                            n_q ^= 1u << s;
                        }
                        if (!ok) break;
                        fence_after();
                        const uint32_t q_lo = desc_lo(q_at + s * S::kTileBytes, 16), k_lo = desc_lo(k_at + k_slot * S::kTileBytes, 16);
                        if (elect()) {
#pragma unroll
                            for (int i = 0; i < DP / 16; ++i) {
                                const uint32_t off = ((i / 4) * kHalfBytes + (i % 4) * 32) >> 4;
                                mma_ss(tmem + s * 256, desc(q_lo + off), desc(k_lo + off), kDescS, i > 0);
                            }
                            mma_commit(bar + B::s_full + 8 * s);
                            if (flags & kUnitRelease) mma_commit(bar + B::k_empty + 8 * k_slot);
                        }
                        __syncwarp();
                    }
                }
                if (flags & kUnitEnd) break;
                old = flags;
                old_v_slot = v_slot;
                old_v_phase = v_phase;
                if (flags & kUnitRelease) {
                    if (++k_slot == S::kK) { k_slot = 0; k_phase ^= 1; }
                    if (++v_slot == S::kV) { v_slot = 0; v_phase ^= 1; }
                }
            }
        }
    } else {
        // ---------------------------------------------------------------- rows: one thread each
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        const int s = warp >> 2, row = tid & 127, group = w.group;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;                 // this warp's quarter of the tensor memory's lanes
        const uint32_t t_s = tmem + lanes + s * 256, t_o = t_s + 128;
        const uint32_t b_s = bar + B::s_full + 8 * s, b_p = bar + B::p_full + 8 * s, b_o = bar + B::o_full + 8 * s;
        const uint32_t b_jf = bar + B::job_full + 8 * kJobs * s, b_je = bar + B::job_empty + 8 * kJobs * s;
        const float c = a.scale * 1.4426950408889634f;
        const int tok_in_tile = row / group, head_in_group = row - tok_in_tile * group;
        const bool loads_q = (warp & 3) == 0;                             // the warp that fetches the stream's queries
        uint32_t count = 0, asked = 0;                                    // units so far; jobs whose queries are on their way
        auto load_q = [&](uint32_t i) {                                   // of job i, which has been read or seen to be there
            const RowJob& j = s_jobs[s][i % kJobs];
            if (lane == 0 && j.tiles) {
                const uint32_t box = j.own ? w.own_box_tokens : w.tile_tokens, to = q_at + s * S::kTileBytes;
                const CUtensorMap* map = j.own ? &p.q_own : &p.q_prefix;
                mbar_expect(bar + B::q_full + 8 * s, box * group * 128 * kHalves);
#pragma unroll
                for (int h = 0; h < kHalves; ++h) load_box3(to + h * kHalfBytes, map, h * 64, j.head * group, j.tok, bar + B::q_full + 8 * s);
            }
            asked = i + 1;
        };
        bool ok = true;
#pragma unroll 1
        for (uint32_t i = 0; ok; ++i) {
            ok = wait(b_jf + 8 * (i % kJobs), i / kJobs & 1, gave_up);
            if (!ok) break;
            if (loads_q && asked == i) load_q(i);
            const RowJob j = s_jobs[s][i % kJobs];
            __syncwarp();
            if (lane == 0) mbar_arrive(b_je + 8 * (i % kJobs));
            if (!j.tiles) break;
            const int tok = j.tok + tok_in_tile;
            const bool warp_on = (warp & 3) * 32 < j.tokens * group;
            int left = min(j.keys, max(0, j.limit + tok));                // keys this row sees from here on
            float top = -INFINITY, sum = 0.f;
#pragma unroll 1
            for (int tile = 0; tile < j.tiles; ++tile, ++count, left -= kTile) {
                ok = wait(b_s, count & 1, gave_up);
                if (!ok) break;
                fence_after();
                // The job's last S is there, so its queries are done with: fetch the next job's, if it is known yet.
                if (loads_q && tile == j.tiles - 1 && __all_sync(~0u, mbar_try(b_jf + 8 * ((i + 1) % kJobs), (i + 1) / kJobs & 1))) load_q(i + 1);
                if (warp_on) {
                    float x[kTile];
#pragma unroll
                    for (int k = 0; k < 4; ++k) tmem_ld32((uint32_t*)x + 32 * k, t_s + 32 * k);
                    tmem_wait_ld();
                    if (__any_sync(~0u, left < kTile)) {
#pragma unroll
                        for (int k = 0; k < kTile; ++k)
                            if (k >= left) x[k] = -INFINITY;
                    }
                    float m0 = x[0], m1 = x[1], m2 = x[2], m3 = x[3];
#pragma unroll
                    for (int k = 4; k < kTile; k += 4) {
                        m0 = fmaxf(m0, x[k]);
                        m1 = fmaxf(m1, x[k + 1]);
                        m2 = fmaxf(m2, x[k + 2]);
                        m3 = fmaxf(m3, x[k + 3]);
                    }
                    const float here = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
                    if (tile == 0) {
                        top = here;
                    } else {
                        const bool grow = (here - top) * c > kGrow;              // also from -inf; never between two of them
                        if (__any_sync(~0u, grow)) {
                            const float f = grow ? exp2_fast((top - here) * c) : 1.f;
                            if (grow) top = here;
                            sum *= f;
                            ok = wait(b_o, (count - 1) & 1, gave_up);
                            if (!ok) break;
                            fence_after();
#pragma unroll 1
                            for (int k = 0; k < DP; k += 16) {
                                float o[16];
                                tmem_ld16((uint32_t*)o, t_o + k);
                                tmem_wait_ld();
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] *= f;
                                tmem_st16(t_o + k, (uint32_t*)o);
                            }
                        }
                    }
                    const float base = top == -INFINITY ? 0.f : top * c;
                    float p0 = 0.f, p1 = 0.f, p2 = 0.f, p3 = 0.f;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t packed[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            const float e0 = exp2_fast(fmaf(x[32 * k + e], c, -base)), e1 = exp2_fast(fmaf(x[32 * k + e + 1], c, -base));
                            const float e2 = exp2_fast(fmaf(x[32 * k + e + 2], c, -base)), e3 = exp2_fast(fmaf(x[32 * k + e + 3], c, -base));
                            p0 += e0;
                            p1 += e1;
                            p2 += e2;
                            p3 += e3;
                            packed[e / 2] = pack2<T>(e0, e1);
                            packed[e / 2 + 1] = pack2<T>(e2, e3);
                        }
                        tmem_st16(t_s + 16 * k, packed);
                    }
                    sum += (p0 + p1) + (p2 + p3);
                    tmem_wait_st();
                }
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(b_p);
            }
            if (!ok) break;
            // ---- the range's result: into the output when it is all there is, else by row (an item's first
            // range) or by stream (one that continues)
            ok = wait(b_o, (count - 1) & 1, gave_up);
            if (!ok) break;
            fence_after();
            if (!warp_on) continue;
            uint8_t* out = nullptr;
            float f = 1.f;
            if (tok_in_tile < j.tokens) {
                uint8_t* ws = (uint8_t*)a.workspace;
                const uint32_t head = j.head * group + head_in_group;
                const uint64_t row_at = (uint64_t)tok * a.q_heads + head;
                if (j.place == kPlaceDirect) {
                    out = (uint8_t*)(a.out + (uint64_t)tok * a.out_token_stride + (uint64_t)head * a.out_head_stride);
                    f = sum == 0.f ? 0.f : 1.f / sum;
                    if (a.lse) ((float*)a.lse)[row_at] = sum == 0.f ? -INFINITY : (top * c + log2f(sum)) * 0.6931471805599453f;
                } else {
                    const bool home = j.place == kPlaceHome;
                    const uint64_t at = home ? home_index(d, j.own, row_at, a.q_heads) : part_index(d, j.own, j.place, row);
                    out = ws + (home ? w.home_o : w.part_o) + 4 * at * a.head_dim;
                    *((float2*)(ws + (home ? w.home_ml : w.part_ml)) + at) = make_float2(top == -INFINITY ? -INFINITY : top * c, sum);
                }
            }
            float o[DP];
#pragma unroll
            for (int k = 0; k < DP; k += 32) tmem_ld32((uint32_t*)o + k, t_o + k);
            tmem_wait_ld();
            fence_before();
            if (!out) continue;
            if (j.place == kPlaceDirect) {
#pragma unroll
                for (int e = 0; e < DP; e += 8)
                    if (e < (int)a.head_dim)                                      // a multiple of 8
                        *(uint4*)(out + 2 * e) = make_uint4(pack2<T>(o[e] * f, o[e + 1] * f), pack2<T>(o[e + 2] * f, o[e + 3] * f),
                                                            pack2<T>(o[e + 4] * f, o[e + 5] * f), pack2<T>(o[e + 6] * f, o[e + 7] * f));
            } else {
#pragma unroll
                for (int e = 0; e < DP; e += 4)
                    if (e < (int)a.head_dim) *(float4*)(out + 4 * e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
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
    p.own_shift = __builtin_ctz(a.cache.page_size);
    p.prefix_shift = a.prefix_len ? __builtin_ctz(a.prefix.page_size) : 0;
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
