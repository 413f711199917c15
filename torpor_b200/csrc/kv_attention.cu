// Attention behind a shared prefix on the fifth-generation tensor cores.
//
// For one key head the rows of a tile are (token, query head of the group) pairs, up to 128 of them; keys come in tiles of
// 128.  S = Q K^T and O += P V are tcgen05.mma chains (M = 128; accumulators in tensor memory, the weights P go back
// into tensor memory over S and are the A operand of the second product).  One thread holds one row of S: maximum,
// exponentials and sum need no exchange between threads.  The maximum that exponentials are taken against
// moves only when it grows by more than 2^8 (fp16: 2^4), so the running output is rarely rescaled; the quotient at the
// end makes the result independent of it.  Weights are rounded to the operands' 16 bits, which the
// tensor cores take; their sum is formed from the unrounded 32-bit values, as are maximum and output.
//
// The work is two lists of (item, key tile) pairs: the prefix with the rows of ALL sequences (this is what makes it
// "computed once for all": a 128-row tile reads each prefix key once for 128 rows), and every sequence's own
// keys with its own rows.  Each list is cut into equal contiguous ranges of tiles, one per stream of
// the grid, wherever the cuts fall: long key axes are split, short ones batched, and no length
// needs to be known on the host.  What a range holds of an item is a partial result (output, maximum,
// sum); combine_kernel joins them.
//
// One CTA per SM runs two streams, a warpgroup of 128 rows and a product thread each, so that one stream's products and
// loads run under the other's exponentials.  The streams take different items (few rows: bound by HBM), or two row
// tiles of one item that share every key tile ("pair": many rows, where a load of 64 KB per 128 rows and tile would
// ask 128 bytes a cycle of the L2).  A stream's S is two buffers of 64 keys: with one of 128 its rows waited 2000
// of 4100 cycles a tile for O and the next S; now there is always one to work on.  Five warps do the rest: one
// thread schedules (units and jobs go to the others through rings in shared memory, so that the lists'
// arithmetic is done and fetched once), two warps load keys and values page by page with TMA, two
// threads issue the products.
//
// Measured, for this kernel alone and thus under ncu, cold: 4096 rows of 32 heads of 128 behind 16384 tokens, 1.88 million
// cycles (1.21 ms at 1.56 GHz, 942 TFLOP/s), the tensor pipe 70 % busy (exponentials: the special function unit at
// 53 %); a causal prompt of 8192 tokens 1.17 million cycles (690 us, 796 TFLOP/s); eight texts of up to 32768 tokens, 86 to
// 89 us, 5.6 to 5.4 TB/s.  Short jobs are bound by what each costs its rows beside the tiles
// (queries, the wait for the last product, storing: some 2000 cycles) and by 5 us before the first key arrives.

#include "kv_kernels.hpp"
#include "kv_device.cuh"
#include "kv_attention.hpp"
#include "kv_dealing.hpp"

#include <atomic>
#include <cstring>
#include <type_traits>

#include <cuda.h>

namespace tsw {

namespace {

constexpr int kThreads = 416;                 // two warpgroups of rows; warps for keys, values, each stream's products, scheduling
constexpr unsigned long long kWaitNs = 2000000000ull, kDrainNs = 5000000ull;
// log2 of the growth of the maximum that is let pass, and of the weight that the maximum's own key has.  bf16 reaches as far down as
// 32 bits do.  fp16 ends at 2^-24, and a weight of 1 for the maximum would leave what lies above unused: a flat tail of a
// million keys behind one that takes 90 % lost an eighth.  Raised by 2^11 (with the growth 2^15, the type ends at 2^16) a weight loses
// bits from 2^-25 of the maximum's on and is lost at 2^-36, where 32-bit sums over as many keys no longer show it.
// A growth of 2^4 instead of 2^8 is exceeded, behind random keys, in 1 of 20 warps and items.
template <typename T> constexpr float kGrow = std::is_same<T, __half>::value ? 4.f : 8.f;
template <typename T> constexpr float kRaise = std::is_same<T, __half>::value ? 11.f : 0.f;

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
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {      // does not wait
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ unsigned long long now() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// Every wait ends: after two seconds, or when another warp of the CTA has given up, it answers false, and the
// caller leaves its loop.  Inlined: the call, though hardly ever made, costs the loops around it registers and
// 2 % (4096 rows behind 16384 tokens).
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile uint32_t* gave_up) {           // a whole warp, one answer
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
__device__ __forceinline__ bool wait_alone(uint32_t bar, uint32_t parity, volatile uint32_t* gave_up) {      // one thread
    if (mbar_try(bar, parity)) return true;
    const unsigned long long t0 = now();
#pragma unroll 1
    while (!mbar_try(bar, parity)) {
        if (now() - t0 > kWaitNs) *gave_up = 1;
        if (*gave_up) return false;
    }
    return true;
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
// Two floats to an instruction.
__device__ __forceinline__ uint64_t two(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 split(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
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

// What the scheduling warp has told the others and they have not yet taken up: loads; takes and rows' jobs of a stream.
constexpr int kLoads = 8, kTakes = 4, kJobs = 4;

// Warps behind the rows' eight.
enum { kWarpK = 8, kWarpV, kWarpSchedule, kWarpProducts };      // kWarpProducts + stream

// mbarriers: byte offsets into the array in shared memory.  Pairs and rings of a stream lie together.
template <int kK, int kV> struct Bars {
    static constexpr int k_full = 0, v_full = k_full + 16 * kK, q_full = v_full + 16 * kV, o_full = q_full + 16, s_full = o_full + 32,
                         load_full = s_full + 32, take_full = load_full + 8 * kLoads, take_empty = take_full + 16 * kTakes,
                         job_full = take_empty + 16 * kTakes,
                         ones = (job_full + 16 * kJobs) / 8,                         // up to here one arrival ends a phase
                         k_empty = 8 * ones, v_empty = k_empty + 8 * kK, load_empty = v_empty + 8 * kV,
                         p_full = load_empty + 8 * kLoads,                           // up to here two, from here four
                         job_empty = p_full + 32, bytes = job_empty + 16 * kJobs;
};

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1) attention_tiles_kernel(const __grid_constant__ Params p) {
    using S = Shape<DP>;
    using B = Bars<S::kK, S::kV>;
    constexpr int kHalves = DP / 64;
    constexpr uint32_t kHalfBytes = kTile * 128;
    extern __shared__ uint8_t s_raw[];
    __shared__ __align__(8) uint64_t s_bars[B::bytes / 8];
    __shared__ Load s_loads[kLoads];
    __shared__ uint32_t s_takes[2][kTakes];
    __shared__ RowJob s_jobs[2][kJobs];
    __shared__ uint32_t s_last[2][2 * kJobs];      // slot of the values of a job's last tile: read up to kJobs jobs later
    __shared__ Prologue s_pro;
    __shared__ uint32_t s_tmem, s_scan[(kThreads + 31) / 32];
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
        mine = add_tiles(mine, sequence_tiles(d, r));
    }
    if (warp == kWarpSchedule) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (warp == kWarpV) {
        for (int i = lane; i < B::bytes / 8; i += 32)
            mbar_init(bar + 8 * i, i < B::ones ? 1 : i < B::p_full / 8 ? 2 : 4);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kWarpK && lane < 6) {
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
        if (lane >= o) before = add_tiles(before, up);
    }
    if (lane == 31) s_scan[warp] = before;
    before -= mine;
    __syncthreads();
    uint32_t total = 0;
#pragma unroll
    for (int i = 0; i < (kThreads + 31) / 32; ++i) {
        if (i == warp) before += total;
        total = add_tiles(total, s_scan[i]);
    }
    const bool too_many = countable(total) != total;
    if (warp == kWarpSchedule) {
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
                if (too_many) atomicOr(p.status, TSW_KV_BAD_ROWS);
                base[batch + 1] = prefix_total;
            }
        }
    }
    if (blockIdx.x == 0) {
        uint32_t* base = (uint32_t*)((uint8_t*)a.workspace + w.own_base);
        uint32_t at = before;
#pragma unroll 1
        for (uint32_t b = b_lo; b < b_hi; ++b) {
            base[b] = too_many ? 0 : at;
            SeqRows r;
            read_rows(a.batch, b, a.max_q, a.cache.page_size, r);
            at += sequence_tiles(d, r);
        }
    }
#pragma unroll 1
    for (int s = 0; s < 2; ++s) {
        const Range g = range_at(d, w.own_pair, countable(total), blockIdx.x, s);
        if (g.end > g.x && g.x >= before && g.x < before + mine) find_start(d, b_lo, b_hi, g.x - before, g.end - g.x, s_pro.own[s]);
    }
    fence_before();
    __syncthreads();
    fence_after();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = uniform(s_tmem);

    if (warp == kWarpSchedule) {
        // ---------------------------------------------------------------- scheduling, by one thread
        if (elect()) {
            Walk walk(d, s_pro);
            Job j;
            int tile;
            uint32_t n = 0, takes[2] = {0, 0}, jobs[2] = {0, 0};
            Ring k{0, 0}, v{0, 0};
            bool use[2], ok = true, more = true;
#pragma unroll 1
            while (ok && more) {
                more = walk.next(d, s_pro, j, tile, use[0], use[1]);
                if (!more) use[0] = use[1] = true;                    // the end is told to everyone
                ok = wait_alone(bar + B::load_empty + 8 * (n % kLoads), (n / kLoads & 1) ^ 1, gave_up);
                if (!ok) break;
                s_loads[n % kLoads] = more ? make_load(j, tile, walk.pair, use[1]) : Load{kLoadEnd, 0, 0, 0};
                mbar_arrive(bar + B::load_full + 8 * (n % kLoads));
                ++n;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    if (!ok || (!use[s] && !walk.pair)) continue;
                    if (use[s]) {
                        if (!more || tile == j.kt0) {
                            const uint32_t i = jobs[s]++, at = s * kJobs + i % kJobs;
                            ok = wait_alone(bar + B::job_empty + 8 * at, (i / kJobs & 1) ^ 1, gave_up);
                            if (!ok) continue;
                            RowJob r = {};
                            if (more) r = make_row_job(d, j, walk.pair, s, blockIdx.x);
                            s_jobs[s][i % kJobs] = r;
                            mbar_arrive(bar + B::job_full + 8 * at);
                        }
                        if (more && tile + 1 == min(j.kt1, seen_by(j, walk.pair, s))) s_last[s][(jobs[s] - 1) % (2 * kJobs)] = v.slot;
                    }
                    const uint32_t i = takes[s]++, at = s * kTakes + i % kTakes;
                    ok = wait_alone(bar + B::take_empty + 8 * at, (i / kTakes & 1) ^ 1, gave_up);
                    if (!ok) continue;
                    s_takes[s][i % kTakes] = more ? make_take(j, tile, use[s], walk.pair, k.slot, v.slot) : (uint32_t)kTakeEnd;
                    mbar_arrive(bar + B::take_full + 8 * at);
                }
                k.step(S::kK);
                v.step(S::kV);
            }
        }
        __syncwarp();
    } else if (warp == kWarpK || warp == kWarpV) {
        // ---------------------------------------------------------------- keys and values
        const bool is_v = warp == kWarpV;
        const uint32_t stages = is_v ? S::kV : S::kK;
        const uint32_t at = is_v ? v_at : k_at, full = bar + (is_v ? B::v_full : B::k_full), empty = bar + (is_v ? B::v_empty : B::k_empty);
        Ring ring{0, 0};
#pragma unroll 1
        for (uint32_t n = 0;; ++n) {
            if (!wait(bar + B::load_full + 8 * (n % kLoads), n / kLoads & 1, gave_up)) break;
            const Load u = s_loads[n % kLoads];
            __syncwarp();
            if (lane == 0) mbar_arrive(bar + B::load_empty + 8 * (n % kLoads));
            if (u.flags & kLoadEnd) break;
            const bool own = u.flags & kLoadOwn;
            const tsw_kv_pages& pg = own ? a.cache : a.prefix;
            const CUtensorMap* map = own ? (is_v ? &p.v_own : &p.k_own) : (is_v ? &p.v_prefix : &p.k_prefix);
            const int shift = own ? p.own_shift : p.prefix_shift, box = min(1 << shift, kTile);
            const int boxes = (load_keys(u.flags) + box - 1) / box, first = u.tile * kTile >> shift, in_page = u.tile * kTile & ((1 << shift) - 1);
            const int* table = (own ? (const int*)a.batch.page_table + (uint64_t)u.b * a.batch.table_stride : (const int*)a.prefix_table) + first;
            int page = lane < boxes ? table[lane] : 0;                // before the wait: its latency passes under it
            if (!wait(empty + 8 * ring.slot, ring.phase ^ 1, gave_up)) break;
            // Each stream has a barrier to a slot: it takes note of every phase of the ones it waits for, so their parities
            // are never mistaken.  Tiles of a list in pairs are on the first stream's for both.
            const uint32_t done = full + 8 * (u.flags & kLoadSecond ? stages + ring.slot : ring.slot);
            if (lane == 0) {
                if (!(u.flags & kLoadPair)) mbar_arrive(empty + 8 * ring.slot);       // the other stream has nothing to do with it
                mbar_expect(done, boxes * box * 128 * kHalves);
            }
            __syncwarp();
#pragma unroll 1
            for (int i = lane; i < boxes; i += 32) {
                if (i >= 32) page = table[i];
                // a number outside the cache is recorded; the copy unit fills such a box with zeros
                if ((uint32_t)page >= pg.pages) { atomicOr(p.status, TSW_KV_BAD_PAGE); page = pg.pages; }
                const uint32_t dst = at + ring.slot * S::kTileBytes + i * box * 128;
#pragma unroll
                for (int h = 0; h < kHalves; ++h)
                    load_box4(dst + h * kHalfBytes, map, h * 64, in_page, load_head(u.flags), page, done);
            }
            ring.step(stages);
        }
    } else if (warp >= kWarpProducts) {
        // ---------------------------------------------------------------- products of one stream, by one thread
        // A stream has two S buffers of half a tile's keys, taken in turn; weights go back over their S.  The S product of a
        // unit goes out in front of the O product of the unit before it, so that there is always one S for the rows to work
        // on; it may overwrite the weights of the unit two before, whose O product is ahead of it in the tensor pipe, which
        // takes them in order.  Nothing waits for a next tile while an O product is held back: where it is not there yet,
        // the O product goes first.
        constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : 1u << 7 | 1u << 10;
        constexpr uint32_t kDescS = 1u << 4 | kType | (kHalf / 8) << 17 | (kTile / 16) << 24;
        constexpr uint32_t kDescO = 1u << 4 | kType | 1u << 16 | (DP / 8) << 17 | (kTile / 16) << 24;
        const int s = warp - kWarpProducts;
        if (elect()) {
            const uint32_t t_s = tmem + s * 256, t_o = t_s + 128, q_lo = desc_lo(q_at + s * S::kTileBytes, 16);
            const uint32_t b_p = bar + B::p_full + 16 * s, b_o = bar + B::o_full + 16 * s, b_s = bar + B::s_full + 16 * s;
            const uint32_t b_tf = bar + B::take_full + 8 * kTakes * s, b_te = bar + B::take_empty + 8 * kTakes * s;
            uint32_t k_ph = 0, v_ph = 0, q_ph = 0;                // phases of the barriers, a bit each
            uint32_t n = 0;                                       // units whose S product has gone out
            uint32_t held_lo = 0, held_slot = 0;                  // the unit before, whose O product has not
            int held_steps = 0;                                   // 0: none
            bool held_first = false, held_last = false, held_wait = false, held_pair = false, ok = true;
            auto see_v = [&](uint32_t slot, bool pair) {
                const uint32_t x = (pair ? 0 : s * S::kV) + slot;
                ok = wait_alone(bar + B::v_full + 8 * x, v_ph >> x & 1, gave_up);
                v_ph ^= 1u << x;
                return ok;
            };
            auto product_o = [&]() {
                const uint32_t buf = (n - 1) & 1, t_p = t_s + buf * kHalf;
                if (held_wait && !see_v(held_slot, held_pair)) return;
                ok = wait_alone(b_p + 8 * buf, (n - 1) >> 1 & 1, gave_up);
                if (!ok) return;
                fence_after();
                if (held_steps == kHalf / 16) {
#pragma unroll
                    for (int i = 0; i < kHalf / 16; ++i) mma_ts(t_o, t_p + i * 8, desc(held_lo + (i * 2048 >> 4)), kDescO, i > 0 || !held_first);
                } else {
#pragma unroll 1
                    for (int i = 0; i < held_steps; ++i) mma_ts(t_o, t_p + i * 8, desc(held_lo + (i * 2048 >> 4)), kDescO, i > 0 || !held_first);
                }
                mma_commit(b_o + 8 * buf);
                if (held_last) mma_commit(bar + B::v_empty + 8 * held_slot);
                held_steps = 0;
            };
#pragma unroll 1
            for (uint32_t t = 0;; ++t) {
                const uint32_t at = t % kTakes, par = t / kTakes & 1;
                if (held_steps && !mbar_test(b_tf + 8 * at, par)) product_o();
                ok = ok && wait_alone(b_tf + 8 * at, par, gave_up);
                if (!ok) break;
                const uint32_t u = s_takes[s][at];
                mbar_arrive(b_te + 8 * at);
                const bool pair = u & kTakePair, first = u & kTakeFirst;
                const uint32_t slot = k_slot(u), x = (pair ? 0 : s * S::kK) + slot;
                if (held_steps && ((u & (kTakeEnd | kTakeSkip | kTakeFirst)) || !mbar_test(bar + B::k_full + 8 * x, k_ph >> x & 1))) product_o();
                if (!ok || (u & kTakeEnd)) break;
                ok = wait_alone(bar + B::k_full + 8 * x, k_ph >> x & 1, gave_up);
                if (!ok) break;
                k_ph ^= 1u << x;
                if (u & kTakeSkip) {                              // the other row tile's alone
                    mbar_arrive(bar + B::k_empty + 8 * slot);
                    if (!see_v(v_slot(u), pair)) break;
                    mbar_arrive(bar + B::v_empty + 8 * v_slot(u));
                    continue;
                }
                if (first) {
                    ok = wait_alone(bar + B::q_full + 8 * s, q_ph, gave_up);
                    if (!ok) break;
                    q_ph ^= 1;
                }
                const int keys = take_keys(u), halves = units_of(keys);
#pragma unroll 1
                for (int h = 0; h < halves; ++h) {
                    const int mine = min(kHalf, keys - h * kHalf);
                    const bool tail = mine & 15;                  // the rows will clear what lies behind: the values have to be there
                    if (tail && (h == 0 || (held_steps && held_wait))) {       // else the O product of the lower half has seen them
                        const uint32_t y = (pair ? 0 : s * S::kV) + v_slot(u);
                        if (held_steps && !mbar_test(bar + B::v_full + 8 * y, v_ph >> y & 1)) product_o();
                        if (ok && (h == 0 || held_steps)) {
                            see_v(v_slot(u), pair);
                            if (h) held_wait = false;
                        }
                        if (!ok) break;
                    }
                    const uint32_t k_lo = desc_lo(k_at + slot * S::kTileBytes + h * kHalf * 128, 16), t_x = t_s + (n & 1) * kHalf;
                    fence_after();
#pragma unroll
                    for (int i = 0; i < DP / 16; ++i) {
                        const uint32_t off = ((i / 4) * kHalfBytes + (i % 4) * 32) >> 4;
                        mma_ss(t_x, desc(q_lo + off), desc(k_lo + off), kDescS, i > 0);
                    }
                    mma_commit(b_s + 8 * (n & 1));
                    if (h + 1 == halves) mma_commit(bar + B::k_empty + 8 * slot);
                    if (held_steps) product_o();
                    if (!ok) break;
                    held_lo = desc_lo(v_at + v_slot(u) * S::kTileBytes + h * kHalf * 128, kHalfBytes);
                    held_slot = v_slot(u);
                    held_steps = (mine + 15) / 16;
                    held_first = first && h == 0;
                    held_last = h + 1 == halves;
                    held_wait = h == 0 && !tail;
                    held_pair = pair;
                    ++n;
                }
                if (!ok) break;
            }
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------------- rows: one thread each
        const int s = warp >> 2, row = tid & 127, group = w.group;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;                 // this warp's quarter of the tensor memory's lanes
        const uint32_t t_s = tmem + lanes + s * 256, t_o = t_s + 128;
        const uint32_t b_s = bar + B::s_full + 16 * s, b_p = bar + B::p_full + 16 * s, b_o = bar + B::o_full + 16 * s;
        const uint32_t b_jf = bar + B::job_full + 8 * kJobs * s, b_je = bar + B::job_empty + 8 * kJobs * s;
        const float c = a.scale * 1.4426950408889634f;
        const int tok_in_tile = row / group, head_in_group = row - tok_in_tile * group;
        const bool loads_q = (warp & 3) == 0;                             // the warp that fetches the stream's queries
        uint32_t count = 0, asked = 0;                                    // units so far; jobs whose queries are on their way
        auto load_q = [&](uint32_t i) {                                   // of job i, which has been read or seen to be there
            const RowJob& j = s_jobs[s][i % kJobs];
            if (lane == 0 && j.units) {
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
            if (!j.units) break;
            const int tok = j.tok + tok_in_tile;
            const bool mine = tok_in_tile < j.tokens;
            const bool warp_on = (warp & 3) * 32 < j.tokens * group;
            int left = keys_seen(j, tok);                                 // keys this row sees from here on
            float top = -INFINITY, sum = 0.f;
#pragma unroll 1
            for (int unit = 0; unit < j.units; ++unit, ++count, left -= kHalf) {
                const uint32_t buf = count & 1, t_x = t_s + buf * kHalf;
                ok = wait(b_s + 8 * buf, count >> 1 & 1, gave_up);
                if (!ok) break;
                fence_after();
                // The job's last S is there, so its queries are done with: fetch the next job's, if it is known yet.
                if (loads_q && unit == j.units - 1 && __all_sync(~0u, mbar_try(b_jf + 8 * ((i + 1) % kJobs), (i + 1) / kJobs & 1))) load_q(i + 1);
                if (warp_on) {
                    float x[kHalf];
#pragma unroll
                    for (int k = 0; k < kHalf; k += 32) tmem_ld32((uint32_t*)x + k, t_x + k);
                    tmem_wait_ld();
                    if (__any_sync(~0u, left < kHalf)) {
#pragma unroll
                        for (int k = 0; k < kHalf; ++k)
                            if (k >= left) x[k] = -INFINITY;
                    }
                    float m0 = x[0], m1 = x[1], m2 = x[2], m3 = x[3];
#pragma unroll
                    for (int k = 4; k < kHalf - 4; k += 8) {
                        m0 = max3(m0, x[k], x[k + 4]);
                        m1 = max3(m1, x[k + 1], x[k + 5]);
                        m2 = max3(m2, x[k + 2], x[k + 6]);
                        m3 = max3(m3, x[k + 3], x[k + 7]);
                    }
                    m0 = max3(m0, x[kHalf - 4], x[kHalf - 3]);
                    const float here = max3(fmaxf(m0, m1), fmaxf(m2, m3), fmaxf(x[kHalf - 2], x[kHalf - 1]));
                    if (unit == 0) {
                        top = here;
                    } else {
                        const bool grow = (here - top) * c > kGrow<T>;              // also from -inf; never between two of them
                        if (__any_sync(~0u, grow)) {
                            const float f = grow ? exp2_fast((top - here) * c) : 1.f;
                            if (grow) top = here;
                            sum *= f;
                            ok = wait(b_o + 8 * ((count - 1) & 1), (count - 1) >> 1 & 1, gave_up);
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
                    // The maximum comes off before the scale: behind it, top c is rounded, from 2^24 on by more than 16 bits can take up,
                    // and weights would be infinite.  32 operations more to 64 keys: 4096 rows behind 16384 tokens 1440 -> 1463 us,
                    // and no less with a branch for the rows that need it.
                    const float off = top == -INFINITY ? 0.f : -top;
                    const uint64_t c2 = two(c, c), off2 = two(off, off), raise2 = two(kRaise<T>, kRaise<T>);
                    uint64_t s0 = 0, s1 = 0;
#pragma unroll
                    for (int k = 0; k < kHalf / 32; ++k) {
                        uint32_t packed[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            const float2 f0 = split(fma2(add2(two(x[32 * k + e], x[32 * k + e + 1]), off2), c2, raise2));
                            const float2 f1 = split(fma2(add2(two(x[32 * k + e + 2], x[32 * k + e + 3]), off2), c2, raise2));
                            const float e0 = exp2_fast(f0.x), e1 = exp2_fast(f0.y), e2 = exp2_fast(f1.x), e3 = exp2_fast(f1.y);
                            s0 = add2(s0, two(e0, e1));
                            s1 = add2(s1, two(e2, e3));
                            packed[e / 2] = pack2<T>(e0, e1);
                            packed[e / 2 + 1] = pack2<T>(e2, e3);
                        }
                        tmem_st16(t_x + 16 * k, packed);
                    }
                    const float2 s01 = split(add2(s0, s1));
                    sum += s01.x + s01.y;
                    tmem_wait_st();
                }
                const int keys = j.keys - unit * kHalf;
                if (keys < kHalf && (keys & 15)) {
                    // Rows of V behind the last key hold whatever their page holds, and a weight of zero does not silence an
                    // infinity: clear what the product's last step would read.  (A pair's streams both do; they write the same.)
                    // They are there: the S product of such a unit waits for them too.
                    const int rows = 16 - (keys & 15);
                    const uint32_t at = v_at + s_last[s][i % (2 * kJobs)] * S::kTileBytes + ((unit & 1) * kHalf + keys) * 128;
#pragma unroll 1
                    for (int e = row; e < rows * 8; e += 128) {
#pragma unroll
                        for (int h = 0; h < kHalves; ++h)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at + h * kHalfBytes + e * 16), "r"(0) : "memory");
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(b_p + 8 * buf);
            }
            if (!ok) break;
            // ---- the range's result: into the output when it is all there is, else by row (an item's first
            // range) or by stream (one that continues)
            ok = wait(b_o + 8 * ((count - 1) & 1), (count - 1) >> 1 & 1, gave_up);
            if (!ok) break;
            fence_after();
            if (!warp_on) continue;
            uint8_t* out = nullptr;
            float f = 1.f;
            if (mine) {
                uint8_t* ws = (uint8_t*)a.workspace;
                const uint32_t head = j.head * group + head_in_group;
                const uint64_t row_at = (uint64_t)tok * a.q_heads + head;
                if (j.place == kPlaceDirect) {
                    out = (uint8_t*)(a.out + (uint64_t)tok * a.out_token_stride + (uint64_t)head * a.out_head_stride);
                    f = sum == 0.f ? 0.f : 1.f / sum;
                    if (a.lse) ((float*)a.lse)[row_at] = sum == 0.f ? -INFINITY : (top * c - kRaise<T> + log2f(sum)) * 0.6931471805599453f;
                } else {
                    const bool home = j.place == kPlaceHome;
                    const uint64_t at = home ? home_index(d, j.own, row_at, a.q_heads) : part_index(d, j.own, j.place, row);
                    out = ws + (home ? w.home_o : w.part_o) + 4 * at * a.head_dim;
                    *((float2*)(ws + (home ? w.home_ml : w.part_ml)) + at) = make_float2(top == -INFINITY ? -INFINITY : top * c - kRaise<T>, sum);
                }
            }
#pragma unroll 1
            for (int k = 0; k < DP; k += 64) {
                float o[64];
                tmem_ld32((uint32_t*)o, t_o + k);
                tmem_ld32((uint32_t*)o + 32, t_o + k + 32);
                tmem_wait_ld();
                if (!out) continue;
                const int left_e = (int)a.head_dim - k;                           // a multiple of 8
                if (j.place == kPlaceDirect) {
#pragma unroll
                    for (int e = 0; e < 64; e += 8)
                        if (e < left_e)
                            *(uint4*)(out + 2 * (k + e)) = make_uint4(pack2<T>(o[e] * f, o[e + 1] * f), pack2<T>(o[e + 2] * f, o[e + 3] * f),
                                                                      pack2<T>(o[e + 4] * f, o[e + 5] * f), pack2<T>(o[e + 6] * f, o[e + 7] * f));
                } else {
#pragma unroll
                    for (int e = 0; e < 64; e += 4)
                        if (e < left_e) *(float4*)(out + 4 * (k + e)) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
            }
            fence_before();
        }
    }
    if (*gave_up) {              // what is in flight lands before the CTA ends
        const unsigned long long t0 = now();
        while (now() - t0 < kDrainNs) {}
    }
    fence_before();
    __syncthreads();
    if (tid == 0 && *gave_up) atomicOr(p.status, TSW_KV_WAIT_GAVE_UP);
    if (warp == kWarpSchedule) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// ---------------------------------------------------------------------------------------------
// Joining the partial results of a row: eight lanes to a row, four rows (heads of one token) to a warp, so that
// a warp has many loads under way: the work is a handful of dependent loads to a row, not arithmetic.  The lanes take
// the parts' maxima and sums side by side, and DP / 8 elements of the head each in the sum over the parts, which
// goes in the order of the ranges: the result does not depend on which finished first.  What does not come from the tile
// kernel is worked out while it still runs.
//
// `many`: a warp takes a token with all its heads.  Without a prefix nearly every row is complete already, and what
// the others cost is the search that finds it so, which is then made once to a token.  Where rows have to be joined, or
// tokens are few, the heads go side by side: 500 rows of an encoder's 22.8 us, 28.7 the other way; 32 sequences behind 2048
// tokens 70.6 and 171.9.  Without a prefix, side by side / a warp to a token, us, 32 heads of 128 in bf16, and 32 on 8:
//   tokens                  1024          2048          4096          8192
//   one causal text         50 / 65       93 / 99       249 / 245     730 / 712
//   on 8 key heads          50 / 67       109 / 116     274 / 268     762 / 738
//   texts of 128 tokens     27.8 / 29.7   39.9 / 37.9   64.5 / 56.4   105 / 87
constexpr int kJoinThreads = 128, kJoinWarps = kJoinThreads / 32;
constexpr uint32_t kManyTokens = 4096;
template <typename T, int DP>
__global__ void __launch_bounds__(kJoinThreads) combine_kernel(const __grid_constant__ tsw_prefix_attention_args a, const __grid_constant__ Deal d, bool many) {
    constexpr int kVec = DP / 32;                    // float4s of a lane: element 4 * (sub + 8 * i)
    const int lane = threadIdx.x & 31, sub = lane & 7, warp = threadIdx.x >> 5;
    const int tok = many ? (int)(blockIdx.x * kJoinWarps) + warp : (int)blockIdx.x;
    const AttentionLayout& w = d.w;
    const int b = tok < (int)a.batch.tokens ? find_sequence((const int*)a.batch.cu_q, a.batch.batch, tok) : -1;
    SeqRows r = {};
    if (b >= 0) read_rows(a.batch, b, a.max_q, a.cache.page_size, r);
    if (b < 0 || tok >= r.first + r.n) {
        // Nothing to join, but what comes behind on the stream is ordered behind this grid alone: it ends after the tile kernel.
        asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    uint32_t before = 0;
#pragma unroll 1
    for (int rt = (int)((uint32_t)(tok - r.first) / (uint32_t)own_item_tokens(d)), i = lane; i < rt; i += 32) {
        const Cut c = cut_own(d, r, i);
        before += max(c.kt_a, c.kt_b);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) before += __shfl_xor_sync(~0u, before, o);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint8_t* ws = (const uint8_t*)a.workspace;
    const uint32_t* base = (const uint32_t*)(ws + w.own_base);
    const uint32_t own_first = base[b], own_total = base[a.batch.batch], prefix_total = base[a.batch.batch + 1];
    const int from = many ? 0 : (int)blockIdx.y * 4 * kJoinWarps + 4 * warp, to = many ? (int)a.q_heads : from + 4;
#pragma unroll 1
    for (int head0 = from; head0 < to; head0 += 4) {
        const int head = head0 + (lane >> 3);
        const uint32_t kv_head = min((uint32_t)head, a.q_heads - 1) / w.group;
        const Parts own = own_parts(d, r, tok, kv_head, own_first, before, own_total);
        Parts pre = {};
        if (a.prefix_len) pre = prefix_parts(d, tok, kv_head, prefix_total);
        // without a prefix, a row that one range holds has been written by the tile kernel itself
        const bool on = head < (int)a.q_heads && (a.prefix_len || !own.has || own.first != own.last);
        if (!__any_sync(~0u, on)) continue;
        const int n0 = on && pre.has ? (int)(pre.last - pre.first) + 1 : 0, n = n0 + (on && own.has ? (int)(own.last - own.first) + 1 : 0);
        int most = n;
        most = max(most, __shfl_xor_sync(~0u, most, 8));
        most = max(most, __shfl_xor_sync(~0u, most, 16));
        const uint64_t row = (uint64_t)tok * a.q_heads + head;
        // The i-th part: of the prefix list first, in each list the one by row, then those of the ranges that continue.
        const uint32_t in_group = head - kv_head * w.group;
        const uint64_t home0 = home_index(d, 0, row, a.q_heads), home1 = home_index(d, 1, row, a.q_heads);
        auto part = [&](int i) -> uint64_t {             // its place; bit 63: among those of the ranges that continue
            const bool l = i >= n0;
            const int k = l ? i - n0 : i;
            if (k == 0) return l ? home1 : home0;
            const Parts& q = l ? own : pre;
            return part_index(d, l, part_place(l ? w.own_pair : w.prefix_pair, q.first + k, q.half), q.place * w.group + in_group) | 1ull << 63;
        };
        float top = -INFINITY, sum = 0.f;
        float4 acc[kVec];
#pragma unroll
        for (int e = 0; e < kVec; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int i0 = 0; i0 < most; i0 += 8) {
            float2 mine = make_float2(-INFINITY, 0.f);
            uint64_t at = 0;
            if (i0 + sub < n) {
                at = part(i0 + sub);
                mine = ((const float2*)(ws + (at >> 63 ? w.part_ml : w.home_ml)))[at & ~(1ull << 63)];
            }
            float next = fmaxf(top, mine.x);
#pragma unroll
            for (int o = 4; o; o >>= 1) next = fmaxf(next, __shfl_xor_sync(~0u, next, o));
            const float base_m = next == -INFINITY ? 0.f : next;
            const float keep = exp2_fast(top - base_m), f = mine.x == -INFINITY && mine.y == 0.f ? 0.f : exp2_fast(mine.x - base_m);
            float add = mine.y * f;
#pragma unroll
            for (int o = 4; o; o >>= 1) add += __shfl_xor_sync(~0u, add, o);
            top = next;
            sum = sum * keep + add;
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                acc[e].x *= keep;
                acc[e].y *= keep;
                acc[e].z *= keep;
                acc[e].w *= keep;
            }
            const int m = min(8, most - i0);
#pragma unroll 4
            for (int i = 0; i < m; ++i) {
                const float fi = __shfl_sync(~0u, f, (lane & 24) + i);
                const uint64_t from = __shfl_sync(~0u, at, (lane & 24) + i);
                if (i0 + i >= n) continue;
                const float* o = (const float*)(ws + (from >> 63 ? w.part_o : w.home_o)) + (from & ~(1ull << 63)) * a.head_dim;
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    const int at_e = 4 * (sub + 8 * e);
                    if (at_e >= (int)a.head_dim) continue;
                    const float4 v = *(const float4*)(o + at_e);
                    acc[e].x = fmaf(v.x, fi, acc[e].x);
                    acc[e].y = fmaf(v.y, fi, acc[e].y);
                    acc[e].z = fmaf(v.z, fi, acc[e].z);
                    acc[e].w = fmaf(v.w, fi, acc[e].w);
                }
            }
        }
        if (!on) continue;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            const int at_e = 4 * (sub + 8 * e);
            if (at_e >= (int)a.head_dim) continue;
            const uint2 v = make_uint2(pack2<T>(acc[e].x * inv, acc[e].y * inv), pack2<T>(acc[e].z * inv, acc[e].w * inv));
            *(uint2*)(a.out + (uint64_t)tok * a.out_token_stride + (uint64_t)head * a.out_head_stride + 2 * at_e) = v;
        }
        if (a.lse && sub == 0) ((float*)a.lse)[row] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
    }
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
cudaError_t launch_tiles(int device, const Params& p, cudaStream_t stream) {
    static std::atomic<uint64_t> ready{0};          // devices on which the kernel has been given its shared memory
    cudaError_t err = cudaSuccess;
    if (!(ready.load(std::memory_order_relaxed) >> device & 1)) {
        err = cudaFuncSetAttribute(attention_tiles_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<DP>::kSmem);
        if (err != cudaSuccess) return err;
        ready.fetch_or(1ull << device, std::memory_order_relaxed);
    }
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
    const bool many = !p.a.prefix_len && p.a.batch.tokens >= kManyTokens;
    cfg.gridDim = many ? dim3((p.a.batch.tokens + kJoinWarps - 1) / kJoinWarps)
                       : dim3(p.a.batch.tokens, (p.a.q_heads + kJoinThreads / 8 - 1) / (kJoinThreads / 8));
    cfg.blockDim = dim3(kJoinThreads);
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, combine_kernel<T, DP>, p.a, p.d, many);
}

}  // namespace

cudaError_t launch_prefix_attention_tiles(int device, const tsw_prefix_attention_args& a, const AttentionLayout& w, uint32_t* status, cudaStream_t stream) {
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
    if (a.head_dim <= 64) return a.dtype == TSW_F16 ? launch_tiles<__half, 64>(device, p, stream) : launch_tiles<__nv_bfloat16, 64>(device, p, stream);
    return a.dtype == TSW_F16 ? launch_tiles<__half, 128>(device, p, stream) : launch_tiles<__nv_bfloat16, 128>(device, p, stream);
}

}  // namespace tsw
