// Key/value cache operators (C ABI): checks of arguments, choice of kernel, translation of a
// function's client addresses.  The kernels are in kv_kernels.cu.

#include "engine_internal.hpp"

#include <algorithm>
#include <atomic>

#include "kv_kernels.hpp"
#include "kv_dealing.hpp"

using namespace tsw;

namespace {

constexpr int kMaxDevices = 64;
constexpr uint32_t kMaxHeadDim = 512;
constexpr int kMaxSms = 160;    // what a workspace is sized for before the device is known

struct DeviceGuard {            // makes a device current; the caller's is put back
    int old = -1;
    cudaError_t err;
    explicit DeviceGuard(int device) {
        err = cudaGetDevice(&old);
        if (err == cudaSuccess && old == device) old = -1;
        else if (err == cudaSuccess) err = cudaSetDevice(device);
    }
    ~DeviceGuard() { if (old >= 0) cudaSetDevice(old); }
};

int sm_count(int device, int* sms) {
    static std::atomic<int> known[kMaxDevices];
    int n = known[device].load(std::memory_order_relaxed);
    if (n == 0) {
        TSW_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device));
        known[device].store(n, std::memory_order_relaxed);
    }
    *sms = n;
    return TSW_OK;
}

// Address of the device's status word; the device is current.
int status_word(int device, uint32_t** word) {
    static std::atomic<uint32_t*> known[kMaxDevices];
    uint32_t* w = known[device].load(std::memory_order_relaxed);
    if (!w) {
        TSW_CUDA(kv_status_symbol(&w));
        known[device].store(w, std::memory_order_relaxed);
    }
    *word = w;
    return TSW_OK;
}

int bad(const char* what) { return fail(TSW_ERR_INVALID, what); }

// Are the rows of an operand that is written apart?  Taken by stride, each dimension has to step over all that the
// ones before it cover; a dimension of one entry steps nowhere.
struct Steps { uint64_t stride, count; };
bool apart(uint64_t row_bytes, Steps x, Steps y, Steps z = {0, 1}) {
    Steps by[3] = {x, y, z};
    std::sort(by, by + 3, [](const Steps& l, const Steps& r) { return l.stride < r.stride; });
    unsigned __int128 covered = row_bytes;
    for (const Steps& s : by) {
        if (s.count <= 1) continue;
        if (s.stride < covered) return false;
        covered += (unsigned __int128)(s.count - 1) * s.stride;
    }
    return true;
}

int check_pages(const tsw_kv_pages& p, uint64_t row_bytes, uint32_t heads, bool written, const char* name) {
    const std::string n(name);
    if (!p.page_size || p.page_size > (1u << 20)) return fail(TSW_ERR_INVALID, n + ": page_size must be 1 to 2^20 tokens");
    if (p.pages > 0x7fffffffu) return fail(TSW_ERR_INVALID, n + ": too many pages");
    if (p.pages && (!p.k || !p.v)) return fail(TSW_ERR_INVALID, n + ": null address");
    if ((p.k | p.v | p.k_page_stride | p.k_token_stride | p.k_head_stride | p.v_page_stride | p.v_token_stride | p.v_head_stride) & 1)
        return fail(TSW_ERR_INVALID, n + ": addresses and strides must be multiples of the element size");
    for (uint64_t s : {p.k_page_stride, p.k_token_stride, p.k_head_stride, p.v_page_stride, p.v_token_stride, p.v_head_stride})
        if (s >> 40) return fail(TSW_ERR_INVALID, n + ": stride out of range");
    if (written && !(apart(row_bytes, {p.k_page_stride, p.pages}, {p.k_token_stride, p.page_size}, {p.k_head_stride, heads}) &&
                     apart(row_bytes, {p.v_page_stride, p.pages}, {p.v_token_stride, p.page_size}, {p.v_head_stride, heads})))
        return fail(TSW_ERR_INVALID, n + ": strides make heads, tokens or pages overlap");
    if (written && p.pages && p.k == p.v) return fail(TSW_ERR_INVALID, n + ": keys and values are the same memory");
    return TSW_OK;
}

int check_batch(const tsw_kv_batch& b) {
    if (b.tokens > 1u << 28 || b.batch > 0xffffffu) return bad("tokens or batch out of range");
    if (b.batch && (!b.seq_lens || !b.cu_q)) return bad("seq_lens and cu_q must be given");
    if (b.table_width && !b.page_table) return bad("page_table is null");
    if (b.batch > 1 && b.table_stride < b.table_width) return bad("table_stride is smaller than table_width");
    if ((b.page_table | b.seq_lens | b.cu_q) & 3) return bad("tables must be 4-byte aligned");
    return TSW_OK;
}

bool has_rows(const tsw_kv_batch& b) { return b.tokens && b.batch; }      // otherwise nothing is launched

int check_heads(uint32_t dtype, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim) {
    if (dtype != TSW_F16 && dtype != TSW_BF16) return bad("dtype must be TSW_F16 or TSW_BF16");
    if (!kv_heads || kv_heads > 4096 || q_heads > 65536) return bad("head counts out of range");
    if (!head_dim || head_dim > kMaxHeadDim) return bad("head_dim must be 1 to 512");
    return TSW_OK;
}

// [tokens][heads][head_dim] operand
int check_rows(const char* name, uint64_t addr, uint64_t tok, uint64_t head, const tsw_kv_batch& b, uint32_t heads, uint64_t row_bytes,
               bool written) {
    const std::string n(name);
    if (b.tokens && heads && !addr) return fail(TSW_ERR_INVALID, n + " is null");
    if ((addr | tok | head) & 1) return fail(TSW_ERR_INVALID, n + ": address and strides must be multiples of the element size");
    if ((tok >> 40) || (head >> 40)) return fail(TSW_ERR_INVALID, n + ": stride out of range");
    if (written && !apart(row_bytes, {tok, b.tokens}, {head, heads}))
        return fail(TSW_ERR_INVALID, n + ": strides make heads or tokens overlap");
    return TSW_OK;
}

#define CHECK(call)                      \
    do {                                 \
        const int _rc = (call);          \
        if (_rc != TSW_OK) return _rc;   \
    } while (0)

int check_append(const tsw_kv_append_args& a) {
    CHECK(check_heads(a.dtype, a.q_heads, a.kv_heads, a.head_dim));
    const uint64_t row = 2ull * a.head_dim;
    if (a.head_dim & 1) return bad("head_dim must be even");
    if ((a.rotary_dim & 1) || a.rotary_dim > a.head_dim) return bad("rotary_dim must be even and at most head_dim");
    if (a.rotary_dim && (!a.inv_freq || (a.inv_freq & 7))) return bad("inv_freq must be an 8-byte aligned device array");
    if (a.position_offset >> 32) return bad("position_offset out of range");
    CHECK(check_batch(a.batch));
    CHECK(check_pages(a.cache, row, a.kv_heads, true, "cache"));
    if ((a.q == 0) != (a.q_out == 0)) return bad("q and q_out go together");
    if (a.q) {
        if (!a.q_heads) return bad("q without heads");
        CHECK(check_rows("q", a.q, a.q_token_stride, a.q_head_stride, a.batch, a.q_heads, row, false));
        CHECK(check_rows("q_out", a.q_out, a.q_out_token_stride, a.q_out_head_stride, a.batch, a.q_heads, row, true));
        if (a.q == a.q_out && (a.q_token_stride != a.q_out_token_stride || a.q_head_stride != a.q_out_head_stride))
            return bad("q_out is q with other strides");
    }
    CHECK(check_rows("k", a.k, a.k_token_stride, a.k_head_stride, a.batch, a.kv_heads, row, false));
    return check_rows("v", a.v, a.v_token_stride, a.v_head_stride, a.batch, a.kv_heads, row, false);
}

int check_attention(const tsw_prefix_attention_args& a) {
    CHECK(check_heads(a.dtype, a.q_heads, a.kv_heads, a.head_dim));
    if (!a.q_heads || a.q_heads % a.kv_heads) return bad("q_heads must be a multiple of kv_heads");
    const uint64_t row = 2ull * a.head_dim;
    CHECK(check_batch(a.batch));
    CHECK(check_pages(a.cache, row, a.kv_heads, false, "cache"));
    if (a.prefix_len) {
        if (a.prefix_len > (uint32_t)kMaxKeys) return bad("prefix_len out of range");
        if (!a.prefix_table || (a.prefix_table & 3)) return bad("prefix_table must be a 4-byte aligned device array");
        CHECK(check_pages(a.prefix, row, a.kv_heads, false, "prefix"));
    }
    if (a.max_q > 0x7fffffffu) return bad("max_q out of range");
    if (!(a.scale == a.scale) || a.scale - a.scale != 0.f) return bad("scale must be finite");
    if (a.lse & 3) return bad("lse must be 4-byte aligned");
    if ((uint64_t)a.batch.tokens * a.q_heads >> 32) return bad("too many rows for one call");
    if (a.batch.tokens && a.out == a.q) return bad("out must not be q");
    CHECK(check_rows("q", a.q, a.q_token_stride, a.q_head_stride, a.batch, a.q_heads, row, false));
    return check_rows("out", a.out, a.out_token_stride, a.out_head_stride, a.batch, a.q_heads, row, true);
}

int use_device(const DeviceGuard& g, int device, int* sms) {
    if (g.err != cudaSuccess) return fail(TSW_ERR_NO_DEVICE, std::string("cudaSetDevice: ") + cudaGetErrorString(g.err));
    return sm_count(device, sms);
}

// No C++ exception leaves a C entry point.
template <typename F> int guarded(F&& f) {
    try {
        return f();
    } catch (const std::exception& ex) {
        return fail(TSW_ERR_INVALID, ex.what());
    } catch (...) {
        return TSW_ERR_INVALID;
    }
}

// The device address of an operand of `bytes` bytes at client address `addr` of a function: it has to lie
// inside one block; parameters in it that are still being swapped in are waited for on the stream.
int operand(tsw_engine* e, const char* func, uint64_t* addr, uint64_t bytes, const char* name, void* stream) {
    if (!*addr || !bytes) return TSW_OK;
    Model* m = repo().find(func);
    if (!m) return fail(TSW_ERR_UNKNOWN_MODEL, std::string("unknown function ") + func);
    auto pit = m->place.find(e->server_id);
    if (pit == m->place.end()) return fail(TSW_ERR_STATE, std::string(func) + " has no memory on this engine");
    for (size_t i = 0; i < m->blocks.size(); ++i) {
        const VBlock& b = m->blocks[i];
        if (!b.alive || *addr < b.vaddr || *addr >= b.vaddr + b.size) continue;
        if (bytes > b.vaddr + b.size - *addr) return fail(TSW_ERR_NOT_FOUND, std::string(name) + " reaches beyond its block");
        Placement& pl = placement(m, e->server_id);
        size_placement(m, pl);
        if (!pl.blocks[i].in_cuda || !pl.blocks[i].cuda) return fail(TSW_ERR_STATE, std::string(name) + ": its block is not on the device");
        for (int p : b.params) {
            const VParam& v = m->params[p];
            if (v.vaddr + v.size <= *addr || v.vaddr >= *addr + bytes) continue;
            uint64_t phys;
            int waited;
            const uint64_t vaddr = v.vaddr;
            if (e->tracking && e->track_func == func) tsw_mark_access(e, vaddr);
            CHECK(tsw_translate_async(e, func, vaddr, stream, &phys, &waited));
        }
        *addr = pl.blocks[i].cuda + (*addr - b.vaddr);
        return TSW_OK;
    }
    return fail(TSW_ERR_NOT_FOUND, std::string(name) + " is not inside any block of the function");
}

// Bytes from the first to the last element of a strided operand.  Counts of 2^31 and strides of 2^40 are legal each and
// together pass 64 bits: what does is longer than any block.
uint64_t span(uint64_t row_bytes, uint64_t n0, uint64_t s0, uint64_t n1, uint64_t s1, uint64_t n2 = 1, uint64_t s2 = 0) {
    using Wide = unsigned __int128;
    if (!n0 || !n1 || !n2) return 0;
    const Wide all = row_bytes + Wide(n0 - 1) * s0 + Wide(n1 - 1) * s1 + Wide(n2 - 1) * s2;
    return all >> 64 ? UINT64_MAX : (uint64_t)all;
}

int operand_pages(tsw_engine* e, const char* func, tsw_kv_pages& p, uint64_t row, uint32_t heads, void* stream) {
    CHECK(operand(e, func, &p.k, span(row, p.pages, p.k_page_stride, p.page_size, p.k_token_stride, heads, p.k_head_stride), "keys", stream));
    return operand(e, func, &p.v, span(row, p.pages, p.v_page_stride, p.page_size, p.v_token_stride, heads, p.v_head_stride), "values", stream);
}

int operand_batch(tsw_engine* e, const char* func, tsw_kv_batch& b, void* stream) {
    if (!b.batch) return TSW_OK;
    CHECK(operand(e, func, &b.page_table, 4 * ((uint64_t)(b.batch - 1) * b.table_stride + b.table_width), "page_table", stream));
    CHECK(operand(e, func, &b.seq_lens, 4ull * b.batch, "seq_lens", stream));
    return operand(e, func, &b.cu_q, 4ull * (b.batch + 1), "cu_q", stream);
}

int engine_ok(tsw_engine* e, const char* func, const void* args) {
    if (!e || !func || !args) return fail(TSW_ERR_INVALID, "null argument");
    if (e->plan) return fail(TSW_ERR_NO_DEVICE, "plan-only engine runs no kernels");
    return TSW_OK;
}

// Blocks lie elsewhere after the next swap-in: a graph would keep the addresses of this one, and write to what lies there by then.
int not_captured(void* stream) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    TSW_CUDA(cudaStreamIsCapturing((cudaStream_t)stream, &status));
    if (status != cudaStreamCaptureStatusNone) return fail(TSW_ERR_STATE, "a function's addresses hold until its next swap: the call cannot be captured");
    return TSW_OK;
}

}  // namespace

extern "C" {

int tsw_kv_append(int device, const tsw_kv_append_args* args, void* stream) {
    return guarded([&]() -> int {
        if (!args) return bad("null argument");
        if (device < 0 || device >= kMaxDevices) return bad("device ordinal out of range");
        CHECK(check_append(*args));
        if (!has_rows(args->batch)) return TSW_OK;
        const DeviceGuard guard(device);
        int sms;
        CHECK(use_device(guard, device, &sms));
        TSW_CUDA(launch_kv_append(*args, sms, (cudaStream_t)stream));
        return TSW_OK;
    });
}

int tsw_prefix_attention_workspace(const tsw_prefix_attention_args* args, uint64_t* bytes) {
    return guarded([&]() -> int {
        if (!args || !bytes) return bad("null argument");
        CHECK(check_attention(*args));
        AttentionLayout w;
        *bytes = attention_layout(*args, kMaxSms, &w) ? w.bytes : 0;
        return TSW_OK;
    });
}

int tsw_prefix_attention(int device, const tsw_prefix_attention_args* args, void* stream) {
    return guarded([&]() -> int {
        if (!args) return bad("null argument");
        if (device < 0 || device >= kMaxDevices) return bad("device ordinal out of range");
        CHECK(check_attention(*args));
        if (!has_rows(args->batch)) return TSW_OK;
        const DeviceGuard guard(device);
        int sms;
        CHECK(use_device(guard, device, &sms));
        AttentionLayout w;
        if (!attention_layout(*args, std::min(sms, kMaxSms), &w)) {
            TSW_CUDA(launch_prefix_attention_rows(*args, (cudaStream_t)stream));
            return TSW_OK;
        }
        if (!args->workspace || (args->workspace & 255)) return bad("workspace must be a 256-byte aligned device address");
        if (args->workspace_bytes < w.bytes) return fail(TSW_ERR_BUFFER, "workspace is smaller than tsw_prefix_attention_workspace asks for");
        uint32_t* word;
        CHECK(status_word(device, &word));
        TSW_CUDA(launch_prefix_attention_tiles(device, *args, w, word, (cudaStream_t)stream));
        return TSW_OK;
    });
}

int tsw_kv_status(int device, void* stream, uint32_t* status, int clear) {
    return guarded([&]() -> int {
        if (!status) return bad("null argument");
        if (device < 0 || device >= kMaxDevices) return bad("device ordinal out of range");
        const DeviceGuard guard(device);
        int sms;
        CHECK(use_device(guard, device, &sms));
        uint32_t* word = nullptr;
        CHECK(status_word(device, &word));
        cudaStream_t s = (cudaStream_t)stream;
        uint32_t seen = 0;
        TSW_CUDA(cudaMemcpyAsync(&seen, word, sizeof(seen), cudaMemcpyDeviceToHost, s));
        TSW_CUDA(cudaStreamSynchronize(s));
        if (clear && seen) {
            TSW_CUDA(launch_kv_status_clear(word, seen, s));      // what was seen, and nothing that came since
            TSW_CUDA(cudaStreamSynchronize(s));
        }
        *status = seen;
        return TSW_OK;
    });
}

int tsw_func_kv_append(tsw_engine* e, const char* func, const tsw_kv_append_args* args, void* stream) {
    return guarded([&]() -> int {
        CHECK(engine_ok(e, func, args));
        CHECK(check_append(*args));
        tsw_kv_append_args a = *args;
        const uint64_t row = 2ull * a.head_dim;
        const DeviceGuard guard(e->cfg.device);
        CHECK(not_captured(stream));
        Lock g1(repo().mu);
        Lock g2(e->mu);
        CHECK(operand_pages(e, func, a.cache, row, a.kv_heads, stream));
        CHECK(operand_batch(e, func, a.batch, stream));
        const bool same = a.q == a.q_out;
        CHECK(operand(e, func, &a.q, span(row, a.batch.tokens, a.q_token_stride, a.q_heads, a.q_head_stride), "q", stream));
        if (same) a.q_out = a.q;
        else CHECK(operand(e, func, &a.q_out, span(row, a.batch.tokens, a.q_out_token_stride, a.q_heads, a.q_out_head_stride), "q_out", stream));
        CHECK(operand(e, func, &a.k, span(row, a.batch.tokens, a.k_token_stride, a.kv_heads, a.k_head_stride), "k", stream));
        CHECK(operand(e, func, &a.v, span(row, a.batch.tokens, a.v_token_stride, a.kv_heads, a.v_head_stride), "v", stream));
        CHECK(operand(e, func, &a.inv_freq, 4ull * a.rotary_dim, "inv_freq", stream));
        const int rc = tsw_kv_append(e->cfg.device, &a, stream);
        if (rc == TSW_OK && has_rows(a.batch)) ++e->kernel_launches;
        return rc;
    });
}

int tsw_func_prefix_attention(tsw_engine* e, const char* func, const tsw_prefix_attention_args* args, void* stream) {
    return guarded([&]() -> int {
        CHECK(engine_ok(e, func, args));
        CHECK(check_attention(*args));
        tsw_prefix_attention_args a = *args;
        const uint64_t row = 2ull * a.head_dim;
        const DeviceGuard guard(e->cfg.device);
        CHECK(not_captured(stream));
        Lock g1(repo().mu);
        Lock g2(e->mu);
        CHECK(operand_pages(e, func, a.cache, row, a.kv_heads, stream));
        if (a.prefix_len) {
            CHECK(operand_pages(e, func, a.prefix, row, a.kv_heads, stream));
            const uint64_t n = ((uint64_t)a.prefix_len + a.prefix.page_size - 1) / a.prefix.page_size;
            CHECK(operand(e, func, &a.prefix_table, 4 * n, "prefix_table", stream));
        }
        CHECK(operand_batch(e, func, a.batch, stream));
        CHECK(operand(e, func, &a.q, span(row, a.batch.tokens, a.q_token_stride, a.q_heads, a.q_head_stride), "q", stream));
        CHECK(operand(e, func, &a.out, span(row, a.batch.tokens, a.out_token_stride, a.q_heads, a.out_head_stride), "out", stream));
        CHECK(operand(e, func, &a.lse, 4ull * a.batch.tokens * a.q_heads, "lse", stream));
        CHECK(operand(e, func, &a.workspace, a.workspace_bytes, "workspace", stream));
        const int rc = tsw_prefix_attention(e->cfg.device, &a, stream);
        AttentionLayout w;
        if (rc == TSW_OK && has_rows(a.batch)) e->kernel_launches += attention_layout(a, kMaxSms, &w) ? 2 : 1;      // tiles and joining, or rows
        return rc;
    });
}

}  // extern "C"
