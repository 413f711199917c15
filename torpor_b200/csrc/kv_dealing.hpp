// How the tile kernel's work is dealt out (kv_attention.cu): plain integer code that the kernel's warps, the
// joining kernel and the host (tests) run alike.
#ifndef TORPOR_KV_DEALING_HPP_
#define TORPOR_KV_DEALING_HPP_

#include <algorithm>
#include <cstdint>
#include <cstring>

#include "kv_attention.hpp"

#ifdef __CUDACC__
#define TSW_HD __host__ __device__ __forceinline__
#define TSW_HD_CALL __host__ __device__ __noinline__      // one copy: the kernels' code is fetched cold at every launch
#else
#define TSW_HD inline
#define TSW_HD_CALL
#endif

#ifdef __CUDA_ARCH__
#define TSW_ROLLED _Pragma("unroll 1")
#else
#define TSW_ROLLED
#endif

namespace tsw {

constexpr int kTile = 128;                    // keys in a step, rows in a tile

TSW_HD int imin(int a, int b) { return a < b ? a : b; }
TSW_HD int imax(int a, int b) { return a > b ? a : b; }

TSW_HD uint32_t trailing_ones(uint32_t x) {
#ifdef __CUDA_ARCH__
    return __clz(__brev(~x));
#else
    return ~x ? __builtin_ctz(~x) : 32;
#endif
}

// Tiles of a list.  Sequences that keep apart stay below this (attention_layout sees to it); rows claimed by many sequences of
// a wild table may not: their sum stops here, and a list that got so far is not dealt out at all.  For the joining kernel
// every sequence then begins at 0 of kMaxTiles, which keeps what it works out inside its tables without a look of its own.
constexpr uint32_t kMaxTiles = 0x7fffffff;
TSW_HD uint32_t add_tiles(uint32_t a, uint32_t b) { return a + b < kMaxTiles ? a + b : kMaxTiles; }      // a, b <= kMaxTiles
TSW_HD uint32_t countable(uint32_t total) { return total < kMaxTiles ? total : 0; }

// Longest sequence: key numbers are 32 bits, and loops step past the end by less than 256.
constexpr int kMaxKeys = 0x7fffff00;

// Rows and length of one sequence, made safe: whatever the tables hold, 0 <= first, first + n <= tokens,
// n <= max_q and 0 <= len <= what the page table covers, kMaxKeys at most.  Returns what had to be changed (TSW_KV_*).
struct SeqRows { int first, n, len; };
TSW_HD uint32_t read_rows(const tsw_kv_batch& t, int b, uint32_t max_q, uint32_t page_size, SeqRows& r) {
    const int* cu = (const int*)t.cu_q;
    const int lo = cu[b], hi = cu[b + 1];
    int len = ((const int*)t.seq_lens)[b];
    uint32_t bad = 0;
    r.first = lo;
    r.n = (int)((uint32_t)hi - (uint32_t)lo);
    if (lo < 0 || hi < lo || hi > (int)t.tokens || (uint32_t)r.n > max_q) {
        bad |= TSW_KV_BAD_ROWS;
        r.first = 0;
        r.n = 0;
    }
    uint64_t room = t.page_table ? (uint64_t)t.table_width * page_size : 0;
    room = room < (uint64_t)kMaxKeys ? room : (uint64_t)kMaxKeys;
    if (len < 0) {
        bad |= TSW_KV_BAD_LENGTH;
        len = 0;
    }
    if ((uint64_t)len > room) {
        bad |= TSW_KV_BAD_LENGTH;
        len = (int)room;
    }
    r.len = len;
    return bad;
}

// The sequence whose rows contain a token, looked for by 32 lanes that narrow the range 32-fold a step.  Whatever the table holds,
// cu_q[lo - 1] <= tok and cu_q[hi] > tok (where there are such entries) hold from step to step, so a sequence that is
// found has cu_q[b] <= tok < cu_q[b + 1]: only the lanes in front of the first one that sees a later row move lo.
struct Search {
    uint32_t lo, hi;
    TSW_HD explicit Search(uint32_t batch) : lo(0), hi(batch + 1) {}
    TSW_HD bool open() const { return lo < hi; }
    TSW_HD uint32_t step() const { return (hi - lo + 31) / 32; }
    TSW_HD bool vote(const int* cu_q, int tok, int lane) const {      // the first entry of this lane's piece
        const uint32_t at = lo + lane * step();
        return at < hi && cu_q[at] <= tok;
    }
    TSW_HD void take(uint32_t votes) {
        const uint32_t by = step(), lead = trailing_ones(votes);
        hi = (uint32_t)imin((int)hi, (int)(lo + lead * by));
        if (lead) lo += (lead - 1) * by + 1;
    }
    TSW_HD int sequence(uint32_t batch) const { return lo <= batch ? (int)lo - 1 : -1; }
};

// ------------------------------------------------------------------ which calls, and their layout

inline bool legal_stride(uint64_t stride, uint64_t count) { return count <= 1 || (stride && !(stride & 15)); }
inline bool legal_pages(const tsw_kv_pages& p, uint32_t heads) {
    return p.pages && p.page_size && !(p.page_size & (p.page_size - 1)) && !((p.k | p.v) & 15) && legal_stride(p.k_page_stride, p.pages) &&
           legal_stride(p.v_page_stride, p.pages) && legal_stride(p.k_token_stride, p.page_size) && legal_stride(p.v_token_stride, p.page_size) &&
           legal_stride(p.k_head_stride, heads) && legal_stride(p.v_head_stride, heads);
}

// False when the tensor-core kernel does not take the call (then the row kernel does).
inline bool attention_layout(const tsw_prefix_attention_args& a, int sms, AttentionLayout* w) {
    const uint32_t group = a.q_heads / a.kv_heads;
    if (a.head_dim > 128 || (a.head_dim & 7) || group > (uint32_t)kTile || !(a.scale > 0.f)) return false;
    // A call without any own page has no cache to describe.
    if (!legal_pages(a.cache, a.kv_heads) || (a.prefix_len && !legal_pages(a.prefix, a.kv_heads))) return false;
    if (((a.q | a.out) & 15) || !legal_stride(a.q_token_stride, a.batch.tokens) || !legal_stride(a.q_head_stride, a.q_heads) ||
        !legal_stride(a.out_token_stride, a.batch.tokens) || !legal_stride(a.out_head_stride, a.q_heads))
        return false;
    memset(w, 0, sizeof(*w));
    w->ctas = sms;
    w->group = group;
    w->tile_tokens = std::min<uint32_t>(kTile / group, a.batch.tokens);
    // max_q is an upper bound and may pass the rows there are.  Cut to them, a list of own rows in pairs means a prefix list in
    // pairs: a pair waits on the first stream's barriers for both, whose phases before it both have to know.
    const uint32_t max_q = std::min(a.max_q, a.batch.tokens);
    w->own_box_tokens = std::min(w->tile_tokens, std::max(1u, max_q));
    w->prefix_tiles = (a.prefix_len + kTile - 1) / kTile;
    // Two row tiles that share their key tiles, where there are two: with one, the streams of a CTA take
    // different key tiles.
    w->prefix_pair = a.batch.tokens > w->tile_tokens;
    w->own_pair = max_q > w->tile_tokens;
    w->part_rows = group * w->tile_tokens;
    // Tile numbers are 32 bits; no sequence is longer than kMaxKeys, however wide its table.
    const uint64_t row_tiles = (uint64_t)a.batch.tokens / w->tile_tokens + 1 + a.batch.batch;
    const uint64_t own_keys = std::min<uint64_t>((uint64_t)a.batch.table_width * a.cache.page_size, kMaxKeys);
    const uint64_t tiles = std::max<uint64_t>((own_keys + kTile - 1) / kTile, w->prefix_tiles);
    if (tiles && a.kv_heads * row_tiles > kMaxTiles / tiles) return false;
    uint64_t at = 0;
    auto part = [&](uint64_t bytes) {
        const uint64_t here = at;
        at += (bytes + 255) & ~255ull;
        return here;
    };
    // Results of one list, and of two behind a prefix.
    const uint64_t lists = a.prefix_len ? 2 : 1, rows = lists * a.batch.tokens * a.q_heads, parts = lists * 2 * w->ctas * w->part_rows;
    w->own_base = part(4ull * (a.batch.batch + 2));
    w->home_ml = part(8 * rows);
    w->home_o = part(4 * rows * a.head_dim);
    w->part_ml = part(8 * parts);
    w->part_o = part(4 * parts * a.head_dim);
    w->bytes = at;
    return true;
}

// ------------------------------------------------------------------ the dealing

struct Deal {                  // what the dealing depends on
    tsw_kv_batch batch;
    uint32_t max_q, page_size, kv_heads, prefix_len, causal;
    AttentionLayout w;
};

// An item of the own list: some rows of one sequence (one row tile, or two when dealt in pairs) and a key head.
struct Cut { int tok, n_a, n_b, kt_a, kt_b; };     // first token, tokens of the two row tiles, key tiles each sees
TSW_HD int tiles_of(int keys) { return (int)(((uint32_t)keys + kTile - 1) / kTile); }     // keys >= 0
TSW_HD int own_item_tokens(const Deal& d) { return d.w.own_pair ? 2 * d.w.tile_tokens : d.w.tile_tokens; }
TSW_HD int prefix_item_tokens(const Deal& d) { return d.w.prefix_pair ? 2 * d.w.tile_tokens : d.w.tile_tokens; }
TSW_HD Cut cut_own(const Deal& d, const SeqRows& r, int rt) {
    Cut c;
    const int per = own_item_tokens(d), lo = rt * per, left = imin(r.n - lo, per);
    c.tok = r.first + lo;
    c.n_a = imin(left, d.w.tile_tokens);
    c.n_b = left - c.n_a;
    const int past = r.len - r.n + lo;              // keys in front of the item's first row
    c.kt_a = tiles_of(d.causal ? imax(0, imin(r.len, past + c.n_a)) : r.len);
    c.kt_b = c.n_b ? tiles_of(d.causal ? imax(0, imin(r.len, past + left)) : r.len) : 0;
    return c;
}
TSW_HD_CALL inline uint32_t sequence_tiles(const Deal& d, const SeqRows& r) {     // over all key heads
    uint32_t sum = 0;
    TSW_ROLLED
    for (int rt = 0, per = own_item_tokens(d); rt * per < r.n; ++rt) {
        const Cut c = cut_own(d, r, rt);
        sum += imax(c.kt_a, c.kt_b);
    }
    return sum * d.kv_heads;
}

// A list of `total` tiles is cut into n ranges, none of them empty; range i starts at i * total / n.  The range that
// holds tile x; how many there are; the range of a CTA's stream (neighbours on different CTAs, so that few ranges
// spread over many); the streams' places for partial results, numbered by range.
TSW_HD_CALL inline uint32_t quotient(uint64_t a, uint32_t b) { return a >> 32 ? (uint32_t)(a / b) : (uint32_t)a / b; }      // 32 bits are the quick way
TSW_HD uint32_t range_start(uint32_t i, uint32_t total, uint32_t n) { return quotient((uint64_t)i * total, n); }
TSW_HD uint32_t range_of(uint32_t x, uint32_t total, uint32_t n) { return quotient(((uint64_t)x + 1) * n - 1, total); }
TSW_HD uint32_t ranges(const Deal& d, bool pair, uint32_t total) {
    const uint32_t n = pair ? d.w.ctas : 2 * d.w.ctas;
    return total < n ? total : n;
}
TSW_HD uint32_t range_index(const Deal& d, bool pair, uint32_t cta, int stream) { return pair ? cta : stream * d.w.ctas + cta; }
TSW_HD uint32_t part_place(bool pair, uint32_t range, int half) { return pair ? 2 * range + half : range; }
struct Range { uint32_t x, end; };
TSW_HD Range range_at(const Deal& d, bool pair, uint32_t total, uint32_t cta, int stream) {
    const uint32_t n = ranges(d, pair, total), i = range_index(d, pair, cta, stream);
    if (i >= n || (pair && stream)) return Range{0, 0};        // pairs: on the first stream's cursor alone
    return Range{range_start(i, total, n), range_start(i + 1, total, n)};
}

struct Job {
    int own;                 // 0: the prefix list, 1: the own list
    int head;                // key head
    int b;
    int tok, n_a, n_b;       // rows: n_a tokens from tok for the first stream, n_b more for the second (pairs only)
    int kt0, kt1;            // key tiles of this range
    int kt_a, kt_b;          // ends of what the two row tiles see
    int keys;                // keys of the whole segment
    int limit;               // row of token t sees keys below limit + t + 1; kNoLimit: all of them
};
constexpr int kNoLimit = 0x7fffffff;          // above every other limit: lengths end at kMaxKeys

struct Start { int b, rt, head, kt; uint32_t left; };      // where a stream's own range begins, and its tiles

struct Prologue {            // what a CTA works out before it starts
    Start own[2];
    Range prefix[2];
    int prefix_rt, tok0, tok1;
};

TSW_HD uint32_t prefix_rows(const Deal& d, int& tok0, int& tok1) {      // row tiles (or pairs) of the whole batch
    const int* cu = (const int*)d.batch.cu_q;
    tok0 = imin(imax(cu[0], 0), (int)d.batch.tokens);
    tok1 = imin(imax(cu[d.batch.batch], tok0), (int)d.batch.tokens);
    const uint32_t per = prefix_item_tokens(d);
    return (tok1 - tok0 + per - 1) / per;
}
// Tile `off` of the own tiles of sequences [lo, hi) begins a range of `left` tiles.
TSW_HD_CALL inline bool find_start(const Deal& d, int lo, int hi, uint32_t off, uint32_t left, Start& s) {
    TSW_ROLLED
    for (int b = lo; b < hi; ++b) {
        SeqRows r;
        read_rows(d.batch, b, d.max_q, d.page_size, r);
        TSW_ROLLED
        for (int rt = 0, per = own_item_tokens(d); rt * per < r.n; ++rt) {
            const Cut c = cut_own(d, r, rt);
            const uint32_t n = imax(c.kt_a, c.kt_b), all = n * d.kv_heads;
            if (off < all) {
                s = Start{b, rt, (int)(off / n), (int)(off % n), left};
                return true;
            }
            off -= all;
        }
    }
    return false;
}

struct Cursor {
    uint32_t x, end;
    Start s;
    SeqRows r;
    int loaded;
    TSW_HD Cursor(const Prologue& pro, int stream) : x(pro.prefix[stream].x), end(pro.prefix[stream].end), s(pro.own[stream]), loaded(-1) {}
    // Next job of the prefix list (own = false) or of the own list.
    TSW_HD bool next(const Deal& d, const Prologue& pro, bool own, Job& j) {
        if (!own) {
            if (x >= end) return false;
            const uint32_t kt_n = d.w.prefix_tiles, item = x / kt_n;
            j.own = 0;
            j.b = 0;
            j.head = item / pro.prefix_rt;
            const int rt = item % pro.prefix_rt;
            j.kt0 = x % kt_n;
            j.kt1 = imin(kt_n, j.kt0 + (end - x));
            x += j.kt1 - j.kt0;
            const int per = prefix_item_tokens(d), lo = rt * per, left = imin(pro.tok1 - pro.tok0 - lo, per);
            j.tok = pro.tok0 + lo;
            j.n_a = imin(left, d.w.tile_tokens);
            j.n_b = left - j.n_a;
            j.kt_a = kt_n;
            j.kt_b = j.n_b ? kt_n : 0;
            j.keys = d.prefix_len;
            j.limit = kNoLimit;
            return true;
        }
        while (s.left) {
            if (loaded != s.b) {
                read_rows(d.batch, s.b, d.max_q, d.page_size, r);
                loaded = s.b;
            }
            if (s.rt * own_item_tokens(d) >= r.n) {
                ++s.b;
                s.rt = 0;
                continue;
            }
            const Cut c = cut_own(d, r, s.rt);
            const int n = imax(c.kt_a, c.kt_b);
            if (n == 0 || s.head == (int)d.kv_heads) {
                ++s.rt;
                s.head = 0;
                s.kt = 0;
                continue;
            }
            j.own = 1;
            j.b = s.b;
            j.head = s.head;
            j.tok = c.tok;
            j.n_a = c.n_a;
            j.n_b = c.n_b;
            j.kt0 = s.kt;
            j.kt1 = imin(n, s.kt + (int)s.left);
            j.kt_a = c.kt_a;
            j.kt_b = c.kt_b;
            j.keys = r.len;
            j.limit = d.causal ? r.len - r.n - r.first : kNoLimit;
            s.left -= j.kt1 - j.kt0;
            s.kt = j.kt1;
            if (s.kt == n) {
                ++s.head;
                s.kt = 0;
            }
            return true;
        }
        return false;
    }
};

// The order in which a CTA's key tiles pass through the rings: first the prefix list, then the own list.  A list that
// is dealt in pairs is on the first cursor alone; otherwise the two streams' tiles take turns while both have some.
struct Walk {
    Cursor c0, c1;
    Job j0, j1;
    int kt0 = 0, kt1 = 0;
    bool live0 = false, live1 = false, need0 = true, need1, last = true, own = false, pair;
    TSW_HD Walk(const Deal& d, const Prologue& pro) : c0(pro, 0), c1(pro, 1) {
        pair = d.w.prefix_pair;
        need1 = !pair;
    }
    // The next tile: its job, its number, and which streams have a product with it.  False at the end.
    TSW_HD bool next(const Deal& d, const Prologue& pro, Job& j, int& tile, bool& use0, bool& use1) {
        need0 = need0 || (!last && live0 && kt0 == j0.kt1);
        need1 = need1 || (last && live1 && kt1 == j1.kt1);
        TSW_ROLLED
        for (;;) {
            if (need0 || need1) {               // one copy of the search for both cursors
                Cursor c = need0 ? c0 : c1;
                const bool live = c.next(d, pro, own, j);
                if (need0) {
                    c0 = c;
                    j0 = j;
                    live0 = live;
                    kt0 = live ? j.kt0 : 0;
                    need0 = false;
                } else {
                    c1 = c;
                    j1 = j;
                    live1 = live;
                    kt1 = live ? j.kt0 : 0;
                    need1 = false;
                }
                continue;
            }
            if (live0 || live1) break;
            if (own) return false;
            own = true;
            pair = d.w.own_pair;
            last = true;
            need0 = true;
            need1 = !pair;
        }
        last = last ? !live0 : live1;
        if (last) {
            j = j1;
            tile = kt1++;
        } else {
            j = j0;
            tile = kt0++;
        }
        use0 = pair ? tile < j.kt_a : !last;
        use1 = pair ? tile < j.kt_b : last;
        return true;
    }
};

// What the warps are told.  A load is one key tile for the loading warps.  A take is the same tile for the products of one
// stream; of a list that is dealt in pairs each stream is told of every tile, also of those that it has no product
// with.  Products go by half tiles (units); a half that lies behind the last key is none.
constexpr int kHalf = kTile / 2;
struct alignas(16) Load {
    uint32_t flags;          // kLoad*, keys of the tile from bit 8, key head from bit 16
    int tile, b, pad;
};
enum { kLoadOwn = 1, kLoadEnd = 2, kLoadPair = 4, kLoadSecond = 8 };      // Second: the second stream's, of a list that is not in pairs
TSW_HD int load_keys(uint32_t flags) { return (flags >> 8 & 0xff) + 1; }
TSW_HD int load_head(uint32_t flags) { return flags >> 16; }
TSW_HD int tile_keys(const Job& j, int tile) { return imin(kTile, j.keys - tile * kTile); }
TSW_HD Load make_load(const Job& j, int tile, bool pair, bool use1) {
    return Load{(j.own ? kLoadOwn : 0u) | (pair ? kLoadPair : use1 ? kLoadSecond : 0u) | (uint32_t)(tile_keys(j, tile) - 1) << 8 | (uint32_t)j.head << 16, tile, j.b, 0};
}
struct Ring {                // place in a ring of n slots
    uint32_t slot, phase;
    TSW_HD void step(uint32_t n) {
        if (++slot == n) {
            slot = 0;
            phase ^= 1;
        }
    }
};
// Bits of a take: kTake*, the tile's keys from bit 8, the slots of its keys and values from bits 16 and 24.
enum { kTakeFirst = 1, kTakeSkip = 2, kTakePair = 4, kTakeEnd = 8 };
TSW_HD int take_keys(uint32_t u) { return (u >> 8 & 0xff) + 1; }
TSW_HD uint32_t k_slot(uint32_t u) { return u >> 16 & 0xff; }
TSW_HD uint32_t v_slot(uint32_t u) { return u >> 24; }
TSW_HD int units_of(int keys) { return keys > kHalf ? 2 : 1; }
TSW_HD uint32_t make_take(const Job& j, int tile, bool use, bool pair, uint32_t k, uint32_t v) {
    return (tile == j.kt0 ? kTakeFirst : 0u) | (use ? 0u : kTakeSkip) | (pair ? kTakePair : 0u) | (uint32_t)(tile_keys(j, tile) - 1) << 8 | k << 16 | v << 24;
}
// A stream's share of a job: its rows, how many units, and where the result goes.
struct alignas(16) RowJob {
    int head, tok, tokens, units;    // units = 0: no more
    int keys, limit;                 // from the range's first key: row of token t sees keys below min(keys, limit + t), or all (kNoLimit)
    int own, place;                  // place >= 0: partial result of a range that continues an item
};
enum { kPlaceDirect = -2, kPlaceHome = -1 };

// End of what stream s sees of the job's keys (pairs: each row tile its own).
TSW_HD int seen_by(const Job& j, bool pair, int s) { return pair && s ? j.kt_b : j.kt_a; }
TSW_HD RowJob make_row_job(const Deal& d, const Job& j, bool pair, int s, uint32_t cta) {
    RowJob r;
    const int seen = seen_by(j, pair, s), end = imin(j.kt1, seen);
    r.head = j.head;
    r.tok = j.tok + (pair && s ? (int)d.w.tile_tokens : 0);
    r.tokens = pair && s ? j.n_b : j.n_a;
    r.units = 2 * (end - j.kt0 - 1) + units_of(tile_keys(j, end - 1));
    r.keys = j.keys - j.kt0 * kTile;
    r.limit = j.limit == kNoLimit ? kNoLimit : j.limit + 1 - j.kt0 * kTile;
    r.own = j.own;
    r.place = j.kt0 ? (int)part_place(pair, range_index(d, pair, cta, s), s) : !d.prefix_len && end == seen ? (int)kPlaceDirect : (int)kPlaceHome;
    return r;
}

// Keys from the range's first one on that the row of token `tok` sees.
TSW_HD int keys_seen(const RowJob& j, int tok) { return j.limit == kNoLimit ? j.keys : imin(j.keys, imax(0, j.limit + tok)); }

// Where the partial results of one row lie: of each list the ranges first .. last, its half of a pair and its
// token's place in the row tile.  `before`: own tiles of the row's sequence in front of its item (one head).
struct Parts { bool has; uint32_t first, last, half, place; };
TSW_HD uint32_t split_rows(const Deal& d, bool pair, uint32_t at, Parts& p) {      // the item of row token `at` of a list
    const uint32_t tile = at / d.w.tile_tokens;
    p.place = at - tile * d.w.tile_tokens;
    p.half = pair ? tile & 1 : 0;
    return pair ? tile >> 1 : tile;
}
TSW_HD Parts prefix_parts(const Deal& d, int tok, int kv_head, uint32_t total) {
    Parts p = {};
    int tok0, tok1;
    const uint32_t rts = prefix_rows(d, tok0, tok1);
    if (!total || tok < tok0 || tok >= tok1) return p;
    const uint32_t item = split_rows(d, d.w.prefix_pair, tok - tok0, p), x = (kv_head * rts + item) * d.w.prefix_tiles;
    const uint32_t n = ranges(d, d.w.prefix_pair, total);
    p.has = true;
    p.first = range_of(x, total, n);
    p.last = range_of(x + d.w.prefix_tiles - 1, total, n);
    return p;
}
TSW_HD Parts own_parts(const Deal& d, const SeqRows& r, int tok, int kv_head, uint32_t base, uint32_t before, uint32_t total) {
    Parts p = {};
    const Cut c = cut_own(d, r, split_rows(d, d.w.own_pair, tok - r.first, p));
    const int seen = p.half ? c.kt_b : c.kt_a;
    if (!seen) return p;
    const uint32_t x = base + before * d.kv_heads + kv_head * imax(c.kt_a, c.kt_b), n = ranges(d, d.w.own_pair, total);
    p.has = true;
    p.first = range_of(x, total, n);
    p.last = range_of(x + seen - 1, total, n);
    return p;
}
TSW_HD int list_place(const Deal& d, int list) { return d.prefix_len ? list : 0; }      // without a prefix the own list is the only one
TSW_HD uint64_t home_index(const Deal& d, int list, uint64_t row, uint32_t q_heads) { return (uint64_t)list_place(d, list) * d.batch.tokens * q_heads + row; }
TSW_HD uint64_t part_index(const Deal& d, int list, uint32_t place, uint32_t row_in_tile) {
    return ((uint64_t)list_place(d, list) * 2 * d.w.ctas + place) * d.w.part_rows + row_in_tile;
}

}  // namespace tsw
#endif
