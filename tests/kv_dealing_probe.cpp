// The dealing of the attention kernel's work (csrc/kv_dealing.hpp), run on the host for random batches: every
// (row tile, head, key tile) is taken exactly once, in whole units; what the joining kernel reads of a row is exactly what was written for it; every index
// stays inside its table or the workspace.
//   kv_dealing_probe SEED CASES
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>

#include "../torpor_b200/csrc/kv_dealing.hpp"

using namespace tsw;

#define REQUIRE(x)                                                              \
    do {                                                                        \
        if (!(x)) {                                                             \
            printf("case %d line %d: %s\n", g_case, __LINE__, #x);              \
            exit(1);                                                            \
        }                                                                       \
    } while (0)
static int g_case;

int main(int argc, char** argv) {
    std::mt19937 rng(argc > 1 ? atoi(argv[1]) : 1);
    const int cases = argc > 2 ? atoi(argv[2]) : 100;
    auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (uint32_t)(hi - lo + 1)); };
    long long tiles_seen = 0, parts_seen = 0;
    for (g_case = 0; g_case < cases; ++g_case) {
        // ---- a batch, sometimes with wild tables
        const int batch = pick(0, 3) ? pick(1, 12) : pick(1, 500), wild = pick(0, 9) == 0;
        const int page_size = 1 << pick(0, 8), kv_heads = pick(1, 6), groups[] = {1, 2, 3, 4, 7, 8, 16, 128}, group = groups[pick(0, 7)];
        const int q_most = pick(0, 2) == 0 ? 1 : pick(0, 1) ? pick(1, 8) : pick(1, 400);
        const int own_most = pick(0, 3) == 0 ? pick(0, 40) : pick(0, 3000), sms = pick(0, 2) ? 148 : pick(1, 20);
        std::vector<int> cu(batch + 1), lens(batch);
        int at = pick(0, 3) ? 0 : pick(0, 5), widest = 0;
        for (int b = 0; b < batch; ++b) {
            cu[b] = at;
            at += pick(0, 4) ? pick(0, q_most) : 0;
            lens[b] = pick(0, 5) ? pick(0, own_most) : 0;
            widest = std::max(widest, lens[b]);
        }
        cu[batch] = at;
        const int tokens = at + pick(0, 4), width = (widest + page_size - 1) / page_size + pick(0, 2);
        if (tokens == 0) continue;
        if (wild)
            for (int i = 0; i < 3; ++i) {
                const int odd[] = {-5, 1 << 30, 0x7fffffff, (int)0x80000000, 7};
                (pick(0, 1) ? cu[pick(0, batch)] : lens[pick(0, batch - 1)]) = odd[pick(0, 4)];
            }
        tsw_prefix_attention_args a = {};
        a.batch.seq_lens = (uint64_t)lens.data();
        a.batch.cu_q = (uint64_t)cu.data();
        a.batch.page_table = width ? 4096 : 0;
        a.batch.batch = batch;
        a.batch.table_width = a.batch.table_stride = width;
        a.batch.tokens = tokens;
        a.head_dim = 64;
        a.kv_heads = kv_heads;
        a.q_heads = kv_heads * group;
        a.cache = tsw_kv_pages{1 << 20, 1 << 21, 4096, 4096, 4096, 4096, 4096, 4096, 100, (uint32_t)page_size};
        a.prefix = a.cache;
        a.prefix_len = pick(0, 2) ? pick(0, 2000) : 0;
        a.q = a.out = 1 << 22;
        a.q_token_stride = a.q_head_stride = a.out_token_stride = a.out_head_stride = 4096;
        a.max_q = pick(0, 9) ? q_most : pick(0, tokens);
        a.causal = pick(0, 1);
        a.scale = 1.f;
        AttentionLayout w;
        REQUIRE(attention_layout(a, sms, &w));
        const Deal d{a.batch, a.max_q, a.cache.page_size, a.kv_heads, a.prefix_len, a.causal, w};
        REQUIRE(w.group * w.tile_tokens <= 128 && w.tile_tokens >= 1 && w.own_box_tokens >= 1 && w.own_box_tokens <= w.tile_tokens);

        // ---- what the first CTA leaves for the joining kernel
        std::vector<uint32_t> base(batch + 1);
        uint32_t total = 0;
        for (int b = 0; b < batch; ++b) {
            SeqRows r;
            read_rows(a.batch, b, a.max_q, page_size, r);
            REQUIRE(r.first >= 0 && r.n >= 0 && r.first + r.n <= tokens && r.len >= 0 && r.len <= (long long)width * page_size && r.n <= (int)a.max_q);
            base[b] = total;
            total += sequence_tiles(d, r);
        }
        base[batch] = total;
        int tok0, tok1;
        const uint32_t rts = prefix_rows(d, tok0, tok1);
        const uint32_t prefix_total = a.kv_heads * rts * w.prefix_tiles;

        std::set<std::tuple<int, int, int, int>> done;                  // list, first token of a row tile, head, key tile
        std::set<uint64_t> home, part;                                  // partial results written, in rows of the workspace
        std::map<uint64_t, int> direct;
        const uint64_t home_rows = 2ull * tokens * a.q_heads, part_rows = 4ull * w.ctas * w.part_rows;
        for (int cta = 0; cta < (int)w.ctas; ++cta) {
            Prologue pro = {};
            for (int s = 0; s < 2; ++s) pro.prefix[s] = range_at(d, w.prefix_pair, prefix_total, cta, s);
            pro.prefix_rt = std::max(1u, rts);
            pro.tok0 = tok0;
            pro.tok1 = tok1;
            for (int s = 0; s < 2; ++s) {
                const Range g = range_at(d, w.own_pair, total, cta, s);
                const uint32_t x = g.x, left = g.end - g.x;
                // the kernel's threads look through pieces of the sequences; one of them holds x
                const int each = (batch + 415) / 416;
                int found = 0;
                for (int lo = 0; left && lo < batch; lo += each) {
                    const int hi = std::min(batch, lo + each);
                    if (x < base[lo] || x >= base[hi]) continue;
                    REQUIRE(find_start(d, lo, hi, x - base[lo], left, pro.own[s]));
                    ++found;
                }
                REQUIRE(found == (left ? 1 : 0));
            }
            // what the scheduling warp tells the others: units and rows' jobs
            Walk walk(d, pro);
            Job j;
            int tile, left[2] = {0, 0};
            bool use[2];
            while (walk.next(d, pro, j, tile, use[0], use[1])) {
                ++tiles_seen;
                REQUIRE(use[0] || use[1]);
                REQUIRE(walk.pair || !(use[0] && use[1]));
                REQUIRE(tile >= j.kt0 && tile < j.kt1 && tile * kTile < j.keys && j.head < 65536);
                const tsw_kv_pages& pg = j.own ? a.cache : a.prefix;
                const Load l = make_load(j, tile, walk.pair, use[1]);
                const int n = load_keys(l.flags), box = std::min((int)pg.page_size, kTile), first = tile * kTile / (int)pg.page_size;
                REQUIRE(n == std::min(kTile, j.keys - tile * kTile) && n >= 1 && load_head(l.flags) == j.head && l.b == j.b && l.tile == tile);
                REQUIRE(first + (n + box - 1) / box - 1 < (j.own ? width : ((int)a.prefix_len + page_size - 1) / page_size));
                REQUIRE(((l.flags & kLoadOwn) != 0) == (j.own == 1) && !(l.flags & kLoadEnd) && ((l.flags & kLoadPair) != 0) == walk.pair);
                REQUIRE(walk.pair || ((l.flags & kLoadSecond) != 0) == use[1]);
                for (int s = 0; s < 2; ++s) {
                    const uint32_t u = make_take(j, tile, use[s], walk.pair, tile % 5, tile % 6);
                    REQUIRE(((u & kTakeSkip) != 0) == !use[s] && ((u & kTakePair) != 0) == walk.pair && !(u & kTakeEnd) && take_keys(u) == n &&
                            k_slot(u) == (uint32_t)tile % 5 && v_slot(u) == (uint32_t)tile % 6);
                    if (!use[s]) continue;
                    const RowJob r = make_row_job(d, j, walk.pair, s, cta);
                    REQUIRE(((u & kTakeFirst) != 0) == (left[s] == 0));
                    if (u & kTakeFirst) {
                        left[s] = r.units;
                        REQUIRE(r.units >= 1 && r.tokens >= 1 && r.tokens <= (int)w.tile_tokens && r.tok >= 0 && r.tok + r.tokens <= tokens);
                        for (int i = 0; i < r.tokens * group; ++i) {
                            const uint64_t row = (uint64_t)(r.tok + i / group) * a.q_heads + r.head * group + i % group;
                            if (r.place == kPlaceDirect) ++direct[row];
                            else if (r.place == kPlaceHome) {
                                const uint64_t h = home_index(d, r.own, row, a.q_heads);
                                REQUIRE(h < home_rows && home.insert(h).second);
                            } else {
                                const uint64_t p = part_index(d, r.own, r.place, i);
                                REQUIRE(p < part_rows && part.insert(p).second);
                            }
                        }
                    }
                    left[s] -= units_of(n);
                    REQUIRE(left[s] >= 0);
                    REQUIRE(done.insert({j.own, r.tok, j.head, tile}).second);
                }
            }
            REQUIRE(left[0] == 0 && left[1] == 0);
        }
        // ---- the joining kernel's view: every row of a sequence
        size_t homes_read = 0;
        std::set<uint64_t> parts_read;
        for (int b = 0; b < batch; ++b) {
            SeqRows r;
            read_rows(a.batch, b, a.max_q, page_size, r);
            for (int i = 0; i < r.n; ++i)
                for (int head = 0; head < (int)a.q_heads; ++head) {
                    const int tok = r.first + i, kv = head / group;
                    const uint64_t row = (uint64_t)tok * a.q_heads + head;
                    uint32_t before = 0;
                    for (int rt = 0; rt < i / own_item_tokens(d); ++rt) {
                        const Cut c = cut_own(d, r, rt);
                        before += std::max(c.kt_a, c.kt_b);
                    }
                    const Parts parts[2] = {prefix_parts(d, tok, kv, prefix_total), own_parts(d, r, tok, kv, base[b], before, total)};
                    const int keys = a.causal ? std::max(0, std::min(r.len, r.len - r.n + i + 1)) : r.len;
                    REQUIRE(wild || parts[0].has == (a.prefix_len > 0));
                    REQUIRE(parts[1].has || keys == 0);
                    if (!wild) {
                        // all of a row's key tiles were taken
                        for (int t = 0; t * kTile < keys; ++t) REQUIRE(done.count({1, tok - (i % (int)w.tile_tokens), kv, t}));
                        for (int t = 0; t < (int)w.prefix_tiles; ++t) REQUIRE(done.count({0, tok - (tok - tok0) % (int)w.tile_tokens, kv, t}));
                    }
                    if (!a.prefix_len && parts[1].has && parts[1].first == parts[1].last) {
                        REQUIRE(wild || direct[row] == 1);
                        continue;
                    }
                    REQUIRE(wild || direct.count(row) == 0);
                    for (int l = 0; l < 2; ++l) {
                        const Parts& q = parts[l];
                        if (!q.has) continue;
                        const uint64_t h = home_index(d, l, row, a.q_heads);
                        REQUIRE(wild || home.count(h));
                        ++homes_read;
                        const bool pair = l ? w.own_pair : w.prefix_pair;
                        for (uint32_t k = q.first + 1; k <= q.last; ++k) {
                            const uint64_t p = part_index(d, l, part_place(pair, k, q.half), q.place * group + head % group);
                            REQUIRE(p < part_rows);
                            REQUIRE(wild || part.count(p));
                            REQUIRE(parts_read.insert(p).second || wild);
                            ++parts_seen;
                        }
                    }
                }
        }
        if (!wild && cu[0] == tok0 && tok1 == cu[batch]) {
            // nothing was written that nobody reads, except for rows of sequences longer than max_q
            bool all = true;
            for (int b = 0; b < batch; ++b) all = all && cu[b + 1] - cu[b] <= (int)a.max_q;
            if (all) {
                REQUIRE(homes_read == home.size());
                REQUIRE(parts_read.size() == part.size());
            }
        }
    }
    printf("ok %d cases, %lld tiles, %lld continued rows\n", cases, tiles_seen, parts_seen);
    return 0;
}
