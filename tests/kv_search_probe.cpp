// Which sequence a row belongs to (Search in csrc/kv_dealing.hpp), on the host with 32 lanes one after the other: for tables in order
// it is the one that contains the row, for any other table one that does, or none.  What the joining kernel works
// out from there stays inside the workspace.
//   kv_search_probe SEED CASES
#include <cstdio>
#include <cstdlib>
#include <random>
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

static int found(const std::vector<int>& cu, int tok) {
    const uint32_t batch = (uint32_t)cu.size() - 1;
    Search s(batch);
    int steps = 0;
    while (s.open()) {
        uint32_t votes = 0;
        for (int lane = 0; lane < 32; ++lane) votes |= (uint32_t)s.vote(cu.data(), tok, lane) << lane;
        s.take(votes);
        REQUIRE(s.lo <= s.hi && s.hi <= batch + 1 && ++steps < 8);
    }
    return s.sequence(batch);
}

int main(int argc, char** argv) {
    std::mt19937 rng(argc > 1 ? atoi(argv[1]) : 1);
    const int cases = argc > 2 ? atoi(argv[2]) : 100;
    auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (uint32_t)(hi - lo + 1)); };
    long long rows = 0;
    for (g_case = 0; g_case < cases; ++g_case) {
        const int batch = pick(0, 2) ? pick(1, 40) : pick(1, 3000), kind = pick(0, 3), each = pick(0, 1) ? 1 : 12;
        std::vector<int> cu(batch + 1), lens(batch);
        cu[0] = pick(0, 4);
        for (int b = 0; b < batch; ++b) {
            cu[b + 1] = cu[b] + pick(0, each);
            lens[b] = pick(0, 400);
        }
        int tokens = cu[batch] + pick(0, 3);
        if (kind == 1) {                                             // a few entries at odd places
            const int odd[] = {-5, 0, 3, 1 << 30, 0x7fffffff, (int)0x80000000, cu[batch] / 2, cu[batch]};
            for (int i = pick(1, 4); i; --i) cu[pick(0, batch)] = odd[pick(0, 7)];
        } else if (kind == 2) {                                      // no order at all
            for (int& x : cu) x = pick(0, tokens);
        } else if (kind == 3 && batch == 3) {
            cu = {0, 10, 12, 5};
            tokens = 12;
        }
        if (!tokens) continue;
        tsw_prefix_attention_args a = {};
        a.batch = tsw_kv_batch{4096, (uint64_t)lens.data(), (uint64_t)cu.data(), (uint32_t)batch, 32, 32, (uint32_t)tokens};
        a.head_dim = 64;
        a.kv_heads = 2;
        a.q_heads = 2 << pick(0, 3);
        a.cache = a.prefix = tsw_kv_pages{1 << 20, 1 << 21, 4096, 4096, 4096, 4096, 4096, 4096, 100, 16};
        a.prefix_len = pick(0, 1) * 300;
        a.q = a.out = 1 << 22;
        a.q_token_stride = a.q_head_stride = a.out_token_stride = a.out_head_stride = 4096;
        a.max_q = pick(0, 1) ? tokens : 12;
        a.causal = pick(0, 1);
        a.scale = 1.f;
        AttentionLayout w;
        REQUIRE(attention_layout(a, 148, &w));
        const Deal d{a.batch, a.max_q, a.cache.page_size, a.kv_heads, a.prefix_len, a.causal, w};
        std::vector<uint32_t> base(batch + 1);
        for (int b = 0; b < batch; ++b) {
            SeqRows r;
            read_rows(a.batch, b, a.max_q, 16, r);
            base[b + 1] = base[b] + sequence_tiles(d, r);
        }
        int tok0, tok1;
        const uint32_t prefix_total = a.kv_heads * prefix_rows(d, tok0, tok1) * w.prefix_tiles;
        const uint64_t part_rows = 4ull * w.ctas * w.part_rows, home_rows = 2ull * tokens * a.q_heads;
        for (int tok = 0; tok < tokens; ++tok, ++rows) {
            const int b = found(cu, tok);
            REQUIRE(b >= -1 && b < batch);
            if (b >= 0) REQUIRE(cu[b] <= tok && tok < cu[b + 1]);
            if (kind == 0 || (kind == 3 && batch != 3)) {            // in order: the one sequence that has the row
                int want = -1;
                for (int i = 0; i < batch; ++i)
                    if (cu[i] <= tok && tok < cu[i + 1]) want = i;
                REQUIRE(b == want);
            }
            if (b < 0) continue;
            SeqRows r;
            read_rows(a.batch, b, a.max_q, 16, r);
            if (tok >= r.first + r.n) continue;
            REQUIRE(tok >= r.first);
            uint32_t before = 0;
            const int rt = (int)((uint32_t)(tok - r.first) / (uint32_t)own_item_tokens(d));
            REQUIRE(rt * own_item_tokens(d) < r.n);
            for (int i = 0; i < rt; ++i) {
                const Cut c = cut_own(d, r, i);
                before += std::max(c.kt_a, c.kt_b);
            }
            for (uint32_t kv = 0; kv < a.kv_heads; ++kv)
                for (int l = 0; l < 2; ++l) {
                    const Parts p = l ? own_parts(d, r, tok, kv, base[b], before, base[batch]) : prefix_parts(d, tok, kv, prefix_total);
                    if (!p.has) continue;
                    const bool pair = l ? w.own_pair : w.prefix_pair;
                    REQUIRE(p.first <= p.last && p.place < w.tile_tokens && p.half < 2);
                    REQUIRE(part_index(d, l, part_place(pair, p.last, p.half), p.place * w.group + w.group - 1) < part_rows);
                    REQUIRE(home_index(d, l, (uint64_t)tok * a.q_heads + a.q_heads - 1, a.q_heads) < home_rows);
                }
        }
    }
    printf("ok %d cases, %lld rows\n", cases, rows);
    return 0;
}
