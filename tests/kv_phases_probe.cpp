// The barriers of the attention kernel's key and value rings, on the host: one to a stream and slot, flipped by the load of
// a tile and waited for by parity.  A stream that has not taken note of a flip takes an old tile for its own, so every
// flip of a barrier that a stream is ever told to wait for has to be among those it was told of before.
//   kv_phases_probe SEED CASES
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

struct Slots {                 // a ring and what has happened to its barriers
    uint32_t stages, at = 0;
    std::vector<long> flips, noted[2];
    explicit Slots(uint32_t n) : stages(n), flips(2 * n) { noted[0].resize(2 * n), noted[1].resize(2 * n); }
    void pass(const Load& l, bool told0, bool told1) {
        const uint32_t done = (l.flags & kLoadSecond ? stages : 0) + at;
        ++flips[done];
        for (int s = 0; s < 2; ++s) {
            if (!(s ? told1 : told0)) continue;
            const uint32_t x = (l.flags & kLoadPair ? 0 : s * stages) + at;
            REQUIRE(x == done);
            REQUIRE(++noted[s][x] == flips[x]);
        }
        at = (at + 1) % stages;
    }
};

static long long check(const tsw_prefix_attention_args& a, int sms) {
    AttentionLayout w;
    REQUIRE(attention_layout(a, sms, &w));
    REQUIRE(!w.own_pair || w.prefix_pair);
    REQUIRE(w.own_box_tokens <= w.tile_tokens);
    const Deal d{a.batch, a.max_q, a.cache.page_size, a.kv_heads, a.prefix_len, a.causal, w};
    uint32_t total = 0;
    for (uint32_t b = 0; b < a.batch.batch; ++b) {
        SeqRows r;
        read_rows(a.batch, b, a.max_q, a.cache.page_size, r);
        total += sequence_tiles(d, r);
    }
    int tok0, tok1;
    const uint32_t rts = prefix_rows(d, tok0, tok1), prefix_total = a.kv_heads * rts * w.prefix_tiles;
    long long tiles = 0;
    for (uint32_t cta = 0; cta < w.ctas; ++cta) {
        Prologue pro = {};
        pro.prefix_rt = std::max(1u, rts);
        pro.tok0 = tok0;
        pro.tok1 = tok1;
        for (int s = 0; s < 2; ++s) {
            pro.prefix[s] = range_at(d, w.prefix_pair, prefix_total, cta, s);
            const Range g = range_at(d, w.own_pair, total, cta, s);
            if (g.end > g.x) REQUIRE(find_start(d, 0, a.batch.batch, g.x, g.end - g.x, pro.own[s]));
        }
        Slots rings[] = {Slots(2), Slots(3), Slots(5), Slots(6)};        // of both head widths
        Walk walk(d, pro);
        Job j;
        int tile;
        bool use[2];
        while (walk.next(d, pro, j, tile, use[0], use[1])) {
            const Load l = make_load(j, tile, walk.pair, use[1]);
            for (Slots& r : rings) r.pass(l, use[0] || walk.pair, use[1] || walk.pair);
            ++tiles;
        }
    }
    return tiles;
}

int main(int argc, char** argv) {
    std::mt19937 rng(argc > 1 ? atoi(argv[1]) : 1);
    const int cases = argc > 2 ? atoi(argv[2]) : 100;
    auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (uint32_t)(hi - lo + 1)); };
    long long tiles = 0;
    for (g_case = 0; g_case < cases; ++g_case) {
        const int batch = pick(1, 6), page_size = 1 << pick(3, 7), groups[] = {1, 2, 4, 16, 128}, q_most = pick(0, 1) ? 1 : pick(1, 300);
        std::vector<int> cu(batch + 1), lens(batch);
        for (int b = 0; b < batch; ++b) {
            cu[b + 1] = cu[b] + pick(pick(0, 1), q_most);
            lens[b] = pick(0, 3000);
        }
        tsw_prefix_attention_args a = {};
        a.batch = tsw_kv_batch{4096, (uint64_t)lens.data(), (uint64_t)cu.data(), (uint32_t)batch, 4096, 4096, (uint32_t)(cu[batch] + pick(0, 2))};
        if (!a.batch.tokens) continue;
        a.head_dim = 64;
        a.kv_heads = pick(1, 32);
        a.q_heads = a.kv_heads * groups[pick(0, 4)];
        a.cache = a.prefix = tsw_kv_pages{1 << 20, 1 << 21, 4096, 4096, 4096, 4096, 4096, 4096, 100, (uint32_t)page_size};
        a.prefix_len = pick(0, 3) ? pick(1, 6000) : 0;
        a.q = a.out = 1 << 22;
        a.q_token_stride = a.q_head_stride = a.out_token_stride = a.out_head_stride = 4096;
        // any upper bound of a sequence's new rows will do: the most there are, the batch's rows, more than those
        const uint32_t bounds[] = {(uint32_t)q_most, a.batch.tokens, a.batch.tokens + 1, a.batch.tokens * 2 + 200, 0x7fffffffu};
        a.max_q = bounds[pick(0, 4)];
        a.causal = pick(0, 1);
        a.scale = 1.f;
        tiles += check(a, pick(0, 2) ? 148 : pick(1, 20));
    }
    printf("ok %d cases, %lld tiles\n", cases, tiles);
    return 0;
}
