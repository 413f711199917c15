// How many keys a row sees, on the host: over all ranges that hold a piece of its keys, as many as its mask leaves it, also where the
// lists are longer than 2^30.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <tuple>
#include <vector>

#include "../torpor_b200/csrc/kv_dealing.hpp"

using namespace tsw;

#define REQUIRE(x)                                                       \
    do {                                                                 \
        if (!(x)) {                                                      \
            printf("case %d line %d: %s\n", g_case, __LINE__, #x);       \
            exit(1);                                                     \
        }                                                                \
    } while (0)
static int g_case;

int main() {
    struct Case { uint32_t prefix; std::vector<int> rows, lens; int first, causal; };
    const Case cases[] = {
        {1000, {1, 3}, {500, 77}, 0, 1}, {1000, {140, 3}, {500, 77}, 2, 1}, {0, {5}, {900}, 0, 0},
        {1u << 30, {1}, {0}, 0, 1}, {(1u << 30) + 4096, {1}, {5}, 0, 1}, {0x7fffff00, {1}, {0}, 0, 1}, {0x7fffff00, {2, 1}, {40, 30}, 7, 1},
        {0x7fffff00, {150}, {150}, 9, 0}, {1073745920, {3}, {3}, 0, 1}, {2147483392, {1}, {1}, 0, 1},
        {0, {1}, {(1 << 30) + 128}, 0, 0}, {0, {2, 1}, {0x7fffff00, 99}, 3, 0}, {0, {1, 3}, {17, 0x7fffff00}, 1, 1}, {3, {200}, {0x7fffff00}, 5, 1},
        {0, {200}, {0x7ffffeff}, 5000, 0}, {0, {200}, {0x7fffff00}, 5000, 1}, {0x7ffffe81, {200}, {1}, 5000, 1}};
    for (const Case& k : cases) {
        const int batch = (int)k.rows.size();
        std::vector<int> cu{k.first};
        for (int n : k.rows) cu.push_back(cu.back() + n);
        tsw_prefix_attention_args a = {};
        a.batch = tsw_kv_batch{4096, (uint64_t)k.lens.data(), (uint64_t)cu.data(), (uint32_t)batch, 2048, 2048, (uint32_t)cu.back() + 1};
        a.head_dim = 8;
        a.kv_heads = a.q_heads = 1;
        a.cache = a.prefix = tsw_kv_pages{1 << 20, 1 << 21, 4096, 4096, 4096, 4096, 4096, 4096, 100, 1 << 20};
        a.q = a.out = 1 << 22;
        a.q_token_stride = a.q_head_stride = a.out_token_stride = a.out_head_stride = 4096;
        a.prefix_len = k.prefix;
        a.max_q = 200;
        a.causal = k.causal;
        a.scale = 1.f;
        AttentionLayout w;
        REQUIRE(attention_layout(a, 148, &w));
        const Deal d{a.batch, a.max_q, a.cache.page_size, a.kv_heads, a.prefix_len, a.causal, w};
        uint32_t total = 0;
        for (int b = 0; b < batch; ++b) {
            SeqRows r;
            REQUIRE(read_rows(a.batch, b, a.max_q, a.cache.page_size, r) == 0);
            total = add_tiles(total, sequence_tiles(d, r));
        }
        int tok0, tok1;
        const uint32_t rts = prefix_rows(d, tok0, tok1), prefix_total = a.kv_heads * rts * w.prefix_tiles;
        std::map<std::pair<int, int>, long long> seen;
        for (uint32_t cta = 0; cta < w.ctas; ++cta) {
            Prologue pro = {};
            pro.prefix_rt = std::max(1u, rts);
            pro.tok0 = tok0;
            pro.tok1 = tok1;
            for (int s = 0; s < 2; ++s) {
                pro.prefix[s] = range_at(d, w.prefix_pair, prefix_total, cta, s);
                const Range g = range_at(d, w.own_pair, total, cta, s);
                if (g.end > g.x) REQUIRE(find_start(d, 0, batch, g.x, g.end - g.x, pro.own[s]));
            }
            for (int list = 0; list < 2; ++list)
                for (int s = 0; s < 2; ++s) {
                    Cursor c(pro, s);
                    Job j;
                    while (c.next(d, pro, list, j)) {
                        const bool pair = list ? w.own_pair : w.prefix_pair;
                        for (int half = 0; half < (pair ? 2 : 1); ++half) {
                            if ((half ? j.n_b : j.n_a) == 0 || seen_by(j, pair, half) <= j.kt0) continue;
                            const RowJob r = make_row_job(d, j, pair, half, cta);
                            for (int i = 0; i < kTile; ++i) {                // rows behind the tile's last are masked like the others
                                const int n = keys_seen(r, r.tok + i);
                                REQUIRE(n >= 0 && n <= r.keys);
                                if (i < r.tokens) seen[{list, r.tok + i}] += std::min<long long>(n, 64ll * r.units);
                            }
                        }
                    }
                }
        }
        for (int b = 0; b < batch; ++b)
            for (int i = 0; i < k.rows[b]; ++i) {
                const int len = k.lens[b], own = k.causal ? std::max(0, len - k.rows[b] + i + 1) : len;
                REQUIRE((seen[{1, cu[b] + i}]) == own);
                REQUIRE((seen[{0, cu[b] + i}]) == (long long)k.prefix);
            }
        ++g_case;
    }
    printf("ok %d\n", g_case);
    return 0;
}
