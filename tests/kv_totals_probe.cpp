// Tile numbers are 32 bits (csrc/kv_dealing.hpp): which calls the layout takes, and tables whose sequences claim the same rows over
// and over, so that their tiles add up to more.  Run on the host as the tile kernel's threads and the joining kernel do it.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../torpor_b200/csrc/kv_dealing.hpp"

using namespace tsw;

#define REQUIRE(x)                                            \
    do {                                                      \
        if (!(x)) {                                           \
            printf("line %d: %s\n", __LINE__, #x);            \
            exit(1);                                          \
        }                                                     \
    } while (0)

static tsw_prefix_attention_args call(uint32_t tokens, uint32_t batch, uint32_t width, uint32_t page_size, uint32_t heads) {
    tsw_prefix_attention_args a = {};
    a.batch = tsw_kv_batch{4096, 0, 0, batch, width, width, tokens};
    a.head_dim = 8;
    a.kv_heads = a.q_heads = heads;
    a.cache = a.prefix = tsw_kv_pages{1 << 20, 1 << 21, 4096, 4096, 4096, 4096, 4096, 4096, 100, page_size};
    a.q = a.out = 1 << 22;
    a.q_token_stride = a.q_head_stride = a.out_token_stride = a.out_head_stride = 4096;
    a.max_q = tokens;
    a.scale = 1.f;
    return a;
}

int main() {
    AttentionLayout w;
    int checks = 0;
    // ---- products that pass 64 bits are not small numbers; tables wider than any sequence are no reason to refuse
    for (uint32_t width : {1u << 26, 1u << 27, 1u << 28}) {
        for (uint32_t heads : {256u, 512u, 1024u, 2048u}) {
            const uint32_t tokens = ((1u << 13) - 2) * 128;
            if ((uint64_t)tokens * heads >> 32) continue;
            REQUIRE(!attention_layout(call(tokens, 1, width, 1u << 20, heads), 148, &w));
            ++checks;
        }
    }
    for (uint32_t width : {1u, 1u << 11, 1u << 20, 0xffffffffu}) {
        REQUIRE(attention_layout(call(128, 1, width, 1u << 20, 32), 148, &w));
        ++checks;
    }
    // ---- sequences on top of one another
    for (uint32_t batch : {16u, 1000u, 30000u, 65536u, 131072u}) {
        const uint32_t tokens = 8192, heads = 32;
        std::vector<int> cu(batch + 1), lens(batch, 32768);
        for (uint32_t b = 0; b <= batch; ++b) cu[b] = b & 1 ? (int)tokens : 0;
        tsw_prefix_attention_args a = call(tokens, batch, 2048, 16, heads);
        a.batch.seq_lens = (uint64_t)lens.data();
        a.batch.cu_q = (uint64_t)cu.data();
        REQUIRE(attention_layout(a, 148, &w));
        const Deal d{a.batch, a.max_q, a.cache.page_size, a.kv_heads, a.prefix_len, a.causal, w};
        unsigned long long all = 0;
        std::vector<uint32_t> base(batch);
        uint32_t sum = 0;
        for (uint32_t b = 0; b < batch; ++b) {
            SeqRows r;
            read_rows(a.batch, b, a.max_q, 16, r);
            base[b] = sum;
            sum = add_tiles(sum, sequence_tiles(d, r));
            all += sequence_tiles(d, r);
        }
        const uint32_t total = countable(sum);
        REQUIRE(total == (all < kMaxTiles ? all : 0));
        if (!total) std::fill(base.begin(), base.end(), 0);
        // no range goes past the last sequence, and no row's parts past the workspace
        for (uint32_t cta = 0; cta < w.ctas; ++cta)
            for (int s = 0; s < 2; ++s) {
                const Range g = range_at(d, w.own_pair, total, cta, s);
                REQUIRE(g.x <= g.end && g.end <= all && (total || g.end == g.x));
            }
        for (uint32_t b = 0; b < batch; b += batch / 8)
            for (int tok = 0; tok < (int)tokens; tok += 97)
                for (uint32_t kv = 0; kv < heads; kv += 5) {
                    SeqRows r;
                    read_rows(a.batch, b, a.max_q, 16, r);
                    if (tok >= r.first + r.n) continue;
                    uint32_t before = 0;
                    for (int i = 0; i < tok / own_item_tokens(d); ++i) {
                        const Cut c = cut_own(d, r, i);
                        before += std::max(c.kt_a, c.kt_b);
                    }
                    const Parts p = own_parts(d, r, tok, kv, base[b], before, sum);
                    REQUIRE(p.has && p.first <= p.last && part_place(w.own_pair, p.last, p.half) < 2 * w.ctas);
                    ++checks;
                }
    }
    printf("ok %d\n", checks);
    return 0;
}
