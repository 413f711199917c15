// What a call asks of its workspace (csrc/kv_dealing.hpp): the parts of a row's results that it can write, apart from one another, and
// not those of a prefix that it does not have.
#include <cstdio>
#include <cstdlib>

#include "../torpor_b200/csrc/kv_dealing.hpp"

using namespace tsw;

#define REQUIRE(x)                                            \
    do {                                                      \
        if (!(x)) {                                           \
            printf("line %d: %s\n", __LINE__, #x);            \
            exit(1);                                          \
        }                                                     \
    } while (0)

int main() {
    int n = 0;
    for (uint32_t tokens : {1u, 7u, 128u, 8192u, 131072u})
        for (uint32_t heads : {1u, 8u, 32u})
            for (uint32_t group : {1u, 4u}) {
                uint64_t bytes[2];
                for (uint32_t prefix : {0u, 1000u}) {
                    tsw_prefix_attention_args a = {};
                    a.batch = tsw_kv_batch{4096, 4096, 4096, 1, 64, 64, tokens};
                    a.head_dim = 128;
                    a.kv_heads = heads;
                    a.q_heads = heads * group;
                    a.cache = a.prefix = tsw_kv_pages{1 << 20, 1 << 21, 4096, 4096, 4096, 4096, 4096, 4096, 100, 16};
                    a.prefix_len = prefix;
                    a.q = a.out = 1 << 22;
                    a.q_token_stride = a.q_head_stride = a.out_token_stride = a.out_head_stride = 4096;
                    a.max_q = tokens;
                    a.scale = 1.f;
                    AttentionLayout w;
                    REQUIRE(attention_layout(a, 148, &w));
                    const Deal d{a.batch, a.max_q, a.cache.page_size, a.kv_heads, a.prefix_len, a.causal, w};
                    const uint64_t rows = (uint64_t)tokens * a.q_heads, o = 4 * 128, lists = prefix ? 2 : 1;
                    // the last row of either list ends before what lies behind it
                    const uint64_t home = home_index(d, 1, rows - 1, a.q_heads), part = part_index(d, 1, 2 * w.ctas - 1, w.part_rows - 1);
                    REQUIRE(home == lists * rows - 1 && part == lists * 2 * w.ctas * w.part_rows - 1);
                    REQUIRE(w.home_ml + 8 * (home + 1) <= w.home_o && w.home_o + o * (home + 1) <= w.part_ml);
                    REQUIRE(w.part_ml + 8 * (part + 1) <= w.part_o && w.part_o + o * (part + 1) <= w.bytes);
                    if (prefix) REQUIRE(home_index(d, 0, rows - 1, a.q_heads) < home_index(d, 1, 0, a.q_heads));
                    if (prefix) REQUIRE(part_index(d, 0, 2 * w.ctas - 1, w.part_rows - 1) < part_index(d, 1, 0, 0));
                    bytes[prefix > 0] = w.bytes;
                    REQUIRE(w.bytes <= lists * (rows + 2 * w.ctas * w.part_rows) * (o + 8) + 8192);
                    ++n;
                }
                REQUIRE(bytes[0] * 2 <= bytes[1] + 8192);
            }
    printf("ok %d\n", n);
    return 0;
}
