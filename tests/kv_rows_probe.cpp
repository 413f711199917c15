// What csrc/kv_dealing.hpp makes of a sequence's length, on the host: never beyond the page table, never so long that a
// loop over its keys leaves 32 bits.
#include <cstdio>

#include "../torpor_b200/csrc/kv_dealing.hpp"

using namespace tsw;

int main() {
    const struct { int len; uint32_t width, page_size; int want; uint32_t wrong; } cases[] = {
        {5, 1, 16, 5, 0}, {16, 1, 16, 16, 0}, {17, 1, 16, 16, TSW_KV_BAD_LENGTH}, {-1, 1, 16, 0, TSW_KV_BAD_LENGTH}, {3, 0, 16, 0, TSW_KV_BAD_LENGTH},
        {0x7fffff00, 2048, 1u << 20, 0x7fffff00, 0}, {0x7fffff01, 2048, 1u << 20, 0x7fffff00, TSW_KV_BAD_LENGTH},
        {0x7fffffff, 2048, 1u << 20, 0x7fffff00, TSW_KV_BAD_LENGTH}, {0x7fffffff, 0xffffffffu, 1u << 20, 0x7fffff00, TSW_KV_BAD_LENGTH},
        {0x7fffffff, 2047, 1u << 20, 2047 << 20, TSW_KV_BAD_LENGTH}};
    int at = 0;
    for (const auto& c : cases) {
        const int cu[2] = {0, 1};
        tsw_kv_batch t = {};
        t.page_table = c.width ? 4096 : 0;
        t.seq_lens = (uint64_t)&c.len;
        t.cu_q = (uint64_t)cu;
        t.batch = 1;
        t.table_width = t.table_stride = c.width;
        t.tokens = 1;
        SeqRows r;
        const uint32_t wrong = read_rows(t, 0, 1, c.page_size, r);
        if (r.len != c.want || wrong != c.wrong || r.n != 1) {
            printf("case %d: length %d, status %u\n", at, r.len, wrong);
            return 1;
        }
        // the steps of the kernels: 32 keys a round, 128 a tile; the counter past the last round still is a number of its own sign
        for (long long step : {32ll, 128ll})
            if ((r.len + step - 1) / step * step + step - 1 > 0x7fffffffll) {
                printf("case %d: steps of %lld pass 32 bits\n", at, step);
                return 1;
            }
        ++at;
    }
    printf("ok %d\n", at);
    return 0;
}
