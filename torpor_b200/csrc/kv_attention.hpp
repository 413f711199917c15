// Launch interface of the tensor-core attention kernel (kv_attention.cu) and the layout of its work.
#ifndef TORPOR_KV_ATTENTION_HPP_
#define TORPOR_KV_ATTENTION_HPP_

#include <cstdint>

#include "../../include/torpor_swap.h"

namespace tsw {

struct AttentionLayout {
    uint32_t ctas;            // one per SM
    uint32_t group;           // query heads to a key head
    uint32_t tile_tokens;     // tokens in a row tile: group * tile_tokens <= 128 rows
    uint32_t own_box_tokens;  // tokens a query load of the own list brings (fewer when max_q is small)
    uint32_t prefix_tiles;    // key tiles of the prefix
    uint32_t prefix_pair, own_pair;   // the list is dealt to the two streams of a CTA together
    uint32_t part_rows;       // rows of a partial result that is not an item's first
    // Workspace, in bytes from its start.  A result that is an item's first range lies by row
    // ([list][token][head], one list without a prefix); the ranges that continue an item (at most one per stream and list) lie by stream.
    uint64_t own_base;        // uint32 [batch + 2]: tiles in front of each sequence's; own total; prefix total
    uint64_t home_ml, home_o; // float2, float [head_dim]
    uint64_t part_ml, part_o;
    uint64_t bytes;
};

#ifdef __CUDART_API_VERSION
cudaError_t launch_prefix_attention_tiles(int device, const tsw_prefix_attention_args& a, const AttentionLayout& w, uint32_t* status, cudaStream_t stream);
#endif

}  // namespace tsw
#endif
