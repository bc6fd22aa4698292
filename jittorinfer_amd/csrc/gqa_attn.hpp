// The kernels of gqa_attn_launch (include/gqa_attn.h) for other operators of the library.
#pragma once

#include "gqa_common.hpp"

namespace mla {
namespace gqa {

// What a launch over the rows behind[b] .. seq_lens[b] - 1 of every sequence leaves of a head: one result in whole_o / whole_ml, or pieces.  Head r of KV head
// kvh's group lies in head block hb = quad ? kvh / 4 : kvh * row_blocks + r / rows, row (quad ? kvh % 4 * group + r : r % rows) of it; items[b * head_blocks + hb] =
// (slot of the first piece, last workgroup), slot / 2 = the first workgroup, the pieces after the first are in the slots 2 * workgroup.  Nothing is left of a sequence without such a row.
struct AttnPieces {
    const float *   part_o;       // [slot][rows][dv], unnormalized
    const float *   whole_o;      // [n_seq][n_head][dv], unnormalized
    const float2 *  part_ml;      // [slot][rows]: reference (log2 units), sum
    const float2 *  whole_ml;     // [n_seq][n_head]
    const int2 *    items;
    const int32_t * seq_lens, * behind;
    int mask_len, cap, rows, row_blocks, head_blocks, quad;
};

// `a`: a call that gqa_attn_check accepts, without weights and window; its dst and workspace are not looked at.  `ws`: attn_behind_size() bytes, 256-byte aligned.
size_t     attn_behind_size(const gqa_attn_args * a);
hipError_t attn_behind(const gqa_attn_args * a, const int32_t * behind, char * ws, AttnPieces & out, hipStream_t st);

}  // namespace gqa
}  // namespace mla
