// Attention of many query rows over the same keys (include/gqa_batch.h): what its host code and its kernels share.
#pragma once

#include "gqa_common.hpp"
#include "../../include/gqa_batch.h"

namespace mla {
namespace gqa {

// "Group": the queries that meet one run of keys -- the new tokens of a sequence, a decoder's over its states, or (own_lens) one token of each of the sequences that
// share a prefix, which is read through the first one's pages.  Its query rows are (token, head of the KV head's group), token-major, cut into blocks of BM.
struct BatchP {
    const char * q; int64_t q_nb1, q_nb2;
    const char * k; int64_t k_page, k_head; int k_row;             // k_page: a page, or (no block table) a group's own part
    const char * v; int64_t v_page, v_head; int v_row;
    const int32_t * block_table; int64_t bt_stride, n_pages;       // block_table == nullptr: rows in one piece
    const int32_t * kv_starts;
    const int32_t * lens;
    const int32_t * q_starts; int per;                             // q_starts == nullptr: `per` tokens a group
    const int32_t * own_lens;     // [n_tok] rows of the token's own sequence, or nullptr
    int32_t * shared, * shared_group;                              // (own_lens) [n_tok]: rows that the token's sequence shares, its group or -1: left for the kernels behind this one
    const char * mask; int64_t mask_nb1; int mask_len;             // mask_len: rows past it are out
    char * dst; int64_t d_nb1, d_nb2;
    float scale_log2;             // |scale| * log2(e)
    float mask_unit;              // 1 / |scale|
    unsigned flip;                // sign bits of a pair of values: Q is negated as it is read where the scale is negative
    float cap_in, cap_out;        // soft cap c: |scale| / c and c * log2(e); cap_out = 0: none
    int causal, window, n_grp, n_tok, n_head, n_head_kv, group;
    double per_head;              // 1 / group
    int cap;                      // rows a group can have
    int n_wg, min_tiles;          // workgroups, and the fewest tiles that are worth one
    float *  part_o;              // [2 * n_wg][BM * dv]: unnormalized sums of the pieces of blocks that several workgroups share, in the lanes' order;
    float2 * part_ml;             // [2 * n_wg][BM]: reference (log2 units), sum; (own_lens) behind them [block number][n_head_kv]: blocks that one workgroup covered
    int4 *   items;               // [block number][n_head_kv]: slot of the first piece, first run, last run
    int4 *   tasks;               // [n_wg]: the block that begins in a run and goes on in others (item, first token of the group, its rows, block), or item -1
    int      blocks, deal;        // block numbers, and a Dealing
};

// Blocks are dealt in equal runs, one to a workgroup, or the one or the other by what the device finds.  Runs cost pieces that are written, read again and joined: as
// much as JOIN_KEYS keys of a block; whole blocks leave workgroups idle at the end.  Both sides, us (32 heads on 8 of 128, bf16, where no other is named): prompts of
// 2 x 512 tokens 40 against 22, 4 x 1024 85 / 60, 1 x 4096 181 / 155, 4 x 1500 to 2048 178 / 141, 32 x 448 tokens over 1500 states (16 heads of 64) 174 / 143; 3 x
// 600 to 1024 over 3000 to 8192 states 371 / 383, 8 x 512 behind 5000 to 16384 rows (16 on 4 of 64) 272 / 367.  Wide heads, masks and caps, runs by 512 (256 for heads of 256) workgroups
// against what is chosen, whole blocks: 2 x 3500 to 4096 tokens, 16 heads of 192, mask 271 / 234; 6 x 300 to 700, 16 on 4 of 256, cap and window 164 to 169 / 167 to 171; 8 x 100 to
// 448 over 300 to 1500 states, 16 of 64, mask 49 to 52 / 53.  (One number for all: a key of heads of 256 costs four times one of 64, and so do its pieces.)
enum Dealing { RUNS, EITHER, WHOLE };
constexpr int JOIN_KEYS = 1280;

// Waves along the query rows and along the keys of a tile, keys of a tile.
enum Shape { FOUR_ROWS, TWO_TWO, FOUR_KEYS };

struct BatchPlan { Shape shape; int bm, n_wg, blocks, deal; size_t off_ml, off_items, off_tasks, bytes; };

// What the three calls have in common.
struct BatchCall {
    int32_t n_tok, n_seq, n_head, n_head_kv, dk, dv, type, n_workgroups;
    float   scale, logit_softcap;
    const void * q; int64_t q_nb1, q_nb2;
    const int32_t * q_starts;
    gqa_pool k, v;
    int64_t cap;                  // rows a sequence can have
    const void * mask; int64_t mask_nb1, mask_ne0;
    void * dst; int64_t d_nb1, d_nb2;
};
int       batch_check(const BatchCall & c);
BatchPlan batch_plan(const BatchCall & c, bool whole_blocks);     // whole_blocks: with room for the blocks that one workgroup covers
void      batch_fill(BatchP & p, const BatchCall & c, const BatchPlan & pl, char * workspace);

template <bool F16> hipError_t batch_launch(const BatchP & p, const BatchPlan & pl, int dk, hipStream_t st);

// Workgroups of a shape that a CU holds, by its registers and its tiles in LDS (plain: no mask, no cap).  Heads of 64, three or two: 8 x 512 tokens behind 5000 to 16384 rows 302 or
// 312 us, although the third one's 168 vector registers spill 36 (none among the products); with a mask more of them do, 8 x 448 tokens over states 68 or 54 us.  Blocks of 128 rows of
// heads of 128 spill 14 of 256 with a mask, 19 with a cap (none among the products either); no other build spills any.
constexpr int batch_wg_per_cu(int dk, Shape s, bool plain) { return s == FOUR_KEYS ? (dk <= 64 ? 2 : 1) : dk == 64 && plain ? 3 : dk <= 128 || (dk == 192 && s == FOUR_ROWS) ? 2 : 1; }

}  // namespace gqa
}  // namespace mla
