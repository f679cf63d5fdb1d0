// What a batch over paged K/V caches is made of: the host plans it (paged_plan.h), the kernels work it off. No CUDA in here.
#pragma once
#include <stdint.h>

namespace llamd {

// A new token: its position and the row of the pools that head 0 of its K and V goes to (head h: `page` rows further each).
struct PagedToken {
    int32_t pos, row;
};

// The batch as the kernels see it: device memory that the batch owns, every index checked against the pools when it was made.
struct PagedView {
    int n_head, n_head_kv, group, hd, page, n_seq, tokens, n_shared, table_stride;
    const PagedToken *token;    // [tokens]
    const int32_t *table;       // [n_seq][table_stride] page ids
};

// One piece of attention: n_tok tokens (all their heads that share kv head `head`; for paged_decode.cu the launch's y) over positions
// [kv_begin, kv_end) of one table.
// Token i of the piece sees positions below limit + i * step. part < 0: the piece is all its rows need, and writes out;
// otherwise its rows' sums go to rows part + ... of the batch's partial results (paged_decode.cu: + head * part_rows).
struct PagedItem {
    int32_t table, kv_begin, kv_end, token, n_tok, limit, step, part, part_rows, head, pad[2];
};
static_assert(sizeof(PagedItem) == 48, "three 16-byte words");

// Where the rows of a token and a kv head find their partial results: entries [begin, begin + count) of the list below.
struct PagedMerge {
    int32_t token, head, begin, count;
};
struct PagedPart {
    int32_t row, token;  // the row of token t and head g of the group: row + (t - token) * group + g
};

// Query rows (tokens x heads of a group) of a piece that paged_decode.cu can take (one token of a wide group), and of one that it is given where a
// stretch has several tokens. Pieces of 16 rows: 32 take 255 registers where 8 take 149 and 16 take 210 (at 128 elements; 203, 93 and 131 at 64) and half the
// CTAs (8 sequences behind 512 shared positions 12.1 us against 6.6, 64 with 3 new tokens behind 3500 102.9 against 90.7), 8 read K and V
// twice as often (102.9).
constexpr int kPagedSmallRows = 32, kPagedPieceRows = 16;

// paged_prompt.cu: two tiles of so many query rows to a piece, positions to a block.
constexpr int kPagedTileRows = 128, kPagedBlock = 128;

}  // namespace llamd
