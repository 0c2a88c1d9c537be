// tree_attn.hip — attention of trees of drafted tokens over the paged KV cache.
//
// As paged_attn.hpp says, over the positions before the tree and those of it whose bits the row's
// mask has: the tree's rows are its sequence's last positions, so a mask matters to the last block or
// two of keys of a tile only, where eight bits at a time are taken from two words.  A row that sees
// nothing has no sum of weights and gives zeros.
//
// 32 trees of 8 to 64 behind 60 to 8100 positions, 32 heads over 8, f32 queries, bf16 cache: 160 us; the
// three products that such queries take are 95 at a large product's rate, the cache 76 at a
// large copy's.  24 trees of 1 to 100 behind a prefix of 4096 and 20 to 600, 16 heads, all bf16:
// 80 us, its 1.5 products 36 (f32 queries 124, f32 cache 274).  26 rows behind 700, 16 heads, all f32: 24.5 us,
// the chain launch - lengths - page - rows - join with six products of 32 keys at a time, in the half
// of a workgroup's waves that has rows.
#include <hip/hip_runtime.h>

#include "drafts.hpp"
#include "paged_attn.hpp"

namespace m1moe {

int launch_tree_attention(const PagedAttnArgs& a, void* stream) {
    return launch_attention<true>(a, static_cast<hipStream_t>(stream));
}

}  // namespace m1moe
