// The built library's plans, which run on the host: workspace and pieces of a call.
#include "drafts.hpp"

using namespace m1moe;

// Floats that a product makes sure of; *used: where its last partial ends, *shared: its counters.
extern "C" int64_t probe_q4(int rows, int cols, int group, int tokens, int x_bf16, int cus, int64_t* used, int* shared) {
    Q4Args a{};
    a.rows = rows;
    a.cols = cols;
    a.group = group;
    a.tokens = tokens;
    a.x_bf16 = x_bf16;
    const int64_t floats = matmul_q4_plan(a, cus);
    const int tiles = tokens > 32 ? 4 : tokens > 16 ? 2 : 1;   // a wave's, each of 256 sums
    const int64_t wgs = a.split > 1 ? a.grid - a.whole : 0;
    *used = a.part_at + wgs * a.waves * tiles * 256;
    *shared = a.split > 1 ? (int)(wgs / a.split) : 0;
    return floats;
}

extern "C" int64_t probe_paged(int rows, int heads, int kv_heads, int head_dim, int x_bf16, int prefix, int cus,
                               int* splits, int64_t* used) {
    PagedAttnArgs a{};
    a.p.num_rows = rows;
    a.p.kv_heads = kv_heads;
    a.p.prefix_len = prefix;
    a.heads = heads;
    a.share = heads / kv_heads;
    a.head_dim = head_dim;
    a.x_bf16 = x_bf16;
    int64_t own = 0;
    const int64_t floats = paged_attention_plan(a, cus, &own);
    *splits = a.splits;
    *used = own + (a.splits ? (int64_t)(a.splits + 1) * rows * heads * (head_dim + 2) : 0);
    return floats;
}
