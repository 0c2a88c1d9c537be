// paged.hpp — kernel arguments of the paged KV cache (paged.hip) and of the
// sampler (sample.hip).
#pragma once

#include <cstdint>

namespace m1moe {

constexpr int kPagedMaxSeqs = 1024;
constexpr int kPagedMaxShare = 64;   // query heads per kv head
constexpr uint32_t kErrPagedBatch = 256u, kErrPagedPage = 512u, kErrTree = 1024u;   // device error flags

// The cache and the batch (m1moe_paged_kv, m1moe_paged_batch).
struct PagedView {
    void *k, *v;
    int32_t num_pages, page_shift, kv_heads;
    int32_t num_seqs, num_rows, table_stride, prefix_len;
    const int32_t *row_start, *kv_len, *pages, *prefix_pages;
    uint32_t* err;
};

struct AppendArgs {
    PagedView p;
    const void *q, *k, *v;
    void* q_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    const uint16_t *q_norm, *k_norm;
    const float* inv_freq;
    float eps, amp;
    int32_t heads, head_dim, rotary, interleaved;
    int32_t x_bf16, cache_bf16;
    const int32_t* depth;   // of a tree's rows, or null: rows at their own positions
};

struct PagedAttnArgs {
    PagedView p;
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    int32_t heads, share, head_dim;   // share: query heads per kv head
    int32_t x_bf16, cache_bf16;
    float scale;
    int32_t grid;        // workgroups the sequences' own positions are shared by
    int32_t splits;      // pieces of the prefix, 0 without one
    int32_t prefix_wgs;  // and the workgroups that take them
    float* part;         // partials: the workgroups' slots
    float* pre;          // and the prefix' pieces, [splits + 1][num_rows * heads][head_dim + 2]
    uint32_t* counters;  // [grid], zero between launches
    // of trees: who sees whom, [num_rows][mask_words] (null: every row sees the earlier ones)
    const uint64_t* mask;
    int32_t mask_words;
};

struct SampleArgs {
    const float* logits;
    int64_t stride;
    int32_t rows, vocab;
    const float *u, *temperature, *top_p, *min_p;
    const int32_t* top_k;
    int32_t* tokens;
    float* probs;
    // workgroups per row and, for more than one, their histograms ([rows * parts][2048]
    // sums and counts) and a counter per row, zero between launches
    int32_t parts;
    unsigned long long* part_sum;
    uint32_t *part_cnt, *counters;
};

int launch_kv_append(const AppendArgs& a, int cus, void* stream);
// Sets grid, splits and prefix_wgs; the floats of partials (slots, then pieces) needed.
int64_t paged_attention_plan(PagedAttnArgs& a, int cus, int64_t* own_floats);
int launch_paged_attention(const PagedAttnArgs& a, void* stream);
int sample_parts(int rows, int vocab, int cus);
int64_t sample_part_words(int cus);   // of part_sum, part_cnt and counters, in this order (sums as two)
int launch_sample(const SampleArgs& a, void* stream);

}  // namespace m1moe
