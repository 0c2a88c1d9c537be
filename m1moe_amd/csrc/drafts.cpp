// drafts.cpp — C ABI of the operators of steps over drafted tokens: their trees' plan, append,
// attention and acceptance, and products with 4-bit weights.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "drafts.hpp"
#include "serving_calls.hpp"

using namespace m1moe;

namespace {

// Memory that a call reads or writes.
struct Range {
    const void* p;
    int64_t bytes;
    const char* what;
};

bool overlap(const Range& a, const Range& b) {
    const intptr_t x = reinterpret_cast<intptr_t>(a.p), y = reinterpret_cast<intptr_t>(b.p);
    return a.p && b.p && x < y + b.bytes && y < x + a.bytes;
}

// Every output apart from every input and from the other outputs.
int32_t check_apart(const Range* outs, const Range* outs_end, const Range* ins, const Range* ins_end) {
    for (const Range* o = outs; o != outs_end; ++o) {
        for (const Range* i = ins; i != ins_end; ++i)
            if (overlap(*o, *i)) return fail(M1MOE_ERR_INVALID, "%s must not overlap %s", o->what, i->what);
        for (const Range* x = outs; x != o; ++x)
            if (overlap(*o, *x)) return fail(M1MOE_ERR_INVALID, "%s must not overlap %s", o->what, x->what);
    }
    return M1MOE_OK;
}
int32_t check_apart(std::initializer_list<Range> outs, std::initializer_list<Range> ins) {
    return check_apart(outs.begin(), outs.end(), ins.begin(), ins.end());
}

int32_t check_mask(const uint64_t* mask, int32_t words) {
    if (!mask) return fail(M1MOE_ERR_INVALID, "d_mask is null");
    if (reinterpret_cast<uintptr_t>(mask) % 8) return fail(M1MOE_ERR_INVALID, "d_mask must be 8-byte aligned");
    if (words < 1 || words > kTreeWords)
        return fail(M1MOE_ERR_INVALID, "mask_words %d out of range [1, %d]", words, kTreeWords);
    return M1MOE_OK;
}

// At least `floats` of the products' workspace.
int32_t ensure_q4_scratch(m1moe_ctx_t ctx, uint64_t floats) {
    ctx->capture_uses_scratch = true;
    if (ctx->q4_cnt && floats <= ctx->q4_part_floats) return M1MOE_OK;
    if (int32_t rc = refuse_growth_in_capture(ctx->stream, "the 4-bit products' scratch")) return rc;
    if (!ctx->q4_cnt) {
        const uint64_t bytes = 4 * (uint64_t)ctx->cus;   // (tiles that are shared are fewer than the CUs)
        if (int32_t rc = device_alloc_zeroed((void**)&ctx->q4_cnt, bytes, "4-bit products' counters", ctx->stream))
            return rc;
        if (floats <= ctx->q4_part_floats) return M1MOE_OK;
    }
    HIP_TRY(hipStreamSynchronize(ctx->stream));
    if (ctx->q4_part) ++ctx->scratch_gen;  // earlier graphs hold the old buffer
    if (ctx->q4_part) HIP_TRY(hipFree(ctx->q4_part));
    ctx->q4_part = nullptr;
    ctx->q4_part_floats = 0;
    if (int32_t rc = device_alloc((void**)&ctx->q4_part, floats * 4, "4-bit products' scratch")) return rc;
    ctx->q4_part_floats = floats;
    return M1MOE_OK;
}

int64_t row_bytes(int64_t stride, int64_t n, int64_t rows, int64_t es) { return ((rows - 1) * stride + n) * es; }

// Of a cache: bytes of a position, and of all of k (or v).
int64_t position_bytes(const m1moe_paged_kv* kv) {
    return (int64_t)kv->num_kv_heads * kv->head_dim * (kv->dtype == M1MOE_BF16 ? 2 : 4);
}
int64_t plane_bytes(const m1moe_paged_kv* kv) { return position_bytes(kv) * kv->page_size * kv->num_pages; }

Range starts_of(const m1moe_paged_batch* b) { return {b->d_row_start, 4 * ((int64_t)b->num_seqs + 1), "d_row_start"}; }
Range lengths_of(const m1moe_paged_batch* b) { return {b->d_kv_len, 4 * (int64_t)b->num_seqs, "d_kv_len"}; }
Range pages_of(const m1moe_paged_batch* b) {
    return {b->d_pages, 4 * (int64_t)b->num_seqs * b->table_stride, "d_pages"};
}

}  // namespace

extern "C" {

int32_t m1moe_tree_plan(m1moe_ctx_t ctx, int32_t num_seqs, int32_t num_rows, const int32_t* d_row_start,
                        const int32_t* d_parents, int32_t mask_words, uint64_t* d_mask, int32_t* d_depth) {
    int32_t rc;
    if (num_seqs < 1 || num_seqs > kPagedMaxSeqs)
        return fail(M1MOE_ERR_INVALID, "num_seqs %d out of range [1, %d]", num_seqs, kPagedMaxSeqs);
    if (num_rows < 1 || num_rows > (1 << 20))
        return fail(M1MOE_ERR_INVALID, "num_rows %d out of range [1, %d]", num_rows, 1 << 20);
    if ((rc = check_i32_ptr(d_row_start, "d_row_start")) || (rc = check_i32_ptr(d_parents, "d_parents")) ||
        (rc = check_mask(d_mask, mask_words)) || (rc = check_i32_ptr(d_depth, "d_depth")))
        return rc;
    if ((rc = check_ctx(ctx))) return rc;
    const int64_t n = num_rows;
    if ((rc = check_apart({{d_mask, 8 * n * mask_words, "d_mask"}, {d_depth, 4 * n, "d_depth"}},
                          {{d_row_start, 4 * (num_seqs + 1), "d_row_start"}, {d_parents, 4 * n, "d_parents"}})))
        return rc;
    if ((rc = set_device(ctx))) return rc;
    TreePlanArgs a{};
    a.num_seqs = num_seqs;
    a.num_rows = num_rows;
    a.words = mask_words;
    a.row_start = d_row_start;
    a.parents = d_parents;
    a.mask = d_mask;
    a.depth = d_depth;
    a.err = ctx->err;
    return launched(launch_tree_plan(a, ctx->stream), "tree_plan");
}

int32_t m1moe_tree_append(m1moe_ctx_t ctx, const m1moe_paged_kv* kv, const m1moe_paged_batch* batch,
                          const m1moe_kv_append_args* args, const int32_t* d_depth) {
    int32_t rc;
    if ((rc = check_kv(kv)) || (rc = check_batch(kv, batch)) || (rc = check_i32_ptr(d_depth, "d_depth"))) return rc;
    AppendArgs a{};
    if ((rc = append_args(ctx, kv, batch, args, a))) return rc;
    const int64_t qd = (int64_t)args->num_heads * kv->head_dim, es = args->dtype == M1MOE_BF16 ? 2 : 4;
    const Range q{args->d_q ? args->d_q_out : nullptr, row_bytes(args->q_out_stride, qd, batch->num_rows, es), "d_q_out"};
    if ((rc = check_apart({q, {kv->d_k, plane_bytes(kv), "the cache's d_k"}, {kv->d_v, plane_bytes(kv), "the cache's d_v"}},
                          {{d_depth, 4 * (int64_t)batch->num_rows, "d_depth"}, starts_of(batch), lengths_of(batch),
                           pages_of(batch)})))
        return rc;
    a.depth = d_depth;
    return launched(launch_kv_append(a, ctx->cus, ctx->stream), "tree_append");
}

int32_t m1moe_tree_attention(m1moe_ctx_t ctx, const m1moe_paged_kv* kv, const m1moe_paged_batch* batch,
                             const uint64_t* d_mask, int32_t mask_words, const void* d_q, int64_t q_stride,
                             void* d_out, int64_t out_stride, int32_t dtype, int32_t num_heads) {
    int32_t rc;
    if ((rc = check_kv(kv)) || (rc = check_batch(kv, batch)) || (rc = check_mask(d_mask, mask_words))) return rc;
    PagedAttnArgs a{};
    if ((rc = attention_args(ctx, kv, batch, d_q, q_stride, d_out, out_stride, dtype, num_heads, a))) return rc;
    const int64_t qd = (int64_t)num_heads * kv->head_dim, es = dtype == M1MOE_BF16 ? 2 : 4;
    if ((rc = check_apart({{d_out, row_bytes(out_stride, qd, batch->num_rows, es), "d_out"}},
                          {{d_mask, 8 * (int64_t)batch->num_rows * mask_words, "d_mask"},
                           starts_of(batch),
                           lengths_of(batch),
                           pages_of(batch),
                           {batch->prefix_len ? batch->d_prefix_pages : nullptr,
                            4 * (((int64_t)batch->prefix_len + kv->page_size - 1) / kv->page_size), "d_prefix_pages"},
                           {kv->d_k, plane_bytes(kv), "the cache's d_k"},
                           {kv->d_v, plane_bytes(kv), "the cache's d_v"}})))
        return rc;
    a.mask = d_mask;
    a.mask_words = mask_words;
    return launched(launch_tree_attention(a, ctx->stream), "tree_attention");
}

int32_t m1moe_tree_accept(m1moe_ctx_t ctx, const m1moe_paged_kv* kvs, int32_t num_caches,
                          const m1moe_paged_batch* batch, const int32_t* d_parents, const int32_t* d_drafts,
                          const int32_t* d_drawn, int32_t* d_path, int32_t* d_accepted, int32_t* d_next,
                          int32_t* d_past) {
    int32_t rc;
    if (num_caches < 1 || num_caches > kMostCaches)
        return fail(M1MOE_ERR_INVALID, "num_caches %d out of range [1, %d]", num_caches, kMostCaches);
    if (!kvs) return fail(M1MOE_ERR_INVALID, "kvs is null");
    for (int i = 0; i < num_caches; ++i) {
        if ((rc = check_kv(kvs + i))) return rc;
        const m1moe_paged_kv &x = kvs[i], &y = kvs[0];
        if (x.dtype != y.dtype || x.num_pages != y.num_pages || x.page_size != y.page_size ||
            x.num_kv_heads != y.num_kv_heads || x.head_dim != y.head_dim)
            return fail(M1MOE_ERR_INVALID, "cache %d differs from cache 0 in its type or sizes", i);
    }
    if ((rc = check_batch(kvs, batch)) || (rc = check_i32_ptr(d_parents, "d_parents")) ||
        (rc = check_i32_ptr(d_drafts, "d_drafts")) || (rc = check_i32_ptr(d_drawn, "d_drawn")) ||
        (rc = check_i32_ptr(d_path, "d_path")) || (rc = check_i32_ptr(d_accepted, "d_accepted")) ||
        (rc = check_i32_ptr(d_next, "d_next")) || (rc = check_i32_ptr(d_past, "d_past")))
        return rc;
    if ((rc = check_ctx(ctx))) return rc;
    const int64_t rows = 4 * (int64_t)batch->num_rows, seqs = 4 * (int64_t)batch->num_seqs;
    const Range outs[4] = {{d_path, rows, "d_path"}, {d_accepted, seqs, "d_accepted"}, {d_next, seqs, "d_next"}, {d_past, seqs, "d_past"}};
    const Range ins[6] = {{d_parents, rows, "d_parents"}, {d_drafts, rows, "d_drafts"}, {d_drawn, rows, "d_drawn"},
                          starts_of(batch), lengths_of(batch), pages_of(batch)};
    if ((rc = check_apart(outs, outs + 4, ins, ins + 6))) return rc;
    TreeAcceptArgs a{};
    const int64_t position = position_bytes(kvs), plane = plane_bytes(kvs);
    for (int i = 0; i < num_caches; ++i) {
        a.planes[2 * i] = kvs[i].d_k;
        a.planes[2 * i + 1] = kvs[i].d_v;
    }
    a.num_planes = 2 * num_caches;
    // (planes that share memory would be moved twice, by workgroups that do not wait for each other)
    void* sorted[2 * kMostCaches];
    std::copy(a.planes, a.planes + a.num_planes, sorted);
    if (!std::is_sorted(sorted, sorted + a.num_planes)) std::sort(sorted, sorted + a.num_planes);
    for (int i = 1; i < a.num_planes; ++i)
        if (static_cast<char*>(sorted[i]) - static_cast<char*>(sorted[i - 1]) < plane)
            return fail(M1MOE_ERR_INVALID, "two of the caches' d_k and d_v overlap");
    // (apart and in order: of those that begin before a range's end, the last one ends last.  The inputs
    // too: every workgroup walks for itself, while others move rows already)
    const auto in_plane = [&](const Range& o) {
        void** after = std::lower_bound(sorted, sorted + a.num_planes, const_cast<char*>(static_cast<const char*>(o.p)) + o.bytes);
        return after != sorted && overlap(o, {after[-1], plane, ""});
    };
    for (const Range& o : outs)
        if (in_plane(o)) return fail(M1MOE_ERR_INVALID, "%s must not overlap a cache's d_k or d_v", o.what);
    for (const Range& i : ins)
        if (in_plane(i)) return fail(M1MOE_ERR_INVALID, "%s must not overlap a cache's d_k or d_v", i.what);
    if ((rc = set_device(ctx))) return rc;
    a.p = view(ctx, kvs, batch);
    a.row_units = (int32_t)(position / 16);
    a.parents = d_parents;
    a.drafts = d_drafts;
    a.drawn = d_drawn;
    a.path = d_path;
    a.accepted = d_accepted;
    a.next = d_next;
    a.past = d_past;
    return launched(launch_tree_accept(a, ctx->stream), "tree_accept");
}

int32_t m1moe_matmul_q4(m1moe_ctx_t ctx, const m1moe_q4_weights* w, const void* d_x, int32_t x_dtype,
                        int64_t x_stride, int32_t tokens, const void* d_residual, void* d_y, int32_t y_dtype,
                        int64_t y_stride) {
    int32_t rc;
    if (!w) return fail(M1MOE_ERR_INVALID, "weights is null");
    if ((rc = check_dev_ptr(w->d_w, "d_w", false)) || (rc = check_dev_ptr(w->d_scales, "d_scales", false)) ||
        (rc = check_dev_ptr(w->d_biases, "d_biases", false)))
        return rc;
    if (w->group_size != 32 && w->group_size != 64 && w->group_size != 128)
        return fail(M1MOE_ERR_INVALID, "group_size %d is not 32, 64 or 128", w->group_size);
    if (w->rows < 1 || w->rows > (1 << 20))
        return fail(M1MOE_ERR_INVALID, "rows %d out of range [1, %d]", w->rows, 1 << 20);
    if (w->cols < 1 || w->cols > 65536 || w->cols % w->group_size)
        return fail(M1MOE_ERR_INVALID, "cols %d is not a multiple of group_size %d up to 65536", w->cols,
                    w->group_size);
    if (tokens < 1 || tokens > 65536) return fail(M1MOE_ERR_INVALID, "tokens %d out of range [1, 65536]", tokens);
    if ((rc = check_dtype(x_dtype)) || (rc = check_rows(d_x, x_stride, w->cols, x_dtype, "d_x"))) return rc;
    if (y_dtype != M1MOE_F32 && y_dtype != M1MOE_BF16)
        return fail(M1MOE_ERR_INVALID, "y_dtype %d is not M1MOE_F32 or M1MOE_BF16", y_dtype);
    if (x_dtype == M1MOE_F32 && y_dtype == M1MOE_BF16)
        return fail(M1MOE_ERR_INVALID, "f32 rows need an f32 result");
    if ((rc = check_rows(d_y, y_stride, w->rows, y_dtype, "d_y")) ||
        (rc = check_dev_ptr(d_residual, "d_residual", true)))
        return rc;
    if ((rc = check_ctx(ctx))) return rc;
    const int64_t xs = x_dtype == M1MOE_BF16 ? 2 : 4, ys = y_dtype == M1MOE_BF16 ? 2 : 4;
    const int64_t n = w->rows, words = n * w->cols / 8, groups = n * (w->cols / w->group_size);
    if (rows_overlap(d_x, xs * x_stride, xs * w->cols, d_y, ys * y_stride, ys * n, tokens))
        return fail(M1MOE_ERR_INVALID, "d_y must not overlap rows of d_x");
    if (d_residual && d_residual != d_y &&
        rows_overlap(d_residual, ys * y_stride, ys * n, d_y, ys * y_stride, ys * n, tokens))
        return fail(M1MOE_ERR_INVALID, "d_residual overlaps rows of d_y and is not d_y itself");
    if ((rc = check_apart({{d_y, row_bytes(y_stride, n, tokens, ys), "d_y"}},
                          {{w->d_w, 4 * words, "d_w"}, {w->d_scales, 2 * groups, "d_scales"},
                           {w->d_biases, 2 * groups, "d_biases"}})))
        return rc;
    if ((rc = set_device(ctx))) return rc;
    Q4Args a{};
    a.w = w->d_w;
    a.scales = w->d_scales;
    a.biases = w->d_biases;
    a.rows = w->rows;
    a.cols = w->cols;
    a.group = w->group_size;
    a.x = d_x;
    a.x_stride = x_stride;
    a.tokens = tokens;
    a.residual = d_residual;
    a.y = d_y;
    a.y_stride = y_stride;
    a.x_bf16 = x_dtype == M1MOE_BF16;
    a.y_bf16 = y_dtype == M1MOE_BF16;
    const int64_t floats = matmul_q4_plan(a, ctx->cus);
    if (floats) {
        if ((rc = ensure_q4_scratch(ctx, (uint64_t)floats))) return rc;
        a.xparts = reinterpret_cast<uint8_t*>(ctx->q4_part);
        a.xsums = reinterpret_cast<uint8_t*>(ctx->q4_part + a.sums_at);
        a.down = ctx->q4_part + a.down_at;
        a.part = ctx->q4_part + a.part_at;
        a.counters = ctx->q4_cnt;
    }
    return launched(launch_matmul_q4(a, ctx->stream), "matmul_q4");
}

}  // extern "C"
