// serving.cpp — C ABI of the operators for several conversations at once: the
// paged KV cache's append and attention, and sampling.
#include <hip/hip_runtime.h>

#include <cmath>

#include "ctx.hpp"
#include "internal.hpp"
#include "m1moe_hip.h"
#include "paged.hpp"

using namespace m1moe;

namespace {

int32_t check_kv(const m1moe_paged_kv* kv) {
    int32_t rc;
    if (!kv) return fail(M1MOE_ERR_INVALID, "kv is null");
    if ((rc = check_dev_ptr(kv->d_k, "d_k", false)) || (rc = check_dev_ptr(kv->d_v, "d_v", false))) return rc;
    if (kv->dtype != M1MOE_F32 && kv->dtype != M1MOE_BF16)
        return fail(M1MOE_ERR_INVALID, "cache dtype %d is not M1MOE_F32 or M1MOE_BF16", kv->dtype);
    if (kv->num_pages < 1) return fail(M1MOE_ERR_INVALID, "num_pages %d must be positive", kv->num_pages);
    if (kv->page_size < 8 || kv->page_size > 4096 || (kv->page_size & (kv->page_size - 1)))
        return fail(M1MOE_ERR_INVALID, "page_size %d is not a power of two from 8 to 4096", kv->page_size);
    if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256)
        return fail(M1MOE_ERR_INVALID, "head_dim %d is not 64, 128 or 256", kv->head_dim);
    if (kv->num_kv_heads < 1 || (int64_t)kv->num_kv_heads * kv->head_dim > 65536)
        return fail(M1MOE_ERR_INVALID, "num_kv_heads %d: need at least 1 and num_kv_heads * head_dim <= 65536",
                    kv->num_kv_heads);
    return M1MOE_OK;
}

int32_t check_i32_ptr(const void* p, const char* what) {
    if (!p) return fail(M1MOE_ERR_INVALID, "%s is null", what);
    if (reinterpret_cast<uintptr_t>(p) % 4) return fail(M1MOE_ERR_INVALID, "%s must be 4-byte aligned", what);
    return M1MOE_OK;
}

int32_t check_batch(const m1moe_paged_kv* kv, const m1moe_paged_batch* b) {
    int32_t rc;
    if (!b) return fail(M1MOE_ERR_INVALID, "batch is null");
    if (b->num_seqs < 1 || b->num_seqs > kPagedMaxSeqs)
        return fail(M1MOE_ERR_INVALID, "num_seqs %d out of range [1, %d]", b->num_seqs, kPagedMaxSeqs);
    if (b->num_rows < 1 || b->num_rows > (1 << 20))
        return fail(M1MOE_ERR_INVALID, "num_rows %d out of range [1, %d]", b->num_rows, 1 << 20);
    if (b->table_stride < 1 || (int64_t)b->table_stride * kv->page_size > (1 << 24))
        return fail(M1MOE_ERR_INVALID, "table_stride %d: need at least 1 and table_stride * page_size <= 2^24",
                    b->table_stride);
    if (b->prefix_len < 0 || (int64_t)b->prefix_len > (int64_t)b->table_stride * kv->page_size)
        return fail(M1MOE_ERR_INVALID, "prefix_len %d out of range [0, table_stride * page_size]", b->prefix_len);
    if ((rc = check_i32_ptr(b->d_row_start, "d_row_start")) || (rc = check_i32_ptr(b->d_kv_len, "d_kv_len")) ||
        (rc = check_i32_ptr(b->d_pages, "d_pages")) ||
        (b->prefix_len > 0 && (rc = check_i32_ptr(b->d_prefix_pages, "d_prefix_pages"))))
        return rc;
    return M1MOE_OK;
}

int32_t check_heads(const m1moe_paged_kv* kv, int32_t heads) {
    if (heads < 1 || heads % kv->num_kv_heads || heads / kv->num_kv_heads > kPagedMaxShare)
        return fail(M1MOE_ERR_INVALID, "num_heads %d must be 1 to %d times num_kv_heads %d", heads,
                    kPagedMaxShare, kv->num_kv_heads);
    if ((int64_t)heads * kv->head_dim > 65536)
        return fail(M1MOE_ERR_INVALID, "num_heads * head_dim = %lld exceeds 65536",
                    (long long)heads * kv->head_dim);
    return M1MOE_OK;
}

// Rows `stride` elements apart, each of n elements, starting at 16-byte bounds.
int32_t check_rows(const void* p, int64_t stride, int64_t n, int32_t dtype, const char* what) {
    int32_t rc;
    if ((rc = check_dev_ptr(p, what, false))) return rc;
    if (stride < n || stride % (dtype == M1MOE_BF16 ? 8 : 4) || stride > (1ll << 32))
        return fail(M1MOE_ERR_INVALID, "%s: a row stride of %lld elements is below the row's %lld or not a "
                    "multiple of 16 bytes", what, (long long)stride, (long long)n);
    return M1MOE_OK;
}

// Whether rows of xn bytes at x, xs bytes apart, share memory with as many of yn bytes at y, ys
// bytes apart (xn <= xs, yn <= ys).  Of different strides: whether their ranges do.
bool rows_overlap(const void* x, int64_t xs, int64_t xn, const void* y, int64_t ys, int64_t yn, int64_t rows) {
    const int64_t d = reinterpret_cast<intptr_t>(y) - reinterpret_cast<intptr_t>(x);
    if (d >= (rows - 1) * xs + xn || -d >= (rows - 1) * ys + yn) return false;
    if (rows == 1 || xs != ys) return true;
    const int64_t at = (d % xs + xs) % xs;   // y's columns from x's on
    return at < xn || at + yn > xs;
}

PagedView view(m1moe_ctx_t ctx, const m1moe_paged_kv* kv, const m1moe_paged_batch* b) {
    PagedView v{};
    v.k = kv->d_k;
    v.v = kv->d_v;
    v.num_pages = kv->num_pages;
    v.page_shift = __builtin_ctz((unsigned)kv->page_size);
    v.kv_heads = kv->num_kv_heads;
    v.num_seqs = b->num_seqs;
    v.num_rows = b->num_rows;
    v.table_stride = b->table_stride;
    v.prefix_len = b->prefix_len;
    v.row_start = b->d_row_start;
    v.kv_len = b->d_kv_len;
    v.pages = b->d_pages;
    v.prefix_pages = b->d_prefix_pages;
    v.err = ctx->err;
    return v;
}

// At least `floats` of paged attention partials.
int32_t ensure_paged_scratch(m1moe_ctx_t ctx, uint64_t floats) {
    ctx->capture_uses_scratch = true;
    if (ctx->paged_cnt && floats <= ctx->paged_part_floats) return M1MOE_OK;
    if (int32_t rc = refuse_growth_in_capture(ctx->stream, "the paged attention scratch")) return rc;
    if (!ctx->paged_cnt) {
        const uint64_t bytes = 4 * (2 * (uint64_t)ctx->cus + 8);   // the largest grid
        if (int32_t rc = device_alloc_zeroed((void**)&ctx->paged_cnt, bytes, "paged attention counters", ctx->stream))
            return rc;
        if (floats <= ctx->paged_part_floats) return M1MOE_OK;
    }
    HIP_TRY(hipStreamSynchronize(ctx->stream));
    if (ctx->paged_part) ++ctx->scratch_gen;  // earlier graphs hold the old buffer
    if (ctx->paged_part) HIP_TRY(hipFree(ctx->paged_part));
    ctx->paged_part = nullptr;
    ctx->paged_part_floats = 0;
    int32_t rc = device_alloc((void**)&ctx->paged_part, floats * 4, "paged attention scratch");
    if (rc) return rc;
    ctx->paged_part_floats = floats;
    return M1MOE_OK;
}

// The histograms of m1moe_sample's workgroups.  Not there yet while the stream is
// captured: the call does without (one workgroup per row, the same results).
int32_t ensure_sample_scratch(m1moe_ctx_t ctx) {
    if (ctx->sample_part) return M1MOE_OK;
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    HIP_TRY(hipStreamIsCapturing(ctx->stream, &cs));
    if (cs != hipStreamCaptureStatusNone) return M1MOE_OK;
    const uint64_t bytes = (uint64_t)sample_part_words(ctx->cus) * 4;
    // (its counters start at zero; cleared on the launches' own stream)
    return device_alloc_zeroed((void**)&ctx->sample_part, bytes, "sampling scratch", ctx->stream);
}

}  // namespace

extern "C" {

int32_t m1moe_check_paged(const m1moe_paged_kv* kv, const m1moe_paged_batch* batch) {
    int32_t rc;
    if ((rc = check_kv(kv)) || (rc = check_batch(kv, batch))) return rc;
    return M1MOE_OK;
}

int32_t m1moe_kv_append(m1moe_ctx_t ctx, const m1moe_paged_kv* kv, const m1moe_paged_batch* batch,
                        const m1moe_kv_append_args* g) {
    int32_t rc;
    if ((rc = check_kv(kv)) || (rc = check_batch(kv, batch))) return rc;
    if (!g) return fail(M1MOE_ERR_INVALID, "args is null");
    if ((rc = check_dtype(g->dtype)) || (rc = check_heads(kv, g->num_heads))) return rc;
    const int64_t qd = (int64_t)g->num_heads * kv->head_dim, kvd = (int64_t)kv->num_kv_heads * kv->head_dim;
    if (!g->d_q != !g->d_q_out)
        return fail(M1MOE_ERR_INVALID, "d_q and d_q_out must both be given or both be null");
    if (g->d_q && ((rc = check_rows(g->d_q, g->q_stride, qd, g->dtype, "d_q")) ||
                   (rc = check_rows(g->d_q_out, g->q_out_stride, qd, g->dtype, "d_q_out"))))
        return rc;
    if (g->d_q && g->d_q == g->d_q_out && g->q_stride != g->q_out_stride)
        return fail(M1MOE_ERR_INVALID, "d_q_out is d_q but its row stride differs");
    if ((rc = check_rows(g->d_k, g->k_stride, kvd, g->dtype, "d_k")) ||
        (rc = check_rows(g->d_v, g->v_stride, kvd, g->dtype, "d_v")) ||
        (rc = check_dev_ptr(g->d_q_norm, "d_q_norm", true)) || (rc = check_dev_ptr(g->d_k_norm, "d_k_norm", true)))
        return rc;
    if (!(g->eps >= 0.f)) return fail(M1MOE_ERR_INVALID, "eps must be >= 0");
    if (g->rotary_dim < 0 || g->rotary_dim % 16 || g->rotary_dim > kv->head_dim)
        return fail(M1MOE_ERR_INVALID, "rotary_dim %d is not a multiple of 16 from 0 to head_dim %d",
                    g->rotary_dim, kv->head_dim);
    if (g->interleaved != 0 && g->interleaved != 1)
        return fail(M1MOE_ERR_INVALID, "interleaved %d is not 0 or 1", g->interleaved);
    if (g->rotary_dim > 0 && (rc = check_i32_ptr(g->d_inv_freq, "d_inv_freq"))) return rc;
    if (g->rotary_dim > 0 && !(std::fabs(g->rope_amplitude) <= 3.4e38f))
        return fail(M1MOE_ERR_INVALID, "rope_amplitude must be finite");
    if ((rc = check_ctx(ctx))) return rc;
    const int64_t es = g->dtype == M1MOE_BF16 ? 2 : 4;
    const auto clash = [&](const void* p, int64_t stride, int64_t n) {
        return rows_overlap(g->d_q_out, es * g->q_out_stride, es * qd, p, es * stride, es * n, batch->num_rows);
    };
    if (g->d_q && ((g->d_q_out != g->d_q && clash(g->d_q, g->q_stride, qd)) || clash(g->d_k, g->k_stride, kvd) ||
                   clash(g->d_v, g->v_stride, kvd)))
        return fail(M1MOE_ERR_INVALID, "d_q_out overlaps rows of d_q, d_k or d_v and is not d_q itself");
    if ((rc = set_device(ctx))) return rc;
    AppendArgs a{};
    a.p = view(ctx, kv, batch);
    a.q = g->d_q;
    a.k = g->d_k;
    a.v = g->d_v;
    a.q_out = g->d_q_out;
    a.q_stride = g->q_stride;
    a.k_stride = g->k_stride;
    a.v_stride = g->v_stride;
    a.q_out_stride = g->q_out_stride;
    a.q_norm = g->d_q_norm;
    a.k_norm = g->d_k_norm;
    a.inv_freq = g->d_inv_freq;
    a.eps = g->eps;
    a.amp = g->rope_amplitude;
    a.heads = g->d_q ? g->num_heads : 0;
    a.head_dim = kv->head_dim;
    a.rotary = g->rotary_dim;
    a.interleaved = g->interleaved;
    a.x_bf16 = g->dtype == M1MOE_BF16;
    a.cache_bf16 = kv->dtype == M1MOE_BF16;
    return launched(launch_kv_append(a, ctx->cus, ctx->stream), "kv_append");
}

int32_t m1moe_paged_attention(m1moe_ctx_t ctx, const m1moe_paged_kv* kv, const m1moe_paged_batch* batch,
                              const void* d_q, int64_t q_stride, void* d_out, int64_t out_stride,
                              int32_t dtype, int32_t num_heads) {
    int32_t rc;
    if ((rc = check_kv(kv)) || (rc = check_batch(kv, batch)) || (rc = check_dtype(dtype)) ||
        (rc = check_heads(kv, num_heads)))
        return rc;
    if (dtype == M1MOE_BF16 && kv->dtype != M1MOE_BF16)
        return fail(M1MOE_ERR_INVALID, "bf16 queries need a bf16 cache");
    const int64_t qd = (int64_t)num_heads * kv->head_dim;
    if ((rc = check_rows(d_q, q_stride, qd, dtype, "d_q")) ||
        (rc = check_rows(d_out, out_stride, qd, dtype, "d_out")))
        return rc;
    if (d_q == d_out) return fail(M1MOE_ERR_INVALID, "d_out must not overlap d_q");
    if ((rc = check_ctx(ctx))) return rc;
    const int64_t es = dtype == M1MOE_BF16 ? 2 : 4;
    if (rows_overlap(d_q, es * q_stride, es * qd, d_out, es * out_stride, es * qd, batch->num_rows))
        return fail(M1MOE_ERR_INVALID, "d_out must not overlap rows of d_q");
    if ((rc = set_device(ctx))) return rc;
    PagedAttnArgs a{};
    a.p = view(ctx, kv, batch);
    a.q = d_q;
    a.out = d_out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.heads = num_heads;
    a.share = num_heads / kv->num_kv_heads;
    a.head_dim = kv->head_dim;
    a.x_bf16 = dtype == M1MOE_BF16;
    a.cache_bf16 = kv->dtype == M1MOE_BF16;
    a.scale = 1.0f / sqrtf((float)kv->head_dim);
    int64_t own = 0;
    const int64_t floats = paged_attention_plan(a, ctx->cus, &own);
    if ((rc = ensure_paged_scratch(ctx, (uint64_t)floats))) return rc;
    a.part = ctx->paged_part;
    a.pre = ctx->paged_part + own;
    a.counters = ctx->paged_cnt;
    return launched(launch_paged_attention(a, ctx->stream), "paged_attention");
}

int32_t m1moe_sample(m1moe_ctx_t ctx, const float* d_logits, int32_t rows, int32_t vocab, int64_t stride,
                     const m1moe_sample_params* s, int32_t* d_tokens, float* d_probs) {
    int32_t rc;
    if ((rc = check_dev_ptr(d_logits, "d_logits", false))) return rc;
    if (rows < 1 || rows > 65536) return fail(M1MOE_ERR_INVALID, "rows %d out of range [1, 65536]", rows);
    if (vocab < 1 || vocab > 262144)
        return fail(M1MOE_ERR_INVALID, "vocab %d out of range [1, 262144]", vocab);
    if (stride < vocab || stride % 4 || stride > (1ll << 32))
        return fail(M1MOE_ERR_INVALID, "a row stride of %lld logits is below the vocabulary's %d or not a "
                    "multiple of 4", (long long)stride, vocab);
    if (!s) return fail(M1MOE_ERR_INVALID, "params is null");
    if ((rc = check_i32_ptr(s->d_u, "d_u")) || (rc = check_i32_ptr(d_tokens, "d_tokens")) ||
        (s->d_temperature && (rc = check_i32_ptr(s->d_temperature, "d_temperature"))) ||
        (s->d_top_k && (rc = check_i32_ptr(s->d_top_k, "d_top_k"))) ||
        (s->d_top_p && (rc = check_i32_ptr(s->d_top_p, "d_top_p"))) ||
        (s->d_min_p && (rc = check_i32_ptr(s->d_min_p, "d_min_p"))) ||
        (d_probs && (rc = check_i32_ptr(d_probs, "d_probs"))))
        return rc;
    if ((rc = check_ctx(ctx)) || (rc = set_device(ctx))) return rc;
    SampleArgs a{};
    a.logits = d_logits;
    a.stride = stride;
    a.rows = rows;
    a.vocab = vocab;
    a.u = s->d_u;
    a.temperature = s->d_temperature;
    a.top_k = s->d_top_k;
    a.top_p = s->d_top_p;
    a.min_p = s->d_min_p;
    a.tokens = d_tokens;
    a.probs = d_probs;
    a.parts = sample_parts(rows, vocab, ctx->cus);
    if (a.parts > 1 && (rc = ensure_sample_scratch(ctx))) return rc;
    if (!ctx->sample_part) a.parts = 1;
    if (a.parts > 1) {
        const uint64_t bins = sample_part_words(ctx->cus) / (3 * (uint64_t)ctx->cus);   // words per part
        a.part_sum = reinterpret_cast<unsigned long long*>(ctx->sample_part);
        a.part_cnt = ctx->sample_part + 2 * bins * ctx->cus;
        a.counters = a.part_cnt + bins * ctx->cus;
    }
    return launched(launch_sample(a, ctx->stream), "sample");
}

}  // extern "C"
