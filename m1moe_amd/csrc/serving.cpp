// serving.cpp — C ABI of the operators for several conversations at once: the
// paged KV cache's append and attention, and sampling.
#include <hip/hip_runtime.h>

#include "serving_calls.hpp"

using namespace m1moe;

namespace {

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
    AppendArgs a{};
    if (int32_t rc = append_args(ctx, kv, batch, g, a)) return rc;
    return launched(launch_kv_append(a, ctx->cus, ctx->stream), "kv_append");
}

int32_t m1moe_paged_attention(m1moe_ctx_t ctx, const m1moe_paged_kv* kv, const m1moe_paged_batch* batch,
                              const void* d_q, int64_t q_stride, void* d_out, int64_t out_stride,
                              int32_t dtype, int32_t num_heads) {
    PagedAttnArgs a{};
    if (int32_t rc = attention_args(ctx, kv, batch, d_q, q_stride, d_out, out_stride, dtype, num_heads, a)) return rc;
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
