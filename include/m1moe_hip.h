/*
 * m1moe_hip.h — C ABI of the MI355X (gfx950) MoE-layer decode library
 * libm1moe_hip.so.
 *
 * This is the boundary that replaces the Metal backend of koaWood/M1MoE for
 * the MoE block of a decoder layer (Sources/M1MoE/InferenceEngine.swift:240-266:
 * CPU router + top-K, pread expert dispatch, matvec4bit x3 + swiGLU per slot,
 * moeCombine).  It is plain C99: no HIP, C++ or torch types cross it, so a
 * SwiftPM .systemLibrary target (or ctypes, cgo, ...) can bind it directly.
 *
 * Conventions
 *  - Every call returns int32_t status; M1MOE_OK (0) is success.  On failure
 *    m1moe_last_error() returns a thread-local message for the last failing
 *    call on this thread.
 *  - A context owns all device memory it allocates (expert arena, routers,
 *    scratch, m1moe_alloc buffers).  Every compute call is enqueued
 *    asynchronously on the context's stream; m1moe_sync() waits for it.  A
 *    context is single-threaded (the reference engine is driven from one
 *    serial queue, Sources/bench/main.swift:58).
 *  - All contexts on one device share one library stream, so the library's
 *    launches on a device never overlap: on a device with at least 256 CUs
 *    the per-CU decode kernels (hidden 2048 and 4096 shapes, see
 *    m1moe_decode_kernel_for) run one workgroup on every CU and each
 *    workgroup waits for every other one, so they need the whole device.
 *    Work of another stream or process on the same GPU can keep some of
 *    their workgroups from starting; the waiting ones then give up after
 *    about a second, and the next m1moe_sync() reports M1MOE_ERR_DEVICE.
 *  - Arguments (shapes, layer/expert ranges, image sizes, dtypes, null
 *    pointers) are validated on the host before anything is enqueued.
 *    Expert indices that arrive in device memory are checked by the kernels;
 *    a bad one sets a sticky device error flag that the next m1moe_sync()
 *    reports (the kernels never read outside the arena).
 *  - Expert weights use the reference's on-disk expert block layout
 *    unchanged (layer_NN.bin): per expert, planar
 *    [gate W|S|B][up W|S|B][down W|S|B]; W = u32 [rows, cols/8] with column
 *    8w+j in bits 4j..4j+3, S/B = bf16 [rows, cols/group_size];
 *    value = nibble*scale + bias (scripts/extract_olmoe.py:20-38,145-150;
 *    ModelSpec.swift:36-52).
 */
#ifndef M1MOE_HIP_H
#define M1MOE_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define M1MOE_ABI_VERSION 1

/* status codes */
enum {
    M1MOE_OK = 0,
    M1MOE_ERR_INVALID = 1, /* bad argument: shape, range, size, null pointer */
    M1MOE_ERR_HIP = 2,     /* the HIP runtime reported an error */
    M1MOE_ERR_OOM = 3,     /* device allocation failed */
    M1MOE_ERR_DEVICE = 4   /* a kernel flagged bad device-side input */
};

/* activation dtypes */
enum { M1MOE_F32 = 0, M1MOE_BF16 = 1 };

/* projections of one expert block */
enum { M1MOE_PROJ_GATE = 0, M1MOE_PROJ_UP = 1, M1MOE_PROJ_DOWN = 2 };

typedef struct m1moe_ctx* m1moe_ctx_t;
typedef struct m1moe_graph* m1moe_graph_t;
typedef struct m1moe_event* m1moe_event_t;

/* MoE dimensions of a model.  Mirrors ModelSpec.hiddenDim/numLayers and
 * MoESpec {numExperts, topK, intermediateDim, normTopkProb} and
 * QuantSpec.groupSize (ModelSpec.swift:19-21,82-94).
 * Constraints: hidden and intermediate are multiples of 64; group_size is
 * 32, 64 or 128 and divides both; 1 <= top_k <= num_experts <= 256;
 * top_k <= 32; hidden <= 16384; intermediate <= 32768. */
typedef struct {
    int32_t hidden;
    int32_t num_experts;
    int32_t top_k;
    int32_t intermediate;
    int32_t group_size;
    int32_t num_layers;
    int32_t norm_topk_prob;
} m1moe_moe_shape;

/* ---- host-only queries (no device needed) ----------------------------- */

int32_t m1moe_abi_version(void);

/* Message of the last failing call on the calling thread ("" if none). */
const char* m1moe_last_error(void);

/* Validates a shape against the constraints above. */
int32_t m1moe_check_shape(const m1moe_moe_shape* shape);

/* ModelSpec.expertBytes4Bit (ModelSpec.swift:36-52). */
int32_t m1moe_expert_bytes(const m1moe_moe_shape* shape, uint64_t* out);

/* Byte offsets of the nine sub-blocks inside one expert block, in the order
 * gate_w, gate_s, gate_b, up_w, up_s, up_b, down_w, down_s, down_b
 * (InferenceEngine.swift:84-97). */
int32_t m1moe_expert_offsets(const m1moe_moe_shape* shape, uint64_t out[9]);

/* The decode kernel a shape runs on a device with `cus` compute units, each
 * holding `blocks_per_cu` workgroups of the per-CU kernels (1 on an
 * MI355X): *kernel = 1 (moe_decode_cu_kernel: hidden 2048, K * I 8192 or
 * 16384) or 2 (moe_decode_cuw_kernel: hidden 4096, K <= 2) when all 256 of
 * the per-CU kernel's workgroups fit on the device at once — these need the
 * whole device (conventions above) — else 0 (moe_decode_kernel, which only
 * waits for lower workgroup ids and shares the device safely).  m1moe_create
 * makes the same choice from the device's CU count and occupancy.  No
 * counterpart in the reference (one Metal path); host only. */
int32_t m1moe_decode_kernel_for(const m1moe_moe_shape* shape, int32_t cus,
                                int32_t blocks_per_cu, int32_t* kernel);

/* ---- context (replaces MetalContext, MetalContext.swift:69-185) -------- */

/* Creates a context on HIP device `device`: allocates the resident expert
 * arena for num_layers layers (num_layers * num_experts * expert_bytes), the
 * bf16 routers and all scratch.  All experts stay resident in HBM; there is
 * no expert cache or streaming (replaces the pread dispatch,
 * InferenceEngine.swift:62-77,271-280). */
int32_t m1moe_create(int32_t device, const m1moe_moe_shape* shape,
                     m1moe_ctx_t* out);

/* Frees everything the context owns.  NULL is a no-op. */
void m1moe_destroy(m1moe_ctx_t ctx);

/* Copies one layer_NN.bin image (num_experts expert blocks, exactly
 * num_experts * expert_bytes bytes) from host memory into the arena.  The
 * reference zero-fills a missing or short expert read
 * (InferenceEngine.swift:274-279); here a wrong size is an error, and so is
 * a non-finite group scale or bias (the layer then stays unloaded). */
int32_t m1moe_upload_layer_experts(m1moe_ctx_t ctx, int32_t layer,
                                   const void* host_image, uint64_t bytes);

/* Copies one layer's router (mlp.gate / block_sparse_moe.gate weight, bf16
 * [num_experts x hidden], InferenceEngine.swift:99-113) from host memory.
 * `count` must be num_experts * hidden.  It stays bf16 in HBM. */
int32_t m1moe_upload_router(m1moe_ctx_t ctx, int32_t layer,
                            const uint16_t* host_router, uint64_t count);

/* Optional per-expert f32 logit bias of one layer, added to the router
 * logits before softmax and top-K.  Absent (the default, or host_bias ==
 * NULL) is the reference's semantics; the reference has no router bias. */
int32_t m1moe_set_logit_bias(m1moe_ctx_t ctx, int32_t layer,
                             const float* host_bias, int32_t count);

/* Device pointer to the first byte of (layer, expert)'s block, for callers
 * that fill the arena on the device.  The decode and prefill kernels also
 * read repacked copies of each layer's blocks; this call marks the layer's
 * copies stale and the next decode or prefill of the layer rebuilds them
 * from the arena (refused during graph capture).  So every write through
 * the pointer must be complete, in order on the context stream (or
 * synchronised), before the next decode or prefill of the layer, and a
 * later write needs this call again first: a write after the rebuild is
 * seen by the arena's gate/up rows but not by the copies. */
int32_t m1moe_expert_block(m1moe_ctx_t ctx, int32_t layer, int32_t expert,
                           void** dev_ptr);

/* ---- memory, streams, events, graphs (so callers never include HIP) ---- */

int32_t m1moe_alloc(m1moe_ctx_t ctx, uint64_t bytes, void** dev_ptr);
int32_t m1moe_free(m1moe_ctx_t ctx, void* dev_ptr);
/* Stream-ordered on the context stream; both return after the copy ends. */
int32_t m1moe_copy_h2d(m1moe_ctx_t ctx, void* dev_dst, const void* host_src,
                       uint64_t bytes);
int32_t m1moe_copy_d2h(m1moe_ctx_t ctx, void* host_dst, const void* dev_src,
                       uint64_t bytes);
int32_t m1moe_copy_d2d(m1moe_ctx_t ctx, void* dev_dst, const void* dev_src,
                       uint64_t bytes);

/* Replaces the context stream with a caller-owned hipStream_t (passed as
 * void*); NULL restores the library stream of the device.  Refused
 * (M1MOE_ERR_INVALID) while another context is live on the same device, and
 * m1moe_create on a device refuses a second context while the first runs on
 * a caller stream: launches on one device stay on one stream. */
int32_t m1moe_set_stream(m1moe_ctx_t ctx, void* hip_stream);
int32_t m1moe_get_stream(m1moe_ctx_t ctx, void** hip_stream);

/* Waits for all work enqueued on the context stream (the reference's
 * commitSync, InferenceEngine.swift:289-294), then reports any sticky device
 * error flag raised by a kernel since the last sync as M1MOE_ERR_DEVICE. */
int32_t m1moe_sync(m1moe_ctx_t ctx);

int32_t m1moe_event_create(m1moe_ctx_t ctx, m1moe_event_t* out);
int32_t m1moe_event_record(m1moe_ctx_t ctx, m1moe_event_t ev);
/* Milliseconds between two recorded events (waits for `end`). */
int32_t m1moe_event_elapsed_ms(m1moe_event_t start, m1moe_event_t end,
                               float* ms);
void m1moe_event_destroy(m1moe_event_t ev);

/* Captures every call enqueued on the context stream between begin and end
 * into a HIP graph (no device work runs during capture).  A graph is
 * launched on the context it was captured on; its launch is refused
 * (M1MOE_ERR_INVALID) once a call has reallocated a scratch buffer of the
 * context since the capture (a prefill, decoder prefill or attention call
 * larger than any before), since the graph holds the freed addresses:
 * capture it again. */
int32_t m1moe_graph_begin(m1moe_ctx_t ctx);
int32_t m1moe_graph_end(m1moe_ctx_t ctx, m1moe_graph_t* out);
int32_t m1moe_graph_launch(m1moe_ctx_t ctx, m1moe_graph_t graph);
void m1moe_graph_destroy(m1moe_graph_t graph);

/* ---- the MoE block ------------------------------------------------------ */

/* Router logits, softmax and top-K for T tokens (computeRouterScores +
 * selectTopK, InferenceEngine.swift:490-519, moved on-GPU).
 * d_x: [T x hidden] in x_dtype.  Logits are exact products accumulated in
 * f64 and rounded once to f32 (plus the optional logit bias); experts are
 * ranked by descending logit with ties to the lower index; weights are the
 * softmax probabilities of the selected experts, renormalised over the
 * selection when norm_topk_prob is set (:514-517).
 * Outputs: d_topk_idx int32 [T x top_k], d_topk_w f32 [T x top_k],
 * d_logits f32 [T x num_experts] (nullable). */
int32_t m1moe_router_topk(m1moe_ctx_t ctx, int32_t layer, int32_t T,
                          const void* d_x, int32_t x_dtype,
                          int32_t* d_topk_idx, float* d_topk_w,
                          float* d_logits);

/* One token through the MoE block of `layer` (batch-1 decode):
 *   out[d] = residual[d] + sum_k w_k * down_k(silu(gate_k x) * up_k x)[d]
 * d_x: [hidden] in x_dtype; d_residual: f32 [hidden] or NULL (zeros);
 * d_out: f32 [hidden].  d_topk_idx / d_topk_w (nullable) receive the routing.
 * Replaces InferenceEngine.swift:240-266 (router, dispatch, the 4K+1 Metal
 * dispatches and the residual hand-off).  Asynchronous. */
int32_t m1moe_moe_decode(m1moe_ctx_t ctx, int32_t layer, const void* d_x,
                         int32_t x_dtype, const float* d_residual,
                         float* d_out, int32_t* d_topk_idx, float* d_topk_w);

/* Same, with the routing given in device memory: d_topk_idx int32 [top_k],
 * d_topk_w f32 [top_k] (InferenceEngine.swift:247-263 without the router). */
int32_t m1moe_moe_decode_given_topk(m1moe_ctx_t ctx, int32_t layer,
                                    const void* d_x, int32_t x_dtype,
                                    const int32_t* d_topk_idx,
                                    const float* d_topk_w,
                                    const float* d_residual, float* d_out);

/* T tokens at once (prefill): routing per token as m1moe_router_topk, the
 * (token, slot) pairs grouped by expert, gate/up/down as MFMA f16 grouped
 * GEMMs with the 4-bit dequant fused, and a deterministic weighted combine.
 * Results equal T independent m1moe_moe_decode calls up to f16 operand
 * rounding (the SwiGLU products in blocks of 32 with a power of two each
 * where they pass the f16 range; a non-finite one is clamped and reported
 * by the next m1moe_sync).  d_x [T x hidden], d_residual f32 [T x hidden]
 * or NULL, d_out f32 [T x hidden], d_topk_idx/d_topk_w [T x top_k]
 * nullable.  T <= the context's prefill capacity (4096 tokens). */
int32_t m1moe_moe_prefill(m1moe_ctx_t ctx, int32_t layer, int32_t T,
                          const void* d_x, int32_t x_dtype,
                          const float* d_residual, float* d_out,
                          int32_t* d_topk_idx, float* d_topk_w);

/* m1moe_moe_prefill with the same arguments, kernels and results, that
 * allocates nothing: no counterpart in the reference.  It is for callers that
 * cannot allocate device memory (code under HIP graph capture without a
 * warm-up call, tight serving loops, harnesses that forbid hipMalloc).  Its
 * scratch is a fixed 64 MiB static device array per GPU (looked up by
 * m1moe_create, held until the process ends) instead of the context's
 * buffers that m1moe_moe_prefill grows; a T whose scratch would not fit is
 * rejected with M1MOE_ERR_INVALID naming the largest T that fits (776
 * tokens at hidden 2048, 8 x 1024 experts; 676 at hidden 4096,
 * 2 x 14336).  Every call on one GPU shares that array, so calls that overlap
 * on one GPU (two streams, or two contexts on one device) race. */
int32_t m1moe_moe_prefill_noalloc(m1moe_ctx_t ctx, int32_t layer, int32_t T,
                                  const void* d_x, int32_t x_dtype,
                                  const float* d_residual, float* d_out,
                                  int32_t* d_topk_idx, float* d_topk_w);

/* Writes the dequantised f32 weights of one projection of one expert,
 * row-major [rows x cols] (gate/up: intermediate x hidden; down: hidden x
 * intermediate), value f32(n)*f32(s)+f32(b), for the bit-exact weight check
 * (Shaders.metal:66-77). */
int32_t m1moe_dequant_debug(m1moe_ctx_t ctx, int32_t layer, int32_t expert,
                            int32_t proj, float* d_out);

/* ---- dense decoder step around the MoE block ---------------------------- */

/* Building blocks (each asynchronous on the context stream; all vectors f32
 * unless stated, weights bf16 row-major). */

/* out[i] = x[i] * rsqrt(sum(x^2)/n + eps) * w[i]   (rmsNormSum + rmsNormApply,
 * Shaders.metal:96-134; InferenceEngine.swift:298-320).  n <= 65536. */
int32_t m1moe_rmsnorm(m1moe_ctx_t ctx, const float* d_x, const uint16_t* d_w,
                      float* d_out, int32_t n, float eps);

/* y[r] = sum_c W[r][c] * x[c] (+ residual[r] when d_residual is non-null)
 * (matvecBF16, Shaders.metal:328-358; residualAdd :152-162).
 * cols % 8 == 0, cols <= 65536. */
int32_t m1moe_matvec_bf16(m1moe_ctx_t ctx, const uint16_t* d_w,
                          const float* d_x, const float* d_residual,
                          float* d_y, int32_t rows, int32_t cols);

/* Decode attention of one query position over seq_len cached positions
 * (attnScores + attnSoftmax + attnValues, Shaders.metal:209-326, dispatched as
 * InferenceEngine.swift:349-399): per head h,
 * s_p = (q_h . k_p[h / hpkv]) / sqrt(head_dim), p_s = softmax(s), out_h =
 * sum_p p_p v_p[h / hpkv].  q f32 [num_heads x head_dim]; caches f32
 * [>= seq_len x num_kv_heads*head_dim]; out f32 [num_heads x head_dim].
 * head_dim is 64, 128 or 256; num_heads % num_kv_heads == 0;
 * 1 <= seq_len <= 65536. */
int32_t m1moe_attention_decode(m1moe_ctx_t ctx, const float* d_q,
                               const float* d_kcache, const float* d_vcache,
                               float* d_out, int32_t num_heads,
                               int32_t num_kv_heads, int32_t head_dim,
                               int32_t seq_len);

/* Index of the largest of n values, ties to the lower index, written to
 * d_idx (greedy sampling, InferenceEngine.swift:550-555: a scan from x[0]
 * with a strict >, so NaN never wins except at index 0). */
int32_t m1moe_argmax(m1moe_ctx_t ctx, const float* d_x, int32_t n,
                     int32_t* d_idx);

/* The whole decode step (InferenceEngine.forward and runLayer,
 * InferenceEngine.swift:125-266, which ran norms/projections/attention on
 * Metal and q/k norms, RoPE, the KV store, router and top-K on the CPU with
 * three syncs per layer): token embedding; per layer input RMSNorm, q/k/v
 * matvecs, per-head q/k RMSNorm (when the model has it), RoPE, f32 KV cache
 * store, attention, o_proj + residual, post-attention RMSNorm, the MoE block
 * of the context; final RMSNorm, lm_head, greedy argmax — all on the GPU with
 * no host sync.  The token and the position live in device memory, so each
 * step reads the previous step's argmax and a greedy loop can be captured in
 * a graph and replayed. */
typedef struct m1moe_dec* m1moe_dec_t;

/* Attention and vocabulary of a model (ModelSpec.swift AttentionSpec and
 * vocabSize).  hidden and num_layers come from the MoE context.
 * head_dim is 64, 128 or 256 (even); num_heads % num_kv_heads == 0;
 * 1 <= max_seq <= 65536; vocab >= 1. */
typedef struct {
    int32_t vocab;
    int32_t num_heads;
    int32_t num_kv_heads;
    int32_t head_dim;
    int32_t max_seq;   /* KV cache positions */
    int32_t qk_norm;   /* per-head q/k RMSNorm before RoPE (OLMoE) */
    float rope_theta;
    float rms_eps;
} m1moe_dec_shape;

/* dense tensors of a model (bf16, row-major) */
enum {
    M1MOE_W_EMBED = 0,      /* [vocab x hidden]                 model.embed_tokens */
    M1MOE_W_LM_HEAD = 1,    /* [vocab x hidden]                 lm_head */
    M1MOE_W_FINAL_NORM = 2, /* [hidden]                         model.norm */
    M1MOE_W_IN_NORM = 3,    /* [hidden]       per layer         input_layernorm */
    M1MOE_W_POST_NORM = 4,  /* [hidden]       per layer         post_attention_layernorm */
    M1MOE_W_Q = 5,          /* [heads*hd x hidden]   per layer  self_attn.q_proj */
    M1MOE_W_K = 6,          /* [kv_heads*hd x hidden]           self_attn.k_proj */
    M1MOE_W_V = 7,          /* [kv_heads*hd x hidden]           self_attn.v_proj */
    M1MOE_W_O = 8,          /* [hidden x heads*hd]              self_attn.o_proj */
    M1MOE_W_Q_NORM = 9,     /* [head_dim]     per layer         self_attn.q_norm (first head_dim
                               values, applied to every head: applyHeadRMSNorm, InferenceEngine.swift:538-548) */
    M1MOE_W_K_NORM = 10     /* [head_dim]     per layer         self_attn.k_norm */
};

/* The decoder uses the MoE context's layers, stream and error flag; destroy
 * it before the context. */
int32_t m1moe_dec_create(m1moe_ctx_t moe, const m1moe_dec_shape* shape,
                         m1moe_dec_t* out);
void m1moe_dec_destroy(m1moe_dec_t dec);
/* count must be the tensor's element count (above); layer is ignored for
 * the model-level tensors. */
int32_t m1moe_dec_upload(m1moe_dec_t dec, int32_t which, int32_t layer,
                         const uint16_t* host_bf16, uint64_t count);
/* Position 0 and an empty KV cache (InferenceEngine.reset, :159-163; the
 * positions past the new one are never read, so only the position is
 * rewritten).  Enqueued on the context stream. */
int32_t m1moe_dec_reset(m1moe_dec_t dec);
/* One step at the current device-side position: reads the token from
 * d_token_in (int32 device), writes the greedy next token to d_token_out
 * (may be the same address) and advances the position.  d_logits (nullable)
 * receives f32 [vocab].  A prompt is fed as steps with d_token_in =
 * &prompt[i]; a greedy loop passes out = in, or &toks[i+1] to keep them.  A token outside
 * [0, vocab) is embedded as token 0, and with the cache full (position ==
 * max_seq) nothing is stored and the position stays; either sets the device
 * error flag, reported by the next m1moe_sync. */
int32_t m1moe_dec_step(m1moe_dec_t dec, const int32_t* d_token_in,
                       int32_t* d_token_out, float* d_logits);
/* Sequence mode: d_seq int32 [seq_cap] holds the prompt in [0, n_prompt).
 * The step at device-side position p embeds d_seq[p] and, when p + 1 >=
 * n_prompt, stores its greedy token at d_seq[p + 1] (if p + 1 < seq_cap).
 * After m1moe_dec_reset, n_prompt + n_gen calls (or replays of one graph
 * captured around one call) run the reference's prefill-then-generate loop
 * (Sources/bench/main.swift:136-163): the prompt forwarded token by token,
 * then each generated token fed back, d_seq[n_prompt .. n_prompt + n_gen]
 * receiving the n_gen + 1 greedy tokens.  p >= seq_cap sets the device error
 * flag (as a token outside the vocabulary). */
int32_t m1moe_dec_step_seq(m1moe_dec_t dec, int32_t* d_seq, int32_t n_prompt,
                           int32_t seq_cap, float* d_logits);
/* The prompt at once: the T tokens d_tokens (int32 device) at positions
 * pos .. pos + T - 1 through every layer in one batch per layer (the
 * reference forwards a prompt token by token, Sources/bench/main.swift:
 * 139-141): q/k/v and o_proj as f32 GEMMs over the T rows, causal attention,
 * the MoE block through the grouped prefill (m1moe_moe_prefill; its f16
 * activations make this path agree with T m1moe_dec_step calls to ~1e-3).
 * Their K/V rows enter the cache, the position advances by T, d_token_out
 * receives the greedy token after the last one and d_logits (nullable) its
 * logits.  1 <= T <= max_seq (prompts longer than 4096 tokens go through in
 * pieces of 4096, each from the position the previous one reached);
 * positions past max_seq set the device error flag.  The first call with a
 * larger piece than any before grows the scratch (make it before capturing a
 * graph). */
int32_t m1moe_dec_prefill(m1moe_dec_t dec, const int32_t* d_tokens, int32_t T,
                          int32_t* d_token_out, float* d_logits);
/* The current position (waits for the context stream). */
int32_t m1moe_dec_position(m1moe_dec_t dec, int32_t* pos);

/* ---- several conversations at once ---------------------------------------
 * Building blocks for callers that run a batch of sequences through a layer
 * (no counterpart in the reference, whose engine holds one conversation): a
 * KV cache in pages, attention over it, and sampling.  Asynchronous on the
 * context stream like the blocks above; lengths, positions and page numbers
 * are read from device memory, so a captured graph serves later steps too. */

/* A KV cache in pages, the caller's memory.  Position p of a sequence lies in
 * page pages[p / page_size] of its page table, at slot p % page_size.
 * Constraints: page_size is a power of two, 8 to 4096; num_pages >= 1;
 * head_dim is 64, 128 or 256; num_kv_heads * head_dim <= 65536. */
typedef struct {
    void* d_k;             /* [num_pages][page_size][num_kv_heads][head_dim] */
    void* d_v;             /* the same */
    int32_t dtype;         /* M1MOE_F32 or M1MOE_BF16 */
    int32_t num_pages;
    int32_t page_size;
    int32_t num_kv_heads;
    int32_t head_dim;
} m1moe_paged_kv;

/* The rows of one call: sequence s has the rows d_row_start[s] ..
 * d_row_start[s + 1] - 1 (none, one, or a whole prompt), which are its last
 * positions: row d_row_start[s] + i is at position d_kv_len[s] - n + i of its
 * n rows.  num_rows is how many rows the caller's buffers hold; those outside
 * every sequence are left as they were.
 * prefix_len > 0: the first prefix_len positions of every sequence lie in the
 * pages d_prefix_pages and are read there (attention computes them once for
 * all; the sequences' own table entries of pages wholly inside the prefix are
 * not read).  Every row is at a position past the prefix.
 * Constraints: 1 <= num_seqs <= 1024; 1 <= num_rows <= 1048576; table_stride
 * >= 1, table_stride * page_size <= 2^24 positions; 0 <= prefix_len <=
 * table_stride * page_size.  In device memory: 0 <= d_row_start[s] <=
 * d_row_start[s + 1] <= num_rows, n <= d_kv_len[s] <= table_stride *
 * page_size, d_kv_len[s] - n >= prefix_len where n > 0.  A sequence that
 * breaks this is skipped, a page outside the cache is not touched (attention
 * reads page 0 in its place); either sets the device error flag, reported by
 * the next m1moe_sync.  (Rows that starts out of order give to two sequences
 * hold either's result.) */
typedef struct {
    int32_t num_seqs;
    int32_t num_rows;
    int32_t table_stride;           /* entries per row of d_pages */
    int32_t prefix_len;
    const int32_t* d_row_start;     /* [num_seqs + 1] */
    const int32_t* d_kv_len;        /* [num_seqs], this call's rows included */
    const int32_t* d_pages;         /* [num_seqs][table_stride] */
    const int32_t* d_prefix_pages;  /* [ceil(prefix_len / page_size)], or NULL */
} m1moe_paged_batch;

/* What m1moe_kv_append reads and writes besides the cache.  Row strides are in
 * elements and multiples of 16 bytes, at least a row's length (q, k and v may
 * be columns of one matrix); pointers are 16-byte aligned. */
typedef struct {
    int32_t dtype;           /* of q, k, v and q_out: M1MOE_F32 or M1MOE_BF16 */
    int32_t num_heads;       /* a multiple of the cache's num_kv_heads */
    const void* d_q;         /* [num_rows][num_heads * head_dim], or NULL: k and v only */
    const void* d_k;         /* [num_rows][num_kv_heads * head_dim] */
    const void* d_v;         /* the same */
    void* d_q_out;           /* as d_q; d_q itself, with its stride, or rows that share no
                              * memory with those of d_q, d_k and d_v; NULL with d_q */
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    const uint16_t* d_q_norm;  /* bf16 [head_dim] per-head RMSNorm weights, or NULL: no norm */
    const uint16_t* d_k_norm;
    float eps;
    int32_t rotary_dim;      /* 0, or a multiple of 16 up to head_dim: rotated dims, from dim 0 */
    int32_t interleaved;     /* pairs (2i, 2i + 1) instead of (i, i + rotary_dim / 2) */
    float rope_amplitude;    /* factor of cos and sin (1 for unscaled RoPE) */
    const float* d_inv_freq; /* f32 [rotary_dim / 2]: angle of pair i = position * inv_freq[i] */
} m1moe_kv_append_args;

/* One row of settings per row of logits, all in device memory; any but d_u may
 * be NULL: temperature 1, no top-k, no top-p, no min-p. */
typedef struct {
    const float* d_u;            /* uniform draws in [0, 1) */
    const float* d_temperature;  /* <= 0 (or NaN): the largest logit */
    const int32_t* d_top_k;      /* <= 0: off */
    const float* d_top_p;        /* >= 1 (or NaN): off */
    const float* d_min_p;        /* <= 0 (or NaN): off */
} m1moe_sample_params;

/* The checks that the calls below make of these descriptions (host only). */
int32_t m1moe_check_paged(const m1moe_paged_kv* kv, const m1moe_paged_batch* batch);

/* For every row of the batch: q and k normalised per head (x * rsqrt(mean(x^2)
 * + eps) * w, where a weight is given), their first rotary_dim dims rotated by
 * the row's position ((a, b) -> (a cos - b sin, a sin + b cos) *
 * rope_amplitude; the angle is formed in 64 bits, all else in f32), q written
 * to d_q_out, k and v to their page and slot.  Two rows must not share a slot. */
int32_t m1moe_kv_append(m1moe_ctx_t ctx, const m1moe_paged_kv* kv,
                        const m1moe_paged_batch* batch,
                        const m1moe_kv_append_args* args);

/* Attention of every row of the batch over its own sequence's positions up to
 * its own: out_h = sum_p softmax_p(q_h . k_p / sqrt(head_dim)) v_p, kv head
 * h / (num_heads / num_kv_heads).  q and out [num_rows][num_heads * head_dim]
 * in dtype (row strides in elements, as above; their rows must not share memory,
 * with different strides not their ranges either); scores, softmax and sums in
 * f32 (dtype M1MOE_BF16: the softmax numerators that multiply v are rounded to
 * two bf16 parts, 16 bits).  dtype M1MOE_BF16 needs a bf16 cache; num_heads is a
 * multiple of num_kv_heads, at most 64 times it, and num_heads * head_dim <=
 * 65536.
 * Later positions take no part, whatever they hold.  The first call of a
 * larger batch may grow the context's workspace (make it before capturing: of
 * the same heads and types, one of as many rows and as long a prefix or less
 * needs no more). */
int32_t m1moe_paged_attention(m1moe_ctx_t ctx, const m1moe_paged_kv* kv,
                              const m1moe_paged_batch* batch, const void* d_q,
                              int64_t q_stride, void* d_out, int64_t out_stride,
                              int32_t dtype, int32_t num_heads);

/* One token per row of d_logits (f32 [rows], stride elements apart, a multiple
 * of 4, >= vocab).  With the logits of a row in descending order, ties to the
 * lower index, and w_i = exp((x_i - x_0) / temperature): the first top_k
 * stay; of these the fewest whose w sum to at least top_p of their total; of
 * these the ones with w_i >= min_p (the first always stays).  With S the sum
 * of what stayed the token is the first whose running sum reaches u * S
 * (m1moe_amd/sampling.py with top-k and min-p; u outside [0, 1] is taken to
 * the nearer end, NaN to 0).  Sums are of whole multiples of 2^-44, so they do
 * not depend on an order; w below 2^-45 counts as 0 and is never drawn.  NaN
 * logits count as -inf; a row with nothing above -inf gives token -1,
 * probability 0.  d_probs (nullable) receives w / S of the token.
 * 1 <= rows <= 65536, 1 <= vocab <= 262144. */
int32_t m1moe_sample(m1moe_ctx_t ctx, const float* d_logits, int32_t rows,
                     int32_t vocab, int64_t stride,
                     const m1moe_sample_params* params, int32_t* d_tokens,
                     float* d_probs);

/* ---- drafted tokens ------------------------------------------------------
 * A step that verifies drafts runs a tree of tokens per sequence through the
 * layers: the rows of a sequence in an m1moe_paged_batch are its tree, row 0 the
 * last token that is certain, every other row a drafted one that hangs on an
 * earlier row, its parent.  Their keys and values are stored row by row behind
 * the conversation's kv_len - n positions; a row sees those and its own
 * ancestors, and its angle is that of its depth.  Then a token is drawn at every
 * row (m1moe_sample), and the drafts that were drawn are taken over.  All
 * asynchronous on the context stream.  m1moe_tree_attention uses
 * m1moe_paged_attention's workspace, m1moe_matmul_q4 one of its own, both the
 * context's; the other calls need none.  A tree has at most 256 rows. */

/* Who sees whom, and depths, from every row's parent: d_parents[row] is the
 * parent's number in the same tree (0 its first row), -1 for none, and lower than
 * the row's own (one that is not counts as none and sets the device error flag,
 * reported by the next m1moe_sync).  Row i of a tree gets in d_mask[row]
 * [mask_words] bit j (word j / 64, bit j % 64) for itself and every ancestor j, in
 * d_depth[row] the number of its ancestors.  Rows outside every sequence are left
 * as they were; a sequence whose starts are out of range or that has more than
 * 64 * mask_words rows is skipped and sets the flag.
 * 1 <= num_seqs <= 1024, 1 <= num_rows <= 1048576, 1 <= mask_words <= 4. */
int32_t m1moe_tree_plan(m1moe_ctx_t ctx, int32_t num_seqs, int32_t num_rows,
                        const int32_t* d_row_start, const int32_t* d_parents,
                        int32_t mask_words, uint64_t* d_mask, int32_t* d_depth);

/* m1moe_kv_append for the rows of trees: a row is stored at its own slot, d_kv_len
 * - n + i for row i, and rotated by the position d_kv_len - n + d_depth[row].  The
 * cache and d_q_out share no memory with d_depth and the batch's arrays. */
int32_t m1moe_tree_append(m1moe_ctx_t ctx, const m1moe_paged_kv* kv,
                          const m1moe_paged_batch* batch,
                          const m1moe_kv_append_args* args, const int32_t* d_depth);

/* m1moe_paged_attention for the rows of trees: row i sees the d_kv_len - n
 * positions before its tree and, of its tree, the rows j <= i whose bit is set in
 * d_mask[row][mask_words] (its own among them only if set).  A row that sees
 * nothing gives zeros, as one whose scores are all -inf does.  A sequence of more
 * than 64 * mask_words rows is skipped and sets the device error flag.  d_out shares
 * no memory with d_mask, the batch's arrays and the cache. */
int32_t m1moe_tree_attention(m1moe_ctx_t ctx, const m1moe_paged_kv* kv,
                             const m1moe_paged_batch* batch, const uint64_t* d_mask,
                             int32_t mask_words, const void* d_q, int64_t q_stride,
                             void* d_out, int64_t out_stride, int32_t dtype,
                             int32_t num_heads);

/* What a sequence keeps of its tree.  From row 0 on the path goes to the lowest
 * child whose token d_drafts[row] is the one drawn at the path's row,
 * d_drawn[row].  The path's rows, in all num_caches caches (the layers', alike in
 * type and sizes, 1 to 64, sharing no memory), move to the places base, base + 1,
 * .. (base = d_kv_len - n); what stood at other places of the tree stays.  Per
 * row: d_path[row_start + i] = the path's row i, -1 past its end.  Per sequence:
 * d_accepted = rows of the path, d_next = the token drawn at its last row (the
 * next tree's row 0), d_past = base + accepted; 0, -1 and d_kv_len for a sequence
 * without rows.  One that is out of range or has more than 256 rows is skipped
 * with the same results, a move from or to a page outside the cache is left out
 * and a parent that is not lower than its row counts as none: each sets the
 * device error flag.  Outputs must not overlap inputs, caches or each other, inputs
 * not the caches. */
int32_t m1moe_tree_accept(m1moe_ctx_t ctx, const m1moe_paged_kv* kvs,
                          int32_t num_caches, const m1moe_paged_batch* batch,
                          const int32_t* d_parents, const int32_t* d_drafts,
                          const int32_t* d_drawn, int32_t* d_path,
                          int32_t* d_accepted, int32_t* d_next, int32_t* d_past);

/* Weights as m1moe_quantize_4bit makes them: [rows][cols / 8] words, column 8w + j
 * in bits 4j..4j+3 of word w, and bf16 scales and biases [rows][cols / group_size];
 * weight = nibble * scale + bias.  group_size is 32, 64 or 128 and divides cols;
 * rows <= 1048576, cols <= 65536; pointers are 16-byte aligned. */
typedef struct {
    const uint32_t* d_w;
    const uint16_t* d_scales;
    const uint16_t* d_biases;
    int32_t rows;
    int32_t cols;
    int32_t group_size;
} m1moe_q4_weights;

/* y[t][r] = sum_c x[t][c] W[r][c] (+ residual[t][r]) for 1 to 65536 tokens t.  x
 * [tokens][cols] in x_dtype, y and residual (NULL: none; d_y itself: in place)
 * [tokens][rows] in y_dtype, y_stride elements apart; row strides are multiples of
 * 16 bytes.  f32 rows give an f32 y, bf16 ones either.  Where it meets the nibbles an
 * f32 x is taken to 22 bits, and x of either type to 2^-39 of the largest value of
 * its row (of at most 32 tokens: of 256 columns for groups of 32, else 512) where that
 * is more: in an f32 row that is what is below 2^-16 of its largest, in a bf16 row
 * below 2^-31.  Products are exact and summed in f32, a group's first.  A row of x that
 * holds an infinity or a NaN gives results that are not finite, the other rows are what
 * they were.  A result does not depend on what else runs, but with the number of tokens
 * its last bits may change, and within those 2^-39 how small values are kept.
 * Calls of more than 32 tokens, or of so few rows of W that their columns are
 * shared by workgroups, use a workspace of the context's, which the first such
 * call of more tokens or longer rows of x makes (behind one of more than 32 tokens
 * none of as many tokens and bytes of a row or fewer needs more): do that before
 * capturing (in a capture it is refused, and graphs from before it are refused
 * afterwards). */
int32_t m1moe_matmul_q4(m1moe_ctx_t ctx, const m1moe_q4_weights* weights,
                        const void* d_x, int32_t x_dtype, int64_t x_stride,
                        int32_t tokens, const void* d_residual, void* d_y,
                        int32_t y_dtype, int64_t y_stride);

/* ---- the converted model directory on disk (host-side) -----------------
 * scripts/extract_olmoe.py writes model_weights.bin (non-expert tensors,
 * 4-byte aligned) + model_weights.json ({name: {offset, shape, dtype}}) and
 * packed_experts/layer_NN.bin (E expert blocks per layer). */
typedef struct m1moe_store* m1moe_store_t;
enum { M1MOE_DT_BF16 = 0, M1MOE_DT_F32 = 1, M1MOE_DT_U32 = 2 };

/* WeightStore.init (WeightStore.swift:47-76): maps the .bin read-only and
 * reads the manifest; every tensor must lie inside the file.  Host only. */
int32_t m1moe_store_open(const char* bin_path, const char* json_path,
                         m1moe_store_t* out);
void m1moe_store_close(m1moe_store_t store);
int32_t m1moe_store_count(m1moe_store_t store, int32_t* n);
/* WeightStore.info / pointer (:86-100): the tensor's bytes inside the
 * mapping, dtype (M1MOE_DT_*), shape (4 entries, unused ones 0) and rank.
 * Each output is nullable. */
int32_t m1moe_store_tensor(m1moe_store_t store, const char* name,
                           const void** data, int32_t* dtype, int64_t* shape,
                           int32_t* ndim);

/* Uploads a converted model directory: every layer_NN.bin of the context's
 * layers (m1moe_upload_layer_experts; the size must be E x expert_bytes),
 * each layer's router (mlp.gate.weight, or block_sparse_moe.gate.weight,
 * InferenceEngine.swift:593-598) and, when dec is non-null, the dense
 * tensors under the reference's weight keys (:580-599; f32 tensors are
 * rounded to bf16; q/k norms: the first head_dim values).  Shapes are
 * checked against the context and decoder.  threads: parallel reads per
 * layer file. */
int32_t m1moe_load_model(m1moe_ctx_t ctx, m1moe_dec_t dec, const char* model_dir,
                         int32_t threads);

/* ---- the converters' 4-bit quantizer (host-only; offline) ---------------
 * quantize_4bit of scripts/extract_olmoe.py:116-159 (extract_mixtral.py
 * :93-116 is the same): per row and group of group_size columns, in f32,
 * lo = min, s = (max - lo) / 15 (1 where that is 0), nibble =
 * clamp(round-half-even((w - lo) / s), 0, 15); scales = bf16(s), biases =
 * bf16(lo), nibbles 8 per u32 (column 8w+j in bits 4j..4j+3).  cols must be
 * a multiple of group_size and of 8 (:130-131); a non-finite weight is
 * refused (M1MOE_ERR_INVALID).  threads: host threads over rows (<= 0: 1). */
int32_t m1moe_quantize_4bit(const float* w, int64_t rows, int64_t cols,
                            int32_t group_size, uint32_t* packed,
                            uint16_t* scales, uint16_t* biases,
                            int32_t threads);
/* One expert block of layer_NN.bin from f32 gate [I, h], up [I, h] and
 * down [h, I] (the per-expert loop of extract_olmoe.py:322-338):
 * [gate W|S|B][up W|S|B][down W|S|B].  block_bytes must be expert_bytes. */
int32_t m1moe_quantize_expert(const m1moe_moe_shape* shape, const float* gate,
                              const float* up, const float* down, void* block,
                              uint64_t block_bytes, int32_t threads);
/* f32_to_bf16 of extract_olmoe.py:104-111: (bits + 0x7FFF + lsb) >> 16. */
int32_t m1moe_f32_to_bf16(const float* x, uint64_t n, uint16_t* out);

/* ---- BPE tokenizer (host-only) -------------------------------------------
 * Tokenizer (Sources/M1MoE/Tokenizer.swift) over a HuggingFace
 * tokenizer.json: byte-level BPE (GPT-2 / OLMoE) or, when
 * model.byte_fallback is true, SentencePiece BPE (Mistral / Mixtral).
 * Text crosses the boundary as UTF-8 bytes (not NUL-terminated). */
typedef struct m1moe_tokenizer* m1moe_tokenizer_t;

/* Tokenizer.init(url:) (:35-62).  M1MOE_ERR_INVALID when the file cannot be
 * read or lacks model.vocab / model.merges (TokenizerError.invalidFormat). */
int32_t m1moe_tokenizer_load(const char* path, m1moe_tokenizer_t* out);
void m1moe_tokenizer_free(m1moe_tokenizer_t tok);
/* Mode (1 = SentencePiece BPE, 0 = byte-level), vocabulary entries and merge
 * pairs.  Each output is nullable. */
int32_t m1moe_tokenizer_info(m1moe_tokenizer_t tok, int32_t* sentencepiece,
                             uint64_t* vocab_size, uint64_t* merges);
/* encode(_:addBOS:bos:) (:66-72): bos first when add_bos.  *n_ids gets the
 * count; ids == NULL only asks for it; a count above cap is an error. */
int32_t m1moe_tokenizer_encode(m1moe_tokenizer_t tok, const char* text,
                               uint64_t text_len, int32_t add_bos,
                               uint32_t bos, uint32_t* ids, uint64_t cap,
                               uint64_t* n_ids);
/* decode(_:skipSpecial:) (:76-81): UTF-8 bytes into out (NUL added when
 * there is room); *out_len gets the length; out == NULL only asks for it. */
int32_t m1moe_tokenizer_decode(m1moe_tokenizer_t tok, const uint32_t* ids,
                               uint64_t n, int32_t skip_special, char* out,
                               uint64_t cap, uint64_t* out_len);

/* ---- seeded synthetic inputs (host-only; bench and test data) ----------
 * Counter-based: value i of tensor `tensor_id` under `seed` is a function of
 * (seed, tensor_id, i) only, so any slice can be generated independently.
 * Normals are Box-Muller in f64, scaled by sigma, rounded to f32, then
 * (bf16 variants) rounded to nearest-even bf16. */
int32_t m1moe_synth_normal_bf16(uint64_t seed, uint64_t tensor_id,
                                uint64_t n, float sigma, int32_t absval,
                                uint16_t* out);
int32_t m1moe_synth_normal_f32(uint64_t seed, uint64_t tensor_id, uint64_t n,
                               float sigma, float* out);
/* One layer_NN.bin image: nibbles uniform in 0..15 (8 per u32), scales
 * bf16 |N(0, scale_sigma)|, biases bf16 N(0, bias_sigma), per expert block.
 * `bytes` must be num_experts * expert_bytes.  Uses up to `threads` host
 * threads (<=0: one). */
int32_t m1moe_synth_layer_image(const m1moe_moe_shape* shape, uint64_t seed,
                                int32_t layer, float scale_sigma,
                                float bias_sigma, void* out, uint64_t bytes,
                                int32_t threads);

#ifdef __cplusplus
}
#endif

#endif /* M1MOE_HIP_H */
