/* crosslane MI355X routed-expert lane: C ABI.
 *
 * One resident expert bank on one GPU; per token and layer, "compute these
 * top-k experts for this vector, then join them in a fixed order". Plain
 * pointers and sizes only. Every call returns int32 status (XL_OK = 0) and,
 * when `err` is non-null, fills it; the context also keeps the last error.
 * A context is driven by one caller thread at a time (the reference drives its
 * HIP lane from one dedicated worker thread, engine/strata/warm/worker.hpp:9-18).
 * Its device work is ordered: every call that enqueues work waits (on the GPU,
 * hipStreamWaitEvent) for the context's previous call when that one named
 * another stream, so calls on one context never overlap, whatever streams they
 * name (they share the context's workspace, exchange buffers and counters).
 * The single-launch layer kernels spin on data other workgroups of the same
 * launch produce: they need all their workgroups resident at once (one per CU)
 * and make progress only while no other kernel holds the CUs they wait for.
 * Two contexts, or another persistent kernel, launched concurrently on other
 * streams can starve them; such a wait ends in the device error flag
 * (XL_E_DEVICE, "layer wait timeout") after about a second, not in a hang.
 * No call allocates device memory after xl_bank_create (the workspace is sized
 * at xl_open, like the reference's arena reservation,
 * engine/strata/sycl/stage/wiring/hip_resident_bank.hpp:63-94).
 *
 * Conventions mirror the reference's DSO ABI (engine/strata/sycl/stage/wiring/
 * abi_v2.h:28-68, abi_backend_plugin.cpp:31-39): a version + struct-size check
 * before anything is written, an int32 code plus a 512-byte message, every
 * exception caught at the boundary, and a context poisoned by a device error
 * (all later compute calls fail until xl_close).
 */
#ifndef CROSSLANE_H
#define CROSSLANE_H
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

#define XL_ABI_VERSION 3u

enum {
    XL_OK = 0,
    XL_E_ARG = 1,        /* invalid argument (shape, id, pointer, finiteness) */
    XL_E_STATE = 2,      /* wrong call order, or a poisoned context */
    XL_E_HIP = 3,        /* HIP runtime error */
    XL_E_DEVICE = 4,     /* a kernel reported an error flag (bad id, non-finite) */
    XL_E_VERSION = 5,    /* ABI version or struct size mismatch */
    XL_E_MEMORY = 6      /* device or host allocation failed */
};

/* ggml block type ids accepted for expert matrices */
enum { XL_IQ2_XXS = 16, XL_IQ2_XS = 17, XL_IQ1_M = 29 };

typedef struct xl_error {
    int32_t code;
    char message[512];
} xl_error;

typedef struct xl_config {
    uint32_t struct_bytes; /* sizeof(xl_config) */
    int32_t device;        /* HIP device ordinal */
    int32_t dim;           /* d_model and d_ff: 256, 512, 768, 1024, 2048, 2304, */
    int32_t ff;            /* 3072, 4096 or 5120 (the real expert: dim 5120, ff 2304) */
    int32_t n_layers;      /* layers in the bank */
    int32_t n_experts;     /* routed experts per layer */
    int32_t max_picks;     /* top-k bound, 1..16 (reference kPicks = 8, model_meta.hpp:18) */
    int32_t max_tokens;    /* grouped-path token bound (0 = grouped path unused). Its
                              workspace, with P = max_tokens * max_picks: about
                              16 * (P / 16 + min(P, n_experts) + 1) * (dim + ff) bytes
                              of per-slot quants plus 4 * P * (dim + ff) bytes of h
                              and per-pick rows (~190 MB at 512 tokens, 8 picks,
                              384 experts, 4096 x 3072). xl_bank_create adds a
                              quarter of the quants' dim part where a gate or up
                              matrix is IQ1_M, of their ff part where a down is */
    float swiglu_limit;    /* SwiGLU limit (model_meta.hpp:34 `lim`, the pack's swiglu_limit):
                              > 0 clamps g to <= lim and u to [-lim, lim] before
                              SiLU(g) * u (q8k_core.hpp:92-95); <= 0: no clamp */
} xl_config;

typedef struct xl_bank_info {
    uint64_t payload_bytes;    /* ggml bytes of every resident matrix */
    uint64_t allocated_bytes;  /* device bytes held by the bank (256-B aligned planes) */
    uint64_t workspace_bytes;  /* device bytes of the per-call workspace (with xl_bank_create's part) */
    int32_t n_layers, n_experts;
    int32_t generated;         /* 1 after xl_bank_generate */
    int32_t reserved;
} xl_bank_info;

typedef struct xl_context xl_context;

uint32_t xl_abi_version(void);

/* Opens a context on cfg->device and sizes its workspace. */
int32_t xl_open(uint32_t abi_version, const xl_config* cfg, xl_context** out, xl_error* err);
/* Drains the context stream, then frees every device allocation. */
void xl_close(xl_context* ctx);
int32_t xl_last_error(const xl_context* ctx, xl_error* err);

/* ---- bank ---------------------------------------------------------------
 * types: n_layers * n_experts * 3 ggml type ids, roles (gate w1, up w3,
 * down w2) fastest; gate and up must share a type (the reference requires the
 * same, hip_resident.hpp:114). Replaces HipResidentBank::load's slab sizing
 * (hip_resident_bank.hpp:38-142, hip_resident.hpp:54-97). */
int32_t xl_bank_create(xl_context* ctx, const int32_t* types, xl_error* err);
/* Fills every matrix on the device from the seeded generator. */
int32_t xl_bank_generate(xl_context* ctx, uint64_t seed, xl_error* err);
/* Uploads / downloads one matrix as raw ggml AoS blocks (host memory); the
 * bank stores it repacked into planes. role: 0 gate, 1 up, 2 down. */
int32_t xl_bank_upload(xl_context* ctx, int32_t layer, int32_t expert, int32_t role, const void* aos, uint64_t bytes,
                       xl_error* err);
int32_t xl_bank_download(xl_context* ctx, int32_t layer, int32_t expert, int32_t role, void* aos, uint64_t bytes,
                         xl_error* err);
int32_t xl_bank_info_get(const xl_context* ctx, xl_bank_info* out);
/* 1 when (layer, expert) is resident (WarmRedirect::warm_contains,
 * engine/strata/warm/runtime.hpp:14). */
int32_t xl_contains(const xl_context* ctx, int32_t layer, int32_t expert);

/* ---- weight pack -------------------------------------------------------------
 * The reference's pack directory (engine/strata/sycl/stage/wiring/
 * pack_source.cpp:144-186): ds4.txt (model_dir, format gguf, hidden_size,
 * moe_intermediate_size, num_hidden_layers, n_routed_experts,
 * num_experts_per_tok, ...) and tensors.txt over shard files; routed experts
 * are layers.<l>.ffn.experts.<e>.w1 / w3 / w2 .weight (gate / up / down) in
 * raw ggml blocks. Host only: xl_pack_meta_get reads the shape, xl_pack_types
 * the block types of a layer window (layout as xl_bank_create takes them);
 * xl_bank_load_pack uploads every expert of the context's n_layers, pack
 * layers first_layer.. (dim, ff and n_experts must match the pack). */
typedef struct xl_pack_meta {
    uint32_t struct_bytes; /* sizeof(xl_pack_meta) */
    int32_t dim, ff, n_layers, n_experts, top_k;
    float swiglu_limit;    /* ds4.txt swiglu_limit, 0 when absent (pack_source.cpp:99) */
} xl_pack_meta;
int32_t xl_pack_meta_get(const char* pack_dir, xl_pack_meta* out, xl_error* err);
int32_t xl_pack_types(const char* pack_dir, int32_t first_layer, int32_t n_layers, int32_t n_experts, int32_t* types,
                      xl_error* err);
int32_t xl_bank_load_pack(xl_context* ctx, const char* pack_dir, int32_t first_layer, xl_error* err);

/* ---- lane calls, host memory, synchronous --------------------------------
 * xl_expert_forward   = WarmRedirect::warm_compute        (runtime.hpp:15)
 * xl_experts_forward  = WarmRedirect::warm_compute_many   (runtime.hpp:13):
 *                       ys is k rows of dim floats in `ids` order
 * xl_layer_forward    = the lane plus the caller's fixed-order combine
 *                       (warm_execute, runtime.cpp:180-188): ascending id,
 *                       out = fma(w, y, out), then out += shared when given.
 * ids must be unique and in [0, n_experts); k in 1..max_picks; x finite. */
int32_t xl_expert_forward(xl_context* ctx, int32_t layer, int32_t expert, const float* x, float* y, xl_error* err);
int32_t xl_experts_forward(xl_context* ctx, int32_t layer, const int32_t* ids, int32_t k, const float* x, float* ys,
                           xl_error* err);
int32_t xl_layer_forward(xl_context* ctx, int32_t layer, const int32_t* ids, const float* w, int32_t k, const float* x,
                         const float* shared_or_null, float* out, xl_error* err);
/* Expert chain with its intermediates (the reference's probe snapshot,
 * parity/hip_resident_check.cpp:56-62,93-104); any output may be null.
 * q8h receives ff/256 Q8_K blocks of 292 bytes. */
int32_t xl_expert_trace(xl_context* ctx, int32_t layer, int32_t expert, const float* x, float* g, float* u, float* h,
                        void* q8h, float* y, xl_error* err);

/* ---- device-resident calls (device pointers, ordered on `stream`; a null
 * stream means the context stream, created non-blocking: it does not wait
 * for work on the legacy default stream). Results are valid after the stream
 * drains; xl_sync drains and reports kernel error flags. Every buffer passed
 * must stay allocated and unwritten by other streams until then: a caching
 * allocator (PyTorch's) that reuses a freed input's memory for work on its own
 * stream races with the call. ids are checked on the device: a bad id sets the flag and
 * that pick contributes nothing. */
int32_t xl_layer_forward_async(xl_context* ctx, int32_t layer, const int32_t* d_ids, const float* d_w, int32_t k,
                               const float* d_x, const float* d_shared_or_null, float* d_out, void* stream,
                               xl_error* err);
int32_t xl_sync(xl_context* ctx, void* stream, xl_error* err);

/* ---- grouped tokens (prefill / batched decode) ------------------------------
 * T tokens, each with its own k picks: ids and w are T x k (token-major), x,
 * shared and out T x dim. The result is that of T xl_layer_forward calls (per
 * token: WarmRedirect::warm_compute_many, engine/strata/warm/runtime.hpp:13,
 * then warm_execute's fixed-order combine, runtime.cpp:180-188) but for the
 * order of the float sums over a row's blocks, with every touched expert's
 * weights read once per task of its (token, pick) pairs on int8 MFMA: IQ2_XXS
 * gate/up + IQ2_XS down layers always, layers of other or mixed types from 13
 * tokens on (below, one layer call per token, with that call's bits). The bits
 * of a token do not depend on the other tokens of a call served by the same
 * kernels. Needs a context opened with max_tokens >= T; picks
 * of one token unique. The async form takes device pointers and checks ids on
 * the device (a bad id sets the flag; that pick contributes nothing). */
int32_t xl_grouped_forward(xl_context* ctx, int32_t layer, int32_t T, int32_t k, const int32_t* ids, const float* w,
                           const float* x, const float* shared_or_null, float* out, xl_error* err);
int32_t xl_grouped_forward_async(xl_context* ctx, int32_t layer, int32_t T, int32_t k, const int32_t* d_ids,
                                 const float* d_w, const float* d_x, const float* d_shared_or_null, float* d_out,
                                 void* stream, xl_error* err);

/* The layer call of xl_layer_forward_async with every float computed in the
 * reference CPU lane's own order: q8k_core.hpp:76-91 (`dot_lane`, `hsum`,
 * `dot`: one exact integer per AVX2 lane and block, one fmaf chain per lane
 * over the blocks, the fixed hsum, IQ1_M's main and delta chains apart) and
 * :92-95 (`swiglu`, whose expf is the host C library's, restated for the
 * device), then the fixed-order combine of runtime.cpp:183-188. Its output
 * equals the CPU reference's bit for bit, so that a pass over many layers can
 * be held to the reference end to end. Separate launches, slower than
 * xl_layer_forward_async; same contract and device pointers. */
int32_t xl_layer_forward_exact_async(xl_context* ctx, int32_t layer, const int32_t* d_ids, const float* d_w,
                                     int32_t k, const float* d_x, const float* d_shared_or_null, float* d_out,
                                     void* stream, xl_error* err);

/* ---- parity trace (device pointers) -------------------------------------------
 * The layer call's own intermediates, written by the kernel that computes it
 * (the reference's probe dumps its lane's Q8_K bytes the same way,
 * parity/hip_resident_check.cpp:91-127): the same single launch
 * xl_layer_forward_async would make, plus
 *   q8x  dim/256 Q8_K blocks (292 bytes: d, qs[256], bsums[16]; q8k_core.hpp:13)
 *        of x, as the launch staged them for its gate/up rows;
 *   q8h  k * ff/256 blocks, pick i's Q8_K(h) as staged for its down rows;
 *   h    k * ff floats, the SwiGLU output the launch quantized;
 *   ints per pick (ids order): gate ff x dim/256, up ff x dim/256, down
 *        dim x ff/256 int32, each row's exact integer per 256-weight block (as
 *        xl_matvec_async's partials; IQ1_M: 8 * main + delta);
 *   y    k * dim floats, every pick's row (ids order) as the launch's own
 *        fixed-order combine read it (so that out can be checked bit for bit
 *        against the combine of these rows);
 * kernel_out (host, may be null): 1 the streaming kernel ran, 3 the all-types
 * kernel. Any of q8x, q8h, h, ints, y may be null (not all).
 * XL_E_ARG when the
 * layer does not run as a single launch. A diagnostic aid (no counterpart in
 * the reference beyond its probe); it runs the traced kernel instances. */
int32_t xl_layer_trace_async(xl_context* ctx, int32_t layer, const int32_t* d_ids, const float* d_w, int32_t k,
                             const float* d_x, const float* d_shared_or_null, float* d_out, void* d_q8x, void* d_q8h,
                             float* d_h, int32_t* d_ints, float* d_y, int32_t* kernel_out, void* stream,
                             xl_error* err);
/* The same for the grouped MFMA path (XL_E_ARG when the layer does not run on
 * it): q8x per token (T x dim/256 blocks), q8h, h, ints and y per pair (P =
 * T * k, token-major), layouts as above. */
int32_t xl_grouped_trace_async(xl_context* ctx, int32_t layer, int32_t T, int32_t k, const int32_t* d_ids,
                               const float* d_w, const float* d_x, const float* d_shared_or_null, float* d_out,
                               void* d_q8x, void* d_q8h, float* d_h, int32_t* d_ints, float* d_y, void* stream,
                               xl_error* err);

/* Fixed-order combine of k per-pick rows on the device (engine/strata/warm/
 * runtime.cpp:183-188; other_combine.hpp:51-73 other_combine): out[c] =
 * fma(w_i, rows[i][c], .) over the picks in ascending expert id (equal ids in
 * pick order) from +0, then + shared[c]. d_rows: k x dim floats (ids order);
 * k in 1..16, dim in 1..2^24; d_shared_or_null may be null. Ordered with the
 * context's other calls; for rows computed elsewhere (xl_experts_forward, the
 * per32 rows). */
int32_t xl_combine_async(xl_context* ctx, const int32_t* d_ids, const float* d_w, int32_t k, const float* d_rows,
                         int32_t dim, const float* d_shared_or_null, float* d_out, void* stream, xl_error* err);

/* ---- router (device pointers) -----------------------------------------------
 * route.cpp:15-37 (route_cpu) on the device, per token: score =
 * sqrt(softplus(logit)) (the logit itself above 20), key = score + bias (a null
 * bias is zeros); k rounds of the first largest key (ties: lower index), each
 * taking the expert out; weight = score / (sum of the picked scores + 1e-20) *
 * scale. logits T x stride (n used, n <= 4096), ids and w T x k (k <= 16).
 * A non-finite logit or key sets the device flag (the reference throws). */
int32_t xl_route_async(xl_context* ctx, const float* d_logits, int32_t T, int32_t stride, const float* d_bias_or_null,
                       int32_t n, int32_t k, float scale, int32_t* d_ids, float* d_w, void* stream, xl_error* err);
/* The router over the layer's n_experts logits, then the layer call on its ids
 * and weights, both on `stream` (no host round trip). Where the streaming
 * kernel has the layer and n_experts <= 512 this is one launch that routes in
 * its prologue, bit-identical to the router followed by the layer call;
 * otherwise the route result lives in the context's workspace (routed calls on
 * one context are stream-ordered). */
int32_t xl_layer_forward_routed_async(xl_context* ctx, int32_t layer, const float* d_logits, const float* d_bias_or_null,
                                      int32_t k, float scale, const float* d_x, const float* d_shared_or_null,
                                      float* d_out, void* stream, xl_error* err);
/* The same for T tokens (logits T x n_experts) into xl_grouped_forward_async. */
int32_t xl_grouped_forward_routed_async(xl_context* ctx, int32_t layer, int32_t T, const float* d_logits,
                                        const float* d_bias_or_null, int32_t k, float scale, const float* d_x,
                                        const float* d_shared_or_null, float* d_out, void* stream, xl_error* err);

/* ---- primitives (device pointers) -----------------------------------------
 * q8k_* : Q8_K quantization of rows x k floats (k a multiple of 256) into
 * rows*k/256 blocks of 292 bytes (q8k_core.hpp:13-38, hip_q8k.hpp:9). */
int32_t xl_quantize_q8k_async(xl_context* ctx, const float* d_x, int32_t rows, int32_t k, void* d_q8k, void* stream,
                              xl_error* err);
/* h[n] = SwiGLU(g, u) with the limit (q8k::activate, hip_q8k.hpp:10;
 * q8k_core.hpp:92-95): limit > 0 clamps g to <= limit and u to [-limit,
 * limit], then g / (1 + exp(-g)) * u on the device's expf. */
int32_t xl_swiglu_async(xl_context* ctx, const float* d_g, const float* d_u, int32_t n, float limit, float* d_h,
                        void* stream, xl_error* err);
/* One planar matrix (n x k) times Q8_K(x): y[n] and, when non-null, the
 * per-block int32 partials (n*k/256 ints: each row's exact integer per
 * 256-weight block, sum of (2s+1) * grid * sign * q over the block; IQ1_M:
 * 8 * main + delta, the integer the decoder forms). Replaces q8k::mv
 * (hip_q8k.hpp:10). d_x is the f32 input vector. */
int32_t xl_matvec_async(xl_context* ctx, int32_t type, const void* d_planar, int32_t n, int32_t k, const float* d_x,
                        float* d_y, int32_t* d_partials, void* stream, xl_error* err);

/* ---- per32 mode (the reference's production HIP lane arithmetic) ----------
 * Replaces hipex::quantize / hipex::project (engine/strata/warm/hip_experts.hpp,
 * hip_experts.hip:43-64) and the SoA branch of enqueue_layer
 * (hip_resident_bank.hpp:185-200), bit for bit: activations quantized per 32
 * values (d = max|x| / 127, q = round-half-even(x / d)); a row is 32 lanes,
 * lane l taking sub-blocks l, l + 32, ...: acc = fma(d_x, (fp16(d) * 0.125) *
 * float(s0 * a + s1 * b), acc), then an xor butterfly 16..1 and lane 0 + 0.
 * SwiGLU g / (1 + exp(-g)) * u on the device's expf (the reference's upstream
 * swiglu kernel is not in its tree).
 * xl_layer_forward_per32: y (k x dim, may be null) the per-pick down outputs
 * (the reference's batch_y), out (dim, may be null, needs w) their fixed-order
 * combine (+ shared). The async form takes device pointers (d_y required). */
int32_t xl_layer_forward_per32(xl_context* ctx, int32_t layer, const int32_t* ids, const float* w, int32_t k,
                               const float* x, const float* shared_or_null, float* y_or_null, float* out_or_null,
                               xl_error* err);
int32_t xl_layer_forward_per32_async(xl_context* ctx, int32_t layer, const int32_t* d_ids, const float* d_w, int32_t k,
                                     const float* d_x, const float* d_shared_or_null, float* d_y,
                                     float* d_out_or_null, void* stream, xl_error* err);
/* rows x k floats (k a multiple of 32) into rows*k int8 d_q and rows*k/32 d_d
 * (hip_experts.hip:17-26, hipex::quantize). */
int32_t xl_quantize_per32_async(xl_context* ctx, const float* d_x, int32_t rows, int32_t k, int8_t* d_q, float* d_d,
                                void* stream, xl_error* err);
/* One matrix (n x k) times per32 activations (d_q 16-byte aligned, k int8;
 * d_d k/32 scales): y[n] (dot_kernel<Type>, hip_experts.hip:27-41; the lane<>
 * of sycl/moe/core.hpp:69-84 for the dense formats). d_planar (16-byte
 * aligned): an IQ matrix in the planar layout of xl_repack, or raw ggml blocks
 * of the dense formats Q8_0 (8), Q4_K (12), Q5_K (13), Q6_K (14). */
int32_t xl_matvec_per32_async(xl_context* ctx, int32_t type, const void* d_planar, int32_t n, int32_t k,
                              const int8_t* d_q, const float* d_d, float* d_y, void* stream, xl_error* err);

/* ---- around the routed experts (device pointers) ----------------------------
 * Shared-expert FFN (hip_backend.cpp:664-666: mv(w1, w3), swiglu, mv(w2), the
 * per32 arithmetic of the production GEMV, SwiGLU with the context's limit)
 * for T tokens: out[T x dim] from x[T x dim]. Matrices: gate and up ff x dim,
 * down dim x ff, each raw ggml blocks of a dense format (Q8_0, Q4_K, Q5_K,
 * Q6_K: the pack's ffn.shared_experts.w1 / w3 / w2 bytes) or planar IQ. The
 * caller's workspace (256-byte aligned, xl_shared_work_bytes(dim, ff, T)
 * bytes) holds the intermediates; nothing is allocated. The result is what
 * xl_layer_forward takes as its shared row. */
uint64_t xl_shared_work_bytes(int32_t dim, int32_t ff, int32_t T);
int32_t xl_shared_forward_async(xl_context* ctx, int32_t type_gate, const void* d_gate, int32_t type_up,
                                const void* d_up, int32_t type_down, const void* d_down, int32_t ff, int32_t T,
                                const float* d_x, float* d_out, void* d_work, uint64_t work_bytes, void* stream,
                                xl_error* err);
/* The shared-expert FFN without a caller workspace: the same kernels and
 * result as xl_shared_forward_async, its intermediates in a static device
 * array of 8 MiB (the library's own, held by every GPU it runs on until the
 * process ends). No counterpart in the reference: it is for callers that
 * cannot allocate device memory (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc). It calls no hipMalloc / hipFree.
 * XL_E_ARG when xl_shared_work_bytes(dim, ff, T) exceeds 8 MiB (T up to 250 at
 * dim 4096 x ff 3072). Every call on one GPU shares that GPU's array: calls
 * that overlap on a GPU (through any context or stream) race. */
int32_t xl_shared_forward_noalloc(xl_context* ctx, int32_t type_gate, const void* d_gate, int32_t type_up,
                                  const void* d_up, int32_t type_down, const void* d_down, int32_t ff, int32_t T,
                                  const float* d_x, float* d_out, void* stream, xl_error* err);
/* Hyper-connection pre + RMS norm that makes the MoE block's input
 * (hip_backend.cpp:629 k4::hc_pre_norm with the layer's ffn_norm; sycl/hc/
 * hc.cpp:89-106, core.hpp:74-80): for T tokens of H <= 4 streams of D,
 * x[t][e] = sum_j mix[t][j] * h[t][j][e] (j ascending), then, when w is not
 * null, x[t][e] = x[t][e] * inv * w[e] with inv = 1 / sqrt(S / D + eps) and S
 * the sum of x^2 in the reference's fixed order (1024 lane sums, 32-lane XOR
 * trees). h T x H x D, mix T x 8, w D, x T x D; bit-identical to the
 * reference. x may not overlap h, mix or w; eps finite and positive. */
int32_t xl_hc_pre_norm_async(xl_context* ctx, const float* d_h, const float* d_mix, const float* d_w_or_null,
                             int32_t D, int32_t H, int32_t T, float eps, float* d_x, void* stream, xl_error* err);
/* The pre-norm and the MoE layer of one token as one call (hip_backend.cpp:629
 * k4::hc_pre_norm, then the routed-expert layer of :635-711): x =
 * xl_hc_pre_norm_async(h, mix, norm_w, D = dim, H, T = 1) is written to d_x
 * and is the layer's input, as xl_layer_forward_async(d_ids, d_w, k, d_x)
 * takes it; out and x bit-identical to those two calls. With H == 1 and a
 * layer the streaming kernel runs, one launch: every workgroup normalizes h
 * in its prologue. h H x dim, mix 8, norm_w dim (null: the pre values only).
 * x may not overlap h, mix or norm_w; out may not overlap h or x. */
int32_t xl_layer_forward_prenorm_async(xl_context* ctx, int32_t layer, const int32_t* d_ids, const float* d_w,
                                       int32_t k, const float* d_h, int32_t H, const float* d_mix,
                                       const float* d_norm_w_or_null, float eps, float* d_x,
                                       const float* d_shared_or_null, float* d_out, void* stream, xl_error* err);
/* Hyper-connection post after the MoE block (hip_backend.cpp:777 k4::hc_post;
 * sycl/hc/hc.cpp:107-115, core.hpp:81-86): for T tokens and H <= 4 streams of
 * D, out[t][k][e] = post[t][k] * y[t][e] + sum_j comb[t][j * H + k] *
 * res[t][j][e] (j ascending, separate roundings). y T x D, res and out T x H x
 * D, post T x 8, comb T x 64. out may be res (in place); other overlaps are
 * rejected. */
int32_t xl_hc_post_async(xl_context* ctx, const float* d_y, const float* d_res, const float* d_post,
                         const float* d_comb, int32_t D, int32_t H, int32_t T, float* d_out, void* stream,
                         xl_error* err);
/* The MoE layer of one token and the hyper-connection post after it as one
 * call (the routed-expert layer of hip_backend.cpp:635-711, then :777
 * k4::hc_post): xl_layer_forward_async(d_ids, d_w, k, d_x, d_shared) writes
 * d_out, and xl_hc_post_async(y = d_out, res, post, comb, D = dim, H, T = 1)
 * writes d_post_out; both bit-identical to those two calls. With a layer the
 * streaming kernel runs, one launch: each workgroup applies hc_post to the
 * output rows it combines. res and post_out H x dim, post 8, comb 64;
 * post_out may be res (in place) and overlaps nothing else. */
int32_t xl_layer_forward_post_async(xl_context* ctx, int32_t layer, const int32_t* d_ids, const float* d_w,
                                    int32_t k, const float* d_x, const float* d_shared_or_null, float* d_out,
                                    const float* d_res, const float* d_post, const float* d_comb, int32_t H,
                                    float* d_post_out, void* stream, xl_error* err);
/* The MoE block of one token as one call (hip_backend.cpp:635-711 with the
 * shared expert of :664-666 added last, then :777 k4::hc_post): d_out and
 * d_post_out bit-identical to xl_shared_forward_async(gate, up, down, ff,
 * T = 1, d_x) into a row s, then xl_layer_forward_post_async(d_ids, d_w, k,
 * d_x, s, d_out, res, post, comb, H, d_post_out). The routed layer runs first
 * and writes d_out; with a layer the streaming kernel runs, that launch also
 * quantizes x per 32 for the shared FFN (no quant32 launch); the shared down
 * rows then add themselves to d_out and apply hc_post in their epilogue.
 * Workspace: xl_shared_work_bytes(dim, ff, 1) bytes, 256-byte aligned,
 * overlapping nothing else. res and post_out H x dim, post 8, comb 64;
 * post_out may be res (in place) and overlaps nothing else; out overlaps no
 * input. */
int32_t xl_moe_block_async(xl_context* ctx, int32_t layer, const int32_t* d_ids, const float* d_w, int32_t k,
                           const float* d_x, int32_t type_gate, const void* d_gate, int32_t type_up, const void* d_up,
                           int32_t type_down, const void* d_down, int32_t ff, void* d_work, uint64_t work_bytes,
                           const float* d_res, const float* d_post, const float* d_comb, int32_t H, float* d_out,
                           float* d_post_out, void* stream, xl_error* err);

/* ---- a block of an 8-bit model around the routed experts (device pointers) ----
 * What a MoE block has around the lane's calls in models with an ordinary
 * residual stream and int8 weights: the norms between blocks, a router over
 * softmax or sigmoid scores, and the int8 product of the dense projections and
 * the shared expert. No counterpart in the reference (its model has the
 * hyper-connection forms and route_cpu above). The calls use neither the bank nor
 * the context's workspace. Element types of activations: XL_F32, XL_F16,
 * XL_BF16 (XL_I8 where a call says so); every stride is in elements, from one
 * token's first value to the next's. Sums and scales are float32 or more. */
enum { XL_F32 = 0, XL_F16 = 1, XL_BF16 = 2, XL_I8 = 3 };
enum { XL_SCORE_SOFTMAX = 0, XL_SCORE_SIGMOID = 1 };

/* Router over scores, per token: s = softmax(logits) or sigmoid(logits); key = s +
 * bias (null: zeros). With n_groups > 1 the experts are n_groups equal groups of
 * consecutive ids, a group is worth the sum of its group_keys (1 or 2) largest
 * keys, and only the top_groups of largest value stay. The k largest keys of what
 * stays are picked, in descending order; all ties go to the lower index. weight =
 * s (without the bias), with renorm divided by (sum of the picked s + 1e-20),
 * times scale. Scores and keys are doubles, the weight rounds to float once.
 * A logit of -inf masks its expert: s = 0, key below every other, so it is picked
 * only where fewer than k others stay, with weight 0 (a row of -inf alone: the
 * lowest ids, weights 0). NaN, +inf or a non-finite bias set the device flag.
 * logits T x stride of type logits_type (n used, n <= 1024); ids and w T x k (k <= 16,
 * k <= top_groups * n / n_groups); T <= 2^19. ids, w go to the layer and grouped
 * calls as they are. */
int32_t xl_route_scored_async(xl_context* ctx, const void* d_logits, int32_t logits_type, int32_t T, int64_t stride,
                              const float* d_bias_or_null, int32_t n, int32_t score, int32_t n_groups,
                              int32_t top_groups, int32_t group_keys, int32_t k, int32_t renorm, float scale,
                              int32_t* d_ids, float* d_w, void* stream, xl_error* err);

/* What lies between two blocks, for T tokens of D values (D <= 32768), one launch:
 *   a = y;  post_w: a = a / sqrt(mean(a^2) + eps) * post_w    (norm after the block)
 *   r = alpha * res + gate * a                                (residual scale, gate)
 *   pre_w: x = r / sqrt(mean(r^2) + eps) * pre_w              (norm before the next)
 * float32 throughout (so values whose squares pass its range, above 1.8e19, leave a
 * norm as 0), x from the unrounded r. y null: r = alpha * res (gate and
 * post_w null too); res null: r = gate * a. gate: T x D, or one row for all tokens
 * (gate_stride 0), or null (1). y, gate and x have element type `type`, res and
 * res_out `res_type`. Outputs, each optional but one needed: res_out (r), x, and q
 * with q_scale: x quantized as xl_quantize_rows_async would quantize it unrounded
 * (q 16-byte aligned, q_stride a multiple of 16). x and q need pre_w. res_out may be
 * res and x may be y (same stride); every other overlap of an output is rejected. */
int32_t xl_block_norm_async(xl_context* ctx, const void* d_y_or_null, int64_t y_stride, const void* d_res_or_null,
                            int64_t res_stride, const void* d_gate_or_null, int64_t gate_stride,
                            const float* d_post_w_or_null, const float* d_pre_w_or_null, int32_t T, int32_t D,
                            int32_t type, int32_t res_type, float alpha, float eps, void* d_res_out_or_null,
                            int64_t res_out_stride, void* d_x_or_null, int64_t x_stride, int8_t* d_q_or_null,
                            int64_t q_stride, float* d_q_scale_or_null, void* stream, xl_error* err);

/* T rows of K values to int8 with a scale each (tokens of activations, or the
 * output channels of a weight matrix): scale = max|x| / 127, q =
 * round-half-even(x / scale), -127..127, separate float roundings. A row of zeros
 * has scale 0. A row with an infinity or NaN sets the device flag and has scale
 * NaN and q = 0. q 16-byte aligned, q_stride a multiple of 16 (the bytes from K to
 * the next multiple of 16 are zeroed); K <= 65536, T <= 2^19. */
int32_t xl_quantize_rows_async(xl_context* ctx, const void* d_x, int32_t type, int32_t T, int32_t K, int64_t x_stride,
                               int8_t* d_q, int64_t q_stride, float* d_scale, void* stream, xl_error* err);

/* Product with int8 weights: out[t][r] = (sum_k x[t][k] * w[r][k]) * x_scale[t] *
 * w_scale[r], the sum exact in int32. x: int8 (x_type XL_I8, with d_x_scale; 16-byte
 * aligned, x_stride a multiple of 16) or float (d_x_scale null): then the call
 * quantizes it as xl_quantize_rows_async does. w: N rows of K, 16-byte aligned,
 * w_stride a multiple of 16 (each row of w and of an int8 x readable up to the next
 * multiple of 16; what lies between is not used). With d_up (as w, same stride) and d_up_scale: SwiGLU
 * of the two products, limit > 0 clamping g to <= limit and u to [-limit, limit]
 * (a NaN stays a NaN), out = g / (1 + exp(-g)) * u (the gate and up of a shared
 * expert; its output is the row that the layer and grouped calls take as
 * `shared`). out: XL_F32, XL_F16 or XL_BF16, one rounding. K <= 65536, N and T <=
 * 2^19. d_work: 256-byte aligned, xl_linear_i8_work_bytes(T, K, N, gated) bytes
 * (needed whatever x_type is), used during the call only. out and work overlap
 * nothing else. */
uint64_t xl_linear_i8_work_bytes(int32_t T, int32_t K, int32_t N, int32_t gated);
int32_t xl_linear_i8_async(xl_context* ctx, const void* d_x, int32_t x_type, const float* d_x_scale_or_null,
                           int64_t x_stride, int32_t T, int32_t K, const int8_t* d_w, const float* d_w_scale,
                           const int8_t* d_up_or_null, const float* d_up_scale_or_null, int64_t w_stride, int32_t N,
                           float limit, void* d_out, int32_t out_type, int64_t out_stride, void* d_work,
                           uint64_t work_bytes, void* stream, xl_error* err);

/* ---- the attention half of a block (device pointers) ----------------------------
 * A cache of pages that holds keys and values in 4 bits, filled with rotary
 * positions applied, read back, and attended to. No counterpart in the reference
 * (its dense stage keeps another attention). The calls use neither the bank nor the
 * context's workspace; element types and strides as in the section above, a row's
 * heads consecutive (head_dim values each). What orders such a call before the context's
 * next one on another stream is recorded by that next call: it then waits for whatever was
 * enqueued on the first stream until there, which must live until then, xl_sync or xl_close, and
 * while that stream is captured (and the next call's is not) the next call is refused. Where
 * one of the context's last 64 calls named another stream than the call before it, it is recorded
 * with the call (5 us of host time; not while the stream is captured), and the next call waits for that call alone.
 *
 * A page holds page_tokens tokens: for each kv head xl_kv_page_bytes(page_tokens,
 * head_dim) bytes, the heads' parts consecutive. A group of 32 values of a head is
 * held as m = float16(min), s = float16((max - m) * float(1/15)) and codes
 * clamp(rint((x - m) * (1 / s)), 0, 15) (s = 0: codes 0), separate float32 roundings, and
 * stands for s * code + m; values past +-32768 are held as +-32768. A row (a token's
 * keys, or values, of one head) with an infinity or a NaN sets the device flag and is held as
 * NaNs. One head's part, P = page_tokens, D = head_dim, G = D / 32:
 *   keys' codes     P x [4][G] words; word (c, g): dims 32g + 8c ..+7, dim 2i of them
 *                   in nibble i, dim 2i + 1 in nibble i + 4
 *   keys' scales    P x [G][2] float16: s, m
 *   values' codes   P/4 x [D/8][2][2][2] halfwords: [c][b][h][e] has dims 8c + 4h ..+3
 *                   of token 2b + e of the four, in order
 *   values' scales  P/4 x [G][2][4] float16: s of the four tokens, then m
 * A kernel of the caller's own may fill it too, if scales are >= 0 and a row's
 * scales are either all finite or all the NaN 0x7e00 with m NaN. (Attention reads values as
 * float16: 15 * s + m and m lie within +-65504 for it.)
 *
 * A batch: sequence b has d_lens[b] tokens, token j in page d_table[b * table_stride
 * + j / page_tokens] at j % page_tokens. Its rows are d_starts[b] .. d_starts[b + 1] - 1
 * of the call's q, k, v and outputs (n_seqs + 1 starts, ascending), the last tokens of the
 * sequence: row i of n is at position d_lens[b] - n + i. A row at a position below 0
 * has no token: nothing is written to the cache for it, and its outputs are zeros.
 * Rows outside every sequence are not read, nor their outputs written. Sequences may share pages
 * (a common prefix) that the call does not write; where two tokens of a
 * write have one place, it ends up with codes and scales of either. A page or a length out of range, or
 * starts that descend or pass `rows`, set the device flag; what they name is skipped, never
 * read or written out of bounds. Only entries of the table that a token needs are read. */
typedef struct xl_kv_batch {
    uint32_t struct_bytes;   /* sizeof(xl_kv_batch) */
    int32_t head_dim;        /* 64, 128 or 256 */
    int32_t kv_heads;        /* 1..256 */
    int32_t page_tokens;     /* a multiple of 16 up to 1024 */
    int32_t n_pages;
    int32_t max_pages;       /* columns of the table; max_pages * page_tokens <= 2^26 */
    int32_t n_seqs;          /* 1..65535 */
    int32_t rows;            /* rows of q, k, v and the outputs, 1..2^23 */
    int32_t max_rows;        /* no sequence has more rows (1..rows); more: the device flag */
    int32_t reserved;        /* 0 */
    int64_t page_stride;     /* bytes from page to page, a multiple of 16 */
    int64_t table_stride;    /* entries from a sequence's row of the table to the next's */
    void* d_pages;           /* 16-byte aligned */
    const int32_t* d_table;
    const int32_t* d_lens;
    const int32_t* d_starts;
} xl_kv_batch;

/* Rotary positions: frequency i turns a pair of dims by the angle position * freq[i],
 * a' = a * cos - b * sin, b' = b * cos + a * sin: the angle in double, its cosine and sine
 * rounded to float, then separate float32 roundings. Pairs are dims (i, i + n_freqs), or (2i, 2i + 1) with
 * `interleaved`; dims from 2 * n_freqs on stay. The first section[0] frequencies go by
 * axis 0's positions, the next section[1] by axis 1's (time, height, width). d_positions: n_axes
 * rows of one position for each row of q and k; null (one axis): the position in the sequence. */
typedef struct xl_rotary {
    uint32_t struct_bytes;   /* sizeof(xl_rotary) */
    int32_t n_freqs;         /* 1..head_dim / 2, the sum of the sections */
    int32_t n_axes;          /* 1..3 */
    int32_t interleaved;
    int32_t section[3];      /* of the first n_axes, each >= 0; the others 0 */
    int32_t reserved;        /* 0 */
    int64_t positions_stride;/* entries from an axis's positions to the next's, >= rows */
    const float* d_freqs;
    const int32_t* d_positions;
} xl_rotary;

/* Bytes of one kv head in a page (0: not a size the cache takes). */
uint64_t xl_kv_page_bytes(int32_t page_tokens, int32_t head_dim);
/* The rows' keys (turned by `rotary`, null: as they are) and values into the cache,
 * and q (turned too) to q_out; q, q_out null: the cache alone (q_out with q, both only with
 * rotary). k, v: rows of kv_heads heads, q and q_out rows of q_heads. q_out overlaps nothing else. */
int32_t xl_kv_write_async(xl_context* ctx, const xl_kv_batch* batch, const void* d_k, int64_t k_stride, const void* d_v,
                          int64_t v_stride, int32_t type, const xl_rotary* rotary_or_null, const void* d_q_or_null,
                          int64_t q_stride, int32_t q_heads, void* d_q_out_or_null, int64_t q_out_stride, void* stream,
                          xl_error* err);
/* What the cache holds at the rows' positions, as floats (one rounding to `type`). k and v may be
 * different columns of the same rows. */
int32_t xl_kv_read_async(xl_context* ctx, const xl_kv_batch* batch, void* d_k, int64_t k_stride, void* d_v,
                         int64_t v_stride, int32_t type, void* stream, xl_error* err);
/* Attention of the rows over the cache: for each row at position i and head h,
 *   score_j = scale * q . key_j, with softcap (1e-20 to 16384; 0: none): softcap * tanh(score_j / softcap)
 *   out = sum_j softmax(score)_j * value_j over j <= i, with window > 0 also j > i - window
 * keys and values of kv head h / (q_heads / kv_heads) (q_heads a multiple of kv_heads, at most 1024). q and out:
 * XL_F16 or XL_BF16. Scores, maxima and sums are float32; keys, values and weights are rounded to float16
 * once. A row that sees no token: zeros. Scores (times log2(e)) past what float32 holds: NaN where
 * they are a row's largest. A token held as NaN makes
 * the outputs of the rows that see it NaN, of no others; so does a value of q that is not finite for its row and head.
 * Tokens that no row of their sequence sees (below the window of its first row) need no page, and what lies in their places may be anything.
 * Outputs of rows that see a token whose page is out of range mean nothing. d_work: 256-byte aligned,
 * xl_attention_work_bytes(batch, q_heads) bytes, used during the call only (0 bytes:
 * may be null). The size goes by the batch's numbers, not by its pointers. out and work overlap nothing else. */
uint64_t xl_attention_work_bytes(const xl_kv_batch* batch, int32_t q_heads);
int32_t xl_attention_async(xl_context* ctx, const xl_kv_batch* batch, const void* d_q, int64_t q_stride, int32_t q_heads,
                           int32_t type, float scale, int32_t window, float softcap, void* d_out, int64_t out_stride,
                           void* d_work, uint64_t work_bytes, void* stream, xl_error* err);

/* ---- stage profiling --------------------------------------------------------
 * Between xl_profile_begin and xl_profile_end, the first max_calls layer calls
 * record a HIP event before and after each kernel on the stream it runs on
 * (the reference's phase marks, hip_experts.hpp:13-20). xl_profile_end drains
 * and returns per-stage totals in ms, the stage and call counts and the stage
 * names (comma separated). Event creation happens in xl_profile_begin. */
int32_t xl_profile_begin(xl_context* ctx, int32_t max_calls, xl_error* err);
int32_t xl_profile_end(xl_context* ctx, float* stage_ms, int32_t max_stages, int32_t* n_stages, int32_t* n_calls,
                       char* names, int32_t names_bytes, xl_error* err);

/* Per-wave timeline of the last single-launch layer call made while profiling
 * was active: 32 words per wave, wave-major over the grid, holding
 * s_memrealtime stamps (100 MHz; zero where a wave did not reach a phase).
 * Words: 0 prologue loads issued, 1 codebooks written, 2 x quantized
 * (barrier), 3 gate/up done, 4 quantizer duty done (all-types kernel),
 * 5 first down pass done, 6 all down passes done, 7 combine done, 8 + j
 * gate/up slot j done; streaming kernel only: 20 + j re-polls of down step j
 * (a count, not a stamp), 24 + 2j step j's h complete, 25 + 2j step j's
 * Q8_K(h) staged. A diagnostic aid: it has no counterpart in the reference. */
int32_t xl_profile_timeline(xl_context* ctx, uint64_t* out, int32_t max_words, int32_t* n_words, xl_error* err);

/* Sets the single-launch kernels' device launch counters (the all-types
 * kernel's epoch and the streaming kernel's launch count, whose parity picks
 * its h exchange buffer) to `launches`, as if that many launches had run. A
 * diagnostic aid for testing the counters' wrap at 2^32; it has no
 * counterpart in the reference. The exchange buffers are reset as at
 * xl_open (h words to the sentinel, tags to zero), so that any count, of
 * either parity and any epoch, leaves the next launch correct. */
int32_t xl_debug_set_launch_count(xl_context* ctx, uint32_t launches, xl_error* err);

/* Layer calls made on the context so far, by how they ran: counts[i] for
 * i < n (kinds past XL_LAUNCH_KINDS read 0). A diagnostic aid (no counterpart
 * in the reference): it shows which launch served a call, e.g. that a routed
 * or pre-normed call ran as one launch rather than as its two-call fallback. */
enum {
    XL_LAUNCH_STREAM = 0,     /* xl_layer_* calls served by the streaming kernel */
    XL_LAUNCH_ALLTYPES = 1,   /* ... by the all-types single launch */
    XL_LAUNCH_SEPARATE = 2,   /* ... by separate launches */
    XL_LAUNCH_ROUTED = 3,     /* routed layer calls that routed inside the streaming launch */
    XL_LAUNCH_PRENORM = 4,    /* pre-normed layer calls that normalized inside the streaming launch */
    XL_LAUNCH_EXACT = 5,      /* xl_layer_forward_exact_async calls */
    XL_LAUNCH_POST = 6,       /* layer + hc_post calls that applied hc_post inside the streaming launch */
    XL_LAUNCH_BLOCK = 7,      /* xl_moe_block_async calls whose streaming launch quantized x for the shared FFN */
    XL_LAUNCH_KINDS = 8
};
int32_t xl_debug_launch_counts(xl_context* ctx, int64_t* counts, int32_t n, xl_error* err);

/* ---- host utilities (no device needed) ------------------------------------ */
uint64_t xl_planar_bytes(int32_t type, int32_t n, int32_t k);
int32_t xl_repack(int32_t type, int32_t n, int32_t k, const void* aos, void* planar);
int32_t xl_restore(int32_t type, int32_t n, int32_t k, const void* planar, void* aos);
/* The generator's AoS bytes of matrix (layer, expert, role), host-side. */
int32_t xl_generate_host(int32_t type, uint64_t seed, int32_t layer, int32_t expert, int32_t role, int32_t n, int32_t k,
                         void* aos);
/* Expanded codebooks: 0 IQ2_XXS grid (256 u64), 1 IQ2_XS grid (512),
 * 2 IQ1 grid (2048), 3 ksigns (128 values widened to u64). */
int32_t xl_codebook(int32_t which, uint64_t* out);

#ifdef __cplusplus
}
#endif
#endif
