/* include/fns_hip.h - C ABI of libfns_hip.so, the MI355X (gfx950) MoE FFN hot path of FlintNSteel.
 *
 * Plain pointers and sizes only: every buffer argument is a device pointer (hipMalloc'd or otherwise GPU-visible)
 * unless stated; `stream` is a hipStream_t passed as void* (NULL = the null stream). Every call is asynchronous on
 * `stream`, allocates nothing, and returns 0 on success or a negative FNS_ERR_* code; fns_hip_last_error() then
 * describes the failure (thread-local). The C++ API of include/fns/ggml_kernels.h and include/fns/kernels.h wraps
 * the same implementations and aborts on error, as the reference does.
 *
 * Each entry point names the reference interface it replaces (paths under the reference repository).
 */
#ifndef FNS_HIP_H
#define FNS_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FNS_OK 0
#define FNS_ERR_TYPE (-1)
#define FNS_ERR_SHAPE (-2)
#define FNS_ERR_LAUNCH (-3)
#define FNS_ERR_NOMEM (-4)
#define FNS_ERR_IO (-5) /* a GGUF file that cannot be opened or is malformed */

/* ggml type ids accepted by the quantized entry points (ggml.h numbering); router dtypes: 0 = f32, 30 = bf16. */
#define FNS_TYPE_F32 0
#define FNS_TYPE_F16 1
#define FNS_TYPE_Q8_1 9
#define FNS_TYPE_Q3_K 11
#define FNS_TYPE_Q4_K 12
#define FNS_TYPE_Q5_K 13
#define FNS_TYPE_Q6_K 14
#define FNS_TYPE_IQ3_XXS 18
#define FNS_TYPE_IQ3_S 21
#define FNS_TYPE_IQ2_S 22
#define FNS_TYPE_IQ4_XS 23
#define FNS_TYPE_BF16 30

#define FNS_GATING_SOFTMAX 0
#define FNS_GATING_SIGMOID 1

int fns_hip_abi_version(void);
const char *fns_hip_last_error(void);

/* --- ggml_kernels.h (reference include/fns/ggml_kernels.h) --- */

/* include/fns/ggml_kernels.h:13-14 q8_1_row_bytes */
size_t fns_hip_q8_1_row_bytes(int64_t ncols);
/* include/fns/ggml_kernels.h:16-17 quantize_q8_1 */
int fns_hip_quantize_q8_1(const float *x, void *xq, int64_t ncols, int64_t nrows, void *stream);
/* include/fns/ggml_kernels.h:19-22 mmvq */
int fns_hip_mmvq(int type, const void *w, int64_t ncols, int64_t nrows, const void *xq, float *dst, int64_t n_cols,
                 void *stream);
/* include/fns/ggml_kernels.h:24-27 mmvq_ids */
int fns_hip_mmvq_ids(int type, const void *w, int64_t ncols, int64_t nrows, int64_t n_mats, const void *xq,
                     int64_t n_xq, const int32_t *ids, int64_t n_ids, float *dst, void *stream);
/* include/fns/ggml_kernels.h:29-31 mmvq_swiglu */
int fns_hip_mmvq_swiglu(int type, const void *w_gate, const void *w_up, int64_t ncols, int64_t nrows, const void *xq,
                        float *dst, void *stream);
/* include/fns/ggml_kernels.h:33-37 mmvq_ids_swiglu_shared (sh_* may be NULL: no shared expert) */
int fns_hip_mmvq_ids_swiglu_shared(int type, const void *w_gate, const void *w_up, int64_t ncols, int64_t nrows,
                                   int64_t n_mats, const void *xq, const int32_t *ids, int64_t n_ids, float *dst,
                                   const void *sh_gate, const void *sh_up, float *sh_dst, void *stream);
/* include/fns/ggml_kernels.h:44-46 mmvq_experts_swiglu; table: device array of expert base pointers */
int fns_hip_mmvq_experts_swiglu(int type, const void *const *table, size_t gate_off, size_t up_off, int64_t ncols,
                                int64_t nrows, const void *xq, int64_t n_xq, const int32_t *ids, int64_t n_ids,
                                float *dst, void *stream);
/* include/fns/ggml_kernels.h:47-48 mmvq_experts */
int fns_hip_mmvq_experts(int type, const void *const *table, size_t off, int64_t ncols, int64_t nrows, const void *xq,
                         int64_t n_xq, const int32_t *ids, int64_t n_ids, float *dst, void *stream);
/* include/fns/ggml_kernels.h:79-80 mmvq_supports */
int fns_hip_mmvq_supports(int type);
/* No counterpart in the reference, whose ggml build compiles the IQ codebooks in: registers ggml's iq3xxs_grid[256],
 * iq3s_grid[512] and iq2s_grid[1024] (the engine's own copies) on the current device; call once per device before
 * any IQ3_XXS / IQ3_S / IQ2_S product. Until then mmvq_supports rejects those three types (IQ4_XS needs no table).
 * Every codebook byte must be 1..127, as ggml's are. Synchronous (hipMemcpyToSymbol); not graph-capturable. */
int fns_hip_set_iq_grids(const uint32_t *iq3xxs, const uint32_t *iq3s, const uint64_t *iq2s);

/* --- kernels.cuh MoE subset (reference src/kernels.cuh, namespace fns::k) --- */

/* src/kernels.cuh:29-32 rms_norm_q8_1 (n any multiple of 32) */
int fns_hip_rms_norm_q8_1(const float *x, const float *w, float *out, void *xq, int n, float eps, int rows,
                          void *stream);
/* src/kernels.cuh:90-91 gemv_bf16, generalised to dtype 0 (f32) or 30 (bf16); cols 1..8 */
int fns_hip_gemv_router(int dtype, const void *w, const float *x, float *y, int ncols, int nrows, int cols,
                        void *stream);
/* src/kernels.cuh:150-153 gemm_bf16_batch (no cuBLAS handle), dtype 0 or 30 */
int fns_hip_gemm_router(int dtype, const void *w, const float *x, float *y, int ncols, int nrows, int n_tok,
                        void *stream);
/* src/kernels.cuh:93-94 route_topk and :155 route_topk_batch; gating FNS_GATING_*, norm 0/1 */
int fns_hip_route_topk(const float *logits, int32_t *ids, float *w, int n_expert, int k, int n_tok, int gating,
                       int norm, void *stream);
/* src/kernels.cuh:96-97 count_routes */
int fns_hip_count_routes(const int32_t *ids, uint32_t *counts, int k, void *stream);
/* src/kernels.cuh:99-100 swiglu */
int fns_hip_swiglu(const float *g, const float *u, float *act, int n, int rows, void *stream);
/* src/kernels.cuh:102-104 glu_mmvq */
int fns_hip_glu_mmvq(const float *g, const float *u, float *act, int n, void *stream);
/* src/kernels.cuh:106-108 amax_guard */
int fns_hip_amax_guard(float *act, float *escale, int n, int rows, void *stream);
/* src/kernels.cuh:110-111 amax_guard_q8_1 (n any multiple of 32) */
int fns_hip_amax_guard_q8_1(const float *act, float *escale, void *xq, int n, int rows, void *stream);
/* src/kernels.cuh:113-115 moe_combine and :156 moe_combine_batch, out-of-place:
 * out[t] = (sum_j (dexp[t][j] * escale[t][j]) * w[t][j] + sh[t]) + x_in[t]; escale, sh, x_in may be NULL;
 * out may alias x_in (the reference's in-place form). */
int fns_hip_moe_combine(const float *dexp, const float *escale, const float *w, const float *sh, const float *x_in,
                        float *out, int n, int k, int n_tok, void *stream);

/* --- fused MoE FFN layer: decode (n_tok = 1) and speculative verify (n_tok <= 4) ---
 * The MoE section of the reference's Engine::ffn_block (src/engine.cu:655-696: router gemv_bf16, route_topk,
 * mmvq_experts_swiglu, amax_guard_q8_1, mmvq_experts, moe_combine) as one call of three kernels:
 *   out[t] = sum_j w[t][j] * e[t][j] * down_{e_j}(q8_1(act[t][j] / e[t][j])) (+ x_resid[t]),
 *   act[t][j] = up_{e_j} . q8_1(x[t]) * silu(gate_{e_j} . q8_1(x[t])), (ids, w) = top-k of gating(router . x[t]).
 * Expert e's slot is table[e] (device array) with gate/up/down matrices at the byte offsets below (GGUF blocks).
 * For n_tok > 1 the selected experts are compacted: each distinct expert's weights are read once per call.
 * workspace: fns_hip_moe_workspace_layout() bytes, device memory, zero-filled once before its first use (it holds an
 * arrival counter that the library keeps consistent from call to call), sections (byte offsets in offsets[6]):
 *   0 logits f32 [n_tok][n_expert], 1 xq Q8_1 [n_tok][q8_1_row_bytes(hidden)], 2 ids i32 [n_tok][k],
 *   3 w f32 [n_tok][k], 4 act f32 [n_tok*k][inter], 5 escale f32 [n_tok*k]. */
typedef struct FnsMoeLayer {
    int hidden, inter, n_expert, k;
    int gating;       /* FNS_GATING_SOFTMAX or FNS_GATING_SIGMOID */
    int norm_w;       /* 1: w = p / max(sum p, 6.103515625e-5) */
    int guard;        /* 1: F16 guard of act before down (reference src/kernels.cu:534-577) */
    int router_dtype; /* FNS_TYPE_F32 or FNS_TYPE_BF16 */
    const void *router_w; /* [n_expert][hidden] */
    int gu_type, down_type;
    const void *const *table;
    size_t gate_off, up_off, down_off;
    const float *router_bias; /* NULL or f32 [n_expert], added to the logits before gating (selection and weights) */
    /* The rest of the reference's Engine::ffn_block (src/engine.cu:655-696; prefill src/engine.cu:331-357); all zero:
     * absent. With ffn_norm the layer input x is the residual stream: h = RMSNorm(x) * ffn_norm (eps norm_eps, as
     * rms_norm_q8_1) feeds the router and the experts. With a shared expert (shexp_inter > 0) its output
     * sh = down_sh . q8_1(up_sh . q8_1(h) * silu(gate_sh . q8_1(h))) joins the combine as the reference's:
     * out = (sum_j w_j e_j dexp_j + sh) + x_resid. */
    const float *ffn_norm;     /* NULL or f32 [hidden] */
    float norm_eps;
    int shexp_inter;           /* 0 or the shared expert's width (a positive multiple of 256) */
    int shexp_gu_type, shexp_down_type;  /* K-quant types of the shared expert's gate/up and down (0: gu_type / down_type) */
    const void *shexp_gate, *shexp_up;   /* [shexp_inter][hidden] blocks */
    const void *shexp_down;              /* [hidden][shexp_inter] blocks */
    /* No counterpart in the reference: a read-ahead hint. NULL, or device bytes the next call will read first
     * (normally the next layer's router_w, prefetch_bytes = its size): the decode router kernel reads them along with
     * its own work so that they sit in the memory-side cache (MI355X Infinity Cache) when the next layer's router
     * reads them. Results do not depend on it. */
    const void *prefetch;
    size_t prefetch_bytes;
} FnsMoeLayer;

int fns_hip_moe_workspace_layout(const FnsMoeLayer *layer, int n_tok, size_t *offsets, size_t *total_bytes);
int fns_hip_moe_layer(const FnsMoeLayer *layer, const float *x, const float *x_resid, float *out, int n_tok,
                      void *workspace, size_t workspace_bytes, void *stream);
/* Same, recording events[0..3] (hipEvent_t, any may be NULL) on `stream` before the router kernel, before the
 * gate/up kernel, before the down kernel and after it: per-kernel durations for measurement. */
int fns_hip_moe_layer_profiled(const FnsMoeLayer *layer, const float *x, const float *x_resid, float *out, int n_tok,
                               void *workspace, size_t workspace_bytes, void *const *events, void *stream);
/* No counterpart in the reference: the same layer as fns_hip_moe_layer for callers that cannot allocate (code under HIP
 * graph capture, serving loops or harnesses that forbid hipMalloc). The workspace is a device array inside the
 * library, fns_hip_moe_noalloc_max_bytes() bytes (4 MiB) per GPU, held until the process ends; a layer whose
 * fns_hip_moe_workspace_layout total exceeds it is rejected with FNS_ERR_NOMEM. The call allocates nothing. Every call
 * on one GPU shares that array and leaves its intermediates there (as fns_hip_moe_layer leaves them in its
 * workspace): calls that overlap on one GPU race, so order them (one stream). The first call on a device clears the
 * array with a kernel on `stream`. */
int fns_hip_moe_layer_noalloc(const FnsMoeLayer *layer, const float *x, const float *x_resid, float *out, int n_tok,
                              void *stream);
size_t fns_hip_moe_noalloc_max_bytes(void);
/* No counterpart in the reference (its kernels have no cross-workgroup wait). The decode kernel's workgroups exchange
 * the act rows through a bounded wait in device memory; a workgroup that gives up (its producers were never
 * scheduled, e.g. other work held the CUs) writes NaN to its output rows and sets FNS_STATUS_EXCHANGE_TIMEOUT in the
 * workspace's status word. The word is sticky across calls (the engine can check once per token or graph replay):
 * this call waits for the stream's work so far, stores the word in *status and, with clear = 1, zeroes it (a kernel
 * on `stream`). workspace NULL: the no-allocation array of the current device. Not graph-capturable (it
 * synchronises). */
#define FNS_STATUS_EXCHANGE_TIMEOUT 1u
int fns_hip_moe_layer_status(const FnsMoeLayer *layer, int n_tok, void *workspace, int clear, uint32_t *status,
                             void *stream);
/* No counterpart in the reference: the graph-capturable form of fns_hip_moe_layer_status for engines that replay a
 * graph per token. Enqueues one single-thread kernel on `stream` that, when the workspace's status word is non-zero,
 * ORs it into *dst (device memory or host memory from hipHostMalloc; the caller zeroes it) and clears the word; a
 * zero word leaves *dst untouched. Layers that share one workspace share its word, so one collect per token covers
 * them. workspace NULL: the no-allocation array of the current device. */
int fns_hip_moe_layer_status_collect(const FnsMoeLayer *layer, int n_tok, void *workspace, uint32_t *dst,
                                     void *stream);
/* Test hook, no counterpart in the reference: the decode kernel's poll limit (0: the default, 65536 polls) and a
 * number of producer arrivals to withhold (> 0: the exchange never completes, every workgroup gives up after
 * spin_limit polls) for the calls that follow; the failure path is then exercised with every kernel exiting normally.
 * Process-wide; set it only while no other thread launches layers. */
int fns_hip_moe_set_test_hooks(int spin_limit, int withhold_arrivals);
/* No counterpart in the reference: how many kernels a call of this layer at n_tok tokens launches on the current
 * device - 2 (n_tok = 1 and a shape the fused kernel holds, all its workgroups resident: router kernel + fused layer
 * kernel) or 3 (router, gate/up, down). Both give the same results bit for bit. */
int fns_hip_moe_layer_kernels(const FnsMoeLayer *layer, int n_tok, int *kernels);
/* Test hook, no counterpart in the reference: restricts the decode path for the calls that follow (0: automatic,
 * 1: never the fused kernel - the three-kernel path). Process-wide, like fns_hip_moe_set_test_hooks. */
int fns_hip_moe_set_path(int path);
/* One of the three kernels of fns_hip_moe_layer (stage 0 router + Q8_1 of x, 1 routing + gate/up + SwiGLU,
 * 2 F16 guard + Q8_1 of act + down + combine), each reading what the previous stage left in the workspace:
 * per-stage tracing (the reference's FNS_TRACE nodes, src/engine.cu:590-599) and per-kernel timing. A call that takes
 * the fused kernel (fns_hip_moe_layer_kernels = 2) launches it at stage 1; stage 2 then launches nothing. */
int fns_hip_moe_layer_stage(const FnsMoeLayer *layer, int stage, const float *x, const float *x_resid, float *out,
                            int n_tok, void *workspace, size_t workspace_bytes, void *stream);

/* --- prefill / batched expert GEMM (MMQ) ---
 * Q8_1 activation rows for the MMQ path are kept as "split images" (q8 * d8 as two f16 halves per value, then the
 * per-32 scaled sums as f16 halves: 4.125 bytes per value; Q8_0, and the layers below for the types scaled every 32
 * columns, use int8 codes, scales and sums, 1.25 bytes per value, in the same room): fns_hip_mmq_q8_1_bytes(ncols, nrows) bytes hold nrows
 * of them plus 4096 bytes of slack (mmq_experts keeps its group lists there). */
/* include/fns/ggml_kernels.h:53-54 mmq_q8_1_bytes */
size_t fns_hip_mmq_q8_1_bytes(int64_t ncols, int64_t nrows);
/* bytes of the expert_bounds buffer of fns_hip_mmq_compact for n_expert experts (bounds + tile-group prefix) */
size_t fns_hip_mmq_bounds_bytes(int64_t n_expert);
/* include/fns/ggml_kernels.h:56-58 mmq: dst[t][nrows] = W . q8_1(x[t]), x f32 [n_tok][ncols]; xq scratch of
 * fns_hip_mmq_q8_1_bytes(ncols, n_tok) bytes. ncols a multiple of 256, nrows of 64. Types (the reference's MMQ set,
 * src/ggml/ggml_mmq.cu:59-66, plus Q3_K): the K-quants, Q8_0 and IQ4_XS / IQ3_XXS / IQ3_S / IQ2_S (the last three once
 * their codebooks are registered) on the tiled MFMA GEMM; Q8_0 takes any nrows: one that is not a multiple of 64 runs on
 * the GEMV kernels, a few token columns per weight pass. */
int fns_hip_mmq(int type, const void *w, int64_t ncols, int64_t nrows, const float *x, int64_t n_tok, void *xq,
                float *dst, void *stream);
/* include/fns/ggml_kernels.h:60-69 MmqIdsScratch + mmq_experts: dst[t][j][nrows] = W_e . q8_1(x[t][j % x_rows_per_tok]),
 * e = ids[t][j]; expert e's matrix at table[e] + off. Scratch (the reference's MmqIdsScratch sizing): ids_src1 /
 * ids_dst n_tok * n_used int32, expert_bounds n_expert + 1 int32, xq fns_hip_mmq_q8_1_bytes(ncols, n_tok * x_rows_per_tok)
 * bytes. */
int fns_hip_mmq_experts(int type, const void *const *table, size_t off, int64_t ncols, int64_t nrows, int64_t n_expert,
                        const float *x, int64_t x_rows_per_tok, int64_t n_tok, const int32_t *ids, int64_t n_used,
                        int32_t *ids_src1, int32_t *ids_dst, int32_t *expert_bounds, void *xq, float *dst, void *stream);
/* Expert-id compaction alone (ggml mm_ids_helper semantics; reference src/ggml/ggml_mmq.cu:110-111): pairs
 * p = t * n_used + j sorted by expert, stable; ids_dst[q] = p, ids_src1[q] = (x_rows_per_tok == 1 ? t : p),
 * expert_bounds[e] = first sorted position of expert e (e <= n_expert), followed by the tile-group prefix
 * (fns_hip_mmq_bounds_bytes(n_expert) bytes in all). */
int fns_hip_mmq_compact(const int32_t *ids, int64_t n_tok, int64_t n_used, int64_t n_expert, int64_t x_rows_per_tok,
                        int32_t *ids_src1, int32_t *ids_dst, int32_t *expert_bounds, void *stream);

/* Prefill MoE layer for n_tok tokens (n_tok * k <= 65536): the MoE section of the reference's Engine::prefill_chunk
 * (src/engine.cu:340-357: batch router, route_topk_batch, mmq_experts gate / up, swiglu, amax_guard, mmq_experts down,
 * moe_combine_batch), out[t] = sum_j w[t][j] * e[t][j] * down_e(q8_1(act[t][j] / e[t][j])) (+ x_resid[t]).
 * workspace: fns_hip_moe_prefill_workspace() bytes; sections (byte offsets in offsets[6]): 0 logits f32 [n_tok][n_expert],
 * 1 ids i32 [n_tok][k], 2 w f32 [n_tok][k], 3 x images, 4 act images [n_tok * k], 5 down outputs f32 [n_tok][k][hidden]. */
int fns_hip_moe_prefill_workspace(const FnsMoeLayer *layer, int64_t n_tok, size_t *offsets, size_t *total_bytes);
/* Byte offset and size of any workspace section of fns_hip_moe_prefill (the six above, then 6 ids_src1, 7 ids_dst
 * (a call whose x or act images have 2 GiB or more runs ranges of tokens in turn; 6 to 8 are then each range's own),
 * 8 expert bounds, group prefix, arrival counters and the status word, 9 f32 act [n_tok * k][inter] (F16 guard
 * only, after the division), 10 guard scales [n_tok * k],
 * 11 RMSNorm output, 12 its Q8_1 blocks, 13 shared-expert act images, 14 shared-expert output). Inspection and tests;
 * the image layouts are internal. */
int fns_hip_moe_prefill_section(const FnsMoeLayer *layer, int64_t n_tok, int section, size_t *offset, size_t *bytes);
/* The form (0: split, 1: int8) and the row stride in bytes of the images in section 3, 4 or 13. They follow from the
 * layer's types alone: a token's result has the same bits in a call of any length. */
int fns_hip_moe_prefill_image(const FnsMoeLayer *layer, int section, int *form, size_t *row_stride);
int fns_hip_moe_prefill(const FnsMoeLayer *layer, const float *x, const float *x_resid, float *out, int64_t n_tok,
                        void *workspace, size_t workspace_bytes, void *stream);
/* No counterpart in the reference. Without the F16 guard and for gate/up and down types from {Q3_K, Q4_K}, gate/up
 * and down (each on the image form of its type) run as one launch whose down workgroups wait (bounded) for their row group's gate/up
 * workgroups; one that gives up writes NaN to its output rows and sets FNS_STATUS_EXCHANGE_TIMEOUT in the workspace's
 * status word (section 8, which the workspace must hold zeroed when first used). As fns_hip_moe_layer_status: waits
 * for the stream's work so far, stores the word in *status and, with clear = 1, zeroes it. The poll limit and
 * withheld arrivals of fns_hip_moe_set_test_hooks apply to this wait too. Not graph-capturable (it synchronises). */
int fns_hip_moe_prefill_status(const FnsMoeLayer *layer, int64_t n_tok, void *workspace, int clear, uint32_t *status,
                               void *stream);
/* No counterpart in the reference: the graph-capturable form of fns_hip_moe_prefill_status, with the behaviour of
 * fns_hip_moe_layer_status_collect. */
int fns_hip_moe_prefill_status_collect(const FnsMoeLayer *layer, int64_t n_tok, void *workspace, uint32_t *dst,
                                       void *stream);

/* --- dense FFN layer (the reference model's leading dense blocks) ---
 * The dense branch of the reference's Engine::ffn_block (src/engine.cu:655-667: rms_norm_q8_1, dense_glu
 * (src/engine.cu:644-653: mmvq_swiglu at one column, else two mmvq and glu_mmvq), gemv of ffn_down (quantize_q8_1 +
 * mmvq, src/engine.cu:585-588), add_inplace) and of Engine::prefill_chunk (src/engine.cu:331-337: rms_norm_mul, mmq of
 * ffn_gate and ffn_up, swiglu, mmq of ffn_down, add_inplace):
 *   out[t] = x[t] + down . q8_1(silu(gate . q8_1(h[t])) * (up . q8_1(h[t]))), h = RMSNorm(x) * ffn_norm (or x).
 * Matrices are GGUF blocks: gate and up [inter][hidden], down [hidden][inter]; any type of the GEMV kernels
 * (fns_hip_mmvq_supports) for the decode form, any type of fns_hip_mmq for the prefill form. out may alias x. */
typedef struct FnsDenseFfn {
    int hidden, inter;                 /* positive multiples of 256 */
    int gate_type, up_type, down_type; /* ggml types */
    const void *gate, *up, *down;
    const float *ffn_norm;             /* NULL or f32 [hidden] */
    float norm_eps;
} FnsDenseFfn;
/* Device bytes of the workspace of either form at n_tok tokens (no zero-fill needed). */
int fns_hip_dense_ffn_workspace(const FnsDenseFfn *ffn, int64_t n_tok, size_t *total_bytes);
/* Decode / verify form (the reference's forward at cols_ = n_tok columns). */
int fns_hip_dense_ffn(const FnsDenseFfn *ffn, const float *x, float *out, int64_t n_tok, void *workspace,
                      size_t workspace_bytes, void *stream);
/* Prefill form (the MMQ GEMMs). */
int fns_hip_dense_ffn_prefill(const FnsDenseFfn *ffn, const float *x, float *out, int64_t n_tok, void *workspace,
                              size_t workspace_bytes, void *stream);
/* src/kernels.cuh:119 add_inplace, out-of-place: out[i] = x[i] + y[i]; out may alias x. */
int fns_hip_add(const float *x, const float *y, float *out, int64_t n, void *stream);

/* --- the attention half of a decoder block ---
 * What an engine runs between the projections (fns_hip_mmvq / fns_hip_mmq of the quantised rows) and the FFN calls above:
 *   Q8_1 rows -> mmvq (q, k, v) -> fns_hip_kv_append -> fns_hip_attn -> quantize_q8_1, mmvq (output projection)
 *   -> fns_hip_add_rms_norm_q8_1 -> gemv_router, mmvq_experts_swiglu ...
 * The reference's counterparts (src/kernels.cuh k::attention*, src/kernels.cu:230-450, flash_attn_prefill of
 * include/fns/ggml_kernels.h:71-77) read a 16-bit cache of one sequence; this cache is paged, holds many sequences and
 * takes 4.25 bits a value. */

/* sum = x + y; out = sum * w / sqrt(mean(sum^2) + eps) per row; xq = Q8_1 blocks of out (rows of
 * fns_hip_q8_1_row_bytes(n), padded with zeros as rms_norm_q8_1's). All f32 [rows][n], n a multiple of 32, w [n]. The bits
 * of fns_hip_add followed by fns_hip_rms_norm_q8_1. sum may be x or y (otherwise no overlaps); out may be NULL. */
int fns_hip_add_rms_norm_q8_1(const float *x, const float *y, const float *w, float *sum, float *out, void *xq, int n,
                              float eps, int rows, void *stream);
/* What Q8_1 rows (fns_hip_q8_1_row_bytes(ncols) apart, ncols a multiple of 32) stand for: x [nrows][ncols] = q * d and,
 * unless NULL, sums [nrows][ncols / 32], the blocks' held sums; both of `dtype` FNS_TYPE_F32 or FNS_TYPE_F16. */
int fns_hip_dequantize_q8_1(const void *xq, int dtype, void *x, void *sums, int64_t ncols, int64_t nrows, void *stream);

/* A paged key/value cache held in 4 bits: blocks of 32 channels of one token and kv head, e2m1 codes (0, .5, 1, 1.5, 2, 3,
 * 4, 6 and their negatives) times 2^(e - 127), one byte e a block, the least with max |block| <= 7 * 2^(e - 127); codes to
 * nearest, ties to even. A block with a NaN or infinity stands for NaNs. `pages`: n_pages * fns_hip_kv_page_bytes bytes,
 * 16-byte aligned; what is never read need not be initialised. */
typedef struct FnsKvCache {
    int n_head_kv;  /* 1..1024 */
    int head_dim;   /* 64, 128 or 256 */
    int page_size;  /* positions of a page: a power of two, 16..4096 */
    int64_t n_pages;
    void *pages;
} FnsKvCache;
/* Bytes of a page; 0 for an unsupported shape. */
size_t fns_hip_kv_page_bytes(int n_head_kv, int head_dim, int page_size);
/* New tokens of n_seq sequences. Tokens q_start[s] .. q_start[s + 1] - 1 are sequence s's last ones: kv_len[s] is its length
 * with them, so token i of n has position kv_len[s] - n + i. Position p lies in page page_table[s * table_stride +
 * p / page_size]; an entry that no position of a call needs may be anything. q_start, kv_len and page_table are device
 * memory (a captured graph takes their values at each replay); the numbers below are the host's:
 *   n_tok   rows of the token arrays: tokens from q_start[n_seq] on are padding and left alone
 *   max_q   at least the new tokens of any sequence (more than this many are not handled)
 *   max_kv  about the longest kv_len: work is divided by it, results hold for any. Far too large (or with a window far shorter)
 *           it leaves fns_hip_attn few workgroups with keys: one token at 4096 keys takes 11 us, with a max_kv of 131072 or a
 *           window of 4096 in 131072 keys 19-21
 * A q_start range outside 0..n_tok or descending is a sequence without tokens. A position whose table entry is outside the
 * table or the cache's pages is never read or written: append leaves it out, attention sees no key there, kv_read gives NaN. */
typedef struct FnsKvBatch {
    int n_seq, max_q;
    int64_t n_tok, max_kv, table_stride;
    const int32_t *q_start;     /* [n_seq + 1] */
    const int32_t *kv_len;      /* [n_seq] */
    const int32_t *page_table;  /* [n_seq][table_stride] */
} FnsKvBatch;

#define FNS_ROPE_NONE 0
#define FNS_ROPE_HALVES 1 /* channel i turns with i + rope_dim / 2 */
#define FNS_ROPE_PAIRS 2  /* channel 2 i turns with 2 i + 1 */
/* k, v [n_tok][n_head_kv][head_dim] (tokens k_stride / v_stride elements apart) into the cache; the first rope_dim channels
 * of k and of q are turned by position * inv_freq[i] on the way (in 64 bits; k is held from the unrounded result). q
 * [n_tok][n_head][head_dim] -> q_out of the same type, n_head a multiple of n_head_kv, or n_head = 0: no queries. q_out may
 * be q (with its stride) and overlaps nothing else. Heads are contiguous within a token; no alignment beyond an element's is
 * needed. Positions that two sequences share (a common page) must not be appended by both in one call. */
typedef struct FnsKvAppend {
    int dtype; /* of k, v, q and q_out: FNS_TYPE_F32 or FNS_TYPE_BF16 */
    int rope;  /* FNS_ROPE_* */
    int rope_dim; /* a multiple of 16 up to head_dim (ignored without a rotation) */
    int n_head;
    const float *inv_freq; /* f32 [rope_dim / 2] */
    const void *k, *v, *q;
    void *q_out;
    int64_t k_stride, v_stride, q_stride, q_out_stride;
} FnsKvAppend;
int fns_hip_kv_append(const FnsKvCache *cache, const FnsKvBatch *batch, const FnsKvAppend *x, void *stream);
/* k, v f32 [n_tok][n_head_kv][head_dim]: what the cache holds of the batch's tokens. */
int fns_hip_kv_read(const FnsKvCache *cache, const FnsKvBatch *batch, float *k, float *v, void *stream);

/* Attention of the batch's tokens over the cache (their own keys included: append first). Query head h reads kv head
 * h / (n_head / n_head_kv). The token at position p sees positions 0..p, with window > 0 the last `window` of them.
 *   out = sum_j p_j V_j, p = softmax over the seen positions of scale * q . K_j; with sinks, exp(sinks[h]) joins the
 *   softmax's denominator (-infinity: nothing; +infinity or a NaN: NaNs). A row that sees nothing is zero; one that sees a token
 *   whose K or V holds a NaN block is NaN.
 * A row of q that holds a NaN or an infinity, or a scale * q beyond f32, gives NaN (where it sees anything); scores beyond f32
 * may.
 * q and out [n_tok][n_head][head_dim], heads contiguous within a token, no overlap, any element alignment. What q enters the
 * products with is within 2^-24 (FNS_TYPE_F32) or 2^-14 (FNS_TYPE_BF16) of its row's largest magnitude (where all of
 * scale * log2(e) * q is below 2^-100: that part of 2^-101), p carries 22 or 11 bits, cut toward zero, and the sum of p counts
 * the same values; softmax statistics and sums are f32. Blocks of V of any size that a row does not see leave its precision alone.
 * One call takes one form for all its sequences, by max_q: decode tokens over long contexts beside a long prompt go undivided
 * (31 at 8000 keys beside a prompt of 512: 222 us, apart 53 and 20), and are better a call of their own.
 * workspace: fns_hip_attn_workspace bytes (they depend on the numbers of the batch and on n_head, not on device memory; fewer
 * tokens can need more), 16-byte aligned, no initialisation; calls that overlap in time need one each. */
typedef struct FnsAttn {
    int dtype; /* of q and out: FNS_TYPE_F32 or FNS_TYPE_BF16 */
    int n_head;
    int window; /* 0: none */
    float scale;
    const float *sinks; /* NULL or f32 [n_head] */
    int64_t q_stride, out_stride; /* elements between tokens */
} FnsAttn;
int fns_hip_attn_workspace(const FnsKvCache *cache, const FnsKvBatch *batch, const FnsAttn *x, size_t *bytes);
int fns_hip_attn(const FnsKvCache *cache, const FnsKvBatch *batch, const FnsAttn *x, const void *q, void *out,
                 void *workspace, size_t workspace_bytes, void *stream);

/* --- trees of drafted tokens, and caches of a bounded length ---
 * A verify step of a tree:  fns_hip_tree_plan -> (projections) -> fns_hip_kv_append_at -> fns_hip_attn_tree -> ... -> the engine
 * picks a path -> fns_hip_kv_keep. A cache kept to a number of positions: fns_hip_attn_tree (its lse) -> fns_hip_kv_weigh every
 * step, fns_hip_kv_evict now and then; after that a token's place in the cache is not its position in the text any more, and
 * fns_hip_kv_append_at takes the latter. No counterparts in the reference, which drafts a line of tokens
 * (src/engine.cu:601-603) and keeps every position. */

/* Host arithmetic: inv_freq [rope_dim / 2] (host memory, f32) of a rotation made for `original` positions with
 * base^(-2 i / rope_dim), scaled to factor * original by the published rule of frequency parts: a pair that turns `fast` times
 * (32, say) or more over the original positions keeps its frequency, one that turns `slow` times (1) or less has it divided by
 * factor, the pairs between go over linearly in their index: from the last pair that keeps it (the first of all where none turns
 * so often) to the first index that would turn `slow` times or less, behind the last pair too, but at most rope_dim - 1.
 * *magnitude = 0.1 ln(factor) + 1, for fns_hip_kv_append_at. A factor of 1 gives the plain frequencies and 1. */
int fns_hip_rope_scaled(int rope_dim, double base, double factor, double original, double fast, double slow, float *inv_freq,
                        float *magnitude);
/* fns_hip_kv_append with the tokens turned by positions of their own: pos int32 [n_tok] (device memory), or NULL: their
 * positions in the cache. What turns is also multiplied by `magnitude` (positive, finite; k and q alike). Without a rotation
 * both are ignored. */
int fns_hip_kv_append_at(const FnsKvCache *cache, const FnsKvBatch *batch, const FnsKvAppend *x, const int32_t *pos,
                         float magnitude, void *stream);

/* What every new token of a batch sees of the new tokens of its sequence: bit j % 64 of sees[t * words + j / 64] for the j-th of
 * them (device memory, [n_tok][words]; bits behind the sequence's tokens are ignored, tokens from 64 * words on are seen by
 * none). */
typedef struct FnsKvTree {
    const uint64_t *sees;
    int words; /* 1..16 */
} FnsKvTree;
/* Those bits from parents, int32 [n_tok]: of a sequence's i-th new token the index j < i of its parent among them, or -1: it
 * follows the sequence's earlier positions. It sees itself and its ancestors. Anything else is no token of the tree (a plan of
 * fixed size is filled up with, say, -2): neither it nor what descends from it sees anything. pos int32 [n_tok] (or NULL) =
 * base[sequence] + its number of ancestors (0 for no token of the tree); base int32 [n_seq], or NULL: the position of the
 * sequence's first new token. 64 * words is at least max_q. Tokens of no sequence are left alone. */
int fns_hip_tree_plan(const FnsKvBatch *batch, const int32_t *parents, const int32_t *base, int words, uint64_t *sees,
                      int32_t *pos, void *stream);
/* fns_hip_attn of a tree, and its denominators. tree: a token sees the positions before its sequence's new tokens and, of these,
 * what its bits say (not the others, itself only with its bit); with a window of W and n bits the last W - n of the earlier
 * positions (none if n >= W: the bits alone say which new tokens it sees). A token without bits sees nothing: its output is
 * zero. NULL: as fns_hip_attn (FNS_TYPE_F32: in the same bits). q enters as f32 does there, whatever its type.
 * lse: NULL or f32 [n_tok][n_head], the logarithm of the softmax's denominator (sinks included) of every row; of one that sees
 * nothing the head's sink, -infinity without sinks. workspace: fns_hip_attn_tree_workspace bytes (with or without a tree; at
 * least fns_hip_attn_workspace's), as fns_hip_attn's. */
int fns_hip_attn_tree_workspace(const FnsKvCache *cache, const FnsKvBatch *batch, const FnsAttn *x, size_t *bytes);
int fns_hip_attn_tree(const FnsKvCache *cache, const FnsKvBatch *batch, const FnsAttn *x, const FnsKvTree *tree, const void *q,
                      void *out, float *lse, void *workspace, size_t workspace_bytes, void *stream);

/* Attention weights of cached positions: f32 [n_pages][n_head_kv][page_size]. For every position j of the sequences that have
 * new tokens, and every kv head,
 *   weights = past (of positions before the new tokens; the new ones start at 0)
 *             + sum over the sequence's new tokens t and the query heads h of the kv head of exp(scale * q[t][h] . K_j - lse[t][h])
 * over the rows that see j (causal or by the tree's bits, the window). past: NULL (zeros), `weights` itself, or another array.
 * x: dtype, n_head, window, scale and q_stride count. A row whose lse is not finite, or whose q is not, adds nothing (so an lse
 * set to infinity leaves a rejected token out); a position whose K holds a NaN block gets nothing. q enters as f32 does in
 * fns_hip_attn, whatever its type; sums are f32, in a fixed order. A position without a page has no weight. Sequences of a call
 * must not share pages. workspace: fns_hip_kv_weigh_workspace bytes, 16-byte aligned, as fns_hip_attn's. */
int fns_hip_kv_weigh_workspace(const FnsKvCache *cache, const FnsKvBatch *batch, const FnsAttn *x, size_t *bytes);
int fns_hip_kv_weigh(const FnsKvCache *cache, const FnsKvBatch *batch, const FnsAttn *x, const FnsKvTree *tree, const void *q,
                     const float *lse, const float *past, float *weights, void *workspace, size_t workspace_bytes,
                     void *stream);

/* Eviction: of every sequence (all its kv_len positions; q_start, n_tok and max_q do not matter) each kv head keeps `budget`
 * positions, or all if there are no more: the first `first`, the last `recent`, and of the others those of the largest weights (a
 * NaN is the largest, of equal ones the earlier is kept). Positions without a page are not there. What is kept moves, in order,
 * to positions 0, 1, ...: K, V (their bytes) and weights; the heads' choices differ, their number does not.
 * They go by the batch's own table (in place: no page may be in it twice, and weights_out is weights) or by `to_table`, with pages
 * none of which any of the call's sequences has; what goes where that table has no page, or behind its end, is lost. What
 * follows the kept positions is undefined in place, left alone elsewhere. kept: int32 [n_seq][n_head_kv][budget], the kept
 * positions in order, then -1. new_len: int32 [n_seq], how many they are; not the batch's kv_len (which the engine sets
 * afterwards). */
typedef struct FnsKvEvict {
    int budget, first, recent; /* budget 1..2^30, first + recent at most that */
    const float *weights;
    float *weights_out;        /* may be weights */
    const int32_t *to_table;   /* NULL: in place; else [n_seq][to_stride] */
    int64_t to_stride;
    int32_t *kept, *new_len;
    void *workspace;           /* fns_hip_kv_evict_workspace bytes, 16-byte aligned; calls that overlap in time need one each */
    size_t workspace_bytes;
} FnsKvEvict;
/* Depends on the numbers of cache and batch alone: 0 where the table has room for at most 32768 positions of a sequence. */
int fns_hip_kv_evict_workspace(const FnsKvCache *cache, const FnsKvBatch *batch, size_t *bytes);
int fns_hip_kv_evict(const FnsKvCache *cache, const FnsKvBatch *batch, const FnsKvEvict *x, void *stream);

/* Of the new tokens of every sequence those listed become its next positions, in the list's order: new token kept[s][i] (its
 * index among the sequence's new tokens) goes to position kv_len - n + i, i < n_kept[s] (at most n and `stride`). Entries that are no
 * new token of the sequence leave that position as it was. weights: NULL, or moved along. new_len int32 [n_seq] =
 * kv_len - n + n_kept (kv_len for a sequence without new tokens); not the batch's kv_len (which the engine sets afterwards). */
typedef struct FnsKvKeep {
    const int32_t *kept;   /* [n_seq][stride] */
    const int32_t *n_kept; /* [n_seq] */
    int64_t stride;        /* 1..1024 */
    float *weights;
    int32_t *new_len;
} FnsKvKeep;
int fns_hip_kv_keep(const FnsKvCache *cache, const FnsKvBatch *batch, const FnsKvKeep *x, void *stream);

/* --- GGUF checkpoints: reader and fully resident MoE layers ---
 * Replaces the reference's loader (src/model.cpp:30-136: gguf header and tensor table, the file mapped without copying)
 * and expert placement (src/engine.cu:375-471: slots [gate | up | down] 256-byte aligned with 4096 zero bytes after the
 * last, a device table of slot pointers); every expert is resident in HBM. The reader is host code (no GPU needed);
 * fns_hip_moe_layer_from_gguf copies with hipMemcpy on the current device. C++ interface: include/fns/gguf.h. */
typedef struct FnsGguf FnsGguf;
typedef struct FnsGgufTensorInfo {
    int type;        /* ggml_type */
    int n_dims;
    int64_t ne[4];   /* ggml order: ne[0] contiguous */
    size_t nbytes;
    size_t offset;   /* from the start of the data section */
    const void *data; /* host pointer into the mapping (valid until fns_hip_gguf_close) */
} FnsGgufTensorInfo;
/* Opens and maps `path`; FNS_ERR_IO (with the reason in fns_hip_last_error) on a missing or malformed file. */
int fns_hip_gguf_open(const char *path, FnsGguf **out);
void fns_hip_gguf_close(FnsGguf *file);
int fns_hip_gguf_info(const FnsGguf *file, uint32_t *version, int64_t *n_tensors, int64_t *n_kv, size_t *data_offset);
/* Tensor by name (FNS_ERR_SHAPE when absent) or by index; *name (optional) points into the reader. */
int fns_hip_gguf_tensor(const FnsGguf *file, const char *name, FnsGgufTensorInfo *info);
int fns_hip_gguf_tensor_at(const FnsGguf *file, int64_t index, FnsGgufTensorInfo *info, const char **name);
/* gguf_get_val_u32 / f32 / bool / str of the reference's loader (src/model.cpp:19-26): FNS_ERR_SHAPE when the key is
 * absent or of another type. *value of _str points into the reader. */
int fns_hip_gguf_get_u32(const FnsGguf *file, const char *key, uint32_t *value);
int fns_hip_gguf_get_f32(const FnsGguf *file, const char *key, float *value);
int fns_hip_gguf_get_bool(const FnsGguf *file, const char *key, int *value);
int fns_hip_gguf_get_str(const FnsGguf *file, const char *key, const char **value);
/* MoE layer `layer` of the file made resident in HBM (blk.N.ffn_{gate,up,down}_exps.weight, ffn_gate_inp.weight,
 * optional exp_probs_b.bias, ffn_norm.weight and ffn_{gate,up,down}_shexp.weight; metadata
 * <arch>.expert_used_count, expert_weights_norm, expert_gating_func (1 softmax, 2 sigmoid; default sigmoid for
 * "flint", the reference's gating), attention.layer_norm_rms_epsilon). Fills *desc for fns_hip_moe_layer /
 * fns_hip_moe_prefill (guard = 1 for "flint", whose blocks apply the F16 guard, else 0); the device memory it points
 * to is owned by *resident. */
typedef struct FnsMoeResident FnsMoeResident;
int fns_hip_moe_layer_from_gguf(const FnsGguf *file, int layer, FnsMoeResident **resident, FnsMoeLayer *desc);
void fns_hip_moe_resident_free(FnsMoeResident *resident);
/* Dense FFN layer `layer` of the file made resident in HBM (reference src/model.cpp:120-125,193-196:
 * blk.N.ffn_{gate,up,down}.weight and ffn_norm.weight, metadata attention.layer_norm_rms_epsilon). Fills *desc for
 * fns_hip_dense_ffn / fns_hip_dense_ffn_prefill; the device memory it points to is owned by *resident. */
typedef struct FnsDenseResident FnsDenseResident;
int fns_hip_dense_ffn_from_gguf(const FnsGguf *file, int layer, FnsDenseResident **resident, FnsDenseFfn *desc);
void fns_hip_dense_resident_free(FnsDenseResident *resident);

/* --- seeded synthetic data on the device (benchmarks and large tests) ---
 * out[i] = mean + std * N(0,1), Philox-4x32-10 counter (offset + i) / 4 and Box-Muller; offset % 4 == 0. */
int fns_hip_fill_normal(float *out, int64_t n, uint64_t seed, uint64_t offset, float mean, float std, void *stream);
/* ggml's reference K-quant quantisers (quantize_row_q{3,4,5,6}_K_ref) on the device: x f32 [nrows][ncols] -> out. */
int fns_hip_quantize_weights(int type, const float *x, void *out, int64_t nrows, int64_t ncols, void *stream);

/* Device self-test of the DPP / lane-permute exchanges the kernels use: writes a bit mask of failing checks to
 * *bad_mask (device int, zero it first); 0 means every exchange matched the LDS-crossbar shuffle. */
int fns_hip_selftest_lanes(int *bad_mask, void *stream);

#ifdef __cplusplus
}
#endif
#endif
