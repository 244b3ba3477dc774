/*
 * rsllm_hip.h — C ABI of the MI355X (gfx950) quantized mat-vec / mat-mul
 * backend for rsLLM.
 *
 * Each entry point replaces one function of the reference's CPU path
 * (citations: paths relative to the rsLLM tree, crates/<crate>/src/...).
 * Arguments keep the reference's meaning and order; slices become
 * (pointer, length) pairs so the same length checks can run here, in the
 * same order, with the same error classes.
 *
 * Two flavours:
 *   - host-pointer entry points: synchronous drop-ins for the Rust functions
 *     (buffers are caller-owned host memory; `out` is valid on return);
 *   - `_dev` entry points: device pointers, enqueued on the caller's
 *     hipStream_t, no host synchronisation.
 *
 * Weights in device memory are in the "device layout" written by
 * rsllm_hip_prepare_weights_dev: for Q4_K it is the GGUF byte stream
 * itself; Q6_K / Q8_0 / Q4_0 / Q2_K / IQ2_XXS matrices are regrouped into
 * 8-block super-tiles of the same total size (see
 * rsllm_hip_prepare_weights_dev).
 *
 * Thread safety: every entry point may be called from any thread, as
 * CpuBackend (backend-cpu/src/lib.rs:42-45) may. Process state (device
 * ordinal, the registry of device copies) is guarded by a mutex, and the
 * registry is a hash map keyed by host address. Each calling thread gets its
 * own stream and host<->device staging for the host-pointer entry points.
 * The kernels' device workspace belongs to a stream: one set per (device,
 * stream), used by every call enqueued on that stream and locked while a
 * call enqueues, so calls on different streams never share workspace and
 * threads sharing a stream take turns. A call that uses a registered or
 * model-resident tensor holds a reference to its device memory until it has
 * synchronised, so a release on another thread never frees memory under it.
 * Device pointers a caller obtained itself (rsllm_hip_model_tensor) are the
 * caller's to keep alive: release a model only after work using them ends.
 */
#ifndef RSLLM_HIP_H
#define RSLLM_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Opaque stream handle: a hipStream_t (NULL = the default stream). */
typedef void *rsllm_hip_stream_t;

/* Status codes. 1..4 mirror rsllm_backend_cpu::Error
 * (backend-cpu/src/error.rs:7-43), 5..6 mirror rsllm_gguf::Error's
 * dequant variants (rsllm-gguf/src/error.rs:69-80). */
typedef enum rsllm_hip_status {
    RSLLM_HIP_OK = 0,
    RSLLM_HIP_ERR_SHAPE_MISMATCH = 1,        /* Error::ShapeMismatch(&str) */
    RSLLM_HIP_ERR_NOT_BLOCK_ALIGNED = 2,     /* Error::NotBlockAligned{what,actual,block} */
    RSLLM_HIP_ERR_NON_FINITE_INPUT = 3,      /* Error::NonFiniteInput(&str) */
    RSLLM_HIP_ERR_UNSUPPORTED_TIER = 4,      /* Error::UnsupportedTier(&str) */
    RSLLM_HIP_ERR_DEQUANT_SIZE_MISMATCH = 5, /* Error::DequantSizeMismatch{src_bytes,expected_bytes} */
    RSLLM_HIP_ERR_UNSUPPORTED_DEQUANT = 6,   /* Error::UnsupportedDequant(name) */
    RSLLM_HIP_ERR_DEVICE = 7,                /* a HIP runtime call failed (no reference counterpart) */
    RSLLM_HIP_ERR_INVALID_ARGUMENT = 8,      /* NULL pointer with nonzero length, or a shape the
                                                reference would panic on (row_len == 0 in
                                                parallel.rs:44) */
    RSLLM_HIP_ERR_UNIMPLEMENTED = 10         /* a call the reference accepts but this backend
                                                does not serve (e.g. the Q4_K-only prefill entry
                                                given another dtype) */
} rsllm_hip_status;

/* GgmlType ids (rsllm-gguf/src/tensor.rs:26-85) used by this ABI. */
enum {
    RSLLM_GGML_F32 = 0, RSLLM_GGML_F16 = 1, RSLLM_GGML_Q4_0 = 2, RSLLM_GGML_Q4_1 = 3,
    RSLLM_GGML_Q8_0 = 8, RSLLM_GGML_Q2_K = 10, RSLLM_GGML_Q4_K = 12, RSLLM_GGML_Q5_K = 13,
    RSLLM_GGML_Q6_K = 14, RSLLM_GGML_Q8_K = 15, RSLLM_GGML_IQ2_XXS = 16, RSLLM_GGML_BF16 = 30
};

/* Details of the last error on the calling thread.
 * what/actual/block: NotBlockAligned (error.rs:18-25);
 * src_bytes/expected_bytes: DequantSizeMismatch (gguf error.rs:71-76). */
typedef struct rsllm_hip_error_detail {
    int32_t status;
    const char *message; /* the reference's message text where it has one */
    const char *what;
    size_t actual, block;
    size_t src_bytes, expected_bytes;
} rsllm_hip_error_detail;

void rsllm_hip_last_error(rsllm_hip_error_detail *out);

/* No reference counterpart; a diagnostic: the number of device allocations
 * (hipMalloc) the library has made in this process so far (workspace sets,
 * staging, registered tensors, model arenas). It only grows. */
uint64_t rsllm_hip_device_allocations(void);

/* Backend handle analogue: CpuBackend::new (backend-cpu/src/lib.rs:50-53)
 * plus device choice. Optional; the first call of any entry point performs
 * it with device 0. */
int rsllm_hip_init(int device_ordinal);

/* BackendCapability analogue (rsllm-cal/src/lib.rs:62-75,
 * backend-cpu/src/capability.rs:119-131). */
typedef struct rsllm_hip_capability {
    const char *backend; /* "rocm" */
    const char *arch;    /* "gfx950" */
    int q4k_matmul, q6k_matmul, q8_0_matmul, q2k_matmul, iq2xxs_matmul, fp8_kv_cache;
} rsllm_hip_capability;
void rsllm_hip_capability_get(rsllm_hip_capability *out);

/* ---- quantized matmul --------------------------------------------------- */

/* matmul_quant_f32 (backend-cpu/src/ops/quant_matmul.rs:45-119).
 * out[t*out_dim + o] = sum_i deq(W)[o, i] * x[t*in_dim + i]; `out` is
 * overwritten. Validation order as :57-92: dtype, in_dim % block,
 * weights_len, x_len, out_len. Accepted dtypes: Q4_K, Q2_K, IQ2_XXS, Q4_0,
 * Q8_0 (the reference's guard), and Q6_K (a deliberate superset: the
 * reference's guard rejects Q6_K). `tier` is
 * accepted and ignored, as the reference ignores it (:55).
 * Weights are uploaded for this call unless the same (pointer, length,
 * dtype, in_dim) was registered with rsllm_hip_register_weights. */
int rsllm_hip_matmul_quant_f32(float *out, size_t out_len, const uint8_t *weights,
                               size_t weights_len, const float *x, size_t x_len, size_t n_tok,
                               size_t in_dim, size_t out_dim, uint32_t dtype, uint32_t tier);

/* Device-pointer matmul_quant_f32: same validation; `weights` in device
 * layout; enqueued on `stream`. */
int rsllm_hip_matmul_quant_f32_dev(float *out, size_t out_len, const uint8_t *weights,
                                   size_t weights_len, const float *x, size_t x_len,
                                   size_t n_tok, size_t in_dim, size_t out_dim, uint32_t dtype,
                                   rsllm_hip_stream_t stream);

/* No counterpart in the reference. For callers that cannot allocate device
 * memory (work under HIP graph capture, serving loops or harnesses that
 * forbid hipMalloc): rsllm_hip_matmul_quant_f32_dev with the same arguments,
 * validation and results, whose activation workspace is a static array of
 * RSLLM_HIP_NOALLOC_SCRATCH_BYTES per GPU (held until the process ends)
 * instead of memory the library allocates; the call itself allocates and
 * frees nothing. A call whose workspace would exceed that size (many tokens
 * of a long row) returns RSLLM_HIP_ERR_INVALID_ARGUMENT. Every call on one
 * GPU shares its array and leaves its contents behind: calls that overlap in
 * time on one GPU (two streams, or two threads) race on it, so enqueue them
 * on one stream. */
#define RSLLM_HIP_NOALLOC_SCRATCH_BYTES ((size_t)48 << 20)
int rsllm_hip_matmul_quant_f32_dev_noalloc(float *out, size_t out_len, const uint8_t *weights,
                                           size_t weights_len, const float *x, size_t x_len,
                                           size_t n_tok, size_t in_dim, size_t out_dim,
                                           uint32_t dtype, rsllm_hip_stream_t stream);

/* Activations pre-quantised for the GEMV kernels, for callers that reuse one
 * x across several weight matrices of the same dtype and in_dim (e.g. an
 * FFN's gate and up projections) or time the GEMV alone. No reference
 * counterpart: matmul_quant_f32 takes f32 x directly. x is re-expressed per
 * 16-element group as s * (256 h + l) with int8 limbs (about 16 bits
 * relative to the group's largest element) in a dtype-specific lane-major
 * layout of rsllm_hip_xq_bytes(dtype, n_tok, in_dim) bytes.
 * rsllm_hip_matmul_prequant_dev is rsllm_hip_matmul_quant_f32_dev with xq in
 * place of x (same validation, x_len replaced by xq_len). The products are
 * the same; the summation order can differ from the one-shot call's kernel,
 * so the two agree to a few ulp, not bit for bit. */
size_t rsllm_hip_xq_bytes(uint32_t dtype, size_t n_tok, size_t in_dim);
int rsllm_hip_quantize_x_dev(uint32_t dtype, const float *x, size_t x_len, size_t n_tok,
                             size_t in_dim, uint8_t *xq, size_t xq_len, rsllm_hip_stream_t stream);
int rsllm_hip_matmul_prequant_dev(float *out, size_t out_len, const uint8_t *weights,
                                  size_t weights_len, const uint8_t *xq, size_t xq_len,
                                  size_t n_tok, size_t in_dim, size_t out_dim, uint32_t dtype,
                                  rsllm_hip_stream_t stream);

/* ---- weights residency ----------------------------------------------------
 * The reference borrows weights from the GGUF mmap for the life of the
 * GgufFile (rsllm-gguf/src/file.rs:81-97, models/src/dsv4/loader.rs:199-216).
 * Registering uploads a tensor once (converted to the device layout);
 * later host-pointer calls with the same (pointer, length, dtype, in_dim)
 * use the device copy. Release removes every registered tensor; the device
 * copy of one that a call on another thread is using is freed when that call
 * ends. */
int rsllm_hip_register_weights(const uint8_t *weights, size_t weights_len, uint32_t dtype,
                               size_t in_dim);
int rsllm_hip_release_weights(void);

/* No reference counterpart (the reference has no streams): frees the device
 * workspace the library keeps for `stream` on the current device, for a
 * caller about to destroy that stream. Work still enqueued there finishes
 * first (hipFree waits for the device); a later call on the stream makes a
 * new set. hipStreamPerThread names a different stream in each thread, so
 * each thread that passes it gets a set of its own, and releasing it frees
 * only the calling thread's set. */
int rsllm_hip_stream_release(rsllm_hip_stream_t stream);

/* ---- whole-model residency ---------------------------------------------------
 * No single reference function: this replaces keeping weights only in the
 * GGUF mmap (GgufFile::open, rsllm-gguf/src/file.rs:81-97; tensor_bytes
 * :181-187; resolve_blob, models/src/dsv4/loader.rs:199-216) when the
 * matmuls run on the GPU. The caller lists every tensor once, after opening
 * the file:
 *   name    TensorInfo::name;
 *   data    GgufFile::tensor_bytes (host memory, e.g. inside the mmap);
 *   len     its byte length;
 *   dtype   TensorInfo::raw_type (GgmlType id);
 *   in_dim  row length (shape[0]) for tensors used as matmul weights (F32 or
 *           a matmul format), else 0.
 * rsllm_hip_model_upload copies all of them into one device allocation, in
 * list order (each 256-byte aligned, so stacked expert tensors stay
 * contiguous), through pinned staging, converting matmul tensors (in_dim !=
 * 0) to the device layout; the rest are copied as is. Matmul tensors are
 * registered under their
 * host range, like rsllm_hip_register_weights, so the host-pointer entry
 * points use the resident copy. An upload whose fingerprint
 * (GgufFile::fingerprint, file.rs:175-177: names, types and shapes only),
 * tensor table and payload match a live model on the same device returns
 * that model, adds a reference and registers the new host ranges, without
 * copying. The payload comparison is a 64-bit hash of every byte (taken by
 * the copy threads during an upload; for a candidate that also matches a
 * 16-window sampled digest, over the new bytes by a host read pass), so
 * files that differ anywhere get separate models. Errors, all before any
 * device work: INVALID_ARGUMENT for
 * NULL arguments or duplicate names, SHAPE_MISMATCH for a matmul tensor
 * whose length is not whole rows of a block-aligned in_dim. Uploads are
 * serialised with each other and with the lookups below.
 * rsllm_hip_model_tensor returns a tensor's device address and length (the
 * device-layout bytes the _dev entry points take). rsllm_hip_model_release
 * drops one reference; the last one removes the registrations, and the
 * allocation is freed once no host-pointer call in flight still uses one of
 * its tensors. `_dev` work on addresses from rsllm_hip_model_tensor must end
 * before the last release. rsllm_hip_release_weights does not touch
 * models. */
typedef struct rsllm_hip_tensor_desc {
    const char *name;
    const uint8_t *data;
    size_t len;
    uint32_t dtype;
    size_t in_dim;
} rsllm_hip_tensor_desc;

typedef struct rsllm_hip_model_info {
    uint64_t device_bytes;   /* size of the model's device allocation */
    uint64_t uploaded_bytes; /* payload bytes copied when it was uploaded */
    double upload_seconds;   /* wall time of that upload */
    uint32_t refs, n_tensors;
} rsllm_hip_model_info;

int rsllm_hip_model_upload(const uint8_t *fingerprint /* 32 bytes */,
                           const rsllm_hip_tensor_desc *tensors, size_t n_tensors,
                           uint64_t *model);
int rsllm_hip_model_tensor(uint64_t model, const char *name, const uint8_t **dev, size_t *len);
int rsllm_hip_model_info_get(uint64_t model, rsllm_hip_model_info *out);
int rsllm_hip_model_release(uint64_t model);

/* GGUF rows -> device layout: `len` bytes holding whole rows of `in_dim`
 * elements (n = len / block_bytes blocks in matrix order, row-major over
 * (row, block)). Q4_K: unchanged (`dst` may equal `src`). Q6_K, Q8_0, Q4_0,
 * Q2_K, IQ2_XXS: the blocks are regrouped into super-tiles of 8 consecutive
 * blocks (the last tile holds the n % 8 remaining blocks, r of them), each
 * tile split into field runs so that every field of every block is aligned:
 *   Q6_K    [ql r*128 | qh r*64 | scales r*16 | d r*2]   (8 blocks: 1680 B)
 *   Q8_0    [qs r*32 | d r*2]                           (8 blocks: 272 B)
 *   Q4_0    [qs r*16 | d r*2]                           (8 blocks: 144 B)
 *   Q2_K    [qs r*64 | scales r*16 | (d, dmin) r*4]     (8 blocks: 672 B)
 *   IQ2_XXS [qs r*64 | d r*2]                           (8 blocks: 528 B)
 * with r = 8 except in the last tile; tile S starts at byte
 * S * 8 * block_bytes. `dst` must not overlap `src`. Enqueued on `stream`. */
int rsllm_hip_prepare_weights_dev(uint8_t *dst, const uint8_t *src, size_t len, uint32_t dtype,
                                  size_t in_dim, rsllm_hip_stream_t stream);

/* ---- prefill GEMM (bf16 activations) ---------------------------------------
 * The prefill form of matmul_quant_f32 (backend-cpu/src/ops/quant_matmul.rs:
 * 45-119, called from models/src/engine_impl.rs:277 prefill with n_tok = T):
 * out[t * out_dim + o] = sum_i deq(W)[o, i] * f32(x[t * in_dim + i]) for a
 * GGUF Q4_K weight (device copy of the GGUF bytes) and bf16 activations
 * (x_len = n_tok * in_dim 16-bit patterns). Runs on the matrix cores
 * (f16 MFMA, fp32 accumulation); within 1e-3 (max|d|/max|y|) of the
 * reference on f32(x). Validation as matmul_quant_f32 (dtype -> in_dim %
 * 256 -> weights -> x -> out); dtypes other than Q4_K return
 * RSLLM_HIP_ERR_UNIMPLEMENTED. Uses a per-thread device workspace of about
 * 2 * n_tok * in_dim bytes; enqueued on `stream`. */
int rsllm_hip_matmul_q4k_bf16_dev(float *out, size_t out_len, const uint8_t *weights,
                                  size_t weights_len, const uint16_t *x_bf16, size_t x_len,
                                  size_t n_tok, size_t in_dim, size_t out_dim, uint32_t dtype,
                                  rsllm_hip_stream_t stream);

/* ---- routed experts (MoE) ---------------------------------------------------
 * accumulate_moe_outputs (models/src/dsv4/moe.rs:648-707) with
 * apply_expert_swiglu (:479-502) and apply_swiglu_clamp (:515-531): for
 * every token t and slot i with weights[t*k+i] != 0 and e = ids[t*k+i]:
 *   out[t] += weights[t*k+i] * down[e] (silu(min(gate[e] x_t, c)) *
 *                                       clamp(up[e] x_t, -c, c))
 * with the clamp applied only when c > 1e-6 (NaN passes through), slots
 * accumulated in i order. `out` [n_tok x n_embd] is ACCUMULATED into (the
 * caller pre-clears or pre-fills it, as the reference's caller does).
 * gate, up: n_expert stacked [n_ff x n_embd] matrices of dtype_gate_up
 * (gate_up_len bytes each blob); down: n_expert stacked [n_embd x n_ff]
 * matrices of dtype_down (StackedExperts::expert, moe.rs:69-108). Q4_K
 * blobs are the GGUF bytes; other dtypes are in the device layout
 * (rsllm_hip_prepare_weights_dev over the whole blob), which needs each
 * expert's block count to be a multiple of 8. ids, weights: n_tok * k.
 * Validation: dtypes, then n_embd % block(gate/up) and n_ff % block(down)
 * (NotBlockAligned), blob lengths, x, out, ids lengths (ShapeMismatch);
 * n_expert <= 16384. Any number of tokens (the reference's prefill passes
 * every token of the forward pass, moe.rs:281,346): calls of more than 8192
 * (token, slot) pairs run in token chunks, each routed and computed on its
 * own, which gives the same result. The reference panics on an expert id
 * out of range: the host entry point returns RSLLM_HIP_ERR_INVALID_ARGUMENT,
 * the device entry point (which cannot inspect ids) skips such slots. Uses
 * the stream's device workspace. */
int rsllm_hip_moe_routed_dev(float *out, size_t out_len, const float *x, size_t x_len,
                             const uint8_t *gate, const uint8_t *up, size_t gate_up_len,
                             const uint8_t *down, size_t down_len, const int32_t *ids,
                             const float *weights, size_t ids_len, size_t n_tok, size_t n_embd,
                             size_t n_ff, size_t n_expert, size_t k, uint32_t dtype_gate_up,
                             uint32_t dtype_down, float clamp, rsllm_hip_stream_t stream);
/* Host-pointer form (synchronous). Expert blobs registered with
 * rsllm_hip_register_weights (in_dim n_embd for gate/up, n_ff for down) are
 * used from the device; otherwise they are uploaded for the call. */
int rsllm_hip_moe_routed(float *out, size_t out_len, const float *x, size_t x_len,
                         const uint8_t *gate, const uint8_t *up, size_t gate_up_len,
                         const uint8_t *down, size_t down_len, const int32_t *ids,
                         const float *weights, size_t ids_len, size_t n_tok, size_t n_embd,
                         size_t n_ff, size_t n_expert, size_t k, uint32_t dtype_gate_up,
                         uint32_t dtype_down, float clamp);

/* ---- expert routing ---------------------------------------------------------
 * No single reference function: the router's product is matmul_weight_f32,
 * and what follows it, the ids and weights rsllm_hip_moe_routed takes, is made
 * here. logits: n_tok rows of n_expert values of `dtype` (F32, F16 or BF16),
 * logits_stride elements apart. Per token, in 64 bits:
 *   s_e   = softmax(l)_e | 1 / (1 + exp(-l_e)) | sqrt(log(1 + exp(l_e)))
 *   key_e = s_e + bias_e     (bias: n_expert values that balance the load and
 *                             take part in the choice alone, or NULL)
 * With n_group > 1, group g holds experts [g n_expert / n_group, ...), counts
 * the sum of its group_top (1 or 2) largest keys (of the experts that can be
 * chosen; the one key where there is only one), and the topk_group groups that
 * count most stay. Of the experts left the k with the largest keys are
 * chosen: ids[t * k + i] in falling order of key, equal keys in rising order of
 * id (groups likewise); without a bias the logits themselves are compared, which
 * is the same order. weights[t * k + i] = scale * s_e, divided by the sum of the
 * chosen experts' s when `renormalise` is nonzero (0 if that sum is 0), rounded
 * once to f32.
 * An expert whose logit or key is NaN or -inf is never chosen (a group without
 * any other neither); places that stay empty get id -1 and weight 0, which
 * rsllm_hip_moe_routed_dev skips. A +inf logit counts as the softmax's limit:
 * the +inf experts share it evenly.
 * Errors: UNIMPLEMENTED for another dtype; INVALID_ARGUMENT for an unknown
 * score, n_expert 0 or above 16384, n_group 0, above 1024 or no divisor of
 * n_expert, topk_group 0 or above n_group, group_top other than 1 and 2, k 0 or
 * above min(64, topk_group * n_expert / n_group), a scale that is not finite,
 * NULL pointers or logits not aligned to their elements; SHAPE_MISMATCH for
 * n_tok above 8388607 (what a launch holds), logits_stride < n_expert, logits_len < (n_tok - 1) * logits_stride + n_expert,
 * bias_len other than 0 and n_expert, ids_len != n_tok * k. Enqueued on
 * `stream`; no workspace. */
enum {
    RSLLM_HIP_SCORE_SOFTMAX = 0, RSLLM_HIP_SCORE_SIGMOID = 1, RSLLM_HIP_SCORE_SQRT_SOFTPLUS = 2
};
int rsllm_hip_moe_route_dev(int32_t *ids, float *weights, size_t ids_len, const void *logits,
                            size_t logits_len, size_t logits_stride, const float *bias,
                            size_t bias_len, size_t n_tok, size_t n_expert, size_t k,
                            size_t n_group, size_t topk_group, size_t group_top, uint32_t score,
                            int renormalise, float scale, uint32_t dtype,
                            rsllm_hip_stream_t stream);

/* ---- caller chain: matmul_weight_f32, matmul_grouped_lora_down ------------
 * rsllm_hip_matmul_weight_f32 replaces matmul_weight_f32
 * (rsllm-models/src/dsv4/weight.rs:113-169): out[t, o] = sum_i W[o, i] x[t, i]
 * for a WeightBlob. dtype 0 (GGML F32) is the F32 arm: `weights` holds
 * out_dim * in_dim f32 values, weights_len counts bytes (out_dim * in_dim *
 * 4). Any other dtype is the Quant arm, matmul_quant_f32 on the blob.
 * Validation in the reference's order:
 *   out_len != n_tok * out_dim            SHAPE_MISMATCH (matmul_weight_f32.out)
 *   x_len != n_tok * in_dim               SHAPE_MISMATCH (matmul_weight_f32.x)
 *   F32: weights_len != out_dim*in_dim*4  SHAPE_MISMATCH (.weight_f32)
 *   Quant: every error of matmul_quant_f32 (dtype, block alignment,
 *          lengths) becomes SHAPE_MISMATCH (.quant), as the reference maps
 *          it; out_dim == 0 (a panic there) is INVALID_ARGUMENT.
 *
 * rsllm_hip_matmul_grouped_lora_down replaces matmul_grouped_lora_down
 * (weight.rs:209-266): x is [n_tok x n_groups * group_dim], out
 * [n_tok x n_groups * rank], weights n_groups stacked [rank x group_dim]
 * row-major matrices (the [n_groups * rank x group_dim] matrix), F32 or a
 * quant dtype as above; out[t, g * rank + o] = sum_i W_g[o, i]
 * x[t, g * group_dim + i]. Validation: x length (.x), out length (.out),
 * then for the groups grouped_weight_slice (weight.rs:271-323: group_dim *
 * rank a multiple of the block (.alignment), each group's slice inside the
 * blob (.f32 / .quant)) and the group's matmul_weight_f32 checks, all
 * SHAPE_MISMATCH; n_groups == 0 is OK. The reference computes group by group
 * and can fail on a later group's slice after writing earlier groups; here
 * every check runs before anything is written.
 *
 * Device forms: weights in this backend's device layout (Quant arm:
 * rsllm_hip_prepare_weights_dev of the [n_groups * rank x group_dim]
 * matrix; F32: as is), x and out on the device, enqueued on `stream`. Each
 * chunk of up to 8 tokens is one launch for all groups (each workgroup holds
 * one group's x in LDS). A group_dim too long for that (over about 60k
 * elements for the 256-element formats) runs each group as its own launch
 * on gathered x, which needs the group to be a whole number of 8-block
 * super-tiles of the device layout (non-Q4_K dtypes: rank * group_dim /
 * block elements a multiple of 8). For such groups that are not, the host
 * form converts each group to the device layout on its own, and the device
 * form returns RSLLM_HIP_ERR_UNIMPLEMENTED (writing nothing). The host form
 * uses a registered copy of the blob only when the groups use all of it and
 * it is not converted group by group. */
int rsllm_hip_matmul_weight_f32(float *out, size_t out_len, const uint8_t *weights,
                                size_t weights_len, const float *x, size_t x_len, size_t n_tok,
                                size_t in_dim, size_t out_dim, uint32_t dtype);
int rsllm_hip_matmul_weight_f32_dev(float *out, size_t out_len, const uint8_t *weights,
                                    size_t weights_len, const float *x, size_t x_len,
                                    size_t n_tok, size_t in_dim, size_t out_dim, uint32_t dtype,
                                    rsllm_hip_stream_t stream);
int rsllm_hip_matmul_grouped_lora_down(float *out, size_t out_len, const uint8_t *weights,
                                       size_t weights_len, const float *x, size_t x_len,
                                       size_t n_tok, size_t n_groups, size_t group_dim,
                                       size_t rank, uint32_t dtype);
int rsllm_hip_matmul_grouped_lora_down_dev(float *out, size_t out_len, const uint8_t *weights,
                                           size_t weights_len, const float *x, size_t x_len,
                                           size_t n_tok, size_t n_groups, size_t group_dim,
                                           size_t rank, uint32_t dtype,
                                           rsllm_hip_stream_t stream);

/* ---- shared expert: apply_shared_expert / apply_expert_swiglu ---------------
 * rsllm_hip_apply_shared_expert replaces apply_shared_expert
 * (rsllm-models/src/dsv4/moe.rs:422-455): every token t of x [n_tok x
 * n_embd] through apply_expert_swiglu (:479-502),
 *   out[t] = down @ (silu(min(gate @ x[t], c)) * clamp(up @ x[t], -c, c)),
 * out [n_tok x n_embd] overwritten. apply_expert_swiglu on one token is the
 * n_tok = 1 call. gate and up are [n_ff x n_embd] and down [n_embd x n_ff]
 * WeightBlobs, each F32 (dtype 0, length in bytes) or a quant dtype of its
 * own; the clamp is skipped when clamp <= 1e-6 (apply_swiglu_clamp
 * :515-531, so 0 stands for the reference's None). Validation:
 * check_moe_shapes (:557-573) x_len then out_len (SHAPE_MISMATCH "moe.x" /
 * "moe.out"), then, if n_tok > 0, matmul_weight_f32's checks of the gate,
 * up and down calls in that order (as for rsllm_hip_matmul_weight_f32).
 * Gate and up of one quant format run as one GEMV launch per chunk of up to
 * 8 tokens (the two matrices as two row groups on the same x), then an
 * elementwise SwiGLU and the down GEMV; other combinations (F32 blobs,
 * mixed formats) run gate and up as separate GEMVs. Host blobs registered with
 * rsllm_hip_register_weights are used from the device.
 *
 * Device form: blobs in the device layout (rsllm_hip_prepare_weights_dev
 * for quant formats; F32 as is), enqueued on `stream`. */
int rsllm_hip_apply_shared_expert(float *out, size_t out_len, const float *x, size_t x_len,
                                  const uint8_t *gate, size_t gate_len, uint32_t dtype_gate,
                                  const uint8_t *up, size_t up_len, uint32_t dtype_up,
                                  const uint8_t *down, size_t down_len, uint32_t dtype_down,
                                  size_t n_tok, size_t n_embd, size_t n_ff, float clamp);
int rsllm_hip_apply_shared_expert_dev(float *out, size_t out_len, const float *x, size_t x_len,
                                      const uint8_t *gate, size_t gate_len, uint32_t dtype_gate,
                                      const uint8_t *up, size_t up_len, uint32_t dtype_up,
                                      const uint8_t *down, size_t down_len, uint32_t dtype_down,
                                      size_t n_tok, size_t n_embd, size_t n_ff, float clamp,
                                      rsllm_hip_stream_t stream);

/* ---- Q8_0 int8-activation path ---------------------------------------------
 * quantize_q8_0_batch (backend-cpu/src/ops/q8_0.rs:95-129, per token
 * quantize_q8_0_activation :42-88): x [n_tok x in_dim] -> xq [n_tok x blocks
 * x 32] int8 and scale [n_tok x blocks], blocks = ceil(in_dim / 32); per
 * block d = amax / 127, q = clamp(round_half_even(x / d), -128, 127) (x * (1
 * / d) exactly as the reference), a partial last block zero-padded.
 * Bit-exact with the reference. Validation order :101-118: x_len, xq_len,
 * scale_len (ShapeMismatch); in_dim == 0 is INVALID_ARGUMENT (the
 * reference's par_chunks_mut(0) panics). A non-finite input returns
 * RSLLM_HIP_ERR_NON_FINITE_INPUT (:67-69); xq and scale are then
 * unspecified. */
int rsllm_hip_quantize_q8_0_batch(const float *x, size_t x_len, int8_t *xq, size_t xq_len,
                                  float *scale, size_t scale_len, size_t n_tok, size_t in_dim);
/* Device-pointer form, enqueued on `stream`. Non-finite inputs cannot be
 * reported synchronously: when `status` (a device int32) is non-NULL it is
 * set to 0, or to 1 if any input was non-finite, once the work completes. */
int rsllm_hip_quantize_q8_0_batch_dev(const float *x, size_t x_len, int8_t *xq, size_t xq_len,
                                      float *scale, size_t scale_len, size_t n_tok,
                                      size_t in_dim, int32_t *status, rsllm_hip_stream_t stream);

/* matmul_q8_0_batch (backend-cpu/src/ops/q8_0.rs:217-263): out[t*out_dim + o]
 * = sum over blocks b, in order, of (wscale[o,b] * xscale[t,b]) * dot_i32(
 * wq[o,b], xq[t,b]) (dot_q8_0_row_scalar :163-193; a non-finite weight scale
 * counts as 0, :143-146; only the first in_dim - 32 b lanes of a partial
 * last block take part). `weights` are raw GGUF Q8_0 rows (out_dim * blocks
 * * 34 bytes, in_dim need not be a multiple of 32). Bit-exact with the
 * reference's scalar tier. Validation order :229-252: weights_len, xq_len,
 * xscale_len, out_len (ShapeMismatch); out_dim == 0 is INVALID_ARGUMENT
 * (parallel.rs:44). `tier` is accepted and ignored (the scalar result is
 * what every call returns). Weights are uploaded (and regrouped into the
 * device layout) for the call unless the same (pointer, length) was
 * registered as Q8_0 with this in_dim. */
int rsllm_hip_matmul_q8_0_batch(float *out, size_t out_len, const uint8_t *weights,
                                size_t weights_len, const int8_t *xq, size_t xq_len,
                                const float *xscale, size_t xscale_len, size_t n_tok,
                                size_t in_dim, size_t out_dim, uint32_t tier);
/* Device-pointer form, enqueued on `stream`: `weights` in the device layout
 * (rsllm_hip_prepare_weights_dev of the GGUF rows with in_dim rounded up to
 * a multiple of 32 — the same bytes matmul_quant_f32_dev takes for Q8_0),
 * weights and xq 16-byte aligned. */
int rsllm_hip_matmul_q8_0_batch_dev(float *out, size_t out_len, const uint8_t *weights,
                                    size_t weights_len, const int8_t *xq, size_t xq_len,
                                    const float *xscale, size_t xscale_len, size_t n_tok,
                                    size_t in_dim, size_t out_dim, rsllm_hip_stream_t stream);

/* ---- int8 product with a scale per token and per channel ---------------------
 * No reference counterpart (its int8 path scales blocks of 32): for weights
 * quantised to int8 with one scale per output row.
 *   d_t       = f32(max_i |x[t, i]| / 127)
 *   q[t, i]   = x[t, i] / d_t to the nearest integer, halves to even (of the
 *               exact quotient; within +-127; 0 where d_t is 0)
 *   out[t, o] = (f32(sum_i q[t, i] w[o, i]) * d_t) * wscale[o] + bias[o]
 * the sum exact in 32-bit integers. A token with a non-finite value gets d_t =
 * NaN and q = 0, so its outputs are NaN and no other token's are touched.
 * Rows of int8 codes (weights, xq) lie rsllm_hip_int8_row_bytes(in_dim) =
 * in_dim rounded up to 64 bytes apart, 16-byte aligned. The quantiser fills the
 * rest of a row with zeros; what a weight row holds there does not matter. It
 * quantises weight rows as well as tokens (n_tok = out_dim).
 * x: n_tok rows of in_dim values of `dtype` / `dtype_x` (F32, F16 or BF16),
 * x_stride elements apart; out: rows of out_dim values of dtype_out (F32, F16 or
 * BF16; rounded once from f32), out_stride elements apart, what lies between
 * rows left as it was. bias: out_dim values or NULL.
 * rsllm_hip_matmul_int8_dev takes x; _quantize_int8_dev and
 * _matmul_int8_prequant_dev are its halves, for one x through several matrices:
 * the same results, bit for bit. `work`: rsllm_hip_int8_work_bytes(n_tok,
 * in_dim, out_dim) bytes of the caller's (it never falls as n_tok grows),
 * 256-byte aligned, used by this call alone until it has run: calls that may
 * overlap, and graphs that may replay at once, get one each. The prequant form
 * also takes NULL with work_len 0 (its products leave nothing between launches).
 * Errors: UNIMPLEMENTED for another dtype; INVALID_ARGUMENT for in_dim 0 or
 * above 131071 (where the sum could leave 32 bits), out_dim 0, NULL or
 * misaligned pointers; SHAPE_MISMATCH for n_tok or out_dim above 8388607 (what a
 * launch holds; work_bytes is then 0), a stride below its row, x_len or out_len below (n_tok - 1) * stride + row, weights_len != out_dim * row bytes,
 * wscale_len != out_dim, bias_len other than 0 and out_dim, xq_len != n_tok *
 * row bytes, scale_len or xscale_len != n_tok, work_len below work_bytes. */
size_t rsllm_hip_int8_row_bytes(size_t in_dim);
size_t rsllm_hip_int8_work_bytes(size_t n_tok, size_t in_dim, size_t out_dim);
int rsllm_hip_quantize_int8_dev(const void *x, size_t x_len, size_t x_stride, int8_t *xq,
                                size_t xq_len, float *scale, size_t scale_len, size_t n_tok,
                                size_t in_dim, uint32_t dtype, rsllm_hip_stream_t stream);
int rsllm_hip_matmul_int8_prequant_dev(void *out, size_t out_len, size_t out_stride,
                                       const int8_t *weights, size_t weights_len,
                                       const float *wscale, size_t wscale_len, const float *bias,
                                       size_t bias_len, const int8_t *xq, size_t xq_len,
                                       const float *xscale, size_t xscale_len, uint8_t *work,
                                       size_t work_len, size_t n_tok, size_t in_dim,
                                       size_t out_dim, uint32_t dtype_out,
                                       rsllm_hip_stream_t stream);
int rsllm_hip_matmul_int8_dev(void *out, size_t out_len, size_t out_stride, const int8_t *weights,
                              size_t weights_len, const float *wscale, size_t wscale_len,
                              const float *bias, size_t bias_len, const void *x, size_t x_len,
                              size_t x_stride, uint8_t *work, size_t work_len, size_t n_tok,
                              size_t in_dim, size_t out_dim, uint32_t dtype_x, uint32_t dtype_out,
                              rsllm_hip_stream_t stream);

/* ---- microscaled 4-bit floating point ------------------------------------------
 * No reference counterpart (the formats it reads are GGUF's): rows of 4-bit codes
 * with an 8-bit scale for every 32 of them, the OCP Microscaling format MXFP4.
 * A code's low three bits stand for 0, 0.5, 1, 1.5, 2, 3, 4, 6, its high bit for the
 * sign; a scale byte s stands for 2^(s - 127), 255 for NaN. Code i of a row is the low
 * (i even) or high half of byte i / 2, scale b that of codes 32 b .. 32 b + 31.
 * Rows of codes lie rsllm_hip_mxfp4_row_bytes(in_dim) = in_dim / 2 rounded up to 64
 * bytes apart, rows of scales rsllm_hip_mxfp4_scale_bytes(in_dim) = a byte a block
 * rounded up to 16; both 16-byte aligned. The quantiser fills the rest of its rows
 * with zeros; of a weight row, what stands behind in_dim does not matter. Both give 0
 * for an in_dim outside 1..1048576.
 * rsllm_hip_quantize_mxfp4_dev: n_rows rows (tokens, or weight channels) of in_dim
 * values of `dtype` (F32, F16 or BF16), x_stride elements apart. Per block
 *   s    = 127 + max(-127, floor(log2(max |x|)) - 2)   (0 for a block of zeros)
 *   code = x / 2^(s - 127) to the nearest, halves to the even code, at most +-6
 * A block with a non-finite value gets s = 255 and codes of 0: it stands for NaN.
 * rsllm_hip_dequantize_mxfp4_dev: the values that codes stand for, in f32 (which holds
 * them exactly up to its largest number) rounded once to `dtype`; what lies between
 * rows of out is left as it was.
 * rsllm_hip_matmul_mxfp4_prequant_dev: the product of two such matrices, xcodes
 * [n_tok x in_dim] and weights [out_dim x in_dim], zeros behind in_dim in xcodes:
 *   out[t, o] = sum_b 2^(sx[t, b] + sw[o, b] - 254) (sum_i x[t, i] w[o, i]) + bias[o]
 * summed in f32 (the matrix cores' order), rows of dtype_out (F32, F16 or BF16; rounded
 * once from f32) out_stride elements apart; bias: out_dim values or NULL. A NaN block
 * makes its token's, or its channel's, outputs NaN.
 * rsllm_hip_matmul_mxfp4_dev takes floats x and quantises them on the way: the same
 * result, bit for bit, as the quantiser and the prequant form. An output must not
 * overlap what its call reads.
 * `work`: rsllm_hip_mxfp4_work_bytes(n_tok, in_dim, out_dim) bytes of the caller's (0
 * for sizes that are refused), 256-byte aligned, used by this call alone until it has run:
 * calls that may overlap, and graphs that may replay at once, get one each. (The prequant
 * form asks for it too, and so far does not write to it.)
 * Errors: UNIMPLEMENTED for another dtype; INVALID_ARGUMENT for in_dim 0 or above
 * 1048576, out_dim 0, NULL or misaligned pointers; SHAPE_MISMATCH for n_rows, n_tok or
 * out_dim above 8388607 (what a launch holds), a stride below its row, x_len or out_len
 * below (rows - 1) * stride + row, code and scale lengths that are not rows * row bytes
 * and rows * scale bytes, bias_len other than 0 and out_dim, work_len below
 * work_bytes. */
size_t rsllm_hip_mxfp4_row_bytes(size_t in_dim);
size_t rsllm_hip_mxfp4_scale_bytes(size_t in_dim);
size_t rsllm_hip_mxfp4_work_bytes(size_t n_tok, size_t in_dim, size_t out_dim);
int rsllm_hip_quantize_mxfp4_dev(const void *x, size_t x_len, size_t x_stride, uint8_t *codes,
                                 size_t codes_len, uint8_t *scales, size_t scales_len,
                                 size_t n_rows, size_t in_dim, uint32_t dtype,
                                 rsllm_hip_stream_t stream);
int rsllm_hip_dequantize_mxfp4_dev(const uint8_t *codes, size_t codes_len, const uint8_t *scales,
                                   size_t scales_len, void *out, size_t out_len,
                                   size_t out_stride, size_t n_rows, size_t in_dim, uint32_t dtype,
                                   rsllm_hip_stream_t stream);
int rsllm_hip_matmul_mxfp4_prequant_dev(void *out, size_t out_len, size_t out_stride,
                                        const uint8_t *weights, size_t weights_len,
                                        const uint8_t *wscales, size_t wscales_len,
                                        const float *bias, size_t bias_len, const uint8_t *xcodes,
                                        size_t xcodes_len, const uint8_t *xscales,
                                        size_t xscales_len, uint8_t *work, size_t work_len,
                                        size_t n_tok, size_t in_dim, size_t out_dim,
                                        uint32_t dtype_out, rsllm_hip_stream_t stream);
int rsllm_hip_matmul_mxfp4_dev(void *out, size_t out_len, size_t out_stride,
                               const uint8_t *weights, size_t weights_len, const uint8_t *wscales,
                               size_t wscales_len, const float *bias, size_t bias_len,
                               const void *x, size_t x_len, size_t x_stride, uint8_t *work,
                               size_t work_len, size_t n_tok, size_t in_dim, size_t out_dim,
                               uint32_t dtype_x, uint32_t dtype_out, rsllm_hip_stream_t stream);

/* ---- a whole mixture-of-experts layer for a few tokens ----------------------------
 * What the reference does between a layer's norm and its residual (the router's product,
 * moe_topk_route, accumulate_moe_outputs, apply_shared_expert; models/src/dsv4/moe.rs:
 * 235-707), for up to 32 tokens and expert weights in MXFP4. Per token:
 *   l_e   = sum_i router[e, i] x[i]                      (in 64 bits)
 *   ids, weights of the k chosen experts: as rsllm_hip_moe_route_dev gives them for
 *           the logits l (in 64 bits), score, bias, groups, renormalise and scale
 *   h_e   = silu(min(gate_e x, c)) * clamp(up_e x, -c, c)  (no clamp when c <= 1e-6)
 *   out   = sum_i weights_i down_{ids_i} h_{ids_i} + sum_j down_{n_expert + j} h_{n_expert + j}
 * the second sum over the n_shared experts that every token takes, which stand behind
 * the others in the weights. Experts of weight 0 are skipped. x and h are not
 * quantised: the products take x exactly (f32 x below 2^-125: to 2^-149), and h rounded
 * to 24 bits (f32 outputs) or 16 (f16 and bf16 ones), and sum in f32; a row's sum that comes
 * out infinite or NaN is made again in 64 bits and rounded to f32. A token with a non-finite value in x gets a row
 * of NaN (its ids and weights by the rules above, whatever its logits became).
 * The layer: `router` [n_expert x n_embd] of dtype_router (F32, F16 or BF16; router_len
 * elements), `bias` n_expert values or NULL (bias_len 0); gate, up: (n_expert +
 * n_shared) * n_ff rows of n_embd codes (gate_up_len bytes each, their scales
 * gate_up_scales_len); down: (n_expert + n_shared) * n_embd rows of n_ff codes. Rows as
 * the quantiser lays them out.
 * out: n_tok rows of n_embd values of dtype_out (F32, F16 or BF16), overwritten,
 * out_stride elements apart; x: rows of dtype_x likewise; ids, weights [n_tok x k] are
 * written. out must not overlap x. `work`: rsllm_hip_moe_mxfp4_work_bytes(layer, n_tok)
 * bytes of the caller's (0 for a NULL layer and for sizes or an n_tok outside the ranges
 * below), 256-byte aligned, used by this call alone until it has run: calls that may
 * overlap, and graphs that may replay at once, get one each. What it holds before does not
 * matter. The struct
 * is read during the call only; what it points to until the work is done.
 * Errors: UNIMPLEMENTED for another dtype; INVALID_ARGUMENT for n_tok above 32, n_embd
 * or n_ff 0 or above 65536, n_expert 0 or above 1024, n_shared above 8, k 0 or above
 * min(32, experts of topk_group groups), n_group that does not divide n_expert,
 * topk_group outside 1..n_group, group_top other than 1 or 2, an unknown score, a
 * scale that is not finite, a NaN clamp, NULL or misaligned pointers; SHAPE_MISMATCH for a stride
 * below its row, lengths below or other than those above, work_len below work_bytes. */
typedef struct rsllm_hip_moe_mxfp4 {
    const void *router;
    size_t router_len;
    const float *bias;
    size_t bias_len;
    const uint8_t *gate, *up;
    size_t gate_up_len;
    const uint8_t *gate_scales, *up_scales;
    size_t gate_up_scales_len;
    const uint8_t *down;
    size_t down_len;
    const uint8_t *down_scales;
    size_t down_scales_len;
    size_t n_embd, n_ff, n_expert, n_shared, k, n_group, topk_group, group_top;
    uint32_t dtype_router;
    uint32_t score; /* RSLLM_HIP_SCORE_* */
    int32_t renormalise;
    float scale;
    float clamp;
} rsllm_hip_moe_mxfp4;
size_t rsllm_hip_moe_mxfp4_work_bytes(const rsllm_hip_moe_mxfp4 *layer, size_t n_tok);
int rsllm_hip_moe_mxfp4_dev(const rsllm_hip_moe_mxfp4 *layer, void *out, size_t out_len,
                            size_t out_stride, int32_t *ids, float *weights, size_t ids_len,
                            const void *x, size_t x_len, size_t x_stride, uint8_t *work,
                            size_t work_len, size_t n_tok, uint32_t dtype_x, uint32_t dtype_out,
                            rsllm_hip_stream_t stream);

/* ---- token log-probabilities --------------------------------------------------
 * No reference counterpart among its compute ops: what a caller reads from the
 * vocabulary projection's product (matmul_weight_f32 or one of the others)
 * beside the token it samples. logits: n_tok rows of `vocab` values of `dtype`
 * (F32, F16 or BF16), logits_stride elements apart. Per row, with m = max l,
 * S = sum exp(l - m), p = exp(l - m) / S:
 *   logprob  = l[token] - m - log S      tokens[t] the given token's id
 *   rank     = 1 + the number of logits above the given token's
 *   entropy  = -sum p log p (natural log)
 *   top_ids, top_logprobs [n_tok x n_top]: the n_top largest logits, in falling
 *              order, equal ones in rising order of id, and their log-
 *              probabilities
 * A logit of -inf (a masked token) has probability 0, adds nothing to the
 * entropy and is never listed; places that stay empty get id -1 and -inf. A row
 * of nothing but -inf: logprob -inf, entropy 0. +inf counts as the limit: the
 * +inf logits share the row evenly. A NaN anywhere in a row makes its logprob,
 * entropy and listed log-probabilities NaN (a NaN logit is not listed or counted).
 * A token id outside [0, vocab) gives logprob NaN and rank 0, a token whose
 * logit is NaN rank 0. The sums are f32, so log-probabilities and entropies are
 * off by a few 2^-24 of 1 beside their own rounding: a token whose p is within
 * 2^-24 of 1 gets logprob 0.
 * tokens (with tokens_len 0) may be NULL: logprob and rank are then not written
 * and may be NULL; rank and entropy may be NULL; n_top 0 takes NULL lists.
 * out_len counts logprob, rank and entropy each. `work`:
 * rsllm_hip_token_logprobs_work_bytes(n_tok, vocab, n_top) bytes of the
 * caller's, 256-byte aligned, used by this call alone until it has run. They do
 * not rise with n_tok (many rows need none): ask for each n_tok that is used.
 * Errors: UNIMPLEMENTED for another dtype; INVALID_ARGUMENT for vocab 0 or above
 * 2^31 - 1, n_top above min(64, vocab), NULL or misaligned pointers;
 * SHAPE_MISMATCH for n_tok above 8388607 (what a launch holds), logits_stride < vocab, logits_len < (n_tok - 1) *
 * logits_stride + vocab, tokens_len other than 0 and n_tok, out_len != n_tok,
 * top_len != n_tok * n_top, work_len below work_bytes. */
size_t rsllm_hip_token_logprobs_work_bytes(size_t n_tok, size_t vocab, size_t n_top);
int rsllm_hip_token_logprobs_dev(float *logprob, float *entropy, int32_t *rank, size_t out_len,
                                 int32_t *top_ids, float *top_logprobs, size_t top_len,
                                 const void *logits, size_t logits_len, size_t logits_stride,
                                 const int32_t *tokens, size_t tokens_len, uint8_t *work,
                                 size_t work_len, size_t n_tok, size_t vocab, size_t n_top,
                                 uint32_t dtype, rsllm_hip_stream_t stream);

/* ---- dequantisation ------------------------------------------------------ */

/* dequant_to_f32 (rsllm-gguf/src/dequant/mod.rs:69-85): decode `src` (GGUF
 * bytes) into dst[dst_len]. Bit-exact with the reference on every arm of its
 * dispatch: F32, F16, BF16, Q4_0, Q4_1, Q4_K, Q5_K, Q6_K, Q8_0, Q2_K, Q8_K,
 * IQ2_XXS; any other dtype is UNSUPPORTED_DEQUANT. Size rule of
 * q4_k.rs:36-49 (and siblings). */
int rsllm_hip_dequant_to_f32(uint32_t dtype, const uint8_t *src, size_t src_len, float *dst,
                             size_t dst_len);
int rsllm_hip_dequant_to_f32_dev(uint32_t dtype, const uint8_t *src, size_t src_len, float *dst,
                                 size_t dst_len, rsllm_hip_stream_t stream);

/* The measurement aids bench.py uses (a streaming read, the matrix-core
 * issue rate) are exported by the same library and declared in
 * rsllm_hip_probe.h: they are not part of the drop-in boundary. */

#ifdef __cplusplus
}
#endif
#endif /* RSLLM_HIP_H */
