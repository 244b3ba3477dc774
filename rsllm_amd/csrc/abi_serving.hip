// C-ABI entry points either side of the matmuls: expert routing, the int8
// product with scales per token and channel, token log-probabilities. Device
// pointers only; nothing is allocated and no library workspace is used (what a
// call needs is the caller's `work`), so every call can be captured.
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>

#include "../../include/rsllm_hip.h"
#include "abi_checks.h"
#include "kernels.h"

using namespace rsllm_hip;
using namespace rsllm_hip::abi;

namespace {

constexpr size_t kI8MaxIn = 131071;  // 128 * 128 * 131071 < 2^31

// The caller's work of an int8 product: codes, then scales.
struct I8Work {
    size_t codes = 0, total = 0;
};
bool i8_work(size_t n_tok, size_t in_dim, size_t out_dim, I8Work *w) {
    if (!counts_ok(n_tok) || !counts_ok(out_dim) || in_dim == 0 || in_dim > kI8MaxIn) return false;
    w->codes = round256(n_tok * i8_row_bytes(in_dim));
    w->total = w->codes + round256(n_tok * sizeof(float));
    return true;
}

// Checks of the product that both forms share.
int check_i8(const void *out, size_t out_len, size_t out_stride, const int8_t *w, size_t w_len,
             const float *wscale, size_t wscale_len, const float *bias, size_t bias_len,
             const uint8_t *work, size_t n_tok, size_t in_dim, size_t out_dim, uint32_t dtype_out) {
    if (!float_type(dtype_out))
        return set_error(RSLLM_HIP_ERR_UNIMPLEMENTED, "matmul_int8: output dtype not implemented");
    if (in_dim == 0 || in_dim > kI8MaxIn)
        return invalid("matmul_int8: in_dim must be 1..131071 (32-bit sums)");
    if (out_dim == 0) return invalid("matmul_int8: out_dim must be non-zero");
    if (!counts_ok(n_tok) || !counts_ok(out_dim))
        return mismatch("matmul_int8: n_tok and out_dim must be at most 8388607");
    if (!product_is(out_dim, i8_row_bytes(in_dim), w_len))
        return mismatch("matmul_int8: weights must be out_dim * int8_row_bytes(in_dim)");
    if (wscale_len != out_dim) return mismatch("matmul_int8: wscale must be out_dim");
    if (bias_len != 0 && bias_len != out_dim)
        return mismatch("matmul_int8: bias must be out_dim or absent");
    if (out_stride < out_dim || !span_ok(n_tok, out_dim, out_stride, out_len))
        return mismatch("matmul_int8: out must hold n_tok rows of out_dim, out_stride apart");
    if (!w || !wscale || (n_tok && !out) || (bias_len && !bias))
        return invalid("NULL pointer with a nonzero length");
    if (!aligned(w, 16) || !aligned(wscale, 4) || !aligned(bias, 4) || !aligned(work, 256) ||
        !aligned(out, elem_bytes(dtype_out)))
        return invalid("matmul_int8: misaligned pointer");
    return RSLLM_HIP_OK;
}

int check_x(const char *what, const void *x, size_t x_len, size_t x_stride, size_t n_tok,
            size_t in_dim, uint32_t dtype) {
    if (!float_type(dtype)) return set_error(RSLLM_HIP_ERR_UNIMPLEMENTED, "int8: x dtype not implemented");
    if (x_stride < in_dim || !span_ok(n_tok, in_dim, x_stride, x_len)) return mismatch(what);
    if (n_tok && !x) return invalid("NULL pointer with a nonzero length");
    if (!aligned(x, elem_bytes(dtype))) return invalid("int8: misaligned x");
    return RSLLM_HIP_OK;
}

}  // namespace

extern "C" {

int rsllm_hip_moe_route_dev(int32_t *ids, float *weights, size_t ids_len, const void *logits,
                            size_t logits_len, size_t logits_stride, const float *bias,
                            size_t bias_len, size_t n_tok, size_t n_expert, size_t k,
                            size_t n_group, size_t topk_group, size_t group_top, uint32_t score,
                            int renormalise, float scale, uint32_t dtype,
                            rsllm_hip_stream_t stream) {
    if (!float_type(dtype))
        return set_error(RSLLM_HIP_ERR_UNIMPLEMENTED, "moe_route: dtype not implemented");
    if (score > RSLLM_HIP_SCORE_SQRT_SOFTPLUS) return invalid("moe_route: unknown score");
    if (n_expert == 0 || n_expert > 16384) return invalid("moe_route: n_expert must be 1..16384");
    if (n_group == 0 || n_group > 1024 || n_expert % n_group != 0)
        return invalid("moe_route: n_group must divide n_expert, at most 1024");
    if (topk_group == 0 || topk_group > n_group)
        return invalid("moe_route: topk_group must be 1..n_group");
    if (group_top != 1 && group_top != 2) return invalid("moe_route: group_top must be 1 or 2");
    if (k == 0 || k > 64 || k > topk_group * (n_expert / n_group))
        return invalid("moe_route: k must be 1..min(64, experts of topk_group groups)");
    if (!std::isfinite(scale)) return invalid("moe_route: scale must be finite");
    if (!counts_ok(n_tok)) return mismatch("moe_route: n_tok must be at most 8388607");
    if (logits_stride < n_expert || !span_ok(n_tok, n_expert, logits_stride, logits_len))
        return mismatch("moe_route: logits must hold n_tok rows of n_expert, logits_stride apart");
    if (bias_len != 0 && bias_len != n_expert)
        return mismatch("moe_route: bias must be n_expert or absent");
    if (!product_is(n_tok, k, ids_len)) return mismatch("moe_route: ids must be n_tok * k");
    if ((n_tok && (!logits || !ids || !weights)) || (bias_len && !bias))
        return invalid("NULL pointer with a nonzero length");
    if (!aligned(logits, elem_bytes(dtype)) || !aligned(ids, 4) || !aligned(weights, 4) ||
        !aligned(bias, 4))
        return invalid("moe_route: misaligned pointer");
    if (n_tok == 0) return abi::ok_status();
    if (const int rc = abi::make_device_current()) return rc;
    const RouteArgs a{logits, logits_stride, bias_len ? bias : nullptr, ids, weights, (int)n_expert,
                      (int)k, (int)n_group, (int)topk_group, (int)group_top, (int)score,
                      renormalise != 0, scale, dtype};
    HIP_TRY(launch_moe_route(a, (int)n_tok, (hipStream_t)stream), "moe_route");
    return abi::ok_status();
}

size_t rsllm_hip_int8_row_bytes(size_t in_dim) {
    return in_dim == 0 || in_dim > kI8MaxIn ? 0 : i8_row_bytes(in_dim);
}

size_t rsllm_hip_int8_work_bytes(size_t n_tok, size_t in_dim, size_t out_dim) {
    I8Work w;
    return i8_work(n_tok, in_dim, out_dim, &w) ? w.total : 0;
}

int rsllm_hip_quantize_int8_dev(const void *x, size_t x_len, size_t x_stride, int8_t *xq,
                                size_t xq_len, float *scale, size_t scale_len, size_t n_tok,
                                size_t in_dim, uint32_t dtype, rsllm_hip_stream_t stream) {
    if (in_dim == 0 || in_dim > kI8MaxIn)
        return invalid("quantize_int8: in_dim must be 1..131071");
    if (!counts_ok(n_tok)) return mismatch("quantize_int8: n_tok must be at most 8388607");
    if (const int rc = check_x("quantize_int8: x must hold n_tok rows of in_dim, x_stride apart", x,
                               x_len, x_stride, n_tok, in_dim, dtype))
        return rc;
    if (!product_is(n_tok, i8_row_bytes(in_dim), xq_len))
        return mismatch("quantize_int8: xq must be n_tok * int8_row_bytes(in_dim)");
    if (scale_len != n_tok) return mismatch("quantize_int8: scale must be n_tok");
    if (n_tok && (!xq || !scale)) return invalid("NULL pointer with a nonzero length");
    if (!aligned(xq, 16) || !aligned(scale, 4)) return invalid("quantize_int8: misaligned pointer");
    if (n_tok == 0) return abi::ok_status();
    if (const int rc = abi::make_device_current()) return rc;
    HIP_TRY(launch_i8_quantize(x, x_stride, xq, scale, (int)n_tok, (int)in_dim, dtype,
                               (hipStream_t)stream),
            "quantize_int8");
    return abi::ok_status();
}

int rsllm_hip_matmul_int8_prequant_dev(void *out, size_t out_len, size_t out_stride,
                                       const int8_t *weights, size_t weights_len,
                                       const float *wscale, size_t wscale_len, const float *bias,
                                       size_t bias_len, const int8_t *xq, size_t xq_len,
                                       const float *xscale, size_t xscale_len, uint8_t *work,
                                       size_t work_len, size_t n_tok, size_t in_dim,
                                       size_t out_dim, uint32_t dtype_out,
                                       rsllm_hip_stream_t stream) {
    (void)work_len;  // (these products leave nothing between launches)
    if (const int rc = check_i8(out, out_len, out_stride, weights, weights_len, wscale, wscale_len,
                                bias, bias_len, work, n_tok, in_dim, out_dim, dtype_out))
        return rc;
    if (!product_is(n_tok, i8_row_bytes(in_dim), xq_len))
        return mismatch("matmul_int8: xq must be n_tok * int8_row_bytes(in_dim)");
    if (xscale_len != n_tok) return mismatch("matmul_int8: xscale must be n_tok");
    if (n_tok && (!xq || !xscale)) return invalid("NULL pointer with a nonzero length");
    if (!aligned(xq, 16) || !aligned(xscale, 4)) return invalid("matmul_int8: misaligned pointer");
    if (n_tok == 0) return abi::ok_status();
    if (const int rc = abi::make_device_current()) return rc;
    const I8Args a{weights, xq, wscale, xscale, bias_len ? bias : nullptr, out, out_stride,
                   (int)n_tok, (int)out_dim, (int)i8_row_bytes(in_dim), dtype_out};
    HIP_TRY(launch_i8_matmul(a, (hipStream_t)stream), "matmul_int8");
    return abi::ok_status();
}

int rsllm_hip_matmul_int8_dev(void *out, size_t out_len, size_t out_stride, const int8_t *weights,
                              size_t weights_len, const float *wscale, size_t wscale_len,
                              const float *bias, size_t bias_len, const void *x, size_t x_len,
                              size_t x_stride, uint8_t *work, size_t work_len, size_t n_tok,
                              size_t in_dim, size_t out_dim, uint32_t dtype_x, uint32_t dtype_out,
                              rsllm_hip_stream_t stream) {
    if (const int rc = check_i8(out, out_len, out_stride, weights, weights_len, wscale, wscale_len,
                                bias, bias_len, work, n_tok, in_dim, out_dim, dtype_out))
        return rc;
    I8Work parts;
    (void)i8_work(n_tok, in_dim, out_dim, &parts);
    if (work_len < parts.total) return mismatch("matmul_int8: work must be int8_work_bytes");
    if (parts.total && !work) return invalid("NULL pointer with a nonzero length");
    if (const int rc = check_x("matmul_int8: x must hold n_tok rows of in_dim, x_stride apart", x,
                               x_len, x_stride, n_tok, in_dim, dtype_x))
        return rc;
    if (n_tok == 0) return abi::ok_status();
    if (const int rc = abi::make_device_current()) return rc;
    int8_t *xq = reinterpret_cast<int8_t *>(work);
    float *xscale = reinterpret_cast<float *>(work + parts.codes);
    const I8Args a{weights, xq, wscale, xscale, bias_len ? bias : nullptr, out, out_stride,
                   (int)n_tok, (int)out_dim, (int)i8_row_bytes(in_dim), dtype_out};
    if (n_tok == 1 && i8_one_supported((int)in_dim)) {
        HIP_TRY(launch_i8_one(a, x, (int)in_dim, dtype_x, (hipStream_t)stream), "matmul_int8");
        return abi::ok_status();
    }
    HIP_TRY(launch_i8_quantize(x, x_stride, xq, xscale, (int)n_tok, (int)in_dim, dtype_x,
                               (hipStream_t)stream),
            "quantize_int8");
    HIP_TRY(launch_i8_matmul(a, (hipStream_t)stream), "matmul_int8");
    return abi::ok_status();
}

size_t rsllm_hip_token_logprobs_work_bytes(size_t n_tok, size_t vocab, size_t n_top) {
    if (!counts_ok(n_tok) || vocab > (size_t)INT_MAX || vocab == 0 || n_top > 64 || n_top > vocab) return 0;
    return logprobs_scratch_bytes((int)n_tok, (int)vocab, (int)n_top);
}

int rsllm_hip_token_logprobs_dev(float *logprob, float *entropy, int32_t *rank, size_t out_len,
                                 int32_t *top_ids, float *top_logprobs, size_t top_len,
                                 const void *logits, size_t logits_len, size_t logits_stride,
                                 const int32_t *tokens, size_t tokens_len, uint8_t *work,
                                 size_t work_len, size_t n_tok, size_t vocab, size_t n_top,
                                 uint32_t dtype, rsllm_hip_stream_t stream) {
    if (!float_type(dtype))
        return set_error(RSLLM_HIP_ERR_UNIMPLEMENTED, "token_logprobs: dtype not implemented");
    if (vocab == 0 || vocab > (size_t)INT_MAX) return invalid("token_logprobs: vocab must be 1..2^31-1");
    if (n_top > 64 || n_top > vocab) return invalid("token_logprobs: n_top must be at most min(64, vocab)");
    if (!counts_ok(n_tok)) return mismatch("token_logprobs: n_tok must be at most 8388607");
    if (logits_stride < vocab || !span_ok(n_tok, vocab, logits_stride, logits_len))
        return mismatch("token_logprobs: logits must hold n_tok rows of vocab, logits_stride apart");
    if (tokens_len != 0 && tokens_len != n_tok)
        return mismatch("token_logprobs: tokens must be n_tok or absent");
    if (out_len != n_tok) return mismatch("token_logprobs: outputs must be n_tok");
    if (!product_is(n_tok, n_top, top_len)) return mismatch("token_logprobs: lists must be n_tok * n_top");
    const size_t need = rsllm_hip_token_logprobs_work_bytes(n_tok, vocab, n_top);
    if (work_len < need) return mismatch("token_logprobs: work must be token_logprobs_work_bytes");
    if ((n_tok && !logits) || (tokens_len && (!tokens || !logprob)) ||
        (top_len && (!top_ids || !top_logprobs)) || (need && !work))
        return invalid("NULL pointer with a nonzero length");
    if (!aligned(logits, elem_bytes(dtype)) || !aligned(tokens, 4) || !aligned(logprob, 4) ||
        !aligned(entropy, 4) || !aligned(rank, 4) || !aligned(top_ids, 4) ||
        !aligned(top_logprobs, 4) || !aligned(work, 256))
        return invalid("token_logprobs: misaligned pointer");
    if (n_tok == 0) return abi::ok_status();
    if (const int rc = abi::make_device_current()) return rc;
    const LogprobArgs a{logits, logits_stride, tokens_len ? tokens : nullptr, logprob, entropy, rank,
                        top_ids, top_logprobs, (int)vocab, (int)n_top, dtype};
    HIP_TRY(launch_logprobs(a, work, (int)n_tok, (hipStream_t)stream), "token_logprobs");
    return abi::ok_status();
}

}  // extern "C"
