// C-ABI entry points of the 4-bit floating-point calls: quantising, decoding, the
// product, the mixture-of-experts layer. Device pointers only; nothing is allocated and
// no library workspace is used (what a call needs is the caller's `work`), so every call
// can be captured.
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/rsllm_hip.h"
#include "abi_checks.h"
#include "kernels.h"

using namespace rsllm_hip;
using namespace rsllm_hip::abi;

namespace {

constexpr size_t kMxMaxIn = (size_t)1 << 20;
bool in_ok(size_t in_dim) { return in_dim != 0 && in_dim <= kMxMaxIn; }

// The caller's work of a product from floats: codes, then scales.
struct MxWork {
    size_t codes = 0, total = 0;
};
bool mx_work(size_t n_tok, size_t in_dim, size_t out_dim, MxWork *w) {
    if (!counts_ok(n_tok) || !counts_ok(out_dim) || !in_ok(in_dim)) return false;
    w->codes = round256(n_tok * mx_row_bytes(in_dim));
    w->total = w->codes + round256(n_tok * mx_scale_bytes(in_dim));
    return true;
}

// Rows of floats: their type, stride, length and alignment.
int check_rows(const char *what, const void *p, size_t len, size_t stride, size_t rows, size_t row,
               uint32_t dtype) {
    if (!float_type(dtype)) return set_error(RSLLM_HIP_ERR_UNIMPLEMENTED, "mxfp4: dtype not implemented");
    if (stride < row || !span_ok(rows, row, stride, len)) return mismatch(what);
    if (rows && !p) return invalid("NULL pointer with a nonzero length");
    if (!aligned(p, elem_bytes(dtype))) return invalid("mxfp4: misaligned pointer");
    return RSLLM_HIP_OK;
}

// Rows of codes and their scales.
int check_codes(const char *what, const uint8_t *codes, size_t codes_len, const uint8_t *scales,
                size_t scales_len, size_t rows, size_t in_dim) {
    if (!product_is(rows, mx_row_bytes(in_dim), codes_len) ||
        !product_is(rows, mx_scale_bytes(in_dim), scales_len))
        return mismatch(what);
    if (rows && (!codes || !scales)) return invalid("NULL pointer with a nonzero length");
    if (!aligned(codes, 16) || !aligned(scales, 16)) return invalid("mxfp4: misaligned pointer");
    return RSLLM_HIP_OK;
}

// Checks of the product that both forms share.
int check_product(const void *out, size_t out_len, size_t out_stride, const uint8_t *w, size_t w_len,
                  const uint8_t *ws, size_t ws_len, const float *bias, size_t bias_len,
                  const uint8_t *work, size_t n_tok, size_t in_dim, size_t out_dim,
                  uint32_t dtype_out) {
    if (!in_ok(in_dim)) return invalid("matmul_mxfp4: in_dim must be 1..1048576");
    if (out_dim == 0) return invalid("matmul_mxfp4: out_dim must be non-zero");
    if (!counts_ok(n_tok) || !counts_ok(out_dim))
        return mismatch("matmul_mxfp4: n_tok and out_dim must be at most 8388607");
    if (const int rc = check_codes("matmul_mxfp4: weights must be out_dim rows of codes and scales", w,
                                   w_len, ws, ws_len, out_dim, in_dim))
        return rc;
    if (bias_len != 0 && bias_len != out_dim)
        return mismatch("matmul_mxfp4: bias must be out_dim or absent");
    if (bias_len && !bias) return invalid("NULL pointer with a nonzero length");
    if (const int rc = check_rows("matmul_mxfp4: out must hold n_tok rows of out_dim, out_stride apart",
                                  out, out_len, out_stride, n_tok, out_dim, dtype_out))
        return rc;
    if (!aligned(bias, 4) || !aligned(work, 256)) return invalid("mxfp4: misaligned pointer");
    return RSLLM_HIP_OK;
}

// A layer's own numbers and matrices (its n_tok apart).
bool layer_sizes_ok(const rsllm_hip_moe_mxfp4 &l) {
    return l.n_embd >= 1 && l.n_embd <= 65536 && l.n_ff >= 1 && l.n_ff <= 65536 && l.n_expert >= 1 &&
           l.n_expert <= 1024 && l.n_shared <= 8 && l.k >= 1 && l.k <= 32;
}
// What is wrong with its groups and k (of sizes that are right), or null.
const char *groups_refused(const rsllm_hip_moe_mxfp4 &l) {
    if (l.n_group == 0 || l.n_expert % l.n_group != 0) return "moe_mxfp4: n_group must divide n_expert";
    if (l.topk_group == 0 || l.topk_group > l.n_group) return "moe_mxfp4: topk_group must be 1..n_group";
    if (l.group_top != 1 && l.group_top != 2) return "moe_mxfp4: group_top must be 1 or 2";
    if (l.k > l.topk_group * (l.n_expert / l.n_group))
        return "moe_mxfp4: k must be at most the experts of topk_group groups";
    return nullptr;
}
int check_layer(const rsllm_hip_moe_mxfp4 &l) {
    if (!float_type(l.dtype_router))
        return set_error(RSLLM_HIP_ERR_UNIMPLEMENTED, "moe_mxfp4: router dtype not implemented");
    if (l.score > RSLLM_HIP_SCORE_SQRT_SOFTPLUS) return invalid("moe_mxfp4: unknown score");
    if (!layer_sizes_ok(l))
        return invalid("moe_mxfp4: n_embd and n_ff must be 1..65536, n_expert 1..1024, n_shared at "
                       "most 8, k 1..32");
    if (const char *why = groups_refused(l)) return invalid(why);
    if (!std::isfinite(l.scale)) return invalid("moe_mxfp4: scale must be finite");
    if (std::isnan(l.clamp)) return invalid("moe_mxfp4: clamp must be a number");
    if (!product_is(l.n_expert, l.n_embd, l.router_len))
        return mismatch("moe_mxfp4: router must be n_expert * n_embd");
    if (l.bias_len != 0 && l.bias_len != l.n_expert)
        return mismatch("moe_mxfp4: bias must be n_expert or absent");
    if (!l.router || (l.bias_len && !l.bias)) return invalid("NULL pointer with a nonzero length");
    if (!aligned(l.router, elem_bytes(l.dtype_router)) || !aligned(l.bias, 4))
        return invalid("moe_mxfp4: misaligned pointer");
    const size_t all = l.n_expert + l.n_shared;
    for (int up = 0; up < 2; up++)
        if (const int rc = check_codes("moe_mxfp4: gate and up must be (n_expert + n_shared) * n_ff rows",
                                       up ? l.up : l.gate, l.gate_up_len, up ? l.up_scales : l.gate_scales,
                                       l.gate_up_scales_len, all * l.n_ff, l.n_embd))
            return rc;
    return check_codes("moe_mxfp4: down must be (n_expert + n_shared) * n_embd rows", l.down,
                       l.down_len, l.down_scales, l.down_scales_len, all * l.n_embd, l.n_ff);
}

}  // namespace

extern "C" {

size_t rsllm_hip_mxfp4_row_bytes(size_t in_dim) { return in_ok(in_dim) ? mx_row_bytes(in_dim) : 0; }

size_t rsllm_hip_mxfp4_scale_bytes(size_t in_dim) { return in_ok(in_dim) ? mx_scale_bytes(in_dim) : 0; }

size_t rsllm_hip_mxfp4_work_bytes(size_t n_tok, size_t in_dim, size_t out_dim) {
    MxWork w;
    return out_dim != 0 && mx_work(n_tok, in_dim, out_dim, &w) ? w.total : 0;
}

int rsllm_hip_quantize_mxfp4_dev(const void *x, size_t x_len, size_t x_stride, uint8_t *codes,
                                 size_t codes_len, uint8_t *scales, size_t scales_len,
                                 size_t n_rows, size_t in_dim, uint32_t dtype,
                                 rsllm_hip_stream_t stream) {
    if (!in_ok(in_dim)) return invalid("quantize_mxfp4: in_dim must be 1..1048576");
    if (!counts_ok(n_rows)) return mismatch("quantize_mxfp4: n_rows must be at most 8388607");
    if (const int rc = check_rows("quantize_mxfp4: x must hold n_rows rows of in_dim, x_stride apart", x,
                                  x_len, x_stride, n_rows, in_dim, dtype))
        return rc;
    if (const int rc = check_codes("quantize_mxfp4: codes and scales must be n_rows rows", codes,
                                   codes_len, scales, scales_len, n_rows, in_dim))
        return rc;
    if (n_rows == 0) return ok_status();
    if (const int rc = make_device_current()) return rc;
    HIP_TRY(launch_mx_quantize(x, x_stride, codes, scales, (int)n_rows, (int)in_dim, dtype,
                               (hipStream_t)stream),
            "quantize_mxfp4");
    return ok_status();
}

int rsllm_hip_dequantize_mxfp4_dev(const uint8_t *codes, size_t codes_len, const uint8_t *scales,
                                   size_t scales_len, void *out, size_t out_len,
                                   size_t out_stride, size_t n_rows, size_t in_dim, uint32_t dtype,
                                   rsllm_hip_stream_t stream) {
    if (!in_ok(in_dim)) return invalid("dequantize_mxfp4: in_dim must be 1..1048576");
    if (!counts_ok(n_rows)) return mismatch("dequantize_mxfp4: n_rows must be at most 8388607");
    if (const int rc = check_codes("dequantize_mxfp4: codes and scales must be n_rows rows", codes,
                                   codes_len, scales, scales_len, n_rows, in_dim))
        return rc;
    if (const int rc = check_rows("dequantize_mxfp4: out must hold n_rows rows of in_dim, out_stride apart",
                                  out, out_len, out_stride, n_rows, in_dim, dtype))
        return rc;
    if (n_rows == 0) return ok_status();
    if (const int rc = make_device_current()) return rc;
    HIP_TRY(launch_mx_dequantize(codes, scales, out, out_stride, (int)n_rows, (int)in_dim, dtype,
                                 (hipStream_t)stream),
            "dequantize_mxfp4");
    return ok_status();
}

int rsllm_hip_matmul_mxfp4_prequant_dev(void *out, size_t out_len, size_t out_stride,
                                        const uint8_t *weights, size_t weights_len,
                                        const uint8_t *wscales, size_t wscales_len,
                                        const float *bias, size_t bias_len, const uint8_t *xcodes,
                                        size_t xcodes_len, const uint8_t *xscales,
                                        size_t xscales_len, uint8_t *work, size_t work_len,
                                        size_t n_tok, size_t in_dim, size_t out_dim,
                                        uint32_t dtype_out, rsllm_hip_stream_t stream) {
    if (const int rc = check_product(out, out_len, out_stride, weights, weights_len, wscales, wscales_len,
                                     bias, bias_len, work, n_tok, in_dim, out_dim, dtype_out))
        return rc;
    if (const int rc = check_codes("matmul_mxfp4: xcodes and xscales must be n_tok rows", xcodes,
                                   xcodes_len, xscales, xscales_len, n_tok, in_dim))
        return rc;
    MxWork parts;
    (void)mx_work(n_tok, in_dim, out_dim, &parts);
    if (work_len < parts.total) return mismatch("matmul_mxfp4: work must be mxfp4_work_bytes");
    if (parts.total && !work) return invalid("NULL pointer with a nonzero length");
    if (n_tok == 0) return ok_status();
    if (const int rc = make_device_current()) return rc;
    const MxArgs a{weights, wscales, xcodes, xscales, bias_len ? bias : nullptr, out, out_stride,
                   (int)n_tok, (int)out_dim, (int)in_dim, dtype_out};
    HIP_TRY(launch_mx_matmul(a, (hipStream_t)stream), "matmul_mxfp4");
    return ok_status();
}

int rsllm_hip_matmul_mxfp4_dev(void *out, size_t out_len, size_t out_stride,
                               const uint8_t *weights, size_t weights_len, const uint8_t *wscales,
                               size_t wscales_len, const float *bias, size_t bias_len,
                               const void *x, size_t x_len, size_t x_stride, uint8_t *work,
                               size_t work_len, size_t n_tok, size_t in_dim, size_t out_dim,
                               uint32_t dtype_x, uint32_t dtype_out, rsllm_hip_stream_t stream) {
    if (const int rc = check_product(out, out_len, out_stride, weights, weights_len, wscales, wscales_len,
                                     bias, bias_len, work, n_tok, in_dim, out_dim, dtype_out))
        return rc;
    if (const int rc = check_rows("matmul_mxfp4: x must hold n_tok rows of in_dim, x_stride apart", x,
                                  x_len, x_stride, n_tok, in_dim, dtype_x))
        return rc;
    MxWork parts;
    (void)mx_work(n_tok, in_dim, out_dim, &parts);
    if (work_len < parts.total) return mismatch("matmul_mxfp4: work must be mxfp4_work_bytes");
    if (parts.total && !work) return invalid("NULL pointer with a nonzero length");
    if (n_tok == 0) return ok_status();
    if (const int rc = make_device_current()) return rc;
    const MxArgs a{weights, wscales, nullptr, nullptr, bias_len ? bias : nullptr, out, out_stride,
                   (int)n_tok, (int)out_dim, (int)in_dim, dtype_out};
    HIP_TRY(launch_mx_matmul_float(a, x, x_stride, dtype_x, work, work + parts.codes, (hipStream_t)stream),
            "matmul_mxfp4");
    return ok_status();
}

size_t rsllm_hip_moe_mxfp4_work_bytes(const rsllm_hip_moe_mxfp4 *layer, size_t n_tok) {
    if (!layer || n_tok > (size_t)kMoeMaxTok || !layer_sizes_ok(*layer)) return 0;
    if (groups_refused(*layer)) return 0;
    return moe_layer_work_bytes((int)n_tok, (int)layer->n_embd, (int)layer->n_ff, (int)layer->n_expert,
                                (int)layer->k, (int)layer->n_shared);
}

int rsllm_hip_moe_mxfp4_dev(const rsllm_hip_moe_mxfp4 *layer, void *out, size_t out_len,
                            size_t out_stride, int32_t *ids, float *weights, size_t ids_len,
                            const void *x, size_t x_len, size_t x_stride, uint8_t *work,
                            size_t work_len, size_t n_tok, uint32_t dtype_x, uint32_t dtype_out,
                            rsllm_hip_stream_t stream) {
    if (!layer) return invalid("moe_mxfp4: NULL layer");
    const rsllm_hip_moe_mxfp4 &l = *layer;
    if (const int rc = check_layer(l)) return rc;
    if (n_tok > (size_t)kMoeMaxTok) return invalid("moe_mxfp4: n_tok must be at most 32");
    if (const int rc = check_rows("moe_mxfp4: out must hold n_tok rows of n_embd, out_stride apart", out,
                                  out_len, out_stride, n_tok, l.n_embd, dtype_out))
        return rc;
    if (const int rc = check_rows("moe_mxfp4: x must hold n_tok rows of n_embd, x_stride apart", x, x_len,
                                  x_stride, n_tok, l.n_embd, dtype_x))
        return rc;
    if (!product_is(n_tok, l.k, ids_len)) return mismatch("moe_mxfp4: ids must be n_tok * k");
    const size_t need = rsllm_hip_moe_mxfp4_work_bytes(layer, n_tok);
    if (work_len < need) return mismatch("moe_mxfp4: work must be moe_mxfp4_work_bytes");
    if (n_tok && (!ids || !weights || !work)) return invalid("NULL pointer with a nonzero length");
    if (!aligned(ids, 4) || !aligned(weights, 4) || !aligned(work, 256))
        return invalid("moe_mxfp4: misaligned pointer");
    if (n_tok == 0) return ok_status();
    if (const int rc = make_device_current()) return rc;
    MoeLayerArgs a{};
    a.router = l.router;
    a.bias = l.bias_len ? l.bias : nullptr;
    a.gate = l.gate;
    a.up = l.up;
    a.down = l.down;
    a.gate_s = l.gate_scales;
    a.up_s = l.up_scales;
    a.down_s = l.down_scales;
    a.n_embd = (int)l.n_embd;
    a.n_ff = (int)l.n_ff;
    a.n_expert = (int)l.n_expert;
    a.n_shared = (int)l.n_shared;
    a.k = (int)l.k;
    a.n_group = (int)l.n_group;
    a.topk_group = (int)l.topk_group;
    a.group_top = (int)l.group_top;
    a.score = (int)l.score;
    a.renormalise = l.renormalise != 0;
    a.scale = l.scale;
    a.clamp = l.clamp;
    a.dtype_router = l.dtype_router;
    a.dtype_x = dtype_x;
    a.dtype_out = dtype_out;
    a.x = x;
    a.x_stride = x_stride;
    a.out = out;
    a.out_stride = out_stride;
    a.ids = ids;
    a.weights = weights;
    a.n_tok = (int)n_tok;
    HIP_TRY(launch_moe_layer(a, work, (hipStream_t)stream), "moe_mxfp4");
    return ok_status();
}

}  // extern "C"
