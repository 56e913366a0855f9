// qdc_linear_w4.hip -- the entry point of the product with 4-bit weights.
#include "qdc_quant.hpp"

using namespace qdc;

static bool product_shape(int64_t rows, int64_t out, int64_t inner, int64_t group, int32_t gated,
                          bool y8) {
    return w4_shape(out, inner, group, gated) && rows >= 0 &&
           ceil_div(rows, (int64_t)16) <= 65535 && !(y8 && (!gated || out / 2 % 16));
}

extern "C" int64_t qdc_linear_w4_workspace(int64_t rows, int64_t out, int64_t inner, int64_t group,
                                           int32_t gated, int32_t y_dtype) {
    const bool y8 = y_dtype == QDC_Q8;
    if (!product_shape(rows, out, inner, group, gated, y8)) return -1;
    return y8 && w4_by_workspace(rows, w4_rows(out, gated), w4_cols(inner)) ? rows * (out / 2) * 4
                                                                           : 0;
}

extern "C" int32_t qdc_linear_w4(void *y, float *y_scales, int32_t y_dtype, const void *x,
                                 const float *x_scales, int32_t x_dtype, const void *packed,
                                 const void *scales, int64_t rows, int64_t out, int64_t inner,
                                 int64_t group, int64_t ld_x, int32_t gated, void *workspace,
                                 int64_t workspace_bytes, hipStream_t stream) {
    const bool x8 = x_dtype == QDC_Q8, y8 = y_dtype == QDC_Q8;
    if ((!valid_dtype(x_dtype) && !x8) || (!valid_dtype(y_dtype) && !(y8 && gated)))
        return QDC_ERR_DTYPE;
    if (!product_shape(rows, out, inner, group, gated, y8)) return QDC_ERR_SHAPE;
    const int64_t cols = gated ? out / 2 : out;
    if (x8 ? inner % 16 != 0 || ld_x != inner : ld_x < inner || ld_x % 8) return QDC_ERR_SHAPE;
    if (ld_x > kW4RowBytes / (x8 ? 1 : elem_size(x_dtype))) return QDC_ERR_SHAPE;
    if (rows == 0) return QDC_OK;
    const int64_t need = qdc_linear_w4_workspace(rows, out, inner, group, gated, y_dtype);
    if (!y || !x || !packed || !scales || (x8 && !x_scales) || (y8 && !y_scales) ||
        (need && !workspace))
        return QDC_ERR_NULL;
    if (!need) workspace = nullptr;
    if (workspace_bytes < need || !aligned16(workspace)) return QDC_ERR_SHAPE;
    if (!x8) x_scales = nullptr;
    if (!y8) y_scales = nullptr;
    if (!aligned16(y) || !aligned16(x) || !aligned16(packed) || !aligned16(scales) ||
        ((uintptr_t)x_scales & 3u) || ((uintptr_t)y_scales & 3u))
        return QDC_ERR_SHAPE;
    const int64_t xe = x8 ? 1 : elem_size(x_dtype), ye = y8 ? 1 : elem_size(y_dtype);
    const QuantRange outs[] = {{y, rows * cols * ye},
                               {y_scales, rows * q8_groups(cols) * 4},
                               {workspace, need}};
    const QuantRange ins[] = {{x, ((rows - 1) * ld_x + inner) * xe},
                              {x_scales, rows * q8_groups(inner) * 4},
                              {packed, w4_bytes(out, inner, gated)},
                              {scales, w4_scale_bytes(out, inner, group, gated)}};
    if (quant_alias(outs, 3, ins, 4)) return QDC_ERR_ALIAS;
    W4Product p{};
    p.x = x;
    p.x_scales = x_scales;
    p.packed = reinterpret_cast<const u32x4 *>(packed);
    p.scales = reinterpret_cast<const u32x2 *>(scales);
    p.y = need ? workspace : y;
    p.y_scales = y_scales;
    p.ld_x = ld_x;
    p.rows = (int)rows;
    p.cols = (int)cols;
    p.inner = (int)inner;
    p.kb = (int)w4_cols(inner);
    p.nb = (int)w4_rows(out, gated);
    p.q8_groups = (int)q8_groups(inner);
    const auto product = x8 ? linear_w4_q8 : x_dtype == QDC_BF16 ? linear_w4_bf16 : linear_w4_f32;
    const int32_t status = product(p, (int)group, gated != 0, need ? QDC_F32 : y_dtype, stream);
    if (status != QDC_OK || !need) return status;
    return qdc_quantize_q8(y, y_scales, workspace, rows, cols, cols, QDC_F32, stream);
}
