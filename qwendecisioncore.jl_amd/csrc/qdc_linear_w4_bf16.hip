// qdc_linear_w4_bf16.hip -- the kernels of qdc_linear_w4.hpp for bf16 rows.
#include "qdc_linear_w4.hpp"

namespace qdc {

int32_t linear_w4_bf16(const W4Product &p, int group, bool gated, int32_t y_dtype, hipStream_t s) {
    return linear_w4<kBf16>(p, group, gated, y_dtype, s);
}

}  // namespace qdc
