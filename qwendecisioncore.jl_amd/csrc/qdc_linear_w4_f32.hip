// qdc_linear_w4_f32.hip -- the kernels of qdc_linear_w4.hpp for f32 rows.
#include "qdc_linear_w4.hpp"

namespace qdc {

int32_t linear_w4_f32(const W4Product &p, int group, bool gated, int32_t y_dtype, hipStream_t s) {
    return linear_w4<kF32>(p, group, gated, y_dtype, s);
}

}  // namespace qdc
