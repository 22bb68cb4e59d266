// field_gated_f32.hip - gated projections of short fp32 rows.
#include "field_gated_short.h"

namespace gs {

size_t gated_short_ws(const GatedArgs& a, bool grad) {
    return ShortPlan(nullptr, a.n, a.hidden, a.dim, a.dtype == 0 ? 3 : 1, grad).bytes;
}
hipError_t gated_short_f32(const GatedArgs& a, bool grad, hipStream_t st) {
    return short_act<float, 3>(a, grad, st);
}

}  // namespace gs
