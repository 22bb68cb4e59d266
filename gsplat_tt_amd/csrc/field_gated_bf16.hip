// field_gated_bf16.hip - gated projections of short bf16 rows.
#include "field_gated_short.h"

namespace gs {

hipError_t gated_short_bf16(const GatedArgs& a, bool grad, hipStream_t st) {
    return short_act<bf16, 1>(a, grad, st);
}

}  // namespace gs
