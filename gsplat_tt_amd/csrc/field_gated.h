// field_gated.h - what the gated projections' kernels share, and the ways that
// field_gated.hip chooses from.
#pragma once

#include <algorithm>

#include "field.h"

#include "field_act.h"
#include "field_device.h"
#include "field_tiles.h"

namespace gs {

constexpr int kShortDim = 128;
size_t gated_short_ws(const GatedArgs& a, bool grad);
hipError_t gated_short_f32(const GatedArgs& a, bool grad, hipStream_t st);
hipError_t gated_short_bf16(const GatedArgs& a, bool grad, hipStream_t st);

// 8 values of a row from column c, zeros past `cols`.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int64_t c, int64_t cols, float* v) {
    if (c + 8 <= cols) {
        load_any<8>(row + c, v);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = c + k < cols ? to_float(row[c + k]) : 0.0f;
    }
}
template <int VEC, typename T>
__device__ __forceinline__ void store_cols(T* row, int64_t c, int64_t cols, const float* v) {
    if (c + VEC <= cols) {
        store_any<VEC>(row + c, v);
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            if (c + k < cols) row[c + k] = from_float<T>(v[k]);
    }
}

}  // namespace gs
