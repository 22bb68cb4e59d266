// field.h - the feature operators (lookup, group norm, label loss, gated projections,
// gradient norm and clipping): arguments
// shared by the entry points (field_api.cpp) and the kernels, and the launchers.
// Every launcher only enqueues kernels on the given stream: no allocation, no
// copy, no memset and no wait, so all of them can be captured into a HIP graph.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

struct gs_ctx;  // include/gsplat_hip.h

namespace gs {

// Bits of the caller's flag word (gs_*'s `flags`).
constexpr uint32_t kFlagIdRange = 1u;  // an id or a label at or past the table's rows

// Element types (GS_F32, GS_BF16) of one operand.
inline int elem_bytes(int dtype) { return dtype == 0 ? 4 : 2; }

struct LookupArgs {
    const void* table;  // (rows, dim), row stride table_stride
    int64_t rows, table_stride;
    int table_dtype;
    const void* ids;  // (n), int32 or int64
    int ids64;
    int64_t n;
    int dim;
    float scale;
    void* out;  // (n, dim), row stride out_stride
    int64_t out_stride;
    int out_dtype;
    uint32_t* flags;
};
hipError_t launch_lookup(const LookupArgs& a, hipStream_t st);

struct LookupGradArgs {
    const void* dout;  // (n, dim), row stride dout_stride
    int64_t dout_stride;
    int dout_dtype;
    const void* ids;
    int ids64;
    int64_t n;
    int dim;
    float scale;
    int accumulate;
    void* dtable;  // (rows, dim), row stride dtable_stride
    int64_t rows, dtable_stride;
    int dtable_dtype;
    void* ws;
    uint32_t* flags;
};
size_t lookup_grad_ws(int64_t n, int64_t rows, int dim);
hipError_t launch_lookup_grad(const LookupGradArgs& a, hipStream_t st);

struct NormArgs {
    const void* x;  // (batch, pixels, channels)
    int64_t x_batch, x_pixel;
    int64_t batch, pixels;
    int channels, groups, act, dtype;
    float eps;
    const float *weight, *bias;  // (channels) or null
    void* y;
    int64_t y_batch, y_pixel;
    float *mean, *rstd;  // (batch, groups)
    void* ws;
    // the gradient's own
    const void* dy;
    int64_t dy_batch, dy_pixel;
    void* dx;
    int64_t dx_batch, dx_pixel;
    float *dweight, *dbias;
};
size_t group_norm_ws(int64_t batch, int channels);
hipError_t launch_group_norm(const NormArgs& a, hipStream_t st);
hipError_t launch_group_norm_grad(const NormArgs& a, hipStream_t st);

struct LossArgs {
    const void* feat;  // (n, dim)
    int64_t n, feat_stride;
    const void* table;  // (rows, dim)
    int64_t rows, table_stride;
    int dim, dtype;
    const void* labels;  // (n)
    int labels64;
    float scale;
    float *loss, *lse;  // (n)
    void* ws;
    uint32_t* flags;
    // the gradients' own
    const float* row_weight;  // (n) or null (1)
    void* dfeat;
    int64_t dfeat_stride;
    void* dtable;
    int64_t dtable_stride;
};
size_t label_loss_ws(int64_t n, int64_t rows, int dim, int dtype, bool grad);
hipError_t launch_label_loss(const LossArgs& a, bool grad, hipStream_t st);

struct GatedArgs {
    const void* x;  // (n, dim)
    int64_t n, x_stride;
    const void *w_gate, *w_up;  // (hidden, dim)
    int64_t hidden, gate_stride, up_stride;
    const float *b_gate, *b_up;  // (hidden) or null
    int dim, dtype, act;
    void* h;  // (n, hidden)
    int64_t h_stride;
    void* ws;
    // the gradients' own
    const void* dh;
    int64_t dh_stride;
    void* dx;
    int64_t dx_stride;
    void *dw_gate, *dw_up;
    int64_t dgate_stride, dup_stride;
    float *db_gate, *db_up;  // (hidden) or null
};
size_t gated_linear_ws(const GatedArgs& a, bool grad);
hipError_t launch_gated_linear(const GatedArgs& a, bool grad, hipStream_t st);

// One tensor of a list: rows of cols values, stride apart.
struct TensorRef {
    void* data;
    int64_t rows, cols, stride;
    int dtype;
};
enum { kNormGiven = -1, kNormL2 = 0, kNormMax = 1 };  // GS_NORM_*
size_t grad_norm_ws(const TensorRef* t, int64_t count);
hipError_t launch_grad_norm(const TensorRef* t, int64_t count, int kind, float* norm, void* ws,
                            hipStream_t st);
hipError_t launch_grad_clip(const TensorRef* in, const TensorRef* out, int64_t count, int kind,
                            float* norm, double max_norm, void* ws, hipStream_t st);

// gs_api.cpp
int ctx_device(const ::gs_ctx* ctx);
hipStream_t ctx_stream(const ::gs_ctx* ctx);

}  // namespace gs
