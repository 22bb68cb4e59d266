// field_api.cpp - the feature operators' C entry points: checks of the
// arguments, then the launchers of field.h on the caller's stream.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <utility>
#include <vector>

#include "../../include/gsplat_hip.h"
#include "field.h"
#include "gs_error.h"

namespace {

using gs::guard;
using gs::GsError;

constexpr int64_t kMaxRows = (int64_t)1 << 30;
constexpr int64_t kMaxIds = ((int64_t)1 << 31) - 2;
constexpr int kMaxDim = 65536;
// a launch takes fewer than 2^32 threads: 2 a sample when the samples are streamed
constexpr int64_t kMaxSamples = ((int64_t)1 << 31) - 256;
constexpr int64_t kMaxLabels = (int64_t)1 << 22;
constexpr int64_t kMaxImages = (int64_t)1 << 20;
constexpr int64_t kMaxPixels = (int64_t)1 << 40;
constexpr int64_t kMaxHidden = (int64_t)1 << 20;
constexpr int64_t kMaxTensors = (int64_t)1 << 20;
constexpr int64_t kMaxValues = (int64_t)1 << 40;

#define LIMIT(cond, msg)                                        \
    do {                                                        \
        if (!(cond)) throw GsError(GS_E_CAPACITY, (msg));       \
    } while (0)

// The context's device for the call, and the caller's again after it.
struct OnDevice {
    int before = -1, here;
    explicit OnDevice(const gs_ctx* ctx) : here(gs::ctx_device(ctx)) {
        HIPCHK(hipGetDevice(&before));
        if (before != here) HIPCHK(hipSetDevice(here));
    }
    ~OnDevice() {
        if (before != here && before >= 0) (void)hipSetDevice(before);
    }
};

void check_dtype(int d, const char* what) {
    REQUIRE(d == GS_F32 || d == GS_BF16, std::string(what) + ": dtype must be GS_F32 or GS_BF16");
}
void check_ptr(const void* p, int dtype, const char* what) {
    REQUIRE(p != nullptr, std::string(what) + " is null");
    REQUIRE(reinterpret_cast<uintptr_t>(p) % (size_t)gs::elem_bytes(dtype) == 0,
            std::string(what) + " is not aligned to its elements");
}
// The rows of an input may overlap (a stride of 0 repeats one row), an output's not.
void check_rows(int64_t rows, int64_t stride, int dim, const char* what, bool output = false) {
    REQUIRE(!output || stride >= dim || rows <= 1,
            std::string(what) + ": rows overlap (stride below dim)");
    REQUIRE(stride >= 0 && stride < ((int64_t)1 << 40), std::string(what) + ": stride out of range");
}
void check_ids(const void* ids, int ids64, const char* what) {
    REQUIRE(ids != nullptr, std::string(what) + " is null");
    REQUIRE(ids64 == 0 || ids64 == 1, std::string(what) + ": ids64 must be 0 or 1");
    REQUIRE(reinterpret_cast<uintptr_t>(ids) % (ids64 ? 8 : 4) == 0,
            std::string(what) + " is not aligned to its elements");
}
void check_words(const void* p, const char* what) {
    REQUIRE(reinterpret_cast<uintptr_t>(p) % 4 == 0,
            std::string(what) + " is not aligned to its elements");
}
void check_ws(const void* ws, int64_t have, size_t want, const char* what) {
    REQUIRE(have >= 0 && (size_t)have >= want, std::string(what) + ": workspace too small");
    REQUIRE(want == 0 || (ws != nullptr && reinterpret_cast<uintptr_t>(ws) % 256 == 0),
            std::string(what) + ": workspace must be 256-byte aligned");
}
void check_dim(int dim, const char* what) {
    REQUIRE(dim >= 1, std::string(what) + ": dim must be at least 1");
    LIMIT(dim <= kMaxDim, std::string(what) + ": dim past 65536");
}

void check_norm(const gs_group_norm* d) {
    REQUIRE(d != nullptr, "group_norm: null description");
    REQUIRE(d->batch >= 0 && d->pixels >= 0, "group_norm: negative size");
    REQUIRE(d->channels >= 1 && d->groups >= 1 && d->channels % d->groups == 0,
            "group_norm: channels must be a positive multiple of groups");
    LIMIT(d->batch <= kMaxImages && d->pixels <= kMaxPixels && d->channels <= kMaxDim,
          "group_norm: at most 2^20 images, 2^40 pixels, 65536 channels");
    LIMIT(d->batch * d->groups < ((int64_t)1 << 31), "group_norm: batch * groups past 2^31");
    REQUIRE(d->act >= GS_ACT_NONE && d->act <= GS_ACT_GELU, "group_norm: unknown activation");
    check_dtype(d->dtype, "group_norm");
    REQUIRE(std::isfinite(d->eps) && d->eps > 0.0f, "group_norm: eps must be positive");
    check_words(d->weight, "group_norm: weight");
    check_words(d->bias, "group_norm: bias");
}
void check_image(const gs_group_norm* d, const void* p, int64_t batch, int64_t pixel,
                 const char* what, bool output = false) {
    if (d->batch == 0 || d->pixels == 0) return;
    check_ptr(p, d->dtype, what);
    REQUIRE(!output || pixel >= d->channels || d->pixels == 1,
            std::string(what) + ": pixels overlap");
    REQUIRE(pixel >= 0 && pixel < ((int64_t)1 << 40) && batch >= 0 && batch < ((int64_t)1 << 50),
            std::string(what) + ": stride out of range");
    REQUIRE(!output || d->batch == 1 || batch >= (d->pixels - 1) * pixel + d->channels,
            std::string(what) + ": images overlap");
}
gs::NormArgs norm_args(const gs_group_norm* d) {
    gs::NormArgs a{};
    a.batch = d->batch;
    a.pixels = d->pixels;
    a.channels = d->channels;
    a.groups = d->groups;
    a.act = d->act;
    a.dtype = d->dtype;
    a.eps = d->eps;
    a.weight = d->weight;
    a.bias = d->bias;
    return a;
}

gs::LossArgs loss_args(const gs_label_loss* d, float* loss, float* lse, void* ws, int64_t ws_bytes,
                       uint32_t* flags, bool grad) {
    REQUIRE(d != nullptr, "label_loss: null description");
    REQUIRE(d->n >= 0, "label_loss: n must not be negative");
    REQUIRE(d->rows >= 1, "label_loss: the table needs a row");
    LIMIT(d->n <= kMaxSamples, "label_loss: n past 2^31 - 256");
    LIMIT(d->rows <= kMaxLabels, "label_loss: rows past 2^22");
    check_dim(d->dim, "label_loss");
    check_dtype(d->dtype, "label_loss");
    REQUIRE(std::isfinite(d->scale), "label_loss: scale must be finite");
    if (d->n > 0) {
        check_ptr(d->feat, d->dtype, "label_loss: feat");
        check_rows(d->n, d->feat_stride, d->dim, "label_loss: feat");
        check_ptr(d->table, d->dtype, "label_loss: table");
        check_rows(d->rows, d->table_stride, d->dim, "label_loss: table");
        check_ids(d->labels, d->labels64, "label_loss: labels");
        check_ws(ws, ws_bytes, gs::label_loss_ws(d->n, d->rows, d->dim, d->dtype, grad),
                 "label_loss");
    }
    check_words(loss, "label_loss: loss");
    check_words(lse, "label_loss: lse");
    check_words(flags, "label_loss: flags");
    gs::LossArgs a{};
    a.feat = d->feat;
    a.n = d->n;
    a.feat_stride = d->feat_stride;
    a.table = d->table;
    a.rows = d->rows;
    a.table_stride = d->table_stride;
    a.dim = d->dim;
    a.dtype = d->dtype;
    a.labels = d->labels;
    a.labels64 = d->labels64;
    a.scale = d->scale;
    a.loss = loss;
    a.lse = lse;
    a.ws = ws;
    a.flags = flags;
    return a;
}


// The description alone, and its pointers if there is a row to compute.
gs::GatedArgs gated_args(const gs_gated_linear* d) {
    REQUIRE(d != nullptr, "gated_linear: null description");
    REQUIRE(d->n >= 0, "gated_linear: n must not be negative");
    REQUIRE(d->hidden >= 1, "gated_linear: hidden must be at least 1");
    LIMIT(d->n <= kMaxSamples, "gated_linear: n past 2^31 - 256");
    LIMIT(d->hidden <= kMaxHidden, "gated_linear: hidden past 2^20");
    check_dim(d->dim, "gated_linear");
    check_dtype(d->dtype, "gated_linear");
    REQUIRE(d->act >= GS_ACT_NONE && d->act <= GS_ACT_GELU, "gated_linear: unknown activation");
    if (d->n > 0) {
        check_ptr(d->x, d->dtype, "gated_linear: x");
        check_rows(d->n, d->x_stride, d->dim, "gated_linear: x");
        check_ptr(d->w_gate, d->dtype, "gated_linear: w_gate");
        check_rows(d->hidden, d->gate_stride, d->dim, "gated_linear: w_gate");
        check_ptr(d->w_up, d->dtype, "gated_linear: w_up");
        check_rows(d->hidden, d->up_stride, d->dim, "gated_linear: w_up");
    }
    check_words(d->b_gate, "gated_linear: b_gate");
    check_words(d->b_up, "gated_linear: b_up");
    gs::GatedArgs a{};
    a.x = d->x;
    a.n = d->n;
    a.x_stride = d->x_stride;
    a.w_gate = d->w_gate;
    a.w_up = d->w_up;
    a.hidden = d->hidden;
    a.gate_stride = d->gate_stride;
    a.up_stride = d->up_stride;
    a.b_gate = d->b_gate;
    a.b_up = d->b_up;
    a.dim = d->dim;
    a.dtype = d->dtype;
    a.act = d->act;
    return a;
}

// A list of tensors, checked; those without values are left out of `to`.
void tensor_list(const gs_tensor* t, int64_t count, const char* what, bool output,
                 std::vector<gs::TensorRef>* to) {
    REQUIRE(count >= 0, std::string(what) + ": negative count");
    LIMIT(count <= kMaxTensors, std::string(what) + ": more than 2^20 tensors");
    REQUIRE(count == 0 || t != nullptr, std::string(what) + ": null list");
    to->reserve((size_t)count);
    for (int64_t k = 0; k < count; ++k) {
        const gs_tensor& one = t[k];
        REQUIRE(one.rows >= 0 && one.cols >= 0, std::string(what) + ": negative size");
        check_dtype(one.dtype, what);
        if (one.rows == 0 || one.cols == 0) continue;
        LIMIT(one.rows <= kMaxValues / one.cols, std::string(what) + ": more than 2^40 values");
        check_ptr(one.data, one.dtype, what);
        REQUIRE(one.rows == 1 || (one.stride >= 0 && one.stride < ((int64_t)1 << 40)),
                std::string(what) + ": stride out of range");
        REQUIRE(!output || one.rows == 1 || one.stride >= one.cols,
                std::string(what) + ": rows overlap (stride below cols)");
        gs::TensorRef r{one.data, one.rows, one.cols, one.stride, one.dtype};
        if (r.rows == 1 || r.stride == r.cols)  // one run of values
            r = {r.data, 1, r.rows * r.cols, r.rows * r.cols, r.dtype};
        to->push_back(r);
    }
}

// Bytes that a tensor reaches over.
struct Span {
    uintptr_t begin, end;
    size_t row, stride;  // bytes of a row and between rows; stride 0: one row
    bool written;
};
Span span_of(const void* data, int64_t rows, int64_t cols, int64_t stride, int dtype,
             bool written) {
    const size_t e = (size_t)gs::elem_bytes(dtype);
    const uintptr_t p = reinterpret_cast<uintptr_t>(data);
    return {p, p + ((size_t)(rows - 1) * (size_t)stride + (size_t)cols) * e, (size_t)cols * e,
            rows > 1 ? (size_t)stride * e : 0, written};
}
Span span_of(const gs::TensorRef& t, bool written) {
    return span_of(t.data, t.rows, t.cols, t.stride, t.dtype, written);
}
// Whether two spans that overlap have no byte in common all the same: columns of one
// matrix.
bool apart(const Span& a, const Span& b) {
    const size_t stride = a.stride != 0 ? a.stride : b.stride;
    if (stride == 0 || (a.stride != 0 && b.stride != 0 && a.stride != b.stride)) return false;
    if (a.row > stride || b.row > stride) return false;
    // b's first byte as a column of a's rows
    const size_t at = b.begin >= a.begin ? (b.begin - a.begin) % stride
                                         : (stride - (a.begin - b.begin) % stride) % stride;
    return at >= a.row && at + b.row <= stride;
}
void check_apart(std::vector<Span>& spans, const char* what) {
    std::sort(spans.begin(), spans.end(),
              [](const Span& a, const Span& b) { return a.begin < b.begin; });
    // `open`: earlier spans that reach past the present one's begin
    std::vector<Span> open;
    for (const Span& s : spans) {
        size_t kept = 0;
        for (const Span& o : open) {
            if (o.end <= s.begin) continue;
            REQUIRE(!(o.written || s.written) || apart(o, s),
                    std::string(what) + ": an output shares memory with another tensor");
            open[kept++] = o;
        }
        open.resize(kept);
        open.push_back(s);
    }
}

// The memory of a gated call: `spans` beside what the description names and the workspace;
// without rows `spans` alone.
void check_gated_apart(const gs::GatedArgs& a, std::vector<Span> spans, const void* ws,
                       size_t ws_bytes, const char* what) {
    if (a.n > 0) {
        spans.push_back(span_of(a.x, a.n, a.dim, a.x_stride, a.dtype, false));
        spans.push_back(span_of(a.w_gate, a.hidden, a.dim, a.gate_stride, a.dtype, false));
        spans.push_back(span_of(a.w_up, a.hidden, a.dim, a.up_stride, a.dtype, false));
        for (const float* b : {a.b_gate, a.b_up})
            if (b != nullptr) spans.push_back(span_of(b, 1, a.hidden, 0, GS_F32, false));
        if (ws_bytes > 0) {
            const uintptr_t at = reinterpret_cast<uintptr_t>(ws);
            spans.push_back({at, at + ws_bytes, ws_bytes, 0, true});
        }
    }
    check_apart(spans, what);
}

}  // namespace

extern "C" {

int gs_stream(gs_ctx* ctx, void** stream) {
    return guard([&] {
        REQUIRE(ctx && stream, "null argument");
        *stream = gs::ctx_stream(ctx);
    });
}

int gs_lookup_dev(gs_ctx* ctx, const void* table, int64_t rows, int64_t table_stride,
                  int table_dtype, const void* ids, int ids64, int64_t n, int dim, float scale,
                  void* out, int64_t out_stride, int out_dtype, uint32_t* flags, void* stream) {
    return guard([&] {
        REQUIRE(ctx, "null ctx");
        REQUIRE(n >= 0 && rows >= 0, "lookup: negative size");
        LIMIT(n <= kMaxIds && rows < kMaxRows, "lookup: n past 2^31 - 2 or rows past 2^30");
        check_dim(dim, "lookup");
        check_dtype(table_dtype, "lookup: table");
        check_dtype(out_dtype, "lookup: out");
        REQUIRE(std::isfinite(scale), "lookup: scale must be finite");
        if (n > 0) {
            if (rows > 0) check_ptr(table, table_dtype, "lookup: table");
            check_rows(rows, table_stride, dim, "lookup: table");
            check_ids(ids, ids64, "lookup: ids");
            check_ptr(out, out_dtype, "lookup: out");
            check_rows(n, out_stride, dim, "lookup: out", true);
        }
        check_words(flags, "lookup: flags");
        const OnDevice on(ctx);
        HIPCHK(gs::launch_lookup({table, rows, table_stride, table_dtype, ids, ids64, n, dim, scale,
                                  out, out_stride, out_dtype, flags},
                                 static_cast<hipStream_t>(stream)));
    });
}

int64_t gs_lookup_grad_workspace(int64_t n, int64_t rows, int dim) {
    if (n < 0 || n > kMaxIds || rows < 0 || rows >= kMaxRows || dim < 1 || dim > kMaxDim) return -1;
    return (int64_t)gs::lookup_grad_ws(n, rows, dim);
}

int gs_lookup_grad_dev(gs_ctx* ctx, const void* dout, int64_t dout_stride, int dout_dtype,
                       const void* ids, int ids64, int64_t n, int dim, float scale,
                       int accumulate, void* dtable, int64_t rows, int64_t dtable_stride,
                       int dtable_dtype, void* workspace, int64_t workspace_bytes,
                       uint32_t* flags, void* stream) {
    return guard([&] {
        REQUIRE(ctx, "null ctx");
        REQUIRE(n >= 0 && rows >= 0, "lookup_grad: negative size");
        LIMIT(n <= kMaxIds && rows < kMaxRows, "lookup_grad: n past 2^31 - 2 or rows past 2^30");
        check_dim(dim, "lookup_grad");
        check_dtype(dout_dtype, "lookup_grad: dout");
        check_dtype(dtable_dtype, "lookup_grad: dtable");
        REQUIRE(std::isfinite(scale), "lookup_grad: scale must be finite");
        REQUIRE(accumulate == 0 || accumulate == 1, "lookup_grad: accumulate must be 0 or 1");
        if (n > 0) {
            check_ptr(dout, dout_dtype, "lookup_grad: dout");
            check_rows(n, dout_stride, dim, "lookup_grad: dout");
            check_ids(ids, ids64, "lookup_grad: ids");
        }
        if (rows > 0) {
            check_ptr(dtable, dtable_dtype, "lookup_grad: dtable");
            check_rows(rows, dtable_stride, dim, "lookup_grad: dtable", true);
            check_ws(workspace, workspace_bytes, gs::lookup_grad_ws(n, rows, dim), "lookup_grad");
        }
        check_words(flags, "lookup_grad: flags");
        const OnDevice on(ctx);
        HIPCHK(gs::launch_lookup_grad({dout, dout_stride, dout_dtype, ids, ids64, n, dim, scale,
                                       accumulate, dtable, rows, dtable_stride, dtable_dtype,
                                       workspace, flags},
                                      static_cast<hipStream_t>(stream)));
    });
}

int64_t gs_group_norm_workspace(int64_t batch, int64_t pixels, int channels) {
    if (batch < 0 || batch > kMaxImages || pixels < 0 || pixels > kMaxPixels || channels < 1 ||
        channels > kMaxDim)
        return -1;
    return (int64_t)gs::group_norm_ws(batch, channels);
}

int gs_group_norm_dev(gs_ctx* ctx, const gs_group_norm* norm, const void* x, int64_t x_batch,
                      int64_t x_pixel, void* y, int64_t y_batch, int64_t y_pixel, float* mean,
                      float* rstd, void* workspace, int64_t workspace_bytes, void* stream) {
    return guard([&] {
        REQUIRE(ctx, "null ctx");
        check_norm(norm);
        check_image(norm, x, x_batch, x_pixel, "group_norm: x");
        check_image(norm, y, y_batch, y_pixel, "group_norm: y", true);
        const bool any = norm->batch > 0 && norm->pixels > 0;
        REQUIRE(!any || (mean && rstd), "group_norm: mean and rstd are needed");
        check_words(mean, "group_norm: mean");
        check_words(rstd, "group_norm: rstd");
        check_ws(workspace, workspace_bytes,
                 gs::group_norm_ws(norm->batch, norm->channels), "group_norm");
        gs::NormArgs a = norm_args(norm);
        a.x = x;
        a.x_batch = x_batch;
        a.x_pixel = x_pixel;
        a.y = y;
        a.y_batch = y_batch;
        a.y_pixel = y_pixel;
        a.mean = mean;
        a.rstd = rstd;
        a.ws = workspace;
        const OnDevice on(ctx);
        HIPCHK(gs::launch_group_norm(a, static_cast<hipStream_t>(stream)));
    });
}

int gs_group_norm_grad_dev(gs_ctx* ctx, const gs_group_norm* norm, const void* dy,
                           int64_t dy_batch, int64_t dy_pixel, const void* x, int64_t x_batch,
                           int64_t x_pixel, const float* mean, const float* rstd, void* dx,
                           int64_t dx_batch, int64_t dx_pixel, float* dweight, float* dbias,
                           void* workspace, int64_t workspace_bytes, void* stream) {
    return guard([&] {
        REQUIRE(ctx, "null ctx");
        check_norm(norm);
        check_image(norm, dy, dy_batch, dy_pixel, "group_norm_grad: dy");
        check_image(norm, x, x_batch, x_pixel, "group_norm_grad: x");
        check_image(norm, dx, dx_batch, dx_pixel, "group_norm_grad: dx", true);
        const bool any = norm->batch > 0 && norm->pixels > 0;
        REQUIRE(!any || (mean && rstd), "group_norm_grad: mean and rstd are needed");
        check_words(mean, "group_norm_grad: mean");
        check_words(rstd, "group_norm_grad: rstd");
        check_words(dweight, "group_norm_grad: dweight");
        check_words(dbias, "group_norm_grad: dbias");
        check_ws(workspace, workspace_bytes,
                 gs::group_norm_ws(norm->batch, norm->channels), "group_norm_grad");
        gs::NormArgs a = norm_args(norm);
        a.x = x;
        a.x_batch = x_batch;
        a.x_pixel = x_pixel;
        a.dy = dy;
        a.dy_batch = dy_batch;
        a.dy_pixel = dy_pixel;
        a.dx = dx;
        a.dx_batch = dx_batch;
        a.dx_pixel = dx_pixel;
        a.mean = const_cast<float*>(mean);
        a.rstd = const_cast<float*>(rstd);
        a.dweight = dweight;
        a.dbias = dbias;
        a.ws = workspace;
        const OnDevice on(ctx);
        HIPCHK(gs::launch_group_norm_grad(a, static_cast<hipStream_t>(stream)));
    });
}

int64_t gs_label_loss_workspace(int64_t n, int64_t rows, int dim, int dtype, int grad) {
    if (n < 0 || n > kMaxSamples || rows < 1 || rows > kMaxLabels || dim < 1 || dim > kMaxDim ||
        (dtype != GS_F32 && dtype != GS_BF16))
        return -1;
    return n == 0 ? 0 : (int64_t)gs::label_loss_ws(n, rows, dim, dtype, grad != 0);
}

int gs_label_loss_dev(gs_ctx* ctx, const gs_label_loss* in, float* loss, float* lse,
                      void* workspace, int64_t workspace_bytes, uint32_t* flags, void* stream) {
    return guard([&] {
        REQUIRE(ctx, "null ctx");
        const gs::LossArgs a = loss_args(in, loss, lse, workspace, workspace_bytes, flags, false);
        const OnDevice on(ctx);
        HIPCHK(gs::launch_label_loss(a, false, static_cast<hipStream_t>(stream)));
    });
}

int gs_label_loss_grad_dev(gs_ctx* ctx, const gs_label_loss* in, const float* row_weight,
                           float* loss, float* lse, void* dfeat, int64_t dfeat_stride,
                           void* dtable, int64_t dtable_stride, void* workspace,
                           int64_t workspace_bytes, uint32_t* flags, void* stream) {
    return guard([&] {
        REQUIRE(ctx, "null ctx");
        gs::LossArgs a = loss_args(in, loss, lse, workspace, workspace_bytes, flags, true);
        check_words(row_weight, "label_loss_grad: row_weight");
        if (in->n > 0) {
            check_ptr(dfeat, in->dtype, "label_loss_grad: dfeat");
            check_rows(in->n, dfeat_stride, in->dim, "label_loss_grad: dfeat", true);
        }
        check_ptr(dtable, in->dtype, "label_loss_grad: dtable");
        check_rows(in->rows, dtable_stride, in->dim, "label_loss_grad: dtable", true);
        a.row_weight = row_weight;
        a.dfeat = dfeat;
        a.dfeat_stride = dfeat_stride;
        a.dtable = dtable;
        a.dtable_stride = dtable_stride;
        const OnDevice on(ctx);
        HIPCHK(gs::launch_label_loss(a, true, static_cast<hipStream_t>(stream)));
    });
}

int64_t gs_gated_linear_workspace(const gs_gated_linear* in, int grad) {
    try {
        return (int64_t)gs::gated_linear_ws(gated_args(in), grad != 0);
    } catch (const std::exception& e) {
        gs::g_err = e.what();
        return -1;
    }
}

int gs_gated_linear_dev(gs_ctx* ctx, const gs_gated_linear* in, void* h, int64_t h_stride,
                        void* workspace, int64_t workspace_bytes, void* stream) {
    return guard([&] {
        gs::GatedArgs a = gated_args(in);
        if (a.n > 0) {
            check_ptr(h, a.dtype, "gated_linear: h");
            check_rows(a.n, h_stride, (int)a.hidden, "gated_linear: h", true);
            const size_t need = gs::gated_linear_ws(a, false);
            check_ws(workspace, workspace_bytes, need, "gated_linear");
            check_gated_apart(a, {span_of(h, a.n, a.hidden, h_stride, a.dtype, true)}, workspace,
                              need, "gated_linear");
        }
        a.h = h;
        a.h_stride = h_stride;
        a.ws = workspace;
        REQUIRE(ctx, "null ctx");  // last: the other checks need no device
        const OnDevice on(ctx);
        HIPCHK(gs::launch_gated_linear(a, false, static_cast<hipStream_t>(stream)));
    });
}

int gs_gated_linear_grad_dev(gs_ctx* ctx, const gs_gated_linear* in, const void* dh,
                             int64_t dh_stride, void* dx, int64_t dx_stride, void* dw_gate,
                             int64_t dw_gate_stride, void* dw_up, int64_t dw_up_stride,
                             float* db_gate, float* db_up, void* workspace,
                             int64_t workspace_bytes, void* stream) {
    return guard([&] {
        gs::GatedArgs a = gated_args(in);
        size_t need = 0;
        if (a.n > 0) {
            check_ptr(dh, a.dtype, "gated_linear_grad: dh");
            check_rows(a.n, dh_stride, (int)a.hidden, "gated_linear_grad: dh");
            check_ptr(dx, a.dtype, "gated_linear_grad: dx");
            check_rows(a.n, dx_stride, a.dim, "gated_linear_grad: dx", true);
            need = gs::gated_linear_ws(a, true);
            check_ws(workspace, workspace_bytes, need, "gated_linear_grad");
        }
        check_ptr(dw_gate, a.dtype, "gated_linear_grad: dw_gate");
        check_rows(a.hidden, dw_gate_stride, a.dim, "gated_linear_grad: dw_gate", true);
        check_ptr(dw_up, a.dtype, "gated_linear_grad: dw_up");
        check_rows(a.hidden, dw_up_stride, a.dim, "gated_linear_grad: dw_up", true);
        check_words(db_gate, "gated_linear_grad: db_gate");
        check_words(db_up, "gated_linear_grad: db_up");
        std::vector<Span> outputs;
        outputs.reserve(12);
        outputs.push_back(span_of(dw_gate, a.hidden, a.dim, dw_gate_stride, a.dtype, true));
        outputs.push_back(span_of(dw_up, a.hidden, a.dim, dw_up_stride, a.dtype, true));
        for (const float* b : {db_gate, db_up})
            if (b != nullptr) outputs.push_back(span_of(b, 1, a.hidden, 0, GS_F32, true));
        if (a.n > 0) {
            outputs.push_back(span_of(dh, a.n, a.hidden, dh_stride, a.dtype, false));
            outputs.push_back(span_of(dx, a.n, a.dim, dx_stride, a.dtype, true));
        }
        check_gated_apart(a, std::move(outputs), workspace, need, "gated_linear_grad");
        a.dh = dh;
        a.dh_stride = dh_stride;
        a.dx = dx;
        a.dx_stride = dx_stride;
        a.dw_gate = dw_gate;
        a.dw_up = dw_up;
        a.dgate_stride = dw_gate_stride;
        a.dup_stride = dw_up_stride;
        a.db_gate = db_gate;
        a.db_up = db_up;
        a.ws = workspace;
        REQUIRE(ctx, "null ctx");  // last: the other checks need no device
        const OnDevice on(ctx);
        HIPCHK(gs::launch_gated_linear(a, true, static_cast<hipStream_t>(stream)));
    });
}

int64_t gs_grad_norm_workspace(const gs_tensor* tensors, int64_t count) {
    try {
        std::vector<gs::TensorRef> t;
        tensor_list(tensors, count, "grad_norm", false, &t);
        return (int64_t)gs::grad_norm_ws(t.data(), (int64_t)t.size());
    } catch (const std::exception& e) {
        gs::g_err = e.what();
        return -1;
    }
}

int gs_grad_norm_dev(gs_ctx* ctx, const gs_tensor* tensors, int64_t count, int kind, float* norm,
                     void* workspace, int64_t workspace_bytes, void* stream) {
    return guard([&] {
        REQUIRE(kind == GS_NORM_L2 || kind == GS_NORM_MAX, "grad_norm: unknown norm");
        std::vector<gs::TensorRef> t;
        tensor_list(tensors, count, "grad_norm", false, &t);
        REQUIRE(norm != nullptr, "grad_norm: norm is null");
        check_words(norm, "grad_norm: norm");
        check_ws(workspace, workspace_bytes, gs::grad_norm_ws(t.data(), (int64_t)t.size()),
                 "grad_norm");
        REQUIRE(ctx, "null ctx");  // last: the other checks need no device
        const OnDevice on(ctx);
        HIPCHK(gs::launch_grad_norm(t.data(), (int64_t)t.size(), kind, norm, workspace,
                                    static_cast<hipStream_t>(stream)));
    });
}

int gs_grad_clip_dev(gs_ctx* ctx, const gs_tensor* in, const gs_tensor* out, int64_t count,
                     int kind, float* norm, double max_norm, void* workspace,
                     int64_t workspace_bytes, void* stream) {
    return guard([&] {
        REQUIRE(kind == GS_NORM_L2 || kind == GS_NORM_MAX || kind == GS_NORM_GIVEN,
                "grad_clip: unknown norm");
        REQUIRE(max_norm >= 0.0, "grad_clip: max_norm must be a number, at least 0");
        std::vector<gs::TensorRef> from, to;
        tensor_list(in, count, "grad_clip: in", false, &from);
        tensor_list(out, count, "grad_clip: out", true, &to);
        bool alike = from.size() == to.size();
        for (int64_t k = 0; k < count; ++k)
            alike &= in[k].rows * in[k].cols == out[k].rows * out[k].cols;
        for (size_t k = 0; alike && k < from.size(); ++k)
            alike = from[k].rows == 1 || to[k].rows == 1 || from[k].rows == to[k].rows;
        REQUIRE(alike, "grad_clip: an output's rows and cols are not its input's");
        REQUIRE(norm != nullptr, "grad_clip: norm is null");
        check_words(norm, "grad_clip: norm");
        if (kind != GS_NORM_GIVEN)
            check_ws(workspace, workspace_bytes, gs::grad_norm_ws(from.data(), (int64_t)from.size()),
                     "grad_clip");
        std::vector<Span> spans;
        spans.reserve(2 * from.size());
        for (size_t k = 0; k < from.size(); ++k) {
            const gs::TensorRef &f = from[k], &t = to[k];
            const bool same = f.data == t.data && f.rows == t.rows && f.cols == t.cols &&
                              f.stride == t.stride && f.dtype == t.dtype;
            if (!same) spans.push_back(span_of(f, false));
            spans.push_back(span_of(t, true));
        }
        const uintptr_t at = reinterpret_cast<uintptr_t>(norm);
        spans.push_back({at, at + 4, 4, 0, kind != GS_NORM_GIVEN});
        check_apart(spans, "grad_clip");
        REQUIRE(ctx, "null ctx");  // last: the other checks need no device
        const OnDevice on(ctx);
        HIPCHK(gs::launch_grad_clip(from.data(), to.data(), (int64_t)from.size(), kind, norm,
                                    max_norm, workspace, static_cast<hipStream_t>(stream)));
    });
}

}  // extern "C"
