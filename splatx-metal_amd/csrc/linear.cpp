// linear.cpp — the C ABI entry points of the linear layers (include/splatx_hip.h): their checks and launches, as learn.cpp's.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "sx_device_args.h"

namespace sxh {
namespace {

constexpr int64_t kMostWidth = int64_t{1} << 24, kMostWeight = int64_t{1} << 40, kMostRows = int64_t{1} << 40, kMostGroups = 32768;

bool sizes_fit(int64_t rows, int64_t in, int64_t out, int64_t groups) {
    return rows >= 0 && rows <= kMostRows && in >= 1 && in <= kMostWidth && out >= 1 && out <= kMostWidth && in * out <= kMostWeight &&
           groups >= 0 && groups <= kMostGroups && rows <= (int64_t{1} << 52) / std::max(in, out);
}

void need_sizes(const char* what, int64_t rows, int64_t in, int64_t out, int64_t groups, const int64_t* ends, uint8_t type,
                uint8_t activation) {
    need_type(what, type, "type");
    if (activation > SXH_ACT_SIGMOID) invalid(what, "activation must be one of SXH_ACT_*");
    if (rows < 0) invalid(what, "negative rows");
    if (in < 1 || in > kMostWidth || out < 1 || out > kMostWidth) invalid(what, "in and out must be 1..16777216");
    if (groups < 0 || groups > kMostGroups) invalid(what, "groups must be 0..32768");
    if (!sizes_fit(rows, in, out, groups)) invalid(what, "rows or in * out are larger than memory");
    if (!ends != !groups) invalid(what, "ends is given with groups, and only then");
}

bool valid(int64_t rows, int64_t in, int64_t out, int64_t groups, uint8_t type) { return sizes_fit(rows, in, out, groups) && type <= SXH_TYPE_F16; }

sxk::LinearFwdArgs arguments(const sxh_linear_inputs& in, const sxh_linear_outputs& out) {
    sxk::LinearFwdArgs a{};
    a.x = in.x; a.weight = in.weight; a.bias = in.bias; a.residual = in.residual;
    a.y = out.y; a.pre = out.pre; a.ends = in.ends;
    a.rows = in.rows; a.in = in.in; a.out = in.out;
    a.x_stride = in.x_stride; a.residual_stride = in.residual_stride; a.y_stride = out.y_stride; a.pre_stride = out.pre_stride;
    a.groups = in.groups ? static_cast<int>(in.groups) : 1;
    a.act = in.activation; a.clear = in.clear != 0; a.workspace = out.workspace;
    return a;
}
sxk::LinearBwdArgs arguments(const sxh_linear_grads_in& in, const sxh_linear_grads& out) {
    sxk::LinearBwdArgs a{};
    a.dy = in.dy; a.pre = in.pre; a.x = in.x; a.weight = in.weight; a.ends = in.ends;
    a.dx = out.dx; a.dweight = out.dweight; a.dbias = out.dbias;
    a.rows = in.rows; a.in = in.in; a.out = in.out;
    a.dy_stride = in.dy_stride; a.pre_stride = in.pre_stride; a.x_stride = in.x_stride; a.dx_stride = out.dx_stride;
    a.groups = in.groups ? static_cast<int>(in.groups) : 1;
    a.act = in.activation; a.clear = in.clear != 0; a.workspace = out.workspace;
    return a;
}

int64_t need_workspace(RowCheck& c, void* workspace, int64_t given, int64_t bytes, const char* function) {
    if (given < bytes) invalid(c.what, "workspace_bytes is " + std::to_string(given) + ", " + function + " " + std::to_string(bytes));
    if (bytes) {
        c.mem.need(workspace, static_cast<size_t>(bytes), 16, "workspace");
        c.out.push_back({"workspace", reinterpret_cast<uintptr_t>(workspace), static_cast<size_t>(bytes), 0, 0});
    }
    return bytes;
}

}  // namespace
}  // namespace sxh

using namespace sxh;

extern "C" {

int64_t sxh_linear_fwd_workspace(const sxh_linear_inputs* in) {
    if (!in || !valid(in->rows, in->in, in->out, in->groups, in->type)) return 0;
    return sxk::linear_fwd_workspace(arguments(*in, sxh_linear_outputs{}), elem(in->type));
}

int32_t sxh_linear_fwd(sxh_backend* b, const sxh_linear_inputs* in, const sxh_linear_outputs* out, const sxh_queue* q) {
    return guarded([&] {
        const char* what = "linear_fwd";
        if (!in || !out) invalid(what, "null inputs/outputs");
        need_sizes(what, in->rows, in->in, in->out, in->groups, in->ends, in->type, in->activation);
        if (in->clear > 1) invalid(what, "clear must be 0 or 1");
        if (!b) invalid(what, "null backend");
        const size_t e = type_size(in->type);
        const int64_t weights = in->groups ? in->groups : 1;
        RowCheck c(what, b->device, in->rows, in->in);
        c.add(in->x, in->x_stride, in->in, e, "x", false);
        c.add_flat(in->weight, weights * in->in * in->out, e, "weight", false);
        if (in->bias) c.add_flat(in->bias, weights * in->out, e, "bias", false);
        if (in->residual) c.add(in->residual, in->residual_stride, in->out, e, "residual", false);
        if (in->groups) c.add_flat(in->ends, in->groups, 8, "ends", false);
        c.add(out->y, out->y_stride, in->out, e, "y", true);
        if (out->pre) c.add(out->pre, out->pre_stride, in->out, e, "pre", true);
        need_workspace(c, out->workspace, out->workspace_bytes, sxh_linear_fwd_workspace(in),
                       "sxh_linear_fwd_workspace");
        c.disjoint();
        if (in->rows == 0) return;
        Queue on(b, q, what);
        sxk::linear_fwd(arguments(*in, *out), elem(in->type), on.stream());
        on.done();
    });
}

int64_t sxh_linear_bwd_workspace(const sxh_linear_grads_in* in) {
    if (!in || !valid(in->rows, in->in, in->out, in->groups, in->type)) return 0;
    char some = 0;  // (not read or written: all gradients are wanted)
    sxh_linear_grads out{};
    out.dx = out.dweight = out.dbias = &some;
    return sxk::linear_bwd_workspace(arguments(*in, out), elem(in->type));
}

int32_t sxh_linear_bwd(sxh_backend* b, const sxh_linear_grads_in* in, const sxh_linear_grads* out, const sxh_queue* q) {
    return guarded([&] {
        const char* what = "linear_bwd";
        if (!in || !out) invalid(what, "null inputs/outputs");
        need_sizes(what, in->rows, in->in, in->out, in->groups, in->ends, in->type, in->activation);
        if (in->clear > 1) invalid(what, "clear must be 0 or 1");
        if (!out->dx && !out->dweight && !out->dbias) invalid(what, "no gradient is wanted");
        if (!in->pre != (in->activation == SXH_ACT_NONE) && in->rows) invalid(what, "pre is given with an activation, and only then");
        if (!b) invalid(what, "null backend");
        const size_t e = type_size(in->type);
        const int64_t weights = in->groups ? in->groups : 1;
        RowCheck c(what, b->device, in->rows, in->in);
        c.add(in->dy, in->dy_stride, in->out, e, "dy", false);
        if (in->pre) c.add(in->pre, in->pre_stride, in->out, e, "pre", false);
        if (out->dweight) c.add(in->x, in->x_stride, in->in, e, "x", false);
        if (out->dx) c.add_flat(in->weight, weights * in->in * in->out, e, "weight", false);
        if (in->groups) c.add_flat(in->ends, in->groups, 8, "ends", false);
        if (out->dx) c.add(out->dx, out->dx_stride, in->in, e, "dx", true);
        if (out->dweight) c.add_flat(out->dweight, weights * in->in * in->out, e, "dweight", true);
        if (out->dbias) c.add_flat(out->dbias, weights * in->out, e, "dbias", true);
        need_workspace(c, out->workspace, out->workspace_bytes, sxh_linear_bwd_workspace(in),
                       "sxh_linear_bwd_workspace");
        c.disjoint();
        Queue on(b, q, what);
        sxk::linear_bwd(arguments(*in, *out), elem(in->type), on.stream());
        on.done();
    });
}

}  // extern "C"
