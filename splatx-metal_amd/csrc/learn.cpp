// learn.cpp — the C ABI entry points of the learned heads' operators: layer norm, gradient norm, AdamW on device
// buffers (include/splatx_hip.h). Each checks its arguments, launches on the caller's queue or on the backend's stream,
// and keeps nothing.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

#include "sx_device_args.h"

namespace sxh {
namespace {

void need_weight_type(const char* what, uint8_t type, uint8_t weight_type) {
    need_type(what, type, "type");
    if (weight_type != SXH_TYPE_F32 && weight_type != type)
        invalid(what, "weight_type must be SXH_TYPE_F32 or the rows' type");
}

}  // namespace
}  // namespace sxh

using namespace sxh;

extern "C" {

int32_t sxh_layer_norm_fwd(sxh_backend* b, const sxh_layer_norm_inputs* in, const sxh_layer_norm_outputs* out,
                           const sxh_queue* q) {
    return guarded([&] {
        const char* what = "layer_norm_fwd";
        if (!in || !out) invalid(what, "null inputs/outputs");
        need_weight_type(what, in->type, in->weight_type);
        if (!(in->eps > 0.0f && std::isfinite(in->eps))) invalid(what, "eps must be positive");
        if (!in->residual != !out->h) invalid(what, "h is written with a residual, and only then");
        if (!out->mean != !out->rstd) invalid(what, "mean and rstd are wanted together or not at all");
        if (!b) invalid(what, "null backend");
        const size_t e = type_size(in->type), we = type_size(in->weight_type);
        RowCheck c(what, b->device, in->rows, in->width);
        c.add(in->x, in->x_stride, e, "x", false);
        if (in->residual) c.add(in->residual, in->residual_stride, e, "residual", false);
        if (in->weight) c.add_flat(in->weight, in->width, we, "weight", false);
        if (in->bias) c.add_flat(in->bias, in->width, we, "bias", false);
        c.add(out->y, out->y_stride, e, "y", true);
        if (out->h) c.add(out->h, out->h_stride, e, "h", true);
        if (out->mean) {
            c.add_flat(out->mean, in->rows, 4, "mean", true);
            c.add_flat(out->rstd, in->rows, 4, "rstd", true);
        }
        c.disjoint();
        if (in->rows == 0) return;
        Queue on(b, q, what);
        sxk::NormFwdArgs a{};
        a.x = in->x; a.residual = in->residual; a.weight = in->weight; a.bias = in->bias;
        a.y = out->y; a.h = out->h; a.mean = out->mean; a.rstd = out->rstd;
        a.rows = in->rows; a.width = static_cast<int>(in->width); a.eps = in->eps;
        a.x_stride = in->x_stride; a.residual_stride = in->residual_stride;
        a.y_stride = out->y_stride; a.h_stride = out->h_stride;
        sxk::layer_norm_fwd(a, elem(in->type), elem(in->weight_type), on.stream());
        on.done();
    });
}

int64_t sxh_layer_norm_bwd_workspace(int64_t rows, int64_t width) {
    if (rows < 0 || width < 1 || width > (int64_t{1} << 24)) return 0;
    int slabs = 0;  // the most that any type needs
    for (const sxk::ElemType t : {sxk::kF32, sxk::kBf16}) slabs = std::max(slabs, sxk::norm_bwd_slabs(rows, width, t, false, false));
    return int64_t{slabs} * 2 * width * 4;
}

int32_t sxh_layer_norm_bwd(sxh_backend* b, const sxh_layer_norm_grads_in* in, const sxh_layer_norm_grads* out,
                           const sxh_queue* q) {
    return guarded([&] {
        const char* what = "layer_norm_bwd";
        if (!in || !out) invalid(what, "null inputs/outputs");
        need_weight_type(what, in->type, in->weight_type);
        if (!out->dx && !out->dweight && !out->dbias) invalid(what, "no gradient is wanted");
        if (in->dh && !out->dx) invalid(what, "dh without dx");
        if (!b) invalid(what, "null backend");
        const size_t e = type_size(in->type), we = type_size(in->weight_type);
        RowCheck c(what, b->device, in->rows, in->width);
        c.add(in->dy, in->dy_stride, e, "dy", false);
        c.add(in->h, in->h_stride, e, "h", false);
        if (in->dh) c.add(in->dh, in->dh_stride, e, "dh", false);
        c.add_flat(in->mean, in->rows, 4, "mean", false);
        c.add_flat(in->rstd, in->rows, 4, "rstd", false);
        if (in->weight) c.add_flat(in->weight, in->width, we, "weight", false);
        if (out->dx) c.add(out->dx, out->dx_stride, e, "dx", true);
        if (out->dweight) c.add_flat(out->dweight, in->width, we, "dweight", true);
        if (out->dbias) c.add_flat(out->dbias, in->width, we, "dbias", true);
        if (out->dweight || out->dbias) {
            const int64_t bytes = sxh_layer_norm_bwd_workspace(in->rows, in->width);
            if (out->workspace_bytes < bytes)
                invalid(what, "workspace_bytes is " + std::to_string(out->workspace_bytes) + ", sxh_layer_norm_bwd_workspace " + std::to_string(bytes));
            c.mem.need(out->workspace, static_cast<size_t>(bytes), 16, "workspace");
            c.out.push_back({"workspace", reinterpret_cast<uintptr_t>(out->workspace), static_cast<size_t>(bytes), 0, 0});
        }
        c.disjoint();
        Queue on(b, q, what);
        sxk::NormBwdArgs a{};
        a.dy = in->dy; a.h = in->h; a.dh = in->dh; a.weight = in->weight; a.mean = in->mean; a.rstd = in->rstd;
        a.dx = out->dx; a.dweight = out->dweight; a.dbias = out->dbias;
        a.partial = static_cast<float*>(out->workspace);
        a.rows = in->rows; a.width = static_cast<int>(in->width);
        a.dy_stride = in->dy_stride; a.h_stride = in->h_stride; a.dh_stride = in->dh_stride; a.dx_stride = out->dx_stride;
        sxk::layer_norm_bwd(a, elem(in->type), elem(in->weight_type), on.stream());
        on.done();
    });
}

int64_t sxh_grad_norm_workspace(int64_t n_tensors) {
    if (n_tensors < 0) return 0;
    return std::max<int64_t>((n_tensors + sxk::kNormTensors - 1) / sxk::kNormTensors, 1) * sxk::kNormSlots * 8;
}

int32_t sxh_grad_norm(sxh_backend* b, const sxh_norm_tensor* tensors, int64_t n_tensors, float* norm, void* workspace,
                      int64_t workspace_bytes, const sxh_queue* q) {
    return guarded([&] {
        const char* what = "grad_norm";
        if (n_tensors < 0 || (n_tensors > 0 && !tensors)) invalid(what, "null tensors, or fewer than none");
        if (!b) invalid(what, "null backend");
        DeviceMemory mem(what, b->device);
        mem.need(norm, 4, 4, "norm");
        const int64_t bytes = sxh_grad_norm_workspace(n_tensors);
        if (workspace_bytes < bytes)
            invalid(what, "workspace_bytes is " + std::to_string(workspace_bytes) + ", sxh_grad_norm_workspace " + std::to_string(bytes));
        mem.need(workspace, static_cast<size_t>(bytes), 16, "workspace");
        const Rows out{"norm", reinterpret_cast<uintptr_t>(norm), 4, 4, 0};
        const Rows work{"workspace", reinterpret_cast<uintptr_t>(workspace), static_cast<size_t>(bytes), static_cast<size_t>(bytes), 0};
        if (!apart(out, work)) invalid(what, "norm overlaps workspace");
        for (int64_t i = 0; i < n_tensors; i++) {
            const sxh_norm_tensor& t = tensors[i];
            need_type(what, t.type, "type");
            if (t.n < 0 || t.n > (int64_t{1} << 40)) invalid(what, "n must be 0..2^40");
            if (!t.n) continue;
            const size_t size = static_cast<size_t>(t.n) * type_size(t.type);
            mem.need(t.grad, size, type_size(t.type), "grad");
            const Rows r{"grad", reinterpret_cast<uintptr_t>(t.grad), size, size, 0};
            if (!apart(out, r)) invalid(what, "norm overlaps a gradient");
            if (!apart(work, r)) invalid(what, "workspace overlaps a gradient");
        }
        Queue on(b, q, what);
        auto* part = static_cast<double*>(workspace);
        int64_t slots = 0;
        for (int64_t i = 0; i < n_tensors;) {
            sxk::NormTable t;
            t.tensors = 0;
            t.first[0] = 0;
            for (; i < n_tensors && t.tensors < sxk::kNormTensors; i++) {
                const sxh_norm_tensor& x = tensors[i];
                const int64_t chunks = (x.n + sxk::kNormChunk - 1) / sxk::kNormChunk;
                if (!chunks) continue;
                if (t.tensors && t.first[t.tensors] + chunks > INT32_MAX) break;
                t.grad[t.tensors] = x.grad;
                t.n[t.tensors] = x.n;
                t.type[t.tensors] = x.type;
                t.first[t.tensors + 1] = t.first[t.tensors] + static_cast<int32_t>(chunks);
                t.tensors++;
            }
            if (!t.tensors) break;
            if (i == n_tensors && slots == 0 && sxk::norm_of_few(t, norm, on.stream())) {
                on.done();
                return;
            }
            slots += sxk::sum_squares(t, part + slots, on.stream());
        }
        sxk::norm_of_sums(part, slots, norm, on.stream());
        on.done();
    });
}

int32_t sxh_adamw(sxh_backend* b, const sxh_adamw_tensor* tensors, int64_t n_tensors, const sxh_adamw_params* p,
                  const sxh_queue* q) {
    return guarded([&] {
        const char* what = "adamw";
        if (!p) invalid(what, "null params");
        if (n_tensors < 0 || (n_tensors > 0 && !tensors)) invalid(what, "null tensors, or fewer than none");
        if (p->step < 1) invalid(what, "step must be 1 or more");
        if (p->state_bits != 32 && p->state_bits != 8) invalid(what, "state_bits must be 32 or 8");
        if (!(p->b1 >= 0.0 && p->b1 < 1.0 && p->b2 >= 0.0 && p->b2 < 1.0)) invalid(what, "b1 and b2 must be in [0, 1)");
        // (the quotient's denominator, roots of floats over roots of 2^-53 at least and eps, and its reciprocal stay normal floats)
        if (!(p->eps >= 1e-30 && p->eps <= 1e30)) invalid(what, "eps must be in [1e-30, 1e30]");
        if (!(p->max_norm >= 0.0f) || !std::isfinite(p->max_norm)) invalid(what, "max_norm must be 0 or more");
        if (!(p->grad_scale > 0.0f) || !std::isfinite(p->grad_scale)) invalid(what, "grad_scale must be positive");
        if (p->adopt != 0 && p->adopt != 1) invalid(what, "adopt must be 0 or 1");
        if (p->max_norm > 0.0f && !p->grad_norm) invalid(what, "max_norm needs grad_norm");
        if (!b) invalid(what, "null backend");
        const bool eight = p->state_bits == 8;
        DeviceMemory mem(what, b->device);
        std::vector<Rows> written, read;
        size_t total = 0;  // bytes of all
        written.reserve(static_cast<size_t>(n_tensors) * (eight ? 7 : 5));
        read.reserve(static_cast<size_t>(n_tensors) + 1);
        auto range = [&](std::vector<Rows>& to, const void* ptr, int64_t n, size_t e, const char* name) {
            const size_t bytes = static_cast<size_t>(n) * e;
            mem.need(ptr, bytes, e, name);
            to.push_back({name, reinterpret_cast<uintptr_t>(ptr), bytes, bytes, 0});
            total += bytes;
        };
        if (p->grad_norm) range(read, p->grad_norm, 1, 4, "grad_norm");
        for (int64_t i = 0; i < n_tensors; i++) {
            const sxh_adamw_tensor& t = tensors[i];
            need_type(what, t.param_type, "param_type");
            need_type(what, t.grad_type, "grad_type");
            if (t.n < 0 || t.n > (int64_t{1} << 40)) invalid(what, "n must be 0..2^40");
            if (!std::isfinite(t.lr) || !std::isfinite(t.weight_decay)) invalid(what, "lr and weight_decay must be finite");
            if ((t.param_type != SXH_TYPE_F32) != (t.master != nullptr) && t.n)
                invalid(what, "master is given with a 16-bit param, and only then");
            if (eight != (t.exp_avg_scale != nullptr) && t.n) invalid(what, "the scales are given with state_bits 8, and only then");
            if (eight != (t.exp_avg_sq_scale != nullptr) && t.n) invalid(what, "the scales are given with state_bits 8, and only then");
            if (!t.n) continue;
            const size_t state = eight ? 1 : 4;
            range(written, t.param, t.n, type_size(t.param_type), "param");
            if (t.master) range(written, t.master, t.n, 4, "master");
            range(written, t.exp_avg, t.n, state, "exp_avg");
            range(written, t.exp_avg_sq, t.n, state, "exp_avg_sq");
            range(read, t.grad, t.n, type_size(t.grad_type), "grad");
            if (t.taken) range(written, t.taken, 2, 8, "taken");
            if (eight) {
                const int64_t blocks = (t.n + sxk::kAdamBlock - 1) / sxk::kAdamBlock;
                range(written, t.exp_avg_scale, blocks, 4, "exp_avg_scale");
                range(written, t.exp_avg_sq_scale, blocks, 4, "exp_avg_sq_scale");
            }
        }
        // no byte is written by two elements, or read as a gradient and written
        std::sort(written.begin(), written.end(), [](const Rows& x, const Rows& y) { return x.at < y.at; });
        for (size_t i = 1; i < written.size(); i++)
            if (!apart(written[i - 1], written[i]))
                invalid(what, std::string(written[i].name) + " overlaps another tensor's " + written[i - 1].name);
        for (const Rows& r : read) {
            auto it = std::upper_bound(written.begin(), written.end(), r, [](const Rows& x, const Rows& y) { return x.at < y.at; });
            if ((it != written.end() && !apart(r, *it)) || (it != written.begin() && !apart(r, *(it - 1))))
                invalid(what, std::string(r.name) + " overlaps what the step writes");
        }
        Queue on(b, q, what);
        sxk::AdamTable t{};
        t.grad_norm = p->grad_norm; t.max_norm = p->max_norm; t.grad_scale = p->grad_scale;
        t.b1 = static_cast<float>(p->b1); t.c1 = static_cast<float>(1.0 - p->b1);
        t.b2 = static_cast<float>(p->b2); t.c2 = static_cast<float>(1.0 - p->b2);
        t.eps = static_cast<float>(p->eps);
        const double step = static_cast<double>(p->step);
        t.root_c2 = static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(p->b2, step)));
        const double by = 1.0 / (1.0 - std::pow(p->b1, step));
        constexpr size_t kKept = size_t{128} << 20;  // half of the last-level cache
        sxk::AdamCounts counts{};  // of the table's tensors
        counts.b1 = p->b1; counts.b2 = p->b2; counts.grad_norm = p->grad_norm; counts.grad_scale = p->grad_scale;
        auto flush = [&] {
            if (counts.tensors) sxk::count_steps(counts, on.stream());
            sxk::adamw(t, eight, total > kKept, p->adopt != 0, on.stream());
            t.tensors = counts.tensors = 0;
        };
        constexpr int64_t kMostChunks = int64_t{1} << 30;  // of a table (a tensor of 2^40 elements has no more, and a lead's one)
        for (int64_t i = 0; i < n_tensors; i++) {
            const sxh_adamw_tensor& x = tensors[i];
            if (!x.n) continue;
            const int64_t chunks = (x.n + (eight ? 0 : sxk::adam_lead(x.exp_avg)) + sxk::kAdamChunk - 1) / sxk::kAdamChunk;
            if (t.tensors == sxk::kAdamTensors || (t.tensors && t.first[t.tensors] + chunks > kMostChunks)) flush();
            sxk::AdamTensor& a = t.t[t.tensors];
            a.param = x.param; a.master = x.master; a.grad = x.grad; a.m = x.exp_avg; a.v = x.exp_avg_sq;
            a.m_scale = x.exp_avg_scale; a.v_scale = x.exp_avg_sq_scale; a.n = x.n;
            a.rates = x.taken ? reinterpret_cast<const float*>(x.taken + 1) : nullptr;
            if (x.taken) {
                counts.taken[counts.tensors] = x.taken;
                counts.lr[counts.tensors++] = x.lr;
            }
            a.decay = static_cast<float>(1.0 - x.lr * x.weight_decay);
            a.rate = static_cast<float>(x.lr * by);
            a.key = eight ? sxk::adam_key(p->seed, p->step, i) : 0;
            a.param_type = x.param_type; a.grad_type = x.grad_type;
            if (t.tensors == 0) t.first[0] = 0;
            t.first[t.tensors + 1] = t.first[t.tensors] + static_cast<int32_t>(chunks);
            t.tensors++;
        }
        if (t.tensors) flush();
        on.done();
    });
}

}  // extern "C"
