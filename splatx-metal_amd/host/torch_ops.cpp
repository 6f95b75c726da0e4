// torch_ops.cpp — the learned heads' operators (include/splatx_hip.h) on torch tensors, for splatx_torch.py.
//
// A Python extension module: it checks the tensors, lets torch's allocator make the outputs and workspaces on the current
// stream, and enqueues the operator there. A small operator takes as long as its call: layer norm of 2000 x 45 takes 6.8 us
// (the same steps in Python with the C entries through ctypes took 11.1), its gradients 9.5 to 10.8 (15.5), an AdamW step of the
// head's ten tensors 7.2 (19.8), the norm of their gradients 6.0 (10.6); what is left is the launch, about 1 us an allocation and
// the pointers' checks. It links the library; torch's own libraries are those of the process, which has imported torch.
#include <ATen/ATen.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <string>
#include <vector>

#include "splatx_hip.h"

namespace {

PyObject* g_invalid = PyExc_ValueError;
PyObject* g_runtime = PyExc_RuntimeError;

// A Python exception that has been set.
struct Raised {};
[[noreturn]] void invalid(const std::string& msg) {
    PyErr_SetString(g_invalid, msg.c_str());
    throw Raised{};
}
void check(int32_t rc) {
    if (rc == SXH_OK) return;
    PyErr_SetString(rc == SXH_ERR_INVALID_ARGUMENT ? g_invalid : g_runtime, sxh_last_error());
    throw Raised{};
}

// Where a call runs: the backend, its device, torch's current stream there.
struct Call {
    sxh_backend* backend;
    int device;
    sxh_queue queue;
};
// An argument whose conversion failed for what it is; any other exception of the conversion (an interrupt, an error of the device
// whose tensor it is) is the caller's as it came.
[[noreturn]] void not_converted(const std::string& msg) {
    if (PyErr_ExceptionMatches(PyExc_TypeError) || PyErr_ExceptionMatches(PyExc_ValueError) || PyErr_ExceptionMatches(PyExc_OverflowError)) {
        PyErr_Clear();
        invalid(msg);
    }
    throw Raised{};
}
bool flag(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Raised{};
    return v != 0;
}
template <class T>
T number(PyObject* o, const char* name);
template <>
double number<double>(PyObject* o, const char* name) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) not_converted(std::string(name) + " must be a number");
    return v;
}
template <>
int64_t number<int64_t>(PyObject* o, const char* name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) not_converted(std::string(name) + " must be a whole number of 64 bits");
    return v;
}
template <>
uint64_t number<uint64_t>(PyObject* o, const char* name) {
    PyObject* whole = PyNumber_Index(o);
    const unsigned long long v = whole ? PyLong_AsUnsignedLongLong(whole) : ~0ull;
    Py_XDECREF(whole);
    if (v == ~0ull && PyErr_Occurred()) not_converted(std::string(name) + " must be a whole number of 0..2^64 - 1");
    return v;
}

// Other Python threads run while the outputs are allocated and the operator is enqueued.
struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    Unlocked() = default;
    Unlocked(const Unlocked&) = delete;
    ~Unlocked() { PyEval_RestoreThread(state); }
};

int type_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return SXH_TYPE_F32;
        case at::kBFloat16: return SXH_TYPE_BF16;
        case at::kHalf: return SXH_TYPE_F16;
        default: return -1;
    }
}

const at::Tensor& tensor(const Call& c, PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) invalid(std::string(name) + " must be a tensor");
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.get_device() != c.device) invalid(std::string(name) + " must be on cuda:" + std::to_string(c.device));
    if (t.layout() != at::kStrided) invalid(std::string(name) + " must be dense");
    return t;
}

// A tensor as rows of its last dimension.
struct Rows {
    const at::Tensor* t;
    void* p;
    int64_t rows, width, stride;
    int type;
};
Rows rows_of(const Call& c, PyObject* o, const char* name, const Rows* like = nullptr) {
    const at::Tensor& t = tensor(c, o, name);
    const int type = type_of(t);
    if (type < 0) invalid(std::string(name) + " must be float32, bfloat16 or float16");
    if (like && (type != like->type || t.sizes() != like->t->sizes())) invalid(std::string(name) + " must have the rows' type and shape");
    const int64_t d = t.dim();
    if (d == 0) invalid(std::string(name) + " has no rows");
    Rows r{&t, t.data_ptr(), 1, t.size(d - 1), 0, type};
    if (r.width > 1 && t.stride(d - 1) != 1) invalid(std::string(name) + ": the elements of a row must lie side by side");
    bool first = true;
    for (int64_t i = d - 2; i >= 0; i--) {  // from the innermost: the rows so far are `stride` apart, and this dimension's go on so
        if (t.size(i) != 1 && t.numel()) {
            if (!first && t.stride(i) != r.stride * r.rows) invalid(std::string(name) + ": rows that are not evenly spaced");
            if (first) r.stride = t.stride(i);
            first = false;
        }
        r.rows *= t.size(i);
    }
    if (r.rows <= 1) r.stride = r.width;
    return r;
}

void* vector(const Call& c, PyObject* o, const char* name, int64_t n, int* type, int allowed) {
    const at::Tensor& t = tensor(c, o, name);
    const int got = type_of(t);
    if ((got != SXH_TYPE_F32 && got != allowed) || got < 0 || t.numel() != n || !t.is_contiguous())
        invalid(std::string(name) + " must be " + std::to_string(n) + " contiguous elements of float32 or the rows' type");
    if (type) *type = got;
    return t.data_ptr();
}

// Contiguous rows like t's.
at::Tensor rows_like(const at::Tensor& t) { return at::empty(t.sizes(), t.options()); }
PyObject* none() { return Py_NewRef(Py_None); }
PyObject* give(const at::Tensor& t) { return t.defined() ? THPVariable_Wrap(t) : none(); }
bool given(PyObject* o) { return o != Py_None; }

Call call_of(PyObject* const* args) {
    return {reinterpret_cast<sxh_backend*>(number<int64_t>(args[0], "backend")), static_cast<int>(number<int64_t>(args[1], "device")),
            {reinterpret_cast<void*>(number<int64_t>(args[2], "stream"))}};
}

// f's result, with its exceptions as Python's; `n` arguments are due.
template <class F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t n, F&& f) {
    HANDLE_TH_ERRORS
    try {
        if (got != n) invalid(std::to_string(n) + " arguments expected");
        return f();
    } catch (const Raised&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// (backend, device, stream, x, weight, bias, eps, residual, stats) -> (y, h, mean, rstd)
PyObject* layer_norm_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 9, [&] {
        const Call c = call_of(a);
        const double eps = number<double>(a[6], "eps");
        const bool add = given(a[7]), stats = flag(a[8]);
        const Rows x = rows_of(c, a[3], "x");
        sxh_layer_norm_inputs in{};
        in.x = x.p; in.rows = x.rows; in.width = x.width; in.x_stride = x.stride;
        in.type = static_cast<uint8_t>(x.type);
        int wt = SXH_TYPE_F32;
        if (given(a[4])) in.weight = vector(c, a[4], "weight", x.width, &wt, x.type);
        if (given(a[5])) {
            int bt = SXH_TYPE_F32;
            in.bias = vector(c, a[5], "bias", x.width, &bt, x.type);
            if (given(a[4]) && bt != wt) invalid("bias must have the weight's type");
            wt = bt;
        }
        in.weight_type = static_cast<uint8_t>(wt);
        in.eps = static_cast<float>(eps);
        if (add) {
            const Rows r = rows_of(c, a[7], "residual", &x);
            in.residual = r.p;
            in.residual_stride = r.stride;
        }
        at::Tensor y, h, mean, rstd;
        int32_t rc;
        {
            const Unlocked unlocked;
            sxh_layer_norm_outputs out{};
            y = rows_like(*x.t);
            out.y = y.data_ptr();
            out.y_stride = out.h_stride = x.width;
            if (add) {
                h = rows_like(*x.t);
                out.h = h.data_ptr();
            }
            if (stats) {
                const auto shape = x.t->sizes().slice(0, x.t->dim() - 1);
                const at::TensorOptions options = x.t->options().dtype(at::kFloat);
                mean = at::empty(shape, options);
                rstd = at::empty(shape, options);
                out.mean = static_cast<float*>(mean.data_ptr());
                out.rstd = static_cast<float*>(rstd.data_ptr());
            }
            rc = sxh_layer_norm_fwd(c.backend, &in, &out, &c.queue);
        }
        check(rc);
        PyObject* t = PyTuple_New(4);
        if (!t) throw Raised{};
        PyTuple_SET_ITEM(t, 0, give(y));
        PyTuple_SET_ITEM(t, 1, add ? give(h) : Py_NewRef(a[3]));
        PyTuple_SET_ITEM(t, 2, give(mean));
        PyTuple_SET_ITEM(t, 3, give(rstd));
        return t;
    });
}

// (backend, device, stream, dy, h, mean, rstd, weight, dh, want_dx, want_dweight, want_dbias) -> (dx, dweight, dbias)
PyObject* layer_norm_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 12, [&] {
        const Call c = call_of(a);
        const bool want_dx = flag(a[9]), want_dweight = flag(a[10]), want_dbias = flag(a[11]);
        const Rows h = rows_of(c, a[4], "h"), dy = rows_of(c, a[3], "dy", &h);
        sxh_layer_norm_grads_in in{};
        in.dy = dy.p; in.h = h.p; in.dy_stride = dy.stride; in.h_stride = h.stride;
        in.rows = h.rows; in.width = h.width; in.type = static_cast<uint8_t>(h.type);
        in.mean = static_cast<float*>(vector(c, a[5], "mean", h.rows, nullptr, SXH_TYPE_F32));
        in.rstd = static_cast<float*>(vector(c, a[6], "rstd", h.rows, nullptr, SXH_TYPE_F32));
        int wt = SXH_TYPE_F32;
        if (given(a[7])) in.weight = vector(c, a[7], "weight", h.width, &wt, h.type);
        in.weight_type = static_cast<uint8_t>(wt);
        if (given(a[8])) {
            const Rows dh = rows_of(c, a[8], "dh", &h);
            in.dh = dh.p;
            in.dh_stride = dh.stride;
        }
        at::Tensor dx, dweight, dbias, work;
        int32_t rc;
        {
            const Unlocked unlocked;
            sxh_layer_norm_grads out{};
            const at::TensorOptions options = h.t->options(), weights = options.dtype(wt == SXH_TYPE_F32 ? at::kFloat : h.t->scalar_type());
            if (want_dx) {
                dx = rows_like(*h.t);
                out.dx = dx.data_ptr();
            }
            out.dx_stride = h.width;
            if (want_dweight) {
                dweight = at::empty({h.width}, weights);
                out.dweight = dweight.data_ptr();
            }
            if (want_dbias) {
                dbias = at::empty({h.width}, weights);
                out.dbias = dbias.data_ptr();
            }
            if (want_dweight || want_dbias) {
                out.workspace_bytes = sxh_layer_norm_bwd_workspace(h.rows, h.width);
                work = at::empty({out.workspace_bytes}, options.dtype(at::kByte));
                out.workspace = work.data_ptr();
            }
            rc = sxh_layer_norm_bwd(c.backend, &in, &out, &c.queue);
        }
        check(rc);
        PyObject* t = PyTuple_New(3);
        if (!t) throw Raised{};
        PyTuple_SET_ITEM(t, 0, give(dx));
        PyTuple_SET_ITEM(t, 1, give(dweight));
        PyTuple_SET_ITEM(t, 2, give(dbias));
        return t;
    });
}

// Item i of a list or tuple, which a number's own conversion to float may have made shorter.
PyObject* item(PyObject* seq, Py_ssize_t i, const char* name) {
    if (i >= PySequence_Fast_GET_SIZE(seq)) invalid(std::string(name) + " has changed during the call");
    return PySequence_Fast_GET_ITEM(seq, i);
}
// Item i of a list or tuple as a number; its conversion may take it out of the list.
double number_of(PyObject* seq, Py_ssize_t i, const char* name) {
    struct Held {
        PyObject* o;
        ~Held() { Py_DECREF(o); }
    } const held{Py_NewRef(item(seq, i, name))};
    return number<double>(held.o, name);
}
// What a call's lists have been asked for: it lives until the call ends, whatever becomes of the lists while other Python threads
// run. (Counted as Python's objects: as many counts of torch's own, which are atomic, take a call of fifty tensors 1 us more.)
struct Kept {
    std::vector<PyObject*> objects;
    explicit Kept(Py_ssize_t most) { objects.reserve(static_cast<size_t>(most)); }
    Kept(const Kept&) = delete;
    ~Kept() {
        for (PyObject* o : objects) Py_DECREF(o);
    }
};
// The tensors of a list or tuple: contiguous, of one of the allowed types.
struct List {
    PyObject* seq = nullptr;
    List(PyObject* o, const char* name) {
        if (!PyList_Check(o) && !PyTuple_Check(o)) invalid(std::string(name) + " must be a list of tensors");
        seq = Py_NewRef(o);
    }
    List(const List&) = delete;
    ~List() { Py_XDECREF(seq); }
    Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(seq); }
    const at::Tensor& at(Kept& kept, const Call& c, Py_ssize_t i, const char* name, const int64_t* numel = nullptr) const {
        PyObject* o = item(seq, i, name);
        const at::Tensor& t = tensor(c, o, name);
        kept.objects.push_back(Py_NewRef(o));
        if (!t.is_contiguous()) invalid(std::string(name) + " must be contiguous");
        if (numel && t.numel() != *numel)
            invalid(std::string(name) + "[" + std::to_string(i) + "]: " + std::to_string(t.numel()) + " elements, wanted are " + std::to_string(*numel));
        return t;
    }
};
void* floats(const at::Tensor& t, const char* name) {
    if (t.scalar_type() != at::kFloat) invalid(std::string(name) + " must be float32");
    return t.data_ptr();
}
uint8_t any_type(const at::Tensor& t, const char* name) {
    const int type = type_of(t);
    if (type < 0) invalid(std::string(name) + " must be float32, bfloat16 or float16");
    return static_cast<uint8_t>(type);
}

// (backend, device, stream, grads) -> norm
PyObject* grad_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 4, [&] {
        const Call c = call_of(a);
        const List grads(a[3], "grads");
        const Py_ssize_t count = grads.size();
        Kept kept(count);
        std::vector<sxh_norm_tensor> table(static_cast<size_t>(count));
        for (Py_ssize_t i = 0; i < count; i++) {
            const at::Tensor& t = grads.at(kept, c, i, "grads");
            table[i] = {t.data_ptr(), t.numel(), any_type(t, "grads")};
        }
        at::Tensor norm, work;
        int32_t rc;
        {
            const Unlocked unlocked;
            const at::TensorOptions options = at::TensorOptions().device(at::kCUDA, c.device);
            const int64_t bytes = sxh_grad_norm_workspace(count);
            norm = at::empty({}, options.dtype(at::kFloat));
            work = at::empty({bytes}, options.dtype(at::kByte));
            rc = sxh_grad_norm(c.backend, table.data(), count, static_cast<float*>(norm.data_ptr()), work.data_ptr(), bytes, &c.queue);
        }
        check(rc);
        return give(norm);
    });
}

// (backend, device, stream, params, grads, exp_avg, exp_avg_sq, step, lr, weight_decay, b1, b2, eps, master, grad_scale,
//  grad_norm, max_norm, exp_avg_scale, exp_avg_sq_scale, seed[, taken, adopt]) -> None
PyObject* adamw(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, std::max<Py_ssize_t>(20, std::min<Py_ssize_t>(n, 22)), [&] {
        const Call c = call_of(a);
        const bool counts = n > 20 && given(a[20]);
        const List params(a[3], "params"), grads(a[4], "grads"), m(a[5], "exp_avg"), v(a[6], "exp_avg_sq");
        const bool masters = given(a[13]), eight = given(a[17]);
        if (eight != given(a[18])) invalid("exp_avg_scale and exp_avg_sq_scale are given together");
        const List master(masters ? a[13] : a[3], "master"), m_scale(eight ? a[17] : a[3], "exp_avg_scale");
        const List v_scale(eight ? a[18] : a[3], "exp_avg_sq_scale"), taken(counts ? a[20] : a[3], "taken");
        const Py_ssize_t count = params.size();
        Kept kept(8 * count);
        std::vector<const at::Tensor*> stepped(static_cast<size_t>(count));
        for (const List* l : {&grads, &m, &v, &master, &m_scale, &v_scale, &taken})
            if (l->size() != count) invalid("as many gradients, moments, masters, scales and counts as params are wanted");
        const bool rates = PyList_Check(a[8]) || PyTuple_Check(a[8]), decays = PyList_Check(a[9]) || PyTuple_Check(a[9]);
        if ((rates && PySequence_Fast_GET_SIZE(a[8]) != count) || (decays && PySequence_Fast_GET_SIZE(a[9]) != count))
            invalid("lr and weight_decay are a number, or one for each tensor");
        const double lr = rates ? 0.0 : number<double>(a[8], "lr"), decay = decays ? 0.0 : number<double>(a[9], "weight_decay");
        std::vector<sxh_adamw_tensor> table(static_cast<size_t>(count));
        for (Py_ssize_t i = 0; i < count; i++) {
            table[i].lr = rates ? number_of(a[8], i, "lr") : lr;
            table[i].weight_decay = decays ? number_of(a[9], i, "weight_decay") : decay;
        }
        sxh_adamw_params p{};
        p.step = number<int64_t>(a[7], "step");
        p.seed = number<uint64_t>(a[19], "seed");
        p.b1 = number<double>(a[10], "b1");
        p.b2 = number<double>(a[11], "b2");
        p.eps = number<double>(a[12], "eps");
        p.grad_scale = static_cast<float>(number<double>(a[14], "grad_scale"));
        p.max_norm = static_cast<float>(number<double>(a[16], "max_norm"));
        p.state_bits = eight ? 8 : 32;
        p.adopt = n > 21 && flag(a[21]);
        // (all the numbers first: their conversions are the caller's code, which may change the lists)
        if (given(a[15])) p.grad_norm = static_cast<float*>(vector(c, a[15], "grad_norm", 1, nullptr, SXH_TYPE_F32));
        for (Py_ssize_t i = 0; i < count; i++) {
            sxh_adamw_tensor& t = table[i];
            const at::Tensor& param = *(stepped[i] = &params.at(kept, c, i, "params"));
            t.n = param.numel();
            t.param = param.data_ptr();
            t.param_type = any_type(param, "params");
            const at::Tensor& g = grads.at(kept, c, i, "grads", &t.n);
            t.grad = g.data_ptr();
            t.grad_type = any_type(g, "grads");
            const at::Tensor &em = m.at(kept, c, i, "exp_avg", &t.n), &ev = v.at(kept, c, i, "exp_avg_sq", &t.n);
            if (eight) {
                for (const at::Tensor* e : {&em, &ev})
                    if (e->scalar_type() != at::kFloat8_e4m3fn && e->scalar_type() != at::kByte)
                        invalid("exp_avg and exp_avg_sq with scales must be float8_e4m3fn or uint8");
                t.exp_avg = em.data_ptr();
                t.exp_avg_sq = ev.data_ptr();
                const int64_t blocks = (t.n + 255) / 256;
                t.exp_avg_scale = static_cast<float*>(floats(m_scale.at(kept, c, i, "exp_avg_scale", &blocks), "exp_avg_scale"));
                t.exp_avg_sq_scale = static_cast<float*>(floats(v_scale.at(kept, c, i, "exp_avg_sq_scale", &blocks), "exp_avg_sq_scale"));
            } else {
                t.exp_avg = floats(em, "exp_avg");
                t.exp_avg_sq = floats(ev, "exp_avg_sq");
            }
            if (counts) {
                constexpr int64_t kWords = 2;
                const at::Tensor& k = taken.at(kept, c, i, "taken", &kWords);
                if (k.scalar_type() != at::kLong) invalid("taken must be int64");
                t.taken = static_cast<int64_t*>(k.data_ptr());
            }
            if (masters) t.master = static_cast<float*>(floats(master.at(kept, c, i, "master", &t.n), "master"));
        }
        int32_t rc;
        {
            const Unlocked unlocked;
            rc = sxh_adamw(c.backend, table.data(), count, &p, &c.queue);
        }
        check(rc);
        // what autograd has saved of a parameter is no longer what it was
        for (const at::Tensor* t : stepped)
            if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
        return none();
    });
}

// A linear layer's activation, weights and groups: weight [out, in], or with ends [groups, out, in].
struct Layer {
    int activation;
    void *weight, *bias = nullptr;
    const at::Tensor* weights;
    const int64_t* ends = nullptr;
    int64_t in, out, groups = 0;
};
Layer layer_of(const Call& c, PyObject* weight, PyObject* bias, PyObject* ends, PyObject* activation, int type) {
    Layer l{};
    l.activation = static_cast<int>(std::clamp<int64_t>(number<int64_t>(activation, "activation"), -1, 255));
    if (l.activation < 0) invalid("activation must be one of SXH_ACT_*");
    const at::Tensor& w = tensor(c, weight, "weight");
    const int64_t lead = given(ends) ? 1 : 0;
    if (w.dim() != 2 + lead) invalid(lead ? "weight must be [groups, out, in]" : "weight must be [out, in]");
    if (type_of(w) != type || !w.is_contiguous()) invalid("weight must be contiguous, of the rows' type");
    l.weights = &w;
    l.weight = w.data_ptr();
    l.out = w.size(lead);
    l.in = w.size(lead + 1);
    if (given(ends)) {
        const at::Tensor& e = tensor(c, ends, "ends");
        l.groups = w.size(0);
        if (l.groups < 1) invalid("weight has no groups");
        if (e.scalar_type() != at::kLong || e.dim() != 1 || e.size(0) != l.groups || !e.is_contiguous())
            invalid("ends must be " + std::to_string(l.groups) + " contiguous elements of int64");
        l.ends = static_cast<const int64_t*>(e.data_ptr());
    }
    if (given(bias)) {
        const at::Tensor& b = tensor(c, bias, "bias");
        if (type_of(b) != type || !b.is_contiguous() || b.numel() != l.out * std::max<int64_t>(l.groups, 1))
            invalid("bias must be contiguous, of the rows' type, an element for each row of weight");
        l.bias = b.data_ptr();
    }
    return l;
}
// Rows of another width beside x's.
Rows rows_beside(const Call& c, PyObject* o, const char* name, const Rows& x, int64_t width) {
    const Rows r = rows_of(c, o, name);
    if (r.type != x.type || r.t->dim() != x.t->dim() || r.width != width || r.t->sizes().slice(0, r.t->dim() - 1) != x.t->sizes().slice(0, r.t->dim() - 1))
        invalid(std::string(name) + " must have the rows' type and shape, " + std::to_string(width) + " wide");
    return r;
}
at::Tensor rows_beside(const at::Tensor& t, int64_t width) {
    std::vector<int64_t> sizes(t.sizes().begin(), t.sizes().end());
    sizes.back() = width;
    return at::empty(sizes, t.options());
}

// (backend, device, stream, x, weight, bias, ends, activation, residual, want_pre) -> (y, pre)
PyObject* linear_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 10, [&] {
        const Call c = call_of(a);
        const bool want_pre = flag(a[9]);
        const Rows x = rows_of(c, a[3], "x");
        const Layer l = layer_of(c, a[4], a[5], a[6], a[7], x.type);
        if (x.width != l.in) invalid("x must be as wide as weight's rows");
        sxh_linear_inputs in{};
        in.x = x.p; in.weight = l.weight; in.bias = l.bias; in.ends = l.ends;
        in.rows = x.rows; in.in = l.in; in.out = l.out; in.groups = l.groups; in.x_stride = x.stride;
        in.type = static_cast<uint8_t>(x.type); in.activation = static_cast<uint8_t>(l.activation); in.clear = 1;
        if (given(a[8])) {
            const Rows r = rows_beside(c, a[8], "residual", x, l.out);
            in.residual = r.p;
            in.residual_stride = r.stride;
        }
        at::Tensor y, pre, work;
        int32_t rc;
        {
            const Unlocked unlocked;
            sxh_linear_outputs out{};
            y = rows_beside(*x.t, l.out);
            out.y = y.data_ptr();
            out.y_stride = out.pre_stride = l.out;
            if (want_pre) {
                pre = rows_beside(*x.t, l.out);
                out.pre = pre.data_ptr();
            }
            out.workspace_bytes = sxh_linear_fwd_workspace(&in);
            if (out.workspace_bytes) {
                work = at::empty({out.workspace_bytes}, x.t->options().dtype(at::kByte));
                out.workspace = work.data_ptr();
            }
            rc = sxh_linear_fwd(c.backend, &in, &out, &c.queue);
        }
        check(rc);
        PyObject* t = PyTuple_New(2);
        if (!t) throw Raised{};
        PyTuple_SET_ITEM(t, 0, give(y));
        PyTuple_SET_ITEM(t, 1, give(pre));
        return t;
    });
}

// (backend, device, stream, dy, x, weight, ends, pre, activation, want_dx, want_dweight, want_dbias) -> (dx, dweight, dbias)
PyObject* linear_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 12, [&] {
        const Call c = call_of(a);
        const bool want_dx = flag(a[9]), want_dweight = flag(a[10]), want_dbias = flag(a[11]);
        const Rows x = rows_of(c, a[4], "x");
        const Layer l = layer_of(c, a[5], Py_None, a[6], a[8], x.type);
        if (x.width != l.in) invalid("x must be as wide as weight's rows");
        const Rows dy = rows_beside(c, a[3], "dy", x, l.out);
        sxh_linear_grads_in in{};
        in.dy = dy.p; in.x = x.p; in.weight = l.weight; in.ends = l.ends;
        in.rows = x.rows; in.in = l.in; in.out = l.out; in.groups = l.groups; in.dy_stride = dy.stride; in.x_stride = x.stride;
        in.type = static_cast<uint8_t>(x.type); in.activation = static_cast<uint8_t>(l.activation); in.clear = 1;
        if (given(a[7])) {
            const Rows p = rows_beside(c, a[7], "pre", x, l.out);
            in.pre = p.p;
            in.pre_stride = p.stride;
        }
        if (given(a[7]) != (l.activation != SXH_ACT_NONE)) invalid("pre is given with an activation, and only then");
        at::Tensor dx, dweight, dbias, work;
        int32_t rc;
        {
            const Unlocked unlocked;
            sxh_linear_grads out{};
            const at::TensorOptions options = x.t->options();
            if (want_dx) {
                dx = rows_beside(*x.t, l.in);
                out.dx = dx.data_ptr();
            }
            out.dx_stride = l.in;
            if (want_dweight) {
                dweight = at::empty(l.weights->sizes(), options);
                out.dweight = dweight.data_ptr();
            }
            if (want_dbias) {
                dbias = at::empty(l.weights->sizes().slice(0, l.weights->dim() - 1), options);
                out.dbias = dbias.data_ptr();
            }
            out.workspace_bytes = sxh_linear_bwd_workspace(&in);
            if (out.workspace_bytes) {
                work = at::empty({out.workspace_bytes}, options.dtype(at::kByte));
                out.workspace = work.data_ptr();
            }
            rc = sxh_linear_bwd(c.backend, &in, &out, &c.queue);
        }
        check(rc);
        PyObject* t = PyTuple_New(3);
        if (!t) throw Raised{};
        PyTuple_SET_ITEM(t, 0, give(dx));
        PyTuple_SET_ITEM(t, 1, give(dweight));
        PyTuple_SET_ITEM(t, 2, give(dbias));
        return t;
    });
}

// (exception for invalid arguments, exception for failures at run time)
PyObject* set_errors(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 2, [&] {
        g_invalid = Py_NewRef(a[0]);
        g_runtime = Py_NewRef(a[1]);
        return none();
    });
}

PyMethodDef kMethods[] = {
    {"layer_norm_fwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(layer_norm_fwd)), METH_FASTCALL, nullptr},
    {"layer_norm_bwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(layer_norm_bwd)), METH_FASTCALL, nullptr},
    {"grad_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(grad_norm)), METH_FASTCALL, nullptr},
    {"adamw", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(adamw)), METH_FASTCALL, nullptr},
    {"linear_fwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear_fwd)), METH_FASTCALL, nullptr},
    {"linear_bwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear_bwd)), METH_FASTCALL, nullptr},
    {"set_errors", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(set_errors)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_splatx_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__splatx_torch() { return PyModule_Create(&kModule); }
