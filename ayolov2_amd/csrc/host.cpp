// CPython helper of the operators whose host side is hot: one pass over a Python list of tensors that fills the ayolo_tensor
// array the C ABI takes (gradient norm, clipping, AdamW: a model has some hundred tensors in five lists per step), and layer
// norm's checks, buffers and autograd node (a norm of a few rows takes the GPU 3 us, a node written in Python 25 us of host time
// forward and, in autograd's own thread, 40 us backward).  No arithmetic here: the kernels are reached through the C ABI, whose
// addresses bind() is given.
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/version.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <stdexcept>
#include <string>

#include "../../include/ayolo.h"

namespace {

using at::Tensor;
using torch::autograd::variable_list;

PyObject* ayolo_error = nullptr;      // _lib.AyoloError
decltype(&ayolo_layer_norm_fwd) f_fwd = nullptr;
decltype(&ayolo_layer_norm_bwd) f_bwd = nullptr;
decltype(&ayolo_layer_norm_bwd_workspace) f_ws = nullptr;
decltype(&ayolo_last_error) f_error = nullptr;

struct Refused : std::runtime_error { using std::runtime_error::runtime_error; };

template <typename... A>
std::string text(const A&... a) { return c10::str(a...); }
#define REFUSE_UNLESS(cond, ...) do { if (!(cond)) throw Refused(text(__VA_ARGS__)); } while (0)

// equal for tensors of equal shape in equal memory order; dimensions of one element have no order
uint64_t layout_of(const Tensor& t) {
    if (!t.is_non_overlapping_and_dense()) return 0;
    uint64_t h = 1469598103934665603ull;
    const at::IntArrayRef size = t.sizes(), stride = t.strides();
    for (size_t d = 0; d < size.size(); ++d) {
        if (size[d] == 1) continue;
        h = (h ^ (uint64_t)size[d]) * 1099511628211ull;
        h = (h ^ (uint64_t)stride[d]) * 1099511628211ull;
    }
    return h | 1;
}

int dtype_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return AYOLO_F32;
        case at::kHalf: return AYOLO_F16;
        case at::kBFloat16: return AYOLO_BF16;
        case at::kByte: return AYOLO_U8;
        default: return -1;
    }
}

// rows(tensors, item=-1, given=None) -> bytes: one ayolo_tensor per entry; None gives an absent one; item >= 0 takes that item of each
// entry.  given, a list: counts up the version of every tensor whose entry there is not None (the kernels write through raw
// addresses, which autograd's version counters do not see; here, where each tensor is at hand, it costs next to nothing).
PyObject* rows(PyObject*, PyObject* args) {
    PyObject *list, *given = Py_None;
    int item = -1;
    if (!PyArg_ParseTuple(args, "O|iO", &list, &item, &given)) return nullptr;
    if (item > 1) {
        PyErr_SetString(PyExc_ValueError, "item: 0 or 1");
        return nullptr;
    }
    if (given != Py_None && !PyList_Check(given)) {
        PyErr_SetString(PyExc_TypeError, "given: a list");
        return nullptr;
    }
    PyObject* seq = PySequence_Fast(list, "a sequence of tensors is needed");
    if (!seq) return nullptr;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
    PyObject* out = PyBytes_FromStringAndSize(nullptr, n * (Py_ssize_t)sizeof(ayolo_tensor));
    bool ok = out != nullptr;
    for (Py_ssize_t i = 0; ok && i < n; ++i) {
        ayolo_tensor row{};
        row.device = -1;
        PyObject* e = PySequence_Fast_GET_ITEM(seq, i);
        if (e != Py_None && item >= 0) {
            const bool tuple = PyTuple_Check(e);
            if (!tuple && !PyList_Check(e)) e = nullptr;
            else if ((tuple ? PyTuple_GET_SIZE(e) : PyList_GET_SIZE(e)) != 2) e = nullptr;
            else e = tuple ? PyTuple_GET_ITEM(e, item) : PyList_GET_ITEM(e, item);
            if (!e) {
                PyErr_Format(PyExc_TypeError, "entry %zd is not a (codes, exponents) pair", i);
                ok = false;
                break;
            }
        }
        if (e != Py_None) {
            if (!THPVariable_Check(e)) {
                PyErr_Format(PyExc_TypeError, "entry %zd is not a tensor", i);
                ok = false;
            } else {
                try {
                    const Tensor& t = THPVariable_Unpack(e);
                    TORCH_CHECK(t.layout() == at::kStrided && !t.is_neg(), "not a strided tensor");
                    row.numel = t.numel();
                    row.dtype = dtype_of(t);
                    row.device = t.is_cuda() ? (int16_t)t.device().index() : (int16_t)-1;
                    row.layout = layout_of(t);
                    row.data = row.numel ? t.mutable_data_ptr() : nullptr;
                    row.present = 1;
                    if (given != Py_None && i < PyList_GET_SIZE(given) && PyList_GET_ITEM(given, i) != Py_None && !t.is_inference())
                        t.unsafeGetTensorImpl()->bump_version();
                } catch (const std::exception&) {
                    PyErr_Format(PyExc_TypeError, "entry %zd is not a strided tensor with memory of its own", i);
                    ok = false;
                }
            }
        }
        if (ok) reinterpret_cast<ayolo_tensor*>(PyBytes_AS_STRING(out))[i] = row;
    }
    Py_DECREF(seq);
    if (!ok) {
        Py_XDECREF(out);
        return nullptr;
    }
    return out;
}

// unlike(rows, model): the places where both arrays that rows() made hold a tensor and the first one's lies in another shape or
// memory order than the second one's, which is a dense block
PyObject* unlike(PyObject*, PyObject* args) {
    PyObject *a, *b;
    if (!PyArg_ParseTuple(args, "SS", &a, &b)) return nullptr;
    const Py_ssize_t n = PyBytes_GET_SIZE(a) / (Py_ssize_t)sizeof(ayolo_tensor);
    if (PyBytes_GET_SIZE(a) != PyBytes_GET_SIZE(b)) {
        PyErr_SetString(PyExc_ValueError, "arrays of different lengths");
        return nullptr;
    }
    const auto *x = reinterpret_cast<const ayolo_tensor*>(PyBytes_AS_STRING(a)), *y = reinterpret_cast<const ayolo_tensor*>(PyBytes_AS_STRING(b));
    PyObject* out = PyList_New(0);
    for (Py_ssize_t i = 0; out && i < n; ++i) {
        if (!x[i].present || !y[i].present || y[i].layout == 0 || x[i].layout == y[i].layout) continue;
        PyObject* k = PyLong_FromSsize_t(i);
        if (!k || PyList_Append(out, k) != 0) Py_CLEAR(out);
        Py_XDECREF(k);
    }
    return out;
}

// bump(tensors, given): counts up the version of every tensor of the first sequence (of every tensor of its pairs) whose entry in the
// second is not None: kernels write through raw addresses, which autograd's version counters do not see.
PyObject* bump(PyObject*, PyObject* args) {
    PyObject *a, *b;
    if (!PyArg_ParseTuple(args, "OO", &a, &b)) return nullptr;
    PyObject* list = PySequence_Fast(a, "a sequence of tensors is needed");
    PyObject* given = list ? PySequence_Fast(b, "a sequence of tensors is needed") : nullptr;
    if (!given) {
        Py_XDECREF(list);
        return nullptr;
    }
    auto one = [](PyObject* e) {
        if (!THPVariable_Check(e)) return;
        const Tensor& t = THPVariable_Unpack(e);
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    };
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(list) && i < PySequence_Fast_GET_SIZE(given); ++i) {
        if (PySequence_Fast_GET_ITEM(given, i) == Py_None) continue;
        PyObject* e = PySequence_Fast_GET_ITEM(list, i);
        if (PyTuple_Check(e)) for (Py_ssize_t k = 0; k < PyTuple_GET_SIZE(e); ++k) one(PyTuple_GET_ITEM(e, k));
        else if (PyList_Check(e)) for (Py_ssize_t k = 0; k < PyList_GET_SIZE(e); ++k) one(PyList_GET_ITEM(e, k));
        else one(e);
    }
    Py_DECREF(list);
    Py_DECREF(given);
    Py_RETURN_NONE;
}

// ------------------------------------------------------------------------------------------------------- layer norm
// Where the rows (the last dimension) of an operand lie.  Leading dimensions may have any strides that two levels describe (a
// channel slice of a wider map, a window of a batch of sequences); anything else is copied, and `t` becomes the copy.
ayolo_rows row_view(Tensor& t) {
    const int64_t C = t.size(-1);
    ayolo_rows r{};
    if (!t.is_contiguous()) {
        int64_t n[2] = {1, 1}, st[2] = {0, 0};
        int levels = 0;
        bool fits = C == 1 || t.stride(-1) == 1;
        for (int64_t d = t.dim() - 2; d >= 0 && fits; --d) {
            if (t.size(d) == 1) continue;
            if (levels > 0 && t.stride(d) == n[levels - 1] * st[levels - 1]) n[levels - 1] *= t.size(d);
            else if (levels == 2) fits = false;
            else { n[levels] = t.size(d); st[levels++] = t.stride(d); }
        }
        if (fits) {
            r.data = t.data_ptr();
            r.stride = levels ? st[0] : C;
            if (levels == 2) { r.outer_stride = st[1]; r.inner = n[0]; }
            return r;
        }
        t = t.contiguous();
    }
    r.data = t.data_ptr();
    r.stride = C;
    return r;
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void checked(int rc, const char* what) {
    if (rc != 0) throw Refused(text(what, " failed (rc=", rc, "): ", f_error()));
}

// The gain and bias as the kernels read them: both of x's type, or both fp32.
at::ScalarType params_type(const Tensor& w, const Tensor& b, at::ScalarType dt) {
    return (w.defined() || b.defined()) && (!w.defined() || w.scalar_type() == dt) && (!b.defined() || b.scalar_type() == dt) ? dt : at::kFloat;
}
Tensor as_param(const Tensor& t, at::ScalarType dt) { return t.defined() ? t.to(dt).contiguous() : t; }      // t itself where it fits

// x laid out so that dimension `dim` is innermost
Tensor empty_along(const Tensor& x, int64_t dim) {
    at::DimVector strides(x.dim());
    int64_t n = 1;
    strides[dim] = 1;
    n *= x.size(dim);
    for (int64_t d = x.dim() - 1; d >= 0; --d) {
        if (d == dim) continue;
        strides[d] = n;
        n *= std::max<int64_t>(x.size(d), 1);
    }
    return at::empty_strided(x.sizes(), strides, x.options());
}
Tensor along(const Tensor& t, int64_t dim) { return !t.defined() || dim == t.dim() - 1 ? t : t.movedim(dim, -1); }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// Below autograd (no views or graph are recorded in here).
struct Norm { Tensor y, s, mean, rstd, w; };
Norm norm_forward(const Tensor& x0, const Tensor& r0, const Tensor& w0, const Tensor& b0, double eps, int64_t dim, bool stats) {
    const at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x0.device());
    const at::ScalarType wdt = params_type(w0, b0, x0.scalar_type());
    Tensor x = along(x0, dim), r = along(r0, dim);
    const int64_t C = x.size(-1), n = x.numel() / C;
    Norm o;
    o.w = as_param(w0, wdt);
    const Tensor b = as_param(b0, wdt);
    o.y = empty_along(x0, dim);
    if (r.defined()) o.s = empty_along(x0, dim);
    if (stats) {
        o.mean = at::empty({n}, x.options().dtype(at::kFloat));
        o.rstd = at::empty({n}, x.options().dtype(at::kFloat));
    }
    const int dt = dtype_of(x);
    const ayolo_rows xr = row_view(x);
    ayolo_rows rr{};
    if (r.defined()) rr = row_view(r);
    checked(f_fwd(dt, &xr, r.defined() ? &rr : nullptr, n, C, ptr(o.w), ptr(b), wdt == at::kFloat ? AYOLO_F32 : dt, (float)eps, ptr(o.y),
                  ptr(o.s), (float*)ptr(o.mean), (float*)ptr(o.rstd), stream_of(x)),
            "ayolo_layer_norm_fwd");
    return o;
}

// Whether torch's calls are recorded to be run later (jit.trace, make_fx and what builds on it): the record would hold the buffers
// that are made in here and not the kernel that fills them.
bool recorded() {
    using c10::impl::TorchDispatchModeKey;
    using c10::impl::TorchDispatchModeTLS;
    if (torch::jit::tracer::isTracing()) return true;
    if (!TorchDispatchModeTLS::any_modes_set()) return false;
    for (const auto k : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL})
        if (TorchDispatchModeTLS::get_mode(k).has_value()) return true;
    return false;
}

// Its edges: x, residual, weight, bias.
struct LayerNormBackward : torch::autograd::Node {
    torch::autograd::SavedVariable s, w, mean, rstd;
    int64_t dim = 0;
    bool sum_kept = false;                                 // s is this node's output (the residual sum), not its input
    at::ScalarType ptype = at::kFloat, wtype = at::kFloat, btype = at::kFloat;

    std::string name() const override { return "LayerNormBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        s.reset_data();
        w.reset_data();
        mean.reset_data();
        rstd.reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        REFUSE_UNLESS(!recorded(), "layer_norm: its backward cannot be traced");
        const bool nx = task_should_compute_output(0), nr = task_should_compute_output(1), nw = task_should_compute_output(2),
                   nb = task_should_compute_output(3);
        Tensor dy = grads[0], q = grads.size() > 1 ? grads[1] : Tensor(), dx, dw, db;
        variable_list out(4);
        if (!dy.defined()) {                               // only the residual sum was used
            out[0] = nx ? q : Tensor();
            out[1] = nr ? q : Tensor();
            return out;
        }
        {
            const Tensor s0 = s.unpack(sum_kept ? shared_from_this() : nullptr), gain = w.unpack(), mu = mean.unpack(), rs = rstd.unpack();
            const at::AutoDispatchBelowADInplaceOrView below;
            const c10::DeviceGuard guard(s0.device());
            Tensor x = along(s0, dim);
            if (dy.is_neg()) dy = dy.resolve_neg();
            if (q.defined() && q.is_neg()) q = q.resolve_neg();
            dy = along(dy.scalar_type() == x.scalar_type() ? dy : dy.to(x.scalar_type()), dim);
            if (q.defined()) q = along(q.scalar_type() == x.scalar_type() ? q : q.to(x.scalar_type()), dim);
            const int64_t C = x.size(-1), n = x.numel() / C;
            const int dt = dtype_of(x);
            if (nx || nr) dx = empty_along(s0, dim);
            if (nw) dw = at::empty({C}, x.options().dtype(ptype));
            if (nb) db = at::empty({C}, x.options().dtype(ptype));
            const size_t need = nw || nb ? f_ws(dt, n, C) : 0;
            const Tensor ws = need ? at::empty({(int64_t)need}, x.options().dtype(at::kByte)) : Tensor();
            const ayolo_rows sr = row_view(x), gr = row_view(dy);
            ayolo_rows qr{};
            if (q.defined()) qr = row_view(q);
            checked(f_bwd(dt, &sr, &gr, q.defined() ? &qr : nullptr, n, C, ptr(gain), ptype == at::kFloat ? AYOLO_F32 : dt, (const float*)ptr(mu),
                          (const float*)ptr(rs), ptr(dx), ptr(dw), ptr(db), ptr(ws), need, stream_of(x)),
                    "ayolo_layer_norm_bwd");
            if (nw && wtype != ptype) dw = dw.to(wtype);
            if (nb && btype != ptype) db = db.to(btype);
        }
        out = {nx ? dx : Tensor(), nr ? dx : Tensor(), dw, db};
        if (at::GradMode::is_enabled()) {                  // create_graph: what was computed here has no derivative
            variable_list given;
            for (auto& t : out)
                if (t.defined()) given.push_back(t.detach().requires_grad_(true));
            const auto stop = std::make_shared<torch::autograd::DelayedError>("layer_norm is differentiable once", (int)given.size());
            const variable_list marked = (*stop)(std::move(given));
            size_t at = 0;
            for (auto& t : out)
                if (t.defined()) t = marked[at++];
        }
        return out;
    }
};

variable_list norm_with_graph(const Tensor& x, const Tensor& r, const Tensor& w, const Tensor& b, double eps, int64_t dim) {
    Norm o = norm_forward(x, r, w, b, eps, dim, true);
    const std::shared_ptr<LayerNormBackward> node(new LayerNormBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, r, w, b));
    node->dim = dim;
    node->sum_kept = r.defined();
    node->ptype = params_type(w, b, x.scalar_type());
    if (w.defined()) node->wtype = w.scalar_type();
    if (b.defined()) node->btype = b.scalar_type();
    variable_list out = {o.y};
    if (r.defined()) out.push_back(o.s);
    torch::autograd::set_history(out, node);
    node->s = torch::autograd::SavedVariable(r.defined() ? out[1] : x, r.defined());
    node->w = torch::autograd::SavedVariable(o.w, false);
    node->mean = torch::autograd::SavedVariable(o.mean, false);
    node->rstd = torch::autograd::SavedVariable(o.rstd, false);
    return out;
}

// layer_norm(x, weight, bias, eps, residual, dim): y, or (y, x + residual)
PyObject* layer_norm(PyObject*, PyObject* args) {
    PyObject *px, *pw, *pb, *pr;
    double eps;
    long long dim;
    if (!PyArg_ParseTuple(args, "OOOdOL", &px, &pw, &pb, &eps, &pr, &dim)) return nullptr;
    try {
        auto take = [](PyObject* o, const char* name, bool needed) -> Tensor {
            if (o == Py_None && !needed) return Tensor();
            REFUSE_UNLESS(THPVariable_Check(o), "layer_norm: ", name, " is not a tensor");
            const Tensor& t = THPVariable_Unpack(o);
            return t.layout() == at::kStrided && t.is_neg() ? t.resolve_neg() : t;       // (a view with its negation still to be done)
        };
        REFUSE_UNLESS(!recorded(), "layer_norm: cannot be traced; run the module that holds it eagerly");
        const Tensor x = take(px, "x", true), w = take(pw, "weight", false), b = take(pb, "bias", false), r = take(pr, "residual", false);
        REFUSE_UNLESS(x.is_cuda(), "layer_norm: the HIP path needs a tensor on the GPU (got ", x.device(), "); there is no CPU fallback");
        const int dt = dtype_of(x);
        REFUSE_UNLESS(x.layout() == at::kStrided && dt >= 0 && dt != AYOLO_U8, "layer_norm: unsupported dtype ", x.scalar_type());
        REFUSE_UNLESS(x.dim() > 0 && -x.dim() <= dim && dim < x.dim(), "layer_norm: no dimension ", dim, " in shape ", x.sizes());
        if (dim < 0) dim += x.dim();
        const int64_t C = x.size(dim);
        REFUSE_UNLESS(C > 0 && C < (1ll << 30) && x.numel() / C < (1ll << 31), "layer_norm: shape ", x.sizes());
        for (const auto& p : {std::make_pair(&w, "weight"), std::make_pair(&b, "bias")}) {
            const Tensor& t = *p.first;
            REFUSE_UNLESS(!t.defined() || (t.dim() == 1 && t.size(0) == C && t.device() == x.device() && t.is_floating_point()),
                          "layer_norm: ", p.second, " must hold ", C, " floating values on ", x.device());
        }
        REFUSE_UNLESS(!r.defined() || (r.sizes() == x.sizes() && r.scalar_type() == x.scalar_type() && r.device() == x.device() && r.layout() == at::kStrided),
                      "layer_norm: residual must have x's shape ", x.sizes(), ", type ", x.scalar_type(), " and device ", x.device());
        REFUSE_UNLESS(eps >= 0.0, "layer_norm: eps=", eps);
        // (a null address would stand for an operand that is not given)
        for (const auto& p : {std::make_pair(&x, "x"), std::make_pair(&w, "weight"), std::make_pair(&b, "bias"), std::make_pair(&r, "residual")}) {
            const Tensor& t = *p.first;
            REFUSE_UNLESS(!t.defined() || t.numel() == 0 || (t.has_storage() && t.storage().data()), "layer_norm: ", p.second, " has no memory of its own");
        }
        for (const Tensor* t : {&x, &w, &b, &r}) REFUSE_UNLESS(!torch::autograd::isFwGradDefined(*t), "layer_norm has no forward-mode derivative");
        variable_list out;
        auto grad = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
        if (at::GradMode::is_enabled() && (grad(x) || grad(r) || grad(w) || grad(b))) {
            out = norm_with_graph(x, r, w, b, eps, dim);
        } else {
            const Norm o = norm_forward(x, r, w, b, eps, dim, false);
            out.push_back(o.y);
            if (r.defined()) out.push_back(o.s);
        }
        PyObject* y = THPVariable_Wrap(out[0]);
        if (out.size() == 1 || !y) return y;
        PyObject* s = THPVariable_Wrap(out[1]);
        PyObject* both = s ? PyTuple_Pack(2, y, s) : nullptr;
        Py_DECREF(y);
        Py_XDECREF(s);
        return both;
    } catch (const Refused& e) {
        PyErr_SetString(ayolo_error ? ayolo_error : PyExc_RuntimeError, e.what());
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}

// bind(AyoloError, address of ayolo_layer_norm_fwd, _bwd, _bwd_workspace, ayolo_last_error)
PyObject* bind(PyObject*, PyObject* args) {
    PyObject* err;
    unsigned long long a, b, c, d;
    if (!PyArg_ParseTuple(args, "OKKKK", &err, &a, &b, &c, &d)) return nullptr;
    Py_INCREF(err);
    Py_XDECREF(ayolo_error);
    ayolo_error = err;
    f_fwd = (decltype(f_fwd))a;
    f_bwd = (decltype(f_bwd))b;
    f_ws = (decltype(f_ws))c;
    f_error = (decltype(f_error))d;
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"rows", rows, METH_VARARGS, "rows(tensors, item=-1, given=None) -> bytes of ayolo_tensor"},
                         {"unlike", unlike, METH_VARARGS, "unlike(rows, model): places in another shape or memory order"},
                         {"bump", bump, METH_VARARGS, "bump(tensors, given): count up the versions of the tensors that are given"},
                         {"layer_norm", layer_norm, METH_VARARGS, "layer_norm(x, weight, bias, eps, residual, dim)"},
                         {"bind", bind, METH_VARARGS, "bind(AyoloError, fwd, bwd, bwd_workspace, last_error)"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() {
    PyObject* m = PyModule_Create(&module);
    if (m && (PyModule_AddStringConstant(m, "built_for_python", PY_VERSION) != 0 || PyModule_AddStringConstant(m, "built_for_torch", TORCH_VERSION) != 0)) Py_CLEAR(m);
    return m;
}
