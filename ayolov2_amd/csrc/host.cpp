// CPython helper of the tensor-list operators (gradient norm, clipping, AdamW): one pass over a Python list of tensors that
// fills the ayolo_tensor array the C ABI takes.  A model has some hundred tensors in five lists per step; asking each for its
// address, size, type and strides from Python costs more host time than the step costs the GPU.  No arithmetic here.
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/ayolo.h"

namespace {

// equal for tensors of equal shape in equal memory order; dimensions of one element have no order
uint64_t layout_of(const at::Tensor& t) {
    if (!t.is_non_overlapping_and_dense()) return 0;
    uint64_t h = 1469598103934665603ull;
    for (int64_t d = 0; d < t.dim(); ++d) {
        if (t.size(d) == 1) continue;
        h = (h ^ (uint64_t)t.size(d)) * 1099511628211ull;
        h = (h ^ (uint64_t)t.stride(d)) * 1099511628211ull;
    }
    return h | 1;
}

int dtype_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return AYOLO_F32;
        case at::kHalf: return AYOLO_F16;
        case at::kBFloat16: return AYOLO_BF16;
        case at::kByte: return AYOLO_U8;
        default: return -1;
    }
}

// rows(tensors, item=-1) -> bytes: one ayolo_tensor per entry; None gives an absent one; item >= 0 takes that item of each entry
PyObject* rows(PyObject*, PyObject* args) {
    PyObject* list;
    int item = -1;
    if (!PyArg_ParseTuple(args, "O|i", &list, &item)) return nullptr;
    PyObject* seq = PySequence_Fast(list, "a sequence of tensors is needed");
    if (!seq) return nullptr;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
    PyObject* out = PyBytes_FromStringAndSize(nullptr, n * (Py_ssize_t)sizeof(ayolo_tensor));
    bool ok = out != nullptr;
    for (Py_ssize_t i = 0; ok && i < n; ++i) {
        ayolo_tensor row{};
        row.device = -1;
        PyObject* e = PySequence_Fast_GET_ITEM(seq, i);
        PyObject* held = nullptr;
        if (e != Py_None && item >= 0) {
            held = PySequence_Check(e) && !THPVariable_Check(e) ? PySequence_GetItem(e, item) : nullptr;
            if (!held) {
                PyErr_Clear();
                PyErr_Format(PyExc_TypeError, "entry %zd is not a (codes, exponents) pair", i);
                ok = false;
                break;
            }
            e = held;
        }
        if (e != Py_None) {
            if (!THPVariable_Check(e)) {
                PyErr_Format(PyExc_TypeError, "entry %zd is not a tensor", i);
                ok = false;
            } else {
                try {
                    const at::Tensor& t = THPVariable_Unpack(e);
                    TORCH_CHECK(t.layout() == at::kStrided, "not a strided tensor");
                    row.numel = t.numel();
                    row.dtype = dtype_of(t);
                    row.device = t.is_cuda() ? (int16_t)t.device().index() : (int16_t)-1;
                    row.layout = layout_of(t);
                    row.data = row.numel ? t.mutable_data_ptr() : nullptr;
                    row.present = 1;
                } catch (const std::exception&) {
                    PyErr_Format(PyExc_TypeError, "entry %zd is not a strided tensor with memory of its own", i);
                    ok = false;
                }
            }
        }
        Py_XDECREF(held);
        if (ok) reinterpret_cast<ayolo_tensor*>(PyBytes_AS_STRING(out))[i] = row;
    }
    Py_DECREF(seq);
    if (!ok) {
        Py_XDECREF(out);
        return nullptr;
    }
    return out;
}

PyMethodDef methods[] = {{"rows", rows, METH_VARARGS, "rows(tensors, item=-1) -> bytes of ayolo_tensor"}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
