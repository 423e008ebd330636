// Python module _host: reads the addresses, lengths and types of a list of tensors in one call.  A model's gradients are hundreds of
// tensors, and asking each for them from Python costs more than the kernels that then work on them (0.6 us a tensor, here 0.02).
// Only this file knows torch's C++ interface; libmsnet_hip.so does not.
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

namespace {

int type_code(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kHalf ? 1 : t == at::kBFloat16 ? 2 : -1; }

const at::Tensor* ordinary(PyObject* o, long device) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || t.get_device() != device || type_code(t.scalar_type()) < 0 || !t.is_contiguous())
        return nullptr;
    return &t;
}

void put(std::string& s, uint64_t v) { s.append(reinterpret_cast<const char*>(&v), 8); }

PyObject* bytes_of(const std::string& s) { return PyBytes_FromStringAndSize(s.data(), (Py_ssize_t)s.size()); }

// tables(tensors, outs or None, device) -> (pointers, out pointers, lengths, types, out types) as bytes objects, or None where any of
// the tensors is not an ordinary one (contiguous, float32 / float16 / bfloat16, on that device; an output of the same shape, of the
// same type or float32, and without a gradient of its own): the caller then finds out what to do or to say.
PyObject* tables(PyObject*, PyObject* args) {
    PyObject *list, *outs;
    long device;
    if (!PyArg_ParseTuple(args, "O!Ol", &PyList_Type, &list, &outs, &device)) return nullptr;
    const bool write = outs != Py_None;
    if (write && (!PyList_Check(outs) || PyList_GET_SIZE(outs) != PyList_GET_SIZE(list))) Py_RETURN_NONE;
    try {
        const Py_ssize_t n = PyList_GET_SIZE(list);
        std::string in, out, lengths, types, out_types;
        in.reserve(8 * n); lengths.reserve(8 * n); types.reserve(n);
        if (write) { out.reserve(8 * n); out_types.reserve(n); }
        for (Py_ssize_t i = 0; i < n; ++i) {
            const at::Tensor* t = ordinary(PyList_GET_ITEM(list, i), device);
            if (!t) Py_RETURN_NONE;
            put(in, (uint64_t)t->const_data_ptr());
            put(lengths, (uint64_t)t->numel());
            types.push_back((char)type_code(t->scalar_type()));
            if (!write) continue;
            const at::Tensor* o = ordinary(PyList_GET_ITEM(outs, i), device);
            if (!o || (o->scalar_type() != t->scalar_type() && o->scalar_type() != at::kFloat) || (o != t && o->sizes() != t->sizes()) ||
                (o->requires_grad() && c10::GradMode::is_enabled()))
                Py_RETURN_NONE;
            put(out, (uint64_t)o->mutable_data_ptr());
            out_types.push_back((char)type_code(o->scalar_type()));
        }
        return Py_BuildValue("(NNNNN)", bytes_of(in), bytes_of(out), bytes_of(lengths), bytes_of(types), bytes_of(out_types));
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// written(tensors): their values changed behind autograd's back; what saved them finds out by their version.
PyObject* written(PyObject*, PyObject* list) {
    if (!PyList_Check(list)) return PyErr_Format(PyExc_TypeError, "written() takes a list of tensors");
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) {
        PyObject* o = PyList_GET_ITEM(list, i);
        if (THPVariable_Check(o) && !THPVariable_Unpack(o).is_inference()) THPVariable_Unpack(o).unsafeGetTensorImpl()->bump_version();
    }
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"tables", tables, METH_VARARGS, "tables(tensors, outs, device)"},
                         {"written", written, METH_O, "written(tensors)"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
