// Python module _host: the group norm and gradient clipping as torch operators over the C ABI (include/msnet_hip.h), the group norm
// with its gradient.  Both work on calls of a few microseconds: reading a list's tensors from Python costs 0.6 us each (here 0.05),
// and a gradient written in Python another 25 us and the interpreter's lock on the autograd thread.  Only this file knows torch's
// C++ interface; libmsnet_hip.so does not, its entry points are handed over by address (bind).
//
// An operator takes ordinary arguments and returns None for all others: hipops.py then lays the tensors out, or says what is wrong.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <cmath>
#include <vector>

#include "../../include/msnet_hip.h"

namespace {

using at::Tensor;

decltype(&msnet_last_error) last_error;
decltype(&msnet_group_norm) norm_forward;
decltype(&msnet_group_norm_workspace_bytes) norm_forward_bytes;
decltype(&msnet_group_norm_backward) norm_backward;
decltype(&msnet_group_norm_backward_workspace_bytes) norm_backward_bytes;
decltype(&msnet_clip_grads) clip_grads;
decltype(&msnet_clip_grads_workspace_bytes) clip_bytes;

void succeed(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed: ", last_error()); }

int type_code(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kHalf ? 1 : t == at::kBFloat16 ? 2 : -1; }

// The type's code, or -1: not an ordinary tensor of the device.
int ordinary_code(const Tensor& t, c10::DeviceIndex device) {
    return t.defined() && t.layout() == at::kStrided && t.is_cuda() && t.get_device() == device && !t.is_neg() ? type_code(t.scalar_type()) : -1;
}

bool ordinary(const Tensor& t, c10::DeviceIndex device) { return ordinary_code(t, device) >= 0; }

// Forward-mode tangents are not carried on: a result without one would stand for a derivative of zero.  A call asks once whether any
// can exist (asking 1000 views and their outputs one by one took 45 us).
bool tangents_exist() { return c10::AutogradState::get_tls_state().get_fw_grad_mode() && torch::autograd::ForwardADLevel::try_get_by_idx(0); }

void refuse_tangent(const Tensor& t, const char* what) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), what,
                                " has no forward-mode derivative (use reverse mode, or hand it tensors without a tangent)");
}

void* stream_of(c10::DeviceIndex device) { return c10::hip::getCurrentHIPStream(device).stream(); }

Tensor workspace(size_t bytes, const Tensor& like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

template <class T = void> T* data(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }

// ---- group norm ------------------------------------------------------------------------------------------------------

struct Rows { int64_t sample = 0, row = 0; };

// As hipops._row_strides: positions at one distance, channels consecutive.
bool rows_of(const Tensor& t, Rows* r) {
    const auto shape = t.sizes(), st = t.strides();
    const int64_t dims = t.dim(), c = shape[dims - 1];
    if (t.is_contiguous()) {
        r->sample = t.numel() / std::max<int64_t>(shape[0], 1);
        r->row = c;
        return true;
    }
    if (c != 1 && st[dims - 1] != 1) return false;
    int64_t row = -1, expected = 0;
    for (int64_t i = dims - 2; i > 0; --i) {
        if (shape[i] == 1) continue;
        if (row < 0) row = expected = st[i];
        else if (st[i] != expected) return false;
        expected *= shape[i];
    }
    r->sample = st[0];
    r->row = row < 0 ? 0 : row;
    return true;
}

struct Dims { int n, c; long s; };

Dims dims_of(const Tensor& x) {
    const int64_t n = x.size(0), c = x.size(-1);
    return {(int)n, (int)c, (long)(n ? x.numel() / (n * c) : 0)};
}

Tensor forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, int64_t groups, double eps, int64_t act,
               const Tensor& stats) {
    const Dims d = dims_of(x);
    Rows xr, rr;
    TORCH_INTERNAL_ASSERT(rows_of(x, &xr) && (!residual.defined() || rows_of(residual, &rr)));
    Tensor y = at::empty(x.sizes(), x.options());
    const int code = type_code(x.scalar_type());
    const size_t bytes = norm_forward_bytes(code, d.n, d.s, d.c, (int)groups);
    const Tensor ws = workspace(bytes, x);
    succeed(norm_forward(data(x), data<float>(weight), data<float>(bias), data(residual), data(y), data<double>(stats), code, (int)act, d.n, d.s, d.c,
                         (int)groups, eps, xr.sample, xr.row, rr.sample, rr.row, d.s * d.c, d.c, data(ws), bytes, stream_of(x.get_device())),
            "msnet_group_norm");
    return y;
}

// While a stream is captured, a leaf must not still be held by a graph that was recorded on another stream: its accumulation node
// belongs to that stream, the captured backward would make the two wait for each other, and torch ends the process there.
void check_capture(const Tensor& t) {
    if (!t.defined() || !t.is_cuda() || !t.requires_grad() || !t.is_leaf()) return;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    if (!node) return;
    const auto theirs = node->stream();
    TORCH_CHECK(!theirs || *theirs == c10::hip::getCurrentHIPStream(t.get_device()).unwrap(),
                "group_norm is being captured while a graph recorded on another stream still holds one of its leaves: drop the results of earlier "
                "eager steps on these tensors first");
}

bool recorded_in_capture() {
    return c10::GradMode::is_enabled() && c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
}

struct GroupNorm : torch::autograd::Function<GroupNorm> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                          const std::optional<Tensor>& residual, int64_t groups, double eps, int64_t act) {
        const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
        const Tensor stats = at::empty({x.size(0), groups, 2}, x.options().dtype(at::kDouble));
        Tensor y = ::forward(x, w, b, r, groups, eps, act, stats);
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["act"] = act;
        ctx->saved_data["residual"] = r.defined();
        ctx->save_for_backward({x, w, b, act ? r : Tensor(), stats});
        return y;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &residual = saved[3], &stats = saved[4];
        const int64_t groups = ctx->saved_data["groups"].toInt(), act = ctx->saved_data["act"].toInt();
        torch::autograd::variable_list out(7);
        if (tangents_exist()) refuse_tangent(grads[0], "the gradient of group_norm");
        {
            c10::AutoGradMode off(false);
            Tensor dy = grads[0].resolve_neg();            // (a view with its sign bit to be applied is none the kernels can read)
            Rows yr, xr, rr;
            if (!rows_of(dy, &yr)) {
                dy = dy.contiguous();
                rows_of(dy, &yr);
            }
            TORCH_INTERNAL_ASSERT(rows_of(x, &xr) && (!residual.defined() || rows_of(residual, &rr)));
            const Dims d = dims_of(x);
            const auto floats = x.options().dtype(at::kFloat);
            size_t input = 0;                              // (only tensors that were given are counted)
            if (ctx->needs_input_grad(input++)) out[0] = at::empty(x.sizes(), x.options());
            if (weight.defined() && ctx->needs_input_grad(input++)) out[1] = at::empty({d.c}, floats);
            if (bias.defined() && ctx->needs_input_grad(input++)) out[2] = at::empty({d.c}, floats);
            if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(input++)) out[3] = act ? at::empty(x.sizes(), x.options()) : dy;
            const int code = type_code(x.scalar_type());
            const size_t bytes = norm_backward_bytes(code, d.n, d.s, d.c, (int)groups);
            const Tensor ws = workspace(bytes, x);
            succeed(norm_backward(data(dy), data(x), data<float>(weight), data<float>(bias), data(residual), data<double>(stats), data(out[0]),
                                  act ? data(out[3]) : nullptr, data<float>(out[1]), data<float>(out[2]), code, (int)act, d.n, d.s, d.c, (int)groups,
                                  yr.sample, yr.row, xr.sample, xr.row, rr.sample, rr.row, data(ws), bytes, stream_of(x.get_device())),
                    "msnet_group_norm_backward");
        }
        if (c10::GradMode::is_enabled()) {                 // the gradients are constants to autograd: differentiating them fails loudly
            auto error = std::make_shared<torch::autograd::DelayedError>("group_norm can be differentiated once only", 4);
            torch::autograd::variable_list known;
            for (auto& t : out)
                if (t.defined()) known.push_back(t.detach().requires_grad_(true));
            known = (*error)(std::move(known));
            size_t k = 0;
            for (auto& t : out)
                if (t.defined()) t = known[k++];
        }
        return out;
    }
};

bool tensor_or_none(PyObject* o, Tensor* t) {
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) return false;
    *t = THPVariable_Unpack(o);
    return t->defined();
}

// group_norm(x, groups, weight, bias, eps, act, residual): the result, or None where an argument is not ordinary.
PyObject* group_norm(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *px, *pw, *pb, *pr;
    long long groups;
    double eps;
    int act;
    if (!PyArg_ParseTuple(args, "OLOOdiO", &px, &groups, &pw, &pb, &eps, &act, &pr)) return nullptr;
    Tensor x, w, b, r;
    if (!tensor_or_none(px, &x) || !x.defined() || !tensor_or_none(pw, &w) || !tensor_or_none(pb, &b) || !tensor_or_none(pr, &r) || !x.is_cuda())
        Py_RETURN_NONE;
    if (tangents_exist())
        for (const Tensor* t : {&x, &w, &b, &r}) refuse_tangent(*t, "group_norm");
    const auto device = c10::hip::current_device();
    Rows any;
    if (!ordinary(x, device) || x.dim() < 2 || !rows_of(x, &any) || x.size(-1) < 1 || groups < 1 || x.size(-1) % groups || !(eps >= 0. && std::isfinite(eps)) ||
        x.size(0) > INT32_MAX || x.size(-1) > INT32_MAX)
        Py_RETURN_NONE;
    for (const Tensor* p : {&w, &b})
        if (p->defined() && (!ordinary(*p, device) || p->scalar_type() != at::kFloat || p->dim() != 1 || p->size(0) != x.size(-1) || !p->is_contiguous()))
            Py_RETURN_NONE;
    if (r.defined() && (!ordinary(r, device) || r.scalar_type() != x.scalar_type() || r.sizes() != x.sizes() || !rows_of(r, &any))) Py_RETURN_NONE;
    const bool grad = c10::GradMode::is_enabled() && (x.requires_grad() || (w.defined() && w.requires_grad()) || (b.defined() && b.requires_grad()) ||
                                                      (r.defined() && r.requires_grad()));
    if (grad && recorded_in_capture())
        for (const Tensor* t : {&x, &w, &b, &r}) check_capture(*t);
    const auto given = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
    return THPVariable_Wrap(grad ? GroupNorm::apply(x, given(w), given(b), given(r), (int64_t)groups, eps, (int64_t)act)
                                 : forward(x, w, b, r, groups, eps, act, Tensor()));
    END_HANDLE_TH_ERRORS
}

// ---- gradient clipping -----------------------------------------------------------------------------------------------

// clip(tensors, outs, max_norm): the norm, or None where a tensor is not ordinary (contiguous, of a known type, on the current
// device, not part of a graph being recorded; an output of its input's shape, and of its type or float32).  outs None: the norm alone.
PyObject* clip(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *list, *outs;
    double max_norm;
    if (!PyArg_ParseTuple(args, "O!Od", &PyList_Type, &list, &outs, &max_norm)) return nullptr;
    const bool write = outs != Py_None, grad = c10::GradMode::is_enabled(), tangents = tangents_exist();
    const Py_ssize_t n = PyList_GET_SIZE(list);
    if (n > INT32_MAX || (write && (!PyList_Check(outs) || PyList_GET_SIZE(outs) != n))) Py_RETURN_NONE;
    if (n && (!THPVariable_Check(PyList_GET_ITEM(list, 0)) || !THPVariable_Unpack(PyList_GET_ITEM(list, 0)).is_cuda())) Py_RETURN_NONE;      // (nothing to ask the GPU)
    const auto device = c10::hip::current_device();
    std::vector<const void*> in(n);
    std::vector<void*> out(write ? n : 0);
    std::vector<int64_t> lengths(n);
    std::vector<uint8_t> types(n), out_types(write ? n : 0);
    std::vector<at::TensorImpl*> written;                  // (the caller's list holds them, and the interpreter's lock is not given up)
    written.reserve(write ? n : 0);
    for (Py_ssize_t i = 0; i < n; ++i) {
        if (!THPVariable_Check(PyList_GET_ITEM(list, i))) Py_RETURN_NONE;
        const Tensor& t = THPVariable_Unpack(PyList_GET_ITEM(list, i));
        if (tangents) refuse_tangent(t, write ? "clip_grads" : "grad_norm");
        const int code = ordinary_code(t, device);
        if (code < 0 || !t.is_contiguous()) Py_RETURN_NONE;
        PyObject* po = write ? PyList_GET_ITEM(outs, i) : nullptr;
        if (grad && t.requires_grad()) Py_RETURN_NONE;
        in[i] = t.const_data_ptr();
        lengths[i] = t.numel();
        types[i] = (uint8_t)code;
        if (!write) continue;
        if (po == PyList_GET_ITEM(list, i)) {              // in place
            out[i] = t.mutable_data_ptr();
            out_types[i] = (uint8_t)code;
            written.push_back(t.unsafeGetTensorImpl());
            continue;
        }
        if (!THPVariable_Check(po)) Py_RETURN_NONE;
        const Tensor& o = THPVariable_Unpack(po);
        if (tangents) refuse_tangent(o, "clip_grads");
        const int out_code = ordinary_code(o, device);
        if (out_code < 0 || !o.is_contiguous() || (out_code != code && out_code != 0) || o.sizes() != t.sizes() || (grad && o.requires_grad()))
            Py_RETURN_NONE;
        out[i] = o.mutable_data_ptr();
        out_types[i] = (uint8_t)out_code;
        written.push_back(o.unsafeGetTensorImpl());
    }
    const auto options = at::TensorOptions().device(at::kCUDA, device);
    Tensor norm = at::empty({}, options.dtype(at::kFloat));
    const size_t bytes = clip_bytes(lengths.data(), (int)n);
    const Tensor ws = at::empty({(int64_t)bytes}, options.dtype(at::kByte));
    succeed(clip_grads(in.data(), write ? out.data() : nullptr, lengths.data(), types.data(), write ? out_types.data() : nullptr, (int)n, max_norm,
                       data<float>(norm), data(ws), bytes, stream_of(device)),
            "msnet_clip_grads");
    for (const auto& o : written)                          // behind autograd's back: what saved them finds out
        if (!o->is_inference()) o->bump_version();
    return THPVariable_Wrap(norm);
    END_HANDLE_TH_ERRORS
}

// refuse_tangents(what, tensors): an error if one of them has a tangent (anything else among them is passed over).
PyObject* refuse_tangents(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    const char* what;
    PyObject* tensors;
    if (!PyArg_ParseTuple(args, "sO", &what, &tensors)) return nullptr;
    const THPObjectPtr items(PySequence_Fast(tensors, "refuse_tangents() takes a sequence"));
    if (!items) return nullptr;
    if (!tangents_exist()) Py_RETURN_NONE;
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(items.get()); ++i)
        if (PyObject* o = PySequence_Fast_GET_ITEM(items.get(), i); THPVariable_Check(o)) refuse_tangent(THPVariable_Unpack(o), what);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// refuse_capture(tensors): an error where group_norm is being captured and one of the tensors must not be (check_capture).  For those
// that are laid out or cast first: what group_norm gets then is no leaf any more, but its graph ends at the same one.
PyObject* refuse_capture(PyObject*, PyObject* tensors) {
    HANDLE_TH_ERRORS
    const THPObjectPtr items(PySequence_Fast(tensors, "refuse_capture() takes a sequence"));
    if (!items) return nullptr;
    if (!recorded_in_capture()) Py_RETURN_NONE;
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(items.get()); ++i)
        if (PyObject* o = PySequence_Fast_GET_ITEM(items.get(), i); THPVariable_Check(o)) check_capture(THPVariable_Unpack(o));
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// bind({name: address}): the library's entry points.
PyObject* bind(PyObject*, PyObject* table) {
    if (!PyDict_Check(table)) return PyErr_Format(PyExc_TypeError, "bind() takes a dict of addresses");
    const auto get = [&](const char* name, auto& f) {
        PyObject* v = PyDict_GetItemString(table, name);
        void* p = v ? PyLong_AsVoidPtr(v) : nullptr;
        f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(p);
        if (!p && !PyErr_Occurred()) PyErr_Format(PyExc_KeyError, "%s", name);
        return p != nullptr;
    };
    if (!get("msnet_last_error", last_error) || !get("msnet_group_norm", norm_forward) || !get("msnet_group_norm_workspace_bytes", norm_forward_bytes) ||
        !get("msnet_group_norm_backward", norm_backward) || !get("msnet_group_norm_backward_workspace_bytes", norm_backward_bytes) ||
        !get("msnet_clip_grads", clip_grads) || !get("msnet_clip_grads_workspace_bytes", clip_bytes))
        return nullptr;
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"bind", bind, METH_O, "bind({name: address})"},
                         {"group_norm", group_norm, METH_VARARGS, "group_norm(x, groups, weight, bias, eps, act, residual)"},
                         {"refuse_tangents", refuse_tangents, METH_VARARGS, "refuse_tangents(what, tensors)"},
                         {"refuse_capture", refuse_capture, METH_O, "refuse_capture(tensors)"},
                         {"clip", clip, METH_VARARGS, "clip(tensors, outs, max_norm)"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
