// The Python mirror's calls between logits and an update on plain torch CUDA
// tensors: reads their descriptors, allocates the outputs and calls the C ABI.
//
// Those calls have many small operands, or long lists of them, beside a kernel
// of a few microseconds: from Python a call with 6 operands took 25 us and a
// list of 38 gradients and outputs 69, most of it in reading attributes one by
// one.  Everything that is refused or out of the ordinary (descriptors that are
// not tensors, other devices or dtypes) gives None here, and the caller's own
// path says why or takes it.
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <vector>

#include "../../include/kernix_b200.h"

namespace {

// The library's entries, as the Python side has loaded them.
struct Entries {
    decltype(&kx_token_log_probs_f32) log_probs32;
    decltype(&kx_token_log_probs_f64) log_probs64;
    decltype(&kx_token_log_probs_backward_f32) backward32;
    decltype(&kx_token_log_probs_backward_f64) backward64;
    decltype(&kx_grad_norm_f32) norm32;
    decltype(&kx_grad_norm_f64) norm64;
    decltype(&kx_clip_grad_norm_f32) clip32;
    decltype(&kx_clip_grad_norm_f64) clip64;
    uint64_t workspace;
} entries;

// A strided tensor on device `dev` that the library can be handed as it lies.
bool plain(PyObject *o, int64_t dev) {
    if (!THPVariable_Check(o)) return false;
    const at::Tensor &t = THPVariable_Unpack(o);
    return t.layout() == at::kStrided && t.is_cuda() && t.get_device() == dev && t.has_storage() && !t.is_neg() &&
           !t.is_conj() && t.dim() <= KX_MAX_RANK;
}
bool plain(PyObject *o, int64_t dev, at::ScalarType type) {
    return plain(o, dev) && THPVariable_Unpack(o).scalar_type() == type;
}

void describe(const at::Tensor &t, kx_tensor *d) {
    *d = kx_tensor{};
    if (t.is_contiguous()) {
        d->data = t.mutable_data_ptr();
        d->storage_len = (uint64_t)t.numel();
    } else {
        d->data = t.storage().mutable_data();
        d->storage_len = t.storage().nbytes() / t.element_size();
        d->origin = (uint64_t)t.storage_offset();
    }
    d->rank = (uint32_t)t.dim();
    for (int64_t i = 0; i < t.dim(); ++i) {
        d->dims[i] = (uint64_t)t.size(i);
        d->strides[i] = t.stride(i);
    }
}
// A C-contiguous tensor's elements as one axis.
void describe_elements(const at::Tensor &t, kx_tensor *d) {
    *d = kx_tensor{};
    d->data = t.mutable_data_ptr();
    d->storage_len = d->dims[0] = (uint64_t)t.numel();
    d->rank = 1;
    d->strides[0] = 1;
}

// An operand that may be None; false if it is something else than asked for.
bool operand(PyObject *o, int64_t dev, at::ScalarType type, kx_tensor *d, const kx_tensor **at) {
    *at = nullptr;
    if (o == Py_None) return true;
    if (!plain(o, dev, type)) return false;
    describe(THPVariable_Unpack(o), d);
    *at = d;
    return true;
}

bool floating(PyObject *o, int64_t dev, at::ScalarType *type) {
    if (!plain(o, dev)) return false;
    *type = THPVariable_Unpack(o).scalar_type();
    return *type == at::kFloat || *type == at::kDouble;
}

PyObject *wrapped(const at::Tensor &t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}

// (handle, device, logits, tokens, temperature, top, entropy, error record) ->
// (status, log_probs, lse, entropy, top_log_probs, top_tokens), or None.
PyObject *token_log_probs(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 8) return PyErr_Format(PyExc_TypeError, "token_log_probs takes 8 arguments");
    auto *h = static_cast<kx_handle *>(PyLong_AsVoidPtr(a[0]));
    const int64_t dev = PyLong_AsLongLong(a[1]);
    const double temperature = PyFloat_AsDouble(a[4]);
    const int64_t top = PyLong_AsLongLong(a[5]);
    const bool entropy = PyObject_IsTrue(a[6]) == 1;
    auto *err = static_cast<kx_error *>(PyLong_AsVoidPtr(a[7]));
    if (PyErr_Occurred()) return nullptr;
    at::ScalarType type;
    kx_tensor d[7];
    const kx_tensor *logits, *tokens, *out[5] = {};
    if (!floating(a[2], dev, &type) || !operand(a[2], dev, type, &d[0], &logits) ||
        !operand(a[3], dev, at::kLong, &d[1], &tokens))
        Py_RETURN_NONE;
    const at::Tensor &x = THPVariable_Unpack(a[2]);
    if (x.dim() == 0) Py_RETURN_NONE;
    std::vector<int64_t> dims(x.sizes().begin(), x.sizes().end() - 1);
    at::Tensor made[5];
    auto make = [&](int i, const at::TensorOptions &options) {
        made[i] = at::empty(dims, options);
        describe(made[i], &d[2 + i]);
        out[i] = &d[2 + i];
    };
    if (tokens) make(0, x.options());
    make(1, x.options());
    if (entropy) make(2, x.options());
    if (top > 0) {
        dims.push_back(top);
        make(3, x.options());
        make(4, x.options().dtype(at::kLong));
    }
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = type == at::kFloat ? entries.log_probs32(h, logits, tokens, (float)temperature, out[0], out[1], out[2], out[3],
                                                  out[4], err)
                            : entries.log_probs64(h, logits, tokens, temperature, out[0], out[1], out[2], out[3],
                                                  out[4], err);
    Py_END_ALLOW_THREADS
    return Py_BuildValue("(iNNNNN)", rc, wrapped(made[0]), wrapped(made[1]), wrapped(made[2]), wrapped(made[3]),
                         wrapped(made[4]));
    END_HANDLE_TH_ERRORS
}

// (handle, device, logits, tokens, lse, entropy, grad_log_probs, grad_entropy,
// grad_lse, temperature, output or None, error record) -> (status, output), or None.
PyObject *token_log_probs_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 12) return PyErr_Format(PyExc_TypeError, "token_log_probs_backward takes 12 arguments");
    auto *h = static_cast<kx_handle *>(PyLong_AsVoidPtr(a[0]));
    const int64_t dev = PyLong_AsLongLong(a[1]);
    const double temperature = PyFloat_AsDouble(a[9]);
    auto *err = static_cast<kx_error *>(PyLong_AsVoidPtr(a[11]));
    if (PyErr_Occurred()) return nullptr;
    at::ScalarType type;
    kx_tensor d[8];
    const kx_tensor *in[7], *to;
    if (!floating(a[2], dev, &type)) Py_RETURN_NONE;
    for (int i = 0; i < 7; ++i)
        if (!operand(a[2 + i], dev, i == 1 ? at::kLong : type, &d[i], &in[i])) Py_RETURN_NONE;
    if (!operand(a[10], dev, type, &d[7], &to)) Py_RETURN_NONE;
    at::Tensor out;
    if (to) {
        out = THPVariable_Unpack(a[10]);
    } else {
        const at::Tensor &x = THPVariable_Unpack(a[2]);
        out = at::empty(x.sizes(), x.options());
        describe(out, &d[7]);
        to = &d[7];
    }
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = type == at::kFloat ? entries.backward32(h, in[0], in[1], in[2], in[3], in[4], in[5], in[6], (float)temperature,
                                                 to, err)
                            : entries.backward64(h, in[0], in[1], in[2], in[3], in[4], in[5], in[6], temperature, to,
                                                 err);
    Py_END_ALLOW_THREADS
    return Py_BuildValue("(iN)", rc, wrapped(out));
    END_HANDLE_TH_ERRORS
}

// (handle, device, list of gradients, list of outputs or None, max_norm, norm or
// None, error record) -> (status, norm), or None.
PyObject *grad_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7) return PyErr_Format(PyExc_TypeError, "grad_norm takes 7 arguments");
    auto *h = static_cast<kx_handle *>(PyLong_AsVoidPtr(a[0]));
    const int64_t dev = PyLong_AsLongLong(a[1]);
    const double max_norm = PyFloat_AsDouble(a[4]);
    auto *err = static_cast<kx_error *>(PyLong_AsVoidPtr(a[6]));
    if (PyErr_Occurred()) return nullptr;
    if (!PyList_CheckExact(a[2]) || (a[3] != Py_None && !PyList_CheckExact(a[3]))) Py_RETURN_NONE;
    const Py_ssize_t count = PyList_GET_SIZE(a[2]);
    const bool clip = a[3] != Py_None;
    if (count == 0 || (clip && PyList_GET_SIZE(a[3]) != count)) Py_RETURN_NONE;
    at::ScalarType type;
    if (!floating(PyList_GET_ITEM(a[2], 0), dev, &type)) Py_RETURN_NONE;
    std::vector<kx_tensor> grads((size_t)count), outs(clip ? (size_t)count : 0);
    for (Py_ssize_t i = 0; i < count; ++i) {
        PyObject *g = PyList_GET_ITEM(a[2], i), *o = clip ? PyList_GET_ITEM(a[3], i) : nullptr;
        if (!plain(g, dev, type) || (o && !plain(o, dev, type))) Py_RETURN_NONE;
        const at::Tensor &tg = THPVariable_Unpack(g);
        if (!o) {
            tg.is_contiguous() ? describe_elements(tg, &grads[i]) : describe(tg, &grads[i]);
            continue;
        }
        const at::Tensor &to = THPVariable_Unpack(o);
        if (tg.sizes() != to.sizes()) Py_RETURN_NONE;
        if (tg.is_contiguous() && to.is_contiguous()) {
            describe_elements(tg, &grads[i]);
            describe_elements(to, &outs[i]);
        } else {
            describe(tg, &grads[i]);
            describe(to, &outs[i]);
        }
    }
    kx_tensor d;
    const kx_tensor *at;
    if (!operand(a[5], dev, type, &d, &at)) Py_RETURN_NONE;
    const auto options = THPVariable_Unpack(PyList_GET_ITEM(a[2], 0)).options();
    at::Tensor norm;
    if (at) {
        norm = THPVariable_Unpack(a[5]);
    } else {
        norm = at::empty({}, options);
        describe(norm, &d);
    }
    const at::Tensor workspace = at::empty({(int64_t)entries.workspace}, options.dtype(at::kByte));
    void *ws = workspace.mutable_data_ptr();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    if (clip)
        rc = (type == at::kFloat ? entries.clip32 : entries.clip64)(h, grads.data(), (uint64_t)count, max_norm,
                                                                    outs.data(), &d, ws, entries.workspace, err);
    else
        rc = (type == at::kFloat ? entries.norm32 : entries.norm64)(h, grads.data(), (uint64_t)count, &d, ws,
                                                                    entries.workspace, err);
    Py_END_ALLOW_THREADS
    return Py_BuildValue("(iN)", rc, wrapped(norm));
    END_HANDLE_TH_ERRORS
}

// The addresses of the eight entries in Entries' order, and of
// kx_grad_norm_workspace.
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
    void *p[9];
    if (n != 9) return PyErr_Format(PyExc_TypeError, "bind takes 9 addresses");
    for (int i = 0; i < 9; ++i)
        if (!(p[i] = PyLong_AsVoidPtr(a[i]))) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
            return nullptr;
        }
    entries.log_probs32 = reinterpret_cast<decltype(entries.log_probs32)>(p[0]);
    entries.log_probs64 = reinterpret_cast<decltype(entries.log_probs64)>(p[1]);
    entries.backward32 = reinterpret_cast<decltype(entries.backward32)>(p[2]);
    entries.backward64 = reinterpret_cast<decltype(entries.backward64)>(p[3]);
    entries.norm32 = reinterpret_cast<decltype(entries.norm32)>(p[4]);
    entries.norm64 = reinterpret_cast<decltype(entries.norm64)>(p[5]);
    entries.clip32 = reinterpret_cast<decltype(entries.clip32)>(p[6]);
    entries.clip64 = reinterpret_cast<decltype(entries.clip64)>(p[7]);
    if (reinterpret_cast<decltype(&kx_grad_norm_workspace)>(p[8])(&entries.workspace) != KX_OK)
        return PyErr_Format(PyExc_RuntimeError, "kx_grad_norm_workspace");
    Py_RETURN_NONE;
}

template <typename F> PyCFunction fast(F f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

PyMethodDef methods[] = {
    {"bind", fast(bind), METH_FASTCALL, "the library's entries"},
    {"token_log_probs", fast(token_log_probs), METH_FASTCALL, "kx_token_log_probs_*"},
    {"token_log_probs_backward", fast(token_log_probs_backward), METH_FASTCALL, "kx_token_log_probs_backward_*"},
    {"grad_norm", fast(grad_norm), METH_FASTCALL, "kx_grad_norm_* and kx_clip_grad_norm_*"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kx_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kx_torch() {
    PyObject *m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch", TORCH_VERSION) < 0) {     // what it was built for
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
