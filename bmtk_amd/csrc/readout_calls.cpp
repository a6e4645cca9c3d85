// The calls of bmtk_amd/readout.py for arguments that are what they should be: checked, results allocated and the C ABI called without the steps in
// between that a Python function takes for each of its arguments (gated_scan of one step: 12.4 us in Python).  Every function
// returns None for what it does not take, errors included: the Python function then goes through it argument by argument.  built_for and
// abi_version: the torch and the library whose headers it was compiled with.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/bmtk_amd.h"

namespace {

// addresses of the library's functions, from set_library
decltype(&bmtk_spike_readout_workspace_bytes) spike_workspace;
decltype(&bmtk_spike_readout_fwd) spike_fwd;
decltype(&bmtk_spike_readout_bwd_weight) spike_bwd_weight;
decltype(&bmtk_spike_readout_bwd_spikes) spike_bwd_spikes;
decltype(&bmtk_gated_scan_workspace_bytes) scan_workspace;
decltype(&bmtk_gated_scan_fwd) scan_fwd;
decltype(&bmtk_gated_scan_bwd) scan_bwd;
decltype(&bmtk_token_logprobs_workspace_bytes) logprobs_workspace;
decltype(&bmtk_token_logprobs_fwd) logprobs_fwd;
decltype(&bmtk_token_logprobs_bwd) logprobs_bwd;
PyObject *raw_stream = nullptr;   // torch._C._cuda_getCurrentRawStream
bool ready = false;

// a call's arguments, as long as all of them are plain
struct Call {
    bool fine = true;
    c10::DeviceIndex device = -1;

    Call(Py_ssize_t nargs, Py_ssize_t wanted)
    {
        fine = ready && nargs == wanted && !c10::impl::TorchDispatchModeTLS::any_modes_set();
    }
    // a device tensor without anything special, that autograd does not ask about
    const at::Tensor *tensor(PyObject *obj)
    {
        if (!fine) return nullptr;
        fine = THPVariable_CheckExact(obj);
        if (!fine) return nullptr;
        const at::Tensor &t = THPVariable_Unpack(obj);
        fine = t.defined() && t.is_cuda();
        if (!fine) return nullptr;
        if (device < 0) device = c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA)->getDevice().index();
        const c10::DispatchKeySet others({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot, c10::DispatchKey::FuncTorchBatched,
                                          c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize, c10::DispatchKey::ZeroTensor,
                                          c10::DispatchKey::Conjugate, c10::DispatchKey::Negative});
        fine = t.layout() == at::kStrided && t.has_storage() && !t.key_set().has_any(others) && t.get_device() == device &&
               !(t.requires_grad() && c10::GradMode::is_enabled()) && !t._fw_grad(0).defined();
        return &t;
    }
    const at::Tensor *tensor(PyObject *obj, at::ScalarType type, c10::IntArrayRef shape)
    {
        const at::Tensor *t = tensor(obj);
        if (fine) fine = t->scalar_type() == type && t->sizes() == shape && t->is_contiguous();
        return t;
    }
    // the same, or None
    const at::Tensor *optional(PyObject *obj, at::ScalarType type, c10::IntArrayRef shape)
    {
        if (obj == Py_None) return nullptr;
        return tensor(obj, type, shape);
    }
    int64_t whole(PyObject *obj, int64_t least, int64_t most)
    {
        if (!fine) return 0;
        int overflow = 1;
        fine = PyLong_CheckExact(obj);
        const int64_t v = fine ? PyLong_AsLongLongAndOverflow(obj, &overflow) : 0;
        fine = fine && overflow == 0 && v >= least && v <= most;
        return v;
    }
    // the current stream's handle
    void *stream()
    {
        if (!fine) return nullptr;
        PyObject *index = PyLong_FromLong(device), *handle = index ? PyObject_CallOneArg(raw_stream, index) : nullptr;
        void *p = handle ? PyLong_AsVoidPtr(handle) : nullptr;
        Py_XDECREF(index);
        Py_XDECREF(handle);
        fine = !PyErr_Occurred();
        return p;
    }
    bool truth(PyObject *obj)
    {
        if (obj != Py_True && obj != Py_False) fine = false;
        return obj == Py_True;
    }
    at::Tensor empty(c10::IntArrayRef shape, at::ScalarType type) { return at::empty(shape, at::TensorOptions().dtype(type).device(c10::Device(c10::DeviceType::CUDA, device))); }
    at::Tensor bytes(int64_t n) { return n > 0 ? empty({n}, at::kByte) : at::Tensor(); }
};

// BMTK_F32 ..., -1 for other types
int code_of(const at::Tensor &t)
{
    switch (t.scalar_type()) {
        case at::kFloat: return BMTK_F32;
        case at::kBFloat16: return BMTK_BF16;
        case at::kHalf: return BMTK_F16;
        default: return -1;
    }
}
void *ptr(const at::Tensor *t) { return t ? t->data_ptr() : nullptr; }
void *ptr(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

PyObject *results(std::initializer_list<at::Tensor> tensors)
{
    PyObject *r = PyTuple_New((Py_ssize_t)tensors.size());
    if (r == nullptr) return nullptr;
    Py_ssize_t k = 0;
    for (const at::Tensor &t : tensors) {
        PyObject *o = t.defined() ? THPVariable_Wrap(t) : (Py_INCREF(Py_None), Py_None);
        if (o == nullptr) {
            Py_DECREF(r);
            return nullptr;
        }
        PyTuple_SET_ITEM(r, k++, o);
    }
    return r;
}

// (what throws, memory that is not there among it, is done again and raised by the Python function)
template <typename F>
PyObject *guarded(F f)
{
    try {
        PyObject *r = f();
        if (r != nullptr) return r;
        if (PyErr_Occurred()) return nullptr;
    } catch (const std::exception &) {
        PyErr_Clear();
    }
    Py_RETURN_NONE;
}

// ---------------------------------------------------------------------------------------------------------------------

struct Spikes {
    const at::Tensor *bits, *weight;
    int64_t steps = 0, n = 0, dim = 0, stride = 0, batch = 0;
    int code = -1;
    Spikes(Call &c, PyObject *bits_obj, PyObject *weight_obj, PyObject *batch_obj)
    {
        bits = c.tensor(bits_obj);
        weight = c.tensor(weight_obj);
        batch = c.whole(batch_obj, 1, 65536);
        if (!c.fine) return;
        code = code_of(*weight);
        c.fine = code >= 0 && bits->scalar_type() == at::kLong && weight->dim() == 2 && bits->dim() == 2 && weight->is_contiguous() && weight->numel() > 0 &&
                 bits->size(0) > 0 && bits->stride(1) == 1 && weight->size(0) < (int64_t{1} << 31) && weight->size(1) <= 65536;
        if (!c.fine) return;
        steps = bits->size(0), n = weight->size(0), dim = weight->size(1);
        stride = steps > 1 ? bits->stride(0) : bits->size(1);
        c.fine = bits->size(1) >= (n * batch + 63) / 64;
    }
};

PyObject *spike_readout(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    return guarded([&]() -> PyObject * {
        Call c(nargs, 3);
        if (!c.fine) return nullptr;
        const Spikes s(c, args[0], args[1], args[2]);
        void *stream = c.stream();
        if (!c.fine) return nullptr;
        const at::Tensor y = c.empty({s.steps, s.batch, s.dim}, s.weight->scalar_type());
        const at::Tensor ws = c.bytes(spike_workspace(s.steps, s.n, (int32_t)s.batch, (int32_t)s.dim, 0));
        if (spike_fwd((const uint64_t *)ptr(s.bits), s.stride, s.steps, s.n, (int32_t)s.batch, ptr(s.weight), (int32_t)s.dim, s.code, ptr(y), (float *)ptr(ws), stream) != 0) return nullptr;
        return THPVariable_Wrap(y);
    });
}

PyObject *spike_readout_bwd(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    return guarded([&]() -> PyObject * {
        Call c(nargs, 5);
        if (!c.fine) return nullptr;
        const Spikes s(c, args[0], args[1], args[3]);
        if (!c.fine) return nullptr;
        const at::Tensor *dy = c.tensor(args[2], s.weight->scalar_type(), {s.steps, s.batch, s.dim});
        const bool spikes = c.truth(args[4]);
        void *stream = c.stream();
        if (!c.fine) return nullptr;
        const at::Tensor d_weight = c.empty({s.n, s.dim}, s.weight->scalar_type());
        const at::Tensor dl_dz = spikes ? c.empty({s.steps, s.n * s.batch}, at::kFloat) : at::Tensor();
        if (spike_bwd_weight((const uint64_t *)ptr(s.bits), s.stride, s.steps, s.n, (int32_t)s.batch, ptr(dy), (int32_t)s.dim, s.code, ptr(d_weight), stream) != 0) return nullptr;
        if (spikes) {
            const at::Tensor ws = c.bytes(s.code == BMTK_F32 ? spike_workspace(s.steps, s.n, (int32_t)s.batch, (int32_t)s.dim, 1) : 0);
            if (spike_bwd_spikes(ptr(s.weight), ptr(dy), s.steps, s.n, (int32_t)s.batch, (int32_t)s.dim, s.code, (float *)ptr(dl_dz), (int32_t *)ptr(ws), stream) != 0) return nullptr;
        }
        return results({d_weight, dl_dz});
    });
}

struct Scan {
    const at::Tensor *x, *decay, *lengths = nullptr;
    int64_t steps = 0, batch = 0, dim = 0, groups = 0, a_t = 0, a_b = 0;
    int code = -1, gate_code = -1;
    Scan(Call &c, PyObject *x_obj, PyObject *decay_obj, PyObject *lengths_obj)
    {
        x = c.tensor(x_obj);
        decay = c.tensor(decay_obj);
        if (!c.fine) return;
        code = code_of(*x), gate_code = code_of(*decay);
        c.fine = code >= 0 && (gate_code == BMTK_F32 || gate_code == code) && x->dim() == 3 && x->numel() > 0 && x->stride(2) == 1;
        if (!c.fine) return;
        steps = x->size(0), batch = x->size(1), dim = x->size(2);
        if (decay->dim() == 1) {
            c.fine = decay->size(0) == dim && decay->is_contiguous();
        } else {
            c.fine = decay->dim() == 3 && decay->size(0) == steps && decay->size(1) == batch && decay->size(2) > 0 && dim % decay->size(2) == 0 && decay->stride(2) == 1;
            if (c.fine) groups = decay->size(2), a_t = decay->stride(0), a_b = decay->stride(1);
        }
        c.fine = c.fine && steps < (int64_t{1} << 31) - 4096 && batch < (int64_t{1} << 31) && batch * dim < (int64_t{1} << 31);
        if (c.fine) lengths = c.optional(lengths_obj, at::kInt, {batch});
    }
};

PyObject *gated_scan(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    return guarded([&]() -> PyObject * {
        Call c(nargs, 5);
        if (!c.fine) return nullptr;
        const Scan s(c, args[0], args[1], args[3]);
        if (!c.fine) return nullptr;
        const at::Tensor *state = c.optional(args[2], at::kFloat, {s.batch, s.dim});
        const bool save = c.truth(args[4]);
        void *stream = c.stream();
        if (!c.fine) return nullptr;
        const at::Tensor h = c.empty({s.steps, s.batch, s.dim}, s.x->scalar_type()), last = c.empty({s.batch, s.dim}, at::kFloat);
        const at::Tensor saved = save ? c.empty({(s.steps + BMTK_SCAN_MARK - 1) / BMTK_SCAN_MARK, s.batch, s.dim}, at::kFloat) : at::Tensor();
        const at::Tensor ws = c.bytes(scan_workspace(s.steps, s.batch, (int32_t)s.dim, (int32_t)s.groups, 0));
        if (scan_fwd(s.steps, s.batch, (int32_t)s.dim, (int32_t)s.groups, s.code, s.gate_code, ptr(s.x), s.x->stride(0), s.x->stride(1), ptr(s.decay), s.a_t, s.a_b,
                     (const float *)ptr(state), (const int32_t *)ptr(s.lengths), ptr(h), (float *)ptr(last), (float *)ptr(saved), (float *)ptr(ws), stream) != 0)
            return nullptr;
        if (save) return results({h, last, saved});
        return results({h, last});
    });
}

PyObject *gated_scan_bwd(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    return guarded([&]() -> PyObject * {
        Call c(nargs, 6);
        if (!c.fine) return nullptr;
        const Scan s(c, args[0], args[1], args[5]);
        if (!c.fine) return nullptr;
        const at::Tensor *saved = c.tensor(args[2], at::kFloat, {(s.steps + BMTK_SCAN_MARK - 1) / BMTK_SCAN_MARK, s.batch, s.dim});
        const at::Tensor *dh = c.tensor(args[3]);
        const at::Tensor *d_last = c.optional(args[4], at::kFloat, {s.batch, s.dim});
        void *stream = c.stream();
        if (!c.fine || dh->scalar_type() != s.x->scalar_type() || dh->sizes() != s.x->sizes() || dh->stride(2) != 1) return nullptr;
        const at::Tensor dx = c.empty({s.steps, s.batch, s.dim}, s.x->scalar_type()), d_decay = c.empty(s.decay->sizes(), s.decay->scalar_type());
        const at::Tensor d_state = c.empty({s.batch, s.dim}, at::kFloat);
        const at::Tensor ws = c.bytes(scan_workspace(s.steps, s.batch, (int32_t)s.dim, (int32_t)s.groups, 1));
        if (scan_bwd(s.steps, s.batch, (int32_t)s.dim, (int32_t)s.groups, s.code, s.gate_code, ptr(s.x), s.x->stride(0), s.x->stride(1), ptr(s.decay), s.a_t, s.a_b,
                     (const float *)ptr(saved), (const int32_t *)ptr(s.lengths), ptr(dh), dh->stride(0), dh->stride(1), (const float *)ptr(d_last), ptr(dx),
                     ptr(d_decay), (float *)ptr(d_state), (float *)ptr(ws), stream) != 0)
            return nullptr;
        return results({dx, d_decay, d_state});
    });
}

// two dimensions: rows of logits and a token for each
struct Logits {
    const at::Tensor *logits, *tokens;
    int64_t rows = 0, vocab = 0, stride = 0;
    int code = -1;
    Logits(Call &c, PyObject *logits_obj, PyObject *tokens_obj)
    {
        logits = c.tensor(logits_obj);
        tokens = c.tensor(tokens_obj);
        if (!c.fine) return;
        code = code_of(*logits);
        c.fine = code >= 0 && logits->dim() == 2 && logits->numel() > 0 && logits->stride(1) == 1 && tokens->scalar_type() == at::kLong && tokens->dim() == 1 &&
                 tokens->is_contiguous() && tokens->size(0) == logits->size(0) && logits->size(0) < (1 << 24) && logits->size(1) < (1 << 30);
        if (!c.fine) return;
        rows = logits->size(0), vocab = logits->size(1);
        stride = rows > 1 ? logits->stride(0) : vocab;
    }
};

PyObject *token_logprobs(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    return guarded([&]() -> PyObject * {
        Call c(nargs, 4);
        if (!c.fine) return nullptr;
        const Logits l(c, args[0], args[1]);
        if (!c.fine) return nullptr;
        const int64_t top = c.whole(args[2], 0, std::min<int64_t>(BMTK_LOGPROBS_MAX_TOP, l.vocab)), ignore = c.whole(args[3], INT64_MIN, INT64_MAX);
        void *stream = c.stream();
        if (!c.fine) return nullptr;
        const at::Tensor logp = c.empty({l.rows}, at::kFloat), entropy = c.empty({l.rows}, at::kFloat), lse = c.empty({l.rows}, at::kFloat);
        at::Tensor top_logp, top_index;
        if (top > 0) top_logp = c.empty({l.rows, top}, at::kFloat), top_index = c.empty({l.rows, top}, at::kLong);
        const at::Tensor ws = c.bytes(logprobs_workspace(l.rows, (int32_t)l.vocab, l.code, (int32_t)top));
        if (logprobs_fwd(l.rows, (int32_t)l.vocab, l.code, ptr(l.logits), l.stride, (const int64_t *)ptr(l.tokens), ignore, (int32_t)top, (float *)ptr(logp),
                         (float *)ptr(entropy), (float *)ptr(lse), (float *)ptr(top_logp), (int64_t *)ptr(top_index), ptr(ws), stream) != 0)
            return nullptr;
        return results({logp, entropy, lse, top_logp, top_index});
    });
}

PyObject *token_logprobs_bwd(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    return guarded([&]() -> PyObject * {
        Call c(nargs, 7);
        if (!c.fine) return nullptr;
        const Logits l(c, args[0], args[1]);
        if (!c.fine) return nullptr;
        const at::Tensor *lse = c.tensor(args[2], at::kFloat, {l.rows}), *entropy = c.tensor(args[3], at::kFloat, {l.rows});
        const at::Tensor *d_logp = c.optional(args[4], at::kFloat, {l.rows}), *d_entropy = c.optional(args[5], at::kFloat, {l.rows});
        const int64_t ignore = c.whole(args[6], INT64_MIN, INT64_MAX);
        void *stream = c.stream();
        if (!c.fine || (d_logp == nullptr && d_entropy == nullptr)) return nullptr;
        const at::Tensor out = c.empty({l.rows, l.vocab}, l.logits->scalar_type());
        if (logprobs_bwd(l.rows, (int32_t)l.vocab, l.code, ptr(l.logits), l.stride, (const int64_t *)ptr(l.tokens), ignore, (const float *)ptr(lse), (const float *)ptr(entropy),
                         (const float *)ptr(d_logp), (const float *)ptr(d_entropy), ptr(out), l.vocab, stream) != 0)
            return nullptr;
        return THPVariable_Wrap(out);
    });
}

template <typename F>
bool take(PyObject *addresses, Py_ssize_t k, F &f)
{
    void *p = PyLong_AsVoidPtr(PyTuple_GET_ITEM(addresses, k));
    f = reinterpret_cast<F>(p);
    return p != nullptr;
}

PyObject *set_library(PyObject *, PyObject *args)
{
    PyObject *addresses, *stream;
    if (!PyArg_ParseTuple(args, "O!O", &PyTuple_Type, &addresses, &stream)) return nullptr;
    if (PyTuple_GET_SIZE(addresses) != 10) {
        PyErr_SetString(PyExc_TypeError, "set_library takes ten addresses");
        return nullptr;
    }
    Py_INCREF(stream);
    Py_XDECREF(raw_stream);
    raw_stream = stream;
    ready = take(addresses, 0, spike_workspace) && take(addresses, 1, spike_fwd) && take(addresses, 2, spike_bwd_weight) && take(addresses, 3, spike_bwd_spikes) &&
            take(addresses, 4, scan_workspace) && take(addresses, 5, scan_fwd) && take(addresses, 6, scan_bwd) && take(addresses, 7, logprobs_workspace) &&
            take(addresses, 8, logprobs_fwd) && take(addresses, 9, logprobs_bwd);
    if (PyErr_Occurred()) return nullptr;
    return PyBool_FromLong(ready);
}

#define BMTK_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, "as bmtk_amd.readout." #name ", or None"}
PyMethodDef methods[] = {BMTK_METHOD(spike_readout), BMTK_METHOD(spike_readout_bwd), BMTK_METHOD(gated_scan), BMTK_METHOD(gated_scan_bwd), BMTK_METHOD(token_logprobs),
                         BMTK_METHOD(token_logprobs_bwd), {"set_library", set_library, METH_VARARGS, "addresses of the C functions, and what says the current stream of a device"}, {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_readout", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__readout()
{
    PyObject *m = PyModule_Create(&module);
    if (m != nullptr && (PyModule_AddStringConstant(m, "built_for", BMTK_AMD_TORCH) != 0 || PyModule_AddIntConstant(m, "abi_version", BMTK_AMD_ABI_VERSION) != 0)) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
