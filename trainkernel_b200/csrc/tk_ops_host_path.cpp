// The short way from a Python call to a launch of libtrainkernel_ops.so.
//
// A small call (a few decoded tokens, a tiny model's update) runs for a few microseconds on the GPU, and checking arguments,
// allocating results and filling structures in Python takes several times that.  The functions here do the same for the
// ordinary call: plain CUDA tensors of matching types and shapes, nothing to record, numbers in range.  Whatever is out of
// the ordinary returns None, and the Python code beside them (losses.py, optim.py) runs instead; it alone knows the errors.
// Nothing is remembered from one call for the next but which devices Python has found usable.
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <iterator>
#include <vector>

#include "trainkernel_ops.h"

namespace {

bool g_usable[64] = {};

// Why a call goes the long way round is decided there, so all of these only say yes or no.
bool plain(PyObject* object) {
    if (!THPVariable_CheckExact(object)) return false;         // a Tensor or a Parameter: a subclass may mean something else by its operations
    const at::Tensor& t = THPVariable_Unpack(object);
    using Key = c10::DispatchKey;
    static const c10::DispatchKeySet special({Key::Python, Key::PythonTLSSnapshot, Key::FuncTorchBatched, Key::FuncTorchGradWrapper, Key::Batched,
                                              Key::Functionalize, Key::Conjugate, Key::Negative, Key::ZeroTensor});
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.is_nested() || t.key_set().has_any(special)) return false;
    return !t._fw_grad(0).defined();                           // a tangent is refused there
}

// Inside a `torch.func` transform, too, what is allocated here would belong to it.
bool tracing() {
    return c10::impl::TorchDispatchModeTLS::any_modes_set() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

bool number(PyObject* object, double* value) {
    if (PyFloat_CheckExact(object)) *value = PyFloat_AS_DOUBLE(object);
    else if (PyLong_CheckExact(object)) *value = PyLong_AsDouble(object);
    else return false;
    if (PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}

bool within(PyObject* object, double low, double high, double* value) { return number(object, value) && *value >= low && *value <= high; }

int type_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return TK_F32;
        case at::kHalf: return TK_F16;
        case at::kBFloat16: return TK_BF16;
        default: return -1;
    }
}

struct Rows {
    tk_token_rows rows;
    at::Tensor logits, targets, mask;
    int device;
    cudaStream_t stream;
};

tk_token_array array_of(const at::Tensor& t) {
    return t.dim() == 2 ? tk_token_array{t.data_ptr(), t.stride(0), t.stride(1)} : tk_token_array{t.data_ptr(), 0, t.stride(0)};
}

bool rows_of(PyObject* logits, PyObject* targets, PyObject* mask, bool records, Rows* r) {
    if (!plain(logits) || !plain(targets) || (mask != Py_None && !plain(mask)) || tracing()) return false;
    r->logits = THPVariable_Unpack(logits);
    r->targets = THPVariable_Unpack(targets);
    const at::Tensor &x = r->logits, &ids = r->targets;
    if (records && x.requires_grad() && c10::GradMode::is_enabled()) return false;
    const int64_t rank = x.dim();
    const int type = type_of(x);
    if (type < 0 || (rank != 2 && rank != 3) || (ids.scalar_type() != at::kLong && ids.scalar_type() != at::kInt) || ids.dim() != rank - 1) return false;
    const int64_t vocab = x.size(-1), length = x.size(-2), batch = rank == 3 ? x.size(0) : 1;
    if (vocab < 1 || length < 1 || batch < 1 || vocab > 0x7ffffff0 || batch > 0x7fffffff / length || (x.stride(-1) != 1 && vocab != 1)) return false;
    if (ids.size(-1) != length || (rank == 3 && ids.size(0) != batch) || ids.device() != x.device()) return false;
    r->device = x.device().index();
    if (r->device < 0 || r->device >= 64 || !g_usable[r->device]) return false;
    r->rows = {x.data_ptr(), rank == 3 ? x.stride(0) : 0, x.stride(-2), batch, length, vocab, type, ids.scalar_type() == at::kLong ? 8 : 4, array_of(ids), {}};
    if (mask != Py_None) {
        r->mask = THPVariable_Unpack(mask);
        if (r->mask.scalar_type() != at::kBool || r->mask.sizes() != ids.sizes() || r->mask.device() != x.device()) return false;
        r->rows.mask = array_of(r->mask);
    }
    r->stream = c10::cuda::getCurrentCUDAStream(r->device).stream();
    return true;
}

// An FP32 constant that broadcasts to the targets' shape.
bool constant_of(PyObject* object, const Rows& r, tk_token_array* to) {
    if (!plain(object)) return false;
    const at::Tensor& t = THPVariable_Unpack(object);
    if (t.scalar_type() != at::kFloat || t.requires_grad() || t.device() != r.logits.device() || t.dim() > r.targets.dim()) return false;
    int64_t strides[2] = {0, 0};                               // batch, token
    for (int64_t i = 0; i < t.dim(); ++i) {                    // from the last dimension
        const int64_t size = t.size(t.dim() - 1 - i), want = r.targets.size(r.targets.dim() - 1 - i);
        if (size != want && size != 1) return false;
        strides[1 - i] = size == 1 ? 0 : t.stride(t.dim() - 1 - i);
    }
    *to = {t.data_ptr(), strides[0], strides[1]};
    return true;
}

at::Tensor empty_like_rows(const Rows& r, at::IntArrayRef shape) { return at::empty(shape, r.logits.options().dtype(at::kFloat).requires_grad(false)); }

// The gradient's room, laid out as losses._grad_like lays it out; only the dense case is made here.
bool grad_of(const Rows& r, double scale, at::Tensor* out, tk_token_grad* grad) {
    const at::Tensor& x = r.logits;
    if (!x.is_contiguous() || reinterpret_cast<uintptr_t>(x.data_ptr()) % 16) return false;
    *out = at::empty(x.sizes(), x.options().requires_grad(false));
    *grad = {out->data_ptr(), x.dim() == 3 ? x.stride(0) : 0, x.stride(-2), nullptr, static_cast<float>(scale), 0};
    return true;
}

PyObject* failed() {
    PyErr_SetString(PyExc_RuntimeError, tk_ops_last_error());
    return nullptr;
}

PyObject* results(std::initializer_list<at::Tensor> list) {
    PyObject* tuple = PyTuple_New(static_cast<Py_ssize_t>(list.size()));
    Py_ssize_t i = 0;
    for (const at::Tensor& t : list) PyTuple_SET_ITEM(tuple, i++, THPVariable_Wrap(t));
    return tuple;
}

// No C++ exception crosses into the interpreter.
template <typename F> PyObject* guarded(F&& body) {
    try {
        return body();
    } catch (const std::exception& e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// (logits, targets, mask) -> logprobs
PyObject* token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        Rows r;
        if (count != 3 || !rows_of(args[0], args[1], args[2], true, &r)) Py_RETURN_NONE;
        at::Tensor logprobs = empty_like_rows(r, r.targets.sizes());
        if (tk_token_logprobs(&r.rows, logprobs.data_ptr<float>(), nullptr, r.device, r.stream)) return failed();
        return THPVariable_Wrap(logprobs);
    });
}

// (logits, targets, weights, mask, grad_scale) -> (logprobs, grad)
PyObject* token_logprobs_and_grad(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        Rows r;
        tk_token_array weights;
        tk_token_grad grad;
        at::Tensor out;
        double scale;
        if (count != 5 || !rows_of(args[0], args[1], args[3], false, &r) || !constant_of(args[2], r, &weights) || !number(args[4], &scale)
            || !grad_of(r, scale, &out, &grad))
            Py_RETURN_NONE;
        at::Tensor logprobs = empty_like_rows(r, r.targets.sizes());
        if (tk_token_logprobs_and_grad(&r.rows, &weights, logprobs.data_ptr<float>(), &grad, r.device, r.stream)) return failed();
        return results({logprobs, out});
    });
}

// (logits, targets, old, advantages, ref, mask, clip, kl_weight, average, grad_scale or None) -> (loss, logprobs[, grad])
PyObject* policy_loss(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        Rows r;
        tk_policy_terms terms{};
        double low, high, kl, scale = 1.0;
        if (count != 10) Py_RETURN_NONE;
        const bool with_grad = args[9] != Py_None;
        if (!rows_of(args[0], args[1], args[5], !with_grad, &r) || !constant_of(args[2], r, &terms.old_logprobs)
            || !constant_of(args[3], r, &terms.advantages) || (args[4] != Py_None && !constant_of(args[4], r, &terms.ref_logprobs)))
            Py_RETURN_NONE;
        if (!PyTuple_CheckExact(args[6]) || PyTuple_GET_SIZE(args[6]) != 2 || !within(PyTuple_GET_ITEM(args[6], 0), 0.0, 1.0, &low)
            || !within(PyTuple_GET_ITEM(args[6], 1), 0.0, 1e30, &high) || !within(args[7], 0.0, 1e30, &kl) || (kl != 0.0 && !terms.ref_logprobs.data)
            || !PyUnicode_CheckExact(args[8]) || (with_grad && !number(args[9], &scale)))
            Py_RETURN_NONE;
        if (PyUnicode_CompareWithASCIIString(args[8], "tokens") == 0) terms.average = TK_AVERAGE_TOKENS;
        else if (PyUnicode_CompareWithASCIIString(args[8], "sequences") == 0) terms.average = TK_AVERAGE_SEQUENCES;
        else Py_RETURN_NONE;
        terms.clip_low = static_cast<float>(low);
        terms.clip_high = static_cast<float>(high);
        terms.kl_weight = static_cast<float>(kl);
        at::Tensor out;
        tk_token_grad grad{};
        if (with_grad && !grad_of(r, scale, &out, &grad)) Py_RETURN_NONE;
        at::Tensor loss = empty_like_rows(r, {}), logprobs = empty_like_rows(r, r.targets.sizes());
        at::Tensor workspace = at::empty({static_cast<int64_t>(tk_policy_workspace_bytes(r.rows.batch, r.rows.length))}, r.logits.options().dtype(at::kByte).requires_grad(false));
        if (tk_policy_loss(&r.rows, &terms, loss.data_ptr<float>(), logprobs.data_ptr<float>(), nullptr, nullptr, &grad, workspace.data_ptr(), r.device, r.stream))
            return failed();
        return with_grad ? results({loss, logprobs, out}) : results({loss, logprobs});
    });
}

// (logits, targets, reference, mask, beta, label_smoothing, grad_scale or None) -> (loss, sums[, grad])
PyObject* preference_loss(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        Rows r;
        double beta, smoothing, scale = 1.0;
        if (count != 7) Py_RETURN_NONE;
        const bool with_grad = args[6] != Py_None;
        if (!rows_of(args[0], args[1], args[3], !with_grad, &r) || r.logits.dim() != 3 || r.rows.batch % 2 || !plain(args[2])) Py_RETURN_NONE;
        const at::Tensor& reference = THPVariable_Unpack(args[2]);
        if (reference.scalar_type() != at::kFloat || reference.requires_grad() || reference.device() != r.logits.device() || reference.dim() != 1
            || reference.size(0) != r.rows.batch || !within(args[4], 0.0, 1e30, &beta) || !within(args[5], 0.0, 1.0, &smoothing)
            || (with_grad && !number(args[6], &scale)))
            Py_RETURN_NONE;
        at::Tensor out;
        tk_token_grad grad{};
        if (with_grad && !grad_of(r, scale, &out, &grad)) Py_RETURN_NONE;
        const int64_t batch = r.rows.batch, tokens = batch * r.rows.length;
        at::Tensor loss = empty_like_rows(r, {}), sums = empty_like_rows(r, {batch});
        // statistics, coefficients and workspace in one piece, none of which is returned
        const int64_t space = static_cast<int64_t>(tk_preference_workspace_bytes(batch, r.rows.length));
        at::Tensor scratch = at::empty({space + 8 * tokens + 4 * batch}, r.logits.options().dtype(at::kByte).requires_grad(false));
        char* at_ = static_cast<char*>(scratch.data_ptr());
        float* stats = reinterpret_cast<float*>(at_ + space);
        if (tk_preference_loss(&r.rows, reference.data_ptr<float>(), reference.stride(0), static_cast<float>(beta), static_cast<float>(smoothing),
                               loss.data_ptr<float>(), sums.data_ptr<float>(), stats, stats + 2 * tokens, &grad, at_, r.device, r.stream))
            return failed();
        return with_grad ? results({loss, sums, out}) : results({loss, sums});
    });
}

bool same_order(const at::Tensor& a, const at::Tensor& b) {
    for (int64_t i = 0; i < a.dim(); ++i)
        if (a.size(i) != 1 && a.stride(i) != b.stride(i)) return false;
    return true;
}

// Bytes of dense tensors, and whether one lies among others that are sorted and apart.
struct Span {
    uintptr_t begin, end;
    bool operator<(const Span& other) const { return begin < other.begin; }
};

Span span_of(const at::Tensor& t) {
    const auto begin = reinterpret_cast<uintptr_t>(t.data_ptr());
    return {begin, begin + static_cast<uintptr_t>(t.numel()) * t.element_size()};
}

bool among(const std::vector<Span>& spans, const Span& s) {
    const auto behind = std::lower_bound(spans.begin(), spans.end(), Span{s.end, 0});       // the first that begins at its end or later
    return s.begin < s.end && behind != spans.begin() && std::prev(behind)->end > s.begin;
}

// (params, grads, sizes, offsets, decay, state struct address, state tensors, bits, lr, betas, eps, seed, grad_scale) -> True
// Only for lists of contiguous tensors of one parameter type and one gradient type.
PyObject* adamw_update(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        if (count != 13 || tracing()) Py_RETURN_NONE;
        PyObject *params = args[0], *grads = args[1], *sizes = args[2], *offsets = args[3], *decay = args[4];
        const auto listed = [](PyObject* o) { return PyList_CheckExact(o) || PyTuple_CheckExact(o); };
        if (!listed(params) || !listed(grads) || !PyTuple_CheckExact(sizes) || !PyTuple_CheckExact(offsets) || !PyTuple_CheckExact(args[6])) Py_RETURN_NONE;
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(params);
        if (n < 1 || PySequence_Fast_GET_SIZE(grads) != n || PyTuple_GET_SIZE(sizes) != n || (PyTuple_CheckExact(decay) && PyTuple_GET_SIZE(decay) != n)) Py_RETURN_NONE;
        tk_adamw_options options{};
        double bits = 0, seed = 0;
        const bool lr_given = number(args[8], &options.lr);
        if ((!lr_given && !plain(args[8])) || !PyTuple_CheckExact(args[9]) || PyTuple_GET_SIZE(args[9]) != 2 || !number(PyTuple_GET_ITEM(args[9], 0), &options.beta1)
            || !number(PyTuple_GET_ITEM(args[9], 1), &options.beta2) || !number(args[10], &options.eps) || !number(args[7], &bits) || !number(args[11], &seed))
            Py_RETURN_NONE;
        options.bits = static_cast<int32_t>(bits);
        options.seed = static_cast<uint32_t>(seed);
        std::vector<tk_adamw_tensor> tensors(static_cast<size_t>(n));
        std::vector<Span> places, gradients;
        places.reserve(static_cast<size_t>(n));
        int param_type = -1, grad_type = -1;
        c10::Device device(c10::kCPU);
        double one_decay = 0.0;
        if (!PyTuple_CheckExact(decay) && !number(decay, &one_decay)) Py_RETURN_NONE;
        for (Py_ssize_t i = 0; i < n; ++i) {
            PyObject *po = PySequence_Fast_GET_ITEM(params, i), *go = PySequence_Fast_GET_ITEM(grads, i);
            if (!plain(po) || !plain(go)) Py_RETURN_NONE;
            const at::Tensor &p = THPVariable_Unpack(po), &g = THPVariable_Unpack(go);
            if (i == 0) {
                param_type = type_of(p);
                grad_type = type_of(g);
                device = p.device();
            }
            if (param_type < 0 || grad_type < 0 || type_of(p) != param_type || type_of(g) != grad_type || p.device() != device || g.device() != device
                || !p.is_contiguous() || p.sizes() != g.sizes() || !same_order(p, g) || (p.requires_grad() && !p.is_leaf()))
                Py_RETURN_NONE;
            const int64_t size = PyLong_AsLongLong(PyTuple_GET_ITEM(sizes, i));
            if (size != p.numel()) Py_RETURN_NONE;
            double d = one_decay;
            if (PyTuple_CheckExact(decay) && !number(PyTuple_GET_ITEM(decay, i), &d)) Py_RETURN_NONE;
            tensors[i] = {p.data_ptr(), g.data_ptr(), PyLong_AsLongLong(PyTuple_GET_ITEM(offsets, i)), size, static_cast<float>(d), 0};
            if (size) places.push_back(span_of(p));
            if (size && (g.data_ptr() != p.data_ptr() || grad_type != param_type)) gradients.push_back(span_of(g));      // its own param's memory is read before it is written
        }
        if (device.index() < 0 || device.index() >= 64 || !g_usable[device.index()]) Py_RETURN_NONE;
        std::sort(places.begin(), places.end());
        if (std::adjacent_find(places.begin(), places.end(), [](const Span& a, const Span& b) { return a.end > b.begin; }) != places.end()) Py_RETURN_NONE;
        for (const Span& gradient : gradients)
            if (among(places, gradient)) Py_RETURN_NONE;
        if (args[12] != Py_None) {
            if (!plain(args[12])) Py_RETURN_NONE;
            const at::Tensor& scale = THPVariable_Unpack(args[12]);
            if (scale.scalar_type() != at::kFloat || scale.numel() != 1 || scale.device() != device || among(places, span_of(scale))) Py_RETURN_NONE;
            options.scale_at = scale.data_ptr<float>();
        }
        if (!lr_given) {
            const at::Tensor& lr = THPVariable_Unpack(args[8]);
            if (lr.scalar_type() != at::kFloat || lr.numel() != 1 || lr.device() != device || among(places, span_of(lr))) Py_RETURN_NONE;
            options.lr_at = lr.data_ptr<float>();
        }
        for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[6]); ++i) {
            if (!plain(PyTuple_GET_ITEM(args[6], i))) Py_RETURN_NONE;
            if (THPVariable_Unpack(PyTuple_GET_ITEM(args[6], i)).device() != device) Py_RETURN_NONE;
        }
        const auto* state = reinterpret_cast<const tk_adamw_state*>(PyLong_AsVoidPtr(args[5]));
        if (PyErr_Occurred()) return nullptr;
        const auto stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
        if (tk_adamw_update(tensors.data(), static_cast<int>(n), param_type, grad_type, state, &options, 1, device.index(), stream)) return failed();
        const auto bump = [](PyObject* o) {
            const at::Tensor& t = THPVariable_Unpack(o);
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
        };
        for (Py_ssize_t i = 0; i < n; ++i) bump(PySequence_Fast_GET_ITEM(params, i));
        for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[6]); ++i) bump(PyTuple_GET_ITEM(args[6], i));
        Py_RETURN_TRUE;
    });
}

// (ordinal): Python has found this device to be an sm_100 one.
PyObject* allow_device(PyObject*, PyObject* ordinal) {
    const long index = PyLong_AsLong(ordinal);
    if (PyErr_Occurred()) return nullptr;
    if (index >= 0 && index < 64) g_usable[index] = true;
    Py_RETURN_NONE;
}

template <typename F> PyMethodDef fast(const char* name, F function) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(function)), METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {
    fast("token_logprobs", token_logprobs),
    fast("token_logprobs_and_grad", token_logprobs_and_grad),
    fast("policy_loss", policy_loss),
    fast("preference_loss", preference_loss),
    fast("adamw_update", adamw_update),
    {"allow_device", allow_device, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_ops_host", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops_host() { return PyModule_Create(&g_module); }
