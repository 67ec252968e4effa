/* gdn_ops_torch.cpp -- the Python binding of the serving operators
 * (gateddeltanet_b200/ops.py): checks torch tensors, allocates outputs and
 * workspaces with torch's allocator and calls the C entries of
 * include/gdn_b200.h on torch's current stream. These calls are made once or
 * more per layer and token, where the same checks in Python took longer than
 * the kernels (13-18 us a call). The C entries' addresses come from the
 * loaded library (bind), so this module does not link against it. */
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <exception>
#include <string>

#include "gdn_b200.h"

namespace {

struct Entries {
    int (*step)(const GdnB200DeltaArgs *);
    int (*chunk)(const GdnB200DeltaArgs *);
    size_t (*chunk_workspace)(uint32_t, uint32_t, uint32_t);
    int (*logits)(const GdnB200LogitsArgs *);
    int (*norm)(const GdnB200NormArgs *);
    int (*linear)(const GdnB200LinearArgs *);
    int (*conv)(const GdnB200ConvArgs *);
    const char *(*last_error)(void);
} g_entry;

/* A refusal on its way to Python. */
struct Refused {
    PyObject *type;
    std::string what;
};
[[noreturn]] __attribute__((format(printf, 1, 2))) void refuse(const char *fmt, ...) {
    char buf[384];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    throw Refused{PyExc_ValueError, buf};
}

std::string text(at::IntArrayRef v) {
    std::string s = "[";
    for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
    return s + "]";
}

/* One tensor argument; the checks name it when they refuse. */
struct Arg {
    const char *who, *what;
    const at::Tensor *t;

    Arg(const char *w, const char *n, PyObject *o) : who(w), what(n), t(nullptr) {
        if (o == Py_None) return;
        if (!THPVariable_Check(o)) refuse("%s: %s is not a tensor", who, what);
        t = &THPVariable_Unpack(o);
    }
    explicit operator bool() const { return t != nullptr; }
    void present() const {
        if (t == nullptr) refuse("%s: %s is missing", who, what);
    }
    void type(at::ScalarType s) const {
        if (t->scalar_type() != s) refuse("%s: %s has type %s, expected %s", who, what, c10::toString(t->scalar_type()), c10::toString(s));
    }
    void on(c10::Device d) const {
        if (!t->is_cuda() || t->device() != d)
            refuse("%s: %s is on %s, all on one CUDA device expected", who, what, t->device().str().c_str());
    }
    void dims(int64_t n) const {
        if (t->dim() != n) refuse("%s: %s has %lld dimensions, expected %lld", who, what, (long long)t->dim(), (long long)n);
    }
    void shape(at::IntArrayRef s) const {
        if (t->sizes() != s) refuse("%s: %s has shape %s, expected %s", who, what, text(t->sizes()).c_str(), text(s).c_str());
    }
    void last_contiguous() const {
        const int64_t n = t->dim();
        if (n > 0 && t->stride(n - 1) != 1 && t->size(n - 1) > 1) refuse("%s: the last dimension of %s is not contiguous", who, what);
    }
    /* Outputs may have any order of dimensions, but no two elements in one place. */
    void disjoint() const {
        std::array<std::pair<int64_t, int64_t>, 4> d;
        size_t n = 0;
        for (int64_t i = 0; i < t->dim(); ++i)
            if (t->size(i) > 1) d[n++] = {t->stride(i), t->size(i)};
        std::sort(d.begin(), d.begin() + n);
        int64_t reach = 1;
        for (size_t i = 0; i < n; ++i) {
            if (d[i].first < reach) refuse("%s: elements of %s overlap (strides %s)", who, what, text(t->strides()).c_str());
            reach = d[i].first * d[i].second;
        }
    }
    /* a gradient or a tangent would end here unseen */
    void no_gradient() const {
        if (t == nullptr) return;
        const bool backward = at::GradMode::is_enabled() && t->requires_grad();
        const bool forward = c10::AutogradState::get_tls_state().get_fw_grad_mode() && t->_fw_grad(0).defined();
        if (backward || forward)
            throw Refused{PyExc_RuntimeError, std::string(who) + ": no gradient is computed for " + what +
                                                  (backward ? " (call it under torch.no_grad())" : "")};
    }
    /* The call wrote it: autograd then notices where it kept the old content.
     * An inference tensor has no version. */
    void written() const {
        if (t != nullptr && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    }
    template <typename T>
    T *ptr() const {
        return t == nullptr ? nullptr : static_cast<T *>(t->data_ptr());
    }
};

/* Stride of dimension d; of a single entry, whose stride torch leaves to
 * chance, that of a contiguous tensor. */
int64_t step(const at::Tensor &t, int64_t d) {
    if (t.size(d) > 1) return t.stride(d);
    int64_t n = 1;
    for (int64_t i = d + 1; i < t.dim(); ++i) n *= t.size(i);
    return n;
}

int dtype_code(const Arg &a) {
    switch (a.t->scalar_type()) {
        case at::kFloat: return 0;
        case at::kBFloat16: return 1;
        default: refuse("%s: %s has type %s, neither float nor bfloat16", a.who, a.what, c10::toString(a.t->scalar_type()));
    }
}

void called(int rc) {
    if (rc != 0) throw Refused{PyExc_RuntimeError, g_entry.last_error()};
}

/* body() with its refusals as Python errors, and C++ exceptions as torch's own
 * (an allocation that fails is a torch.OutOfMemoryError) */
template <typename F>
PyObject *guarded(F body) {
    try {
        return body();
    } catch (const Refused &r) {
        PyErr_SetString(r.type, r.what.c_str());
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}

/* (q, k, v, g, beta, state, starts, slots, fresh, scale, normalize, out) -> out */
PyObject *delta(PyObject *const *args, Py_ssize_t nargs, bool chunk) {
    return guarded([&]() -> PyObject * {
        const char *who = chunk ? "delta_chunk" : "delta_step";
        if (nargs != 12) refuse("%s: 12 arguments expected", who);
        if (g_entry.step == nullptr) throw Refused{PyExc_RuntimeError, "the library is not bound"};
        const Arg q(who, "q", args[0]), k(who, "k", args[1]), v(who, "v", args[2]), g(who, "g", args[3]), beta(who, "beta", args[4]),
            state(who, "state", args[5]), starts(who, "starts", args[6]), slots(who, "slots", args[7]), fresh(who, "fresh", args[8]),
            out(who, "out", args[11]);
        for (const Arg *a : {&q, &k, &v, &g, &beta, &state}) a->present();
        for (const Arg *a : {&q, &k, &v, &g, &beta, &state, &out}) a->no_gradient();
        q.dims(3);
        v.dims(3);
        state.dims(4);
        GdnB200DeltaArgs a = {};
        a.dtype = dtype_code(q);
        const at::ScalarType type = q.t->scalar_type();
        const c10::Device device = q.t->device();
        const int64_t tokens = q.t->size(0), heads = q.t->size(1), key_dim = q.t->size(2);
        const int64_t v_heads = v.t->size(1), value_dim = v.t->size(2), n_slots = state.t->size(0);
        for (const Arg *x : {&k, &v}) x->type(type);
        for (const Arg *x : {&g, &beta, &state}) x->type(at::kFloat);
        k.shape(q.t->sizes());
        v.shape({tokens, v_heads, value_dim});
        g.shape({tokens, v_heads});
        beta.shape({tokens, v_heads});
        state.shape({n_slots, v_heads, value_dim, key_dim});
        for (const Arg *x : {&q, &k, &v, &state}) x->last_contiguous();
        for (const Arg *x : {&q, &k, &v, &g, &beta, &state}) x->on(device);
        const auto ss = state.t->strides();
        if ((ss[2] != key_dim && value_dim > 1) || (ss[1] != value_dim * key_dim && v_heads > 1))
            refuse("%s: a slot of state is not one block [v_heads, value_dim, key_dim]", who);
        int64_t sequences = tokens;
        if (starts) {
            starts.type(at::kInt);
            starts.dims(1);
            starts.on(device);
            starts.last_contiguous();
            sequences = starts.t->size(0) - 1;
            if (sequences < 0) refuse("%s: starts has shape [0], expected [sequences + 1]", who);
        }
        if (slots) {
            slots.type(at::kInt);
            slots.shape({sequences});
            slots.on(device);
            slots.last_contiguous();
        }
        if (fresh) {
            if (fresh.t->scalar_type() != at::kByte) fresh.type(at::kBool);
            fresh.shape({sequences});
            fresh.on(device);
            fresh.last_contiguous();
        }
        for (int64_t x : {tokens, sequences, heads, v_heads, key_dim, value_dim, n_slots})
            if (x > 0x7fffffff) refuse("%s: a size of %lld is too large", who, (long long)x);
        at::Tensor result;
        if (out) {
            out.type(type);
            out.shape(v.t->sizes());
            out.on(device);
            out.last_contiguous();
            out.disjoint();
            result = *out.t;
        } else {
            result = at::empty({tokens, v_heads, value_dim}, q.t->options().requires_grad(false));
        }
        double scale = 0.0;
        if (args[9] == Py_None) {
            scale = key_dim > 0 ? 1.0 / std::sqrt((double)key_dim) : 0.0;
        } else {
            scale = PyFloat_AsDouble(args[9]);
            if (PyErr_Occurred()) return nullptr;
        }
        const int normalize = PyObject_IsTrue(args[10]);
        if (normalize < 0) return nullptr;
        a.q = q.ptr<const void>();
        a.k = k.ptr<const void>();
        a.v = v.ptr<const void>();
        a.g = g.ptr<const float>();
        a.beta = beta.ptr<const float>();
        a.state = state.ptr<float>();
        a.out = result.data_ptr();
        a.starts = starts.ptr<const int32_t>();
        a.slots = slots.ptr<const int32_t>();
        a.fresh = fresh.ptr<const uint8_t>();
        a.stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
        a.q_token = step(*q.t, 0), a.q_head = step(*q.t, 1);
        a.k_token = step(*k.t, 0), a.k_head = step(*k.t, 1);
        a.v_token = step(*v.t, 0), a.v_head = step(*v.t, 1);
        a.g_token = step(*g.t, 0), a.g_head = step(*g.t, 1);
        a.beta_token = step(*beta.t, 0), a.beta_head = step(*beta.t, 1);
        a.out_token = step(result, 0), a.out_head = step(result, 1);
        a.state_slot = step(*state.t, 0);
        a.sequences = (uint32_t)sequences, a.tokens = (uint32_t)tokens;
        a.heads = (uint32_t)heads, a.v_heads = (uint32_t)v_heads;
        a.key_dim = (uint32_t)key_dim, a.value_dim = (uint32_t)value_dim;
        a.state_slots = (uint32_t)n_slots;
        a.normalize = normalize;
        a.device = device.index();
        a.scale = (float)scale;
        if (chunk) {
            a.workspace_bytes = g_entry.chunk_workspace(a.tokens, a.sequences, a.v_heads);
            const at::Tensor workspace = at::empty({(int64_t)a.workspace_bytes}, q.t->options().dtype(at::kByte));
            a.workspace = workspace.data_ptr();
            called(g_entry.chunk(&a));
        } else {
            called(g_entry.step(&a));
        }
        state.written();
        out.written();
        if (out) {
            Py_INCREF(args[11]);
            return args[11];
        }
        return THPVariable_Wrap(result);
    });
}

PyObject *delta_step(PyObject *, PyObject *const *args, Py_ssize_t nargs) { return delta(args, nargs, false); }
PyObject *delta_chunk(PyObject *, PyObject *const *args, Py_ssize_t nargs) { return delta(args, nargs, true); }

/* (logits, tokens, lens, prompt_lens, repetition, presence, frequency,
 *  bias_ids, bias, mask, out) -> (out, picks) */
PyObject *constrain_logits(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        const char *who = "constrain_logits";
        if (nargs != 11) refuse("%s: 11 arguments expected", who);
        if (g_entry.logits == nullptr) throw Refused{PyExc_RuntimeError, "the library is not bound"};
        const Arg logits(who, "logits", args[0]), tokens(who, "tokens", args[1]), lens(who, "lens", args[2]),
            prompt_lens(who, "prompt_lens", args[3]), repetition(who, "repetition", args[4]), presence(who, "presence", args[5]),
            frequency(who, "frequency", args[6]), bias_ids(who, "bias_ids", args[7]), bias(who, "bias", args[8]),
            mask(who, "mask", args[9]), out(who, "out", args[10]);
        logits.present();
        for (const Arg *a : {&logits, &repetition, &presence, &frequency, &bias, &out}) a->no_gradient();
        logits.dims(2);
        logits.last_contiguous();
        GdnB200LogitsArgs a = {};
        a.dtype = dtype_code(logits);
        const c10::Device device = logits.t->device();
        logits.on(device);
        const int64_t rows = logits.t->size(0), vocab = logits.t->size(1);
        auto each = [&](const Arg &x, at::ScalarType type) {
            if (!x) return;
            x.type(type);
            x.shape({rows});
            x.on(device);
            x.last_contiguous();
        };
        auto table = [&](const Arg &x, at::ScalarType type, int64_t width) {
            x.type(type);
            x.dims(2);
            x.shape({rows, width});
            x.on(device);
            x.last_contiguous();
        };
        int64_t history = 0, biases = 0;
        if (tokens) {
            tokens.dims(2);
            history = tokens.t->size(1);
            table(tokens, at::kInt, history);
        } else if (lens || prompt_lens || repetition || presence || frequency) {
            refuse("%s: lens, prompt_lens and penalties need tokens", who);
        }
        each(lens, at::kInt);
        each(prompt_lens, at::kInt);
        each(repetition, at::kFloat);
        each(presence, at::kFloat);
        each(frequency, at::kFloat);
        if ((bool)bias != (bool)bias_ids) refuse("%s: bias and bias_ids go together", who);
        if (bias) {
            bias.dims(2);
            biases = bias.t->size(1);
            table(bias, at::kFloat, biases);
            table(bias_ids, at::kInt, biases);
        }
        if (mask) table(mask, at::kInt, (vocab + 31) / 32);
        for (int64_t x : {rows, vocab, history, biases})
            if (x > 0x7fffffff) refuse("%s: a size of %lld is too large", who, (long long)x);
        at::Tensor result;
        if (out) {
            table(out, logits.t->scalar_type(), vocab);
            if (args[10] != args[0]) out.disjoint();
            result = *out.t;
        } else {
            result = at::empty({rows, vocab}, logits.t->options().requires_grad(false));
        }
        at::Tensor picks = at::empty({rows}, logits.t->options().dtype(at::kInt).requires_grad(false));
        a.logits = logits.ptr<const void>();
        a.out = result.data_ptr();
        a.picks = static_cast<int32_t *>(picks.data_ptr());
        a.tokens = tokens.ptr<const int32_t>();
        a.lens = lens.ptr<const int32_t>();
        a.prompt_lens = prompt_lens.ptr<const int32_t>();
        a.repetition = repetition.ptr<const float>();
        a.presence = presence.ptr<const float>();
        a.frequency = frequency.ptr<const float>();
        a.bias_ids = bias_ids.ptr<const int32_t>();
        a.bias = bias.ptr<const float>();
        a.mask = mask.ptr<const uint32_t>();
        a.stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
        a.logits_row = logits.t->stride(0);
        a.out_row = result.stride(0);
        if (tokens) a.tokens_row = tokens.t->stride(0);
        if (bias) a.bias_row = bias.t->stride(0), a.bias_ids_row = bias_ids.t->stride(0);
        if (mask) a.mask_row = mask.t->stride(0);
        a.rows = (uint32_t)rows, a.vocab = (uint32_t)vocab;
        a.history = (uint32_t)history, a.biases = (uint32_t)biases;
        a.device = device.index();
        called(g_entry.logits(&a));
        out.written();
        PyObject *first = out ? Py_NewRef(args[10]) : THPVariable_Wrap(result);
        if (first == nullptr) return nullptr;
        PyObject *second = THPVariable_Wrap(picks);
        if (second == nullptr) {
            Py_DECREF(first);
            return nullptr;
        }
        PyObject *both = PyTuple_Pack(2, first, second);
        Py_DECREF(first);
        Py_DECREF(second);
        return both;
    });
}

/* the code of a result's type: that of `out`, else `dtype`'s, else `standard` */
int result_type(const char *who, PyObject *dtype, const Arg &out, at::ScalarType standard, bool eight_bits, at::ScalarType &type) {
    type = out ? out.t->scalar_type() : standard;
    if (dtype != Py_None) {
        if (!THPDtype_Check(dtype)) refuse("%s: dtype is not a torch.dtype", who);
        type = reinterpret_cast<THPDtype *>(dtype)->scalar_type;
        if (out) out.type(type);
    }
    switch (type) {
        case at::kFloat: return 0;
        case at::kBFloat16: return 1;
        case at::kFloat8_e4m3fn:
            if (eight_bits) return 2;
            [[fallthrough]];
        default: refuse("%s: results of type %s are not computed", who, c10::toString(type));
    }
}

/* (x, weight, residual, gate, eps, dtype, out, scales) -> out, or (out, scales) in 8 bits */
PyObject *rms_norm(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        const char *who = "rms_norm";
        if (nargs != 8) refuse("%s: 8 arguments expected", who);
        if (g_entry.norm == nullptr) throw Refused{PyExc_RuntimeError, "the library is not bound"};
        const Arg x(who, "x", args[0]), weight(who, "weight", args[1]), residual(who, "residual", args[2]), gate(who, "gate", args[3]),
            out(who, "out", args[6]), scales(who, "scales", args[7]);
        x.present();
        for (const Arg *a : {&x, &weight, &residual, &gate, &out, &scales}) a->no_gradient();
        const int64_t n = x.t->dim();
        if (n != 2) x.dims(3);
        GdnB200NormArgs a = {};
        a.dtype = dtype_code(x);
        const c10::Device device = x.t->device();
        x.on(device);
        x.last_contiguous();
        const int64_t tokens = x.t->size(0), heads = n == 3 ? x.t->size(1) : 1, dim = x.t->size(n - 1);
        for (int64_t v : {tokens, heads, dim})
            if (v > 0x7fffffff) refuse("%s: a size of %lld is too large", who, (long long)v);
        if (weight) {
            a.weight_dtype = dtype_code(weight);
            weight.shape({dim});
            weight.on(device);
            weight.last_contiguous();
        }
        if (residual) {
            a.residual_dtype = dtype_code(residual);
            residual.shape(x.t->sizes());
            residual.on(device);
            residual.last_contiguous();
            residual.disjoint();
        }
        if (gate) {
            gate.type(x.t->scalar_type());
            gate.shape(x.t->sizes());
            gate.on(device);
            gate.last_contiguous();
        }
        const double eps = PyFloat_AsDouble(args[4]);
        if (PyErr_Occurred()) return nullptr;
        at::ScalarType type;
        a.out_dtype = result_type(who, args[5], out, x.t->scalar_type(), true, type);
        at::Tensor result, factors;
        if (out) {
            out.shape(x.t->sizes());
            out.on(device);
            out.last_contiguous();
            if (args[6] != args[0]) out.disjoint();
            result = *out.t;
        } else {
            result = at::empty(x.t->sizes(), x.t->options().dtype(type).requires_grad(false));
        }
        if (a.out_dtype == 2) {
            if (scales) {
                scales.type(at::kFloat);
                scales.shape({tokens});
                scales.on(device);
                scales.last_contiguous();
                factors = *scales.t;
            } else {
                factors = at::empty({tokens}, x.t->options().dtype(at::kFloat).requires_grad(false));
            }
            a.scales = static_cast<float *>(factors.data_ptr());
        } else if (scales) {
            refuse("%s: scales are those of 8-bit results", who);
        }
        auto head = [&](const at::Tensor &t) { return n == 3 ? step(t, 1) : dim; };
        a.x = x.ptr<const void>();
        a.gate = gate.ptr<const void>();
        a.weight = weight.ptr<const void>();
        a.residual = residual.ptr<void>();
        a.out = result.data_ptr();
        a.stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
        a.x_token = step(*x.t, 0), a.x_head = head(*x.t);
        if (gate) a.gate_token = step(*gate.t, 0), a.gate_head = head(*gate.t);
        if (residual) a.residual_token = step(*residual.t, 0), a.residual_head = head(*residual.t);
        a.out_token = step(result, 0), a.out_head = head(result);
        a.tokens = (uint32_t)tokens, a.heads = (uint32_t)heads, a.dim = (uint32_t)dim;
        a.device = device.index();
        a.eps = (float)eps;
        called(g_entry.norm(&a));
        residual.written();
        out.written();
        scales.written();
        PyObject *first = out ? Py_NewRef(args[6]) : THPVariable_Wrap(result);
        if (a.out_dtype != 2 || first == nullptr) return first;
        PyObject *second = scales ? Py_NewRef(args[7]) : THPVariable_Wrap(factors);
        PyObject *both = second == nullptr ? nullptr : PyTuple_Pack(2, first, second);
        Py_DECREF(first);
        Py_XDECREF(second);
        return both;
    });
}

/* the number of an activation's name in `names` (None: 0) */
int activation_code(const char *who, PyObject *o, std::initializer_list<const char *> names) {
    if (o == Py_None) return 0;
    const char *name = PyUnicode_Check(o) ? PyUnicode_AsUTF8(o) : nullptr;
    int code = 0;
    std::string all;
    for (const char *n : names) {
        ++code;
        if (name != nullptr && std::string(n) == name) return code;
        all += std::string(all.empty() ? "" : ", ") + n;
    }
    PyErr_Clear();
    refuse("%s: activation is neither None nor one of %s", who, all.c_str());
}

/* (x, weight, bias, activation, residual, x_scales, weight_scales, dtype, out) -> out */
PyObject *linear(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        const char *who = "linear";
        if (nargs != 9) refuse("%s: 9 arguments expected", who);
        if (g_entry.linear == nullptr) throw Refused{PyExc_RuntimeError, "the library is not bound"};
        const Arg x(who, "x", args[0]), weight(who, "weight", args[1]), bias(who, "bias", args[2]), residual(who, "residual", args[4]),
            x_scales(who, "x_scales", args[5]), weight_scales(who, "weight_scales", args[6]), out(who, "out", args[8]);
        x.present();
        weight.present();
        for (const Arg *a : {&x, &weight, &bias, &residual, &x_scales, &weight_scales, &out}) a->no_gradient();
        GdnB200LinearArgs a = {};
        a.activation = activation_code(who, args[3], {"silu", "gelu", "swiglu"});
        x.dims(2);
        weight.dims(2);
        const bool eight = x.t->scalar_type() == at::kFloat8_e4m3fn;
        if (!eight && x.t->scalar_type() != at::kBFloat16)
            refuse("%s: x has type %s, neither bfloat16 nor float8_e4m3fn", who, c10::toString(x.t->scalar_type()));
        a.dtype = eight ? 2 : 1;
        const c10::Device device = x.t->device();
        const int64_t tokens = x.t->size(0), inputs = x.t->size(1), rows = weight.t->size(0);
        for (int64_t v : {tokens, inputs, rows})
            if (v > 0x7fffffff) refuse("%s: a size of %lld is too large", who, (long long)v);
        if (a.activation == 3 && rows % 2 != 0) refuse("%s: swiglu takes the two halves of weight, which has %lld rows", who, (long long)rows);
        const int64_t outputs = a.activation == 3 ? rows / 2 : rows;
        weight.type(x.t->scalar_type());
        weight.shape({rows, inputs});
        for (const Arg *t : {&x, &weight}) {
            t->on(device);
            t->last_contiguous();
        }
        auto vector = [&](const Arg &t, int64_t size) {
            t.shape({size});
            t.on(device);
            t.last_contiguous();
        };
        if ((bool)x_scales != eight || (bool)weight_scales != eight)
            refuse(eight ? "%s: 8-bit x and weight need x_scales and weight_scales" : "%s: x_scales and weight_scales are those of 8-bit operands", who);
        if (eight) {
            x_scales.type(at::kFloat);
            weight_scales.type(at::kFloat);
            vector(x_scales, tokens);
            vector(weight_scales, rows);
        }
        if (bias) {
            a.bias_dtype = dtype_code(bias);
            vector(bias, rows);
        }
        if (residual) {
            a.residual_dtype = dtype_code(residual);
            residual.shape({tokens, outputs});
            residual.on(device);
            residual.last_contiguous();
        }
        at::ScalarType type;
        a.out_dtype = result_type(who, args[7], out, at::kBFloat16, false, type);
        at::Tensor result;
        if (out) {
            out.shape({tokens, outputs});
            out.on(device);
            out.last_contiguous();
            out.disjoint();
            result = *out.t;
        } else {
            result = at::empty({tokens, outputs}, x.t->options().dtype(type).requires_grad(false));
        }
        a.x = x.ptr<const void>();
        a.weight = weight.ptr<const void>();
        a.bias = bias.ptr<const void>();
        a.residual = residual.ptr<const void>();
        a.x_scales = x_scales.ptr<const float>();
        a.weight_scales = weight_scales.ptr<const float>();
        a.out = result.data_ptr();
        a.stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
        a.x_row = step(*x.t, 0), a.weight_row = step(*weight.t, 0), a.out_row = step(result, 0);
        if (residual) a.residual_row = step(*residual.t, 0);
        a.tokens = (uint32_t)tokens, a.inputs = (uint32_t)inputs, a.outputs = (uint32_t)outputs;
        a.device = device.index();
        called(g_entry.linear(&a));
        out.written();
        return out ? Py_NewRef(args[8]) : THPVariable_Wrap(result);
    });
}

/* (x, weight, tails, bias, activation, starts, slots, fresh, out) -> out */
PyObject *short_conv(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        const char *who = "short_conv";
        if (nargs != 9) refuse("%s: 9 arguments expected", who);
        if (g_entry.conv == nullptr) throw Refused{PyExc_RuntimeError, "the library is not bound"};
        const Arg x(who, "x", args[0]), weight(who, "weight", args[1]), tails(who, "tails", args[2]), bias(who, "bias", args[3]),
            starts(who, "starts", args[5]), slots(who, "slots", args[6]), fresh(who, "fresh", args[7]), out(who, "out", args[8]);
        for (const Arg *a : {&x, &weight, &tails}) a->present();
        for (const Arg *a : {&x, &weight, &tails, &bias, &out}) a->no_gradient();
        GdnB200ConvArgs a = {};
        a.activation = activation_code(who, args[4], {"silu"});
        x.dims(2);
        weight.dims(2);
        tails.dims(3);
        a.dtype = dtype_code(x);
        a.weight_dtype = dtype_code(weight);
        a.tail_dtype = dtype_code(tails);
        const c10::Device device = x.t->device();
        const int64_t tokens = x.t->size(0), channels = x.t->size(1), width = weight.t->size(1), n_slots = tails.t->size(0);
        weight.shape({channels, width});
        tails.shape({n_slots, width - 1, channels});
        if (!weight.t->is_contiguous()) refuse("%s: weight is not contiguous", who);
        for (const Arg *t : {&x, &tails}) t->last_contiguous();
        for (const Arg *t : {&x, &weight, &tails}) t->on(device);
        if (bias) {
            bias.type(weight.t->scalar_type());
            bias.shape({channels});
            bias.on(device);
            bias.last_contiguous();
        }
        int64_t sequences = tokens;
        if (starts) {
            starts.type(at::kInt);
            starts.dims(1);
            starts.on(device);
            starts.last_contiguous();
            sequences = starts.t->size(0) - 1;
            if (sequences < 0) refuse("%s: starts has shape [0], expected [sequences + 1]", who);
        }
        if (slots) {
            slots.type(at::kInt);
            slots.shape({sequences});
            slots.on(device);
            slots.last_contiguous();
        }
        if (fresh) {
            if (fresh.t->scalar_type() != at::kByte) fresh.type(at::kBool);
            fresh.shape({sequences});
            fresh.on(device);
            fresh.last_contiguous();
        }
        for (int64_t v : {tokens, sequences, channels, width, n_slots})
            if (v > 0x7fffffff) refuse("%s: a size of %lld is too large", who, (long long)v);
        at::Tensor result;
        if (out) {
            out.type(x.t->scalar_type());
            out.shape(x.t->sizes());
            out.on(device);
            out.last_contiguous();
            out.disjoint();
            result = *out.t;
        } else {
            result = at::empty({tokens, channels}, x.t->options().requires_grad(false));
        }
        a.x = x.ptr<const void>();
        a.weight = weight.ptr<const void>();
        a.bias = bias.ptr<const void>();
        a.tails = tails.ptr<void>();
        a.out = result.data_ptr();
        a.starts = starts.ptr<const int32_t>();
        a.slots = slots.ptr<const int32_t>();
        a.fresh = fresh.ptr<const uint8_t>();
        a.stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
        a.x_token = step(*x.t, 0), a.out_token = step(result, 0);
        a.tails_slot = step(*tails.t, 0), a.tails_row = step(*tails.t, 1);
        a.sequences = (uint32_t)sequences, a.tokens = (uint32_t)tokens, a.channels = (uint32_t)channels;
        a.width = (uint32_t)width, a.tail_slots = (uint32_t)n_slots;
        a.device = device.index();
        called(g_entry.conv(&a));
        tails.written();
        out.written();
        return out ? Py_NewRef(args[8]) : THPVariable_Wrap(result);
    });
}

/* bind(step, chunk, chunk_workspace, logits, norm, linear, conv, last_error): addresses of the C entries */
PyObject *bind(PyObject *, PyObject *args) {
    unsigned long long p[8];
    if (!PyArg_ParseTuple(args, "KKKKKKKK", p, p + 1, p + 2, p + 3, p + 4, p + 5, p + 6, p + 7)) return nullptr;
    g_entry.step = reinterpret_cast<decltype(g_entry.step)>(p[0]);
    g_entry.chunk = reinterpret_cast<decltype(g_entry.chunk)>(p[1]);
    g_entry.chunk_workspace = reinterpret_cast<decltype(g_entry.chunk_workspace)>(p[2]);
    g_entry.logits = reinterpret_cast<decltype(g_entry.logits)>(p[3]);
    g_entry.norm = reinterpret_cast<decltype(g_entry.norm)>(p[4]);
    g_entry.linear = reinterpret_cast<decltype(g_entry.linear)>(p[5]);
    g_entry.conv = reinterpret_cast<decltype(g_entry.conv)>(p[6]);
    g_entry.last_error = reinterpret_cast<decltype(g_entry.last_error)>(p[7]);
    Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"delta_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(delta_step)), METH_FASTCALL, nullptr},
    {"delta_chunk", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(delta_chunk)), METH_FASTCALL, nullptr},
    {"constrain_logits", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(constrain_logits)), METH_FASTCALL, nullptr},
    {"rms_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rms_norm)), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear)), METH_FASTCALL, nullptr},
    {"short_conv", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(short_conv)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_ops_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops_torch(void) { return PyModule_Create(&g_module); }
