// The short way from Python's lists of tensors to the calls of include/cista_optim.h: one call reads
// the tensors, allocates, and launches.  Reading 25 gradients from Python (address, size, type,
// device, strides) takes 12 us, which is more than the kernels' own time at the default network's
// size; here it takes 0.6 us.
//
// Whatever is not plain (a type, layout, device or state that needs a check, a message or a copy)
// makes the entry return NotImplemented before anything has been launched or changed; the Python
// caller (v2e2v_amd/optim.py) then takes its own way, which handles or refuses it.  No C++ exception
// leaves an entry.  Called through ctypes.PyDLL, with the GIL held.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <cmath>
#include <vector>

#include "../../include/cista_lstc.h"
#include "../../include/cista_optim.h"

namespace {

struct NotPlain {};
struct Failed {                          // a status that the caller turns into its error
    int status;
};

int type_of(const at::Tensor &t) {
    switch (t.scalar_type()) {
    case at::kFloat: return CISTA_F32;
    case at::kBFloat16: return CISTA_BF16;
    case at::kHalf: return CISTA_F16;
    default: throw NotPlain();
    }
}

const at::Tensor &tensor_of(PyObject *o) {
    if (!o || !THPVariable_Check(o)) throw NotPlain();
    return THPVariable_Unpack(o);
}

// a dense tensor on the device of the others
void plain(const at::Tensor &t, int &device) {
    if (t.layout() != at::kStrided || !t.is_cuda() || t.is_neg() || t.is_inference() ||
        t.unsafeGetTensorImpl()->is_python_dispatch() || t._is_zerotensor() || !t.is_non_overlapping_and_dense())
        throw NotPlain();
    if (device < 0) device = t.get_device();
    if (t.get_device() != device) throw NotPlain();
}

struct List {                            // a list's or tuple's items
    PyObject *const *items;
    Py_ssize_t n;
    explicit List(PyObject *o) {
        if (!o || !(PyList_CheckExact(o) || PyTuple_CheckExact(o))) throw NotPlain();
        items = PySequence_Fast_ITEMS(o);
        n = PySequence_Fast_GET_SIZE(o);
    }
};

std::vector<cista_tensor> read(PyObject *list, bool grads, int &device) {
    const List l(list);
    std::vector<cista_tensor> out;
    out.reserve(l.n);
    for (Py_ssize_t i = 0; i < l.n; ++i) {
        const at::Tensor &x = tensor_of(l.items[i]);
        if (grads && !x.is_leaf()) throw NotPlain();
        const at::Tensor &t = grads ? x.grad() : x;
        if (!t.defined()) {
            if (!grads) throw NotPlain();
            continue;
        }
        plain(t, device);
        out.push_back({t.numel() ? t.data_ptr() : nullptr, t.numel(), type_of(t)});
    }
    if (out.empty()) throw NotPlain();
    return out;
}

void changed(PyObject *list) {
    const List l(list);
    for (Py_ssize_t i = 0; i < l.n; ++i) {
        const at::Tensor &g = THPVariable_Unpack(l.items[i]).grad();
        if (g.defined()) g.unsafeGetTensorImpl()->bump_version();
    }
}

struct Call {                            // device, stream and memory of one call
    c10::DeviceGuard guard;
    at::Tensor norm, workspace;
    void *stream;
    Call(int device, size_t n, bool has_norm)
        : guard(c10::Device(c10::kCUDA, (c10::DeviceIndex)device)),
          stream(c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream()) {
        const auto on = at::TensorOptions().device(c10::Device(c10::kCUDA, (c10::DeviceIndex)device));
        if (has_norm) norm = at::empty({}, on.dtype(at::kFloat));
        workspace = at::empty({(int64_t)cista_optim_workspace_bytes((int)n)}, on.dtype(at::kByte));
    }
    float *norm_at() { return norm.defined() ? norm.data_ptr<float>() : nullptr; }
    PyObject *result() {
        if (norm.defined()) return THPVariable_Wrap(norm);
        Py_RETURN_NONE;
    }
};

void must(int status) {
    if (status != CISTA_OK) throw Failed{status};
}

// `f`'s result; NotImplemented for what is not plain, the status as an int for a refused call
template <typename F> PyObject *guarded(F f) {
    try {
        return f();
    } catch (const Failed &e) {
        return PyLong_FromLong(e.status);
    } catch (...) {
        PyErr_Clear();
        Py_RETURN_NOTIMPLEMENTED;
    }
}

PyObject *item(PyObject *dict, PyObject *key) {
    PyObject *o = PyDict_GetItemWithError(dict, key);
    if (!o) throw NotPlain();
    return o;
}

bool has(PyObject *dict, PyObject *key) {
    const int found = PyDict_Contains(dict, key);
    if (found < 0) throw NotPlain();
    return found;
}

double number(PyObject *o) {
    if (PyFloat_CheckExact(o)) return PyFloat_AS_DOUBLE(o);
    if (!PyLong_Check(o)) throw NotPlain();
    const double x = PyLong_AsDouble(o);
    if (x == -1.0 && PyErr_Occurred()) throw NotPlain();
    return x;
}

int truth(PyObject *o) {
    const int x = PyObject_IsTrue(o);
    if (x < 0) throw NotPlain();
    return x;
}

struct Keys {
    PyObject *params, *lr, *betas, *eps, *weight_decay, *decoupled, *maximize, *step, *exp_avg, *exp_avg_sq, *master;
    Keys() {
        auto s = [](const char *t) { return PyUnicode_InternFromString(t); };
        params = s("params"), lr = s("lr"), betas = s("betas"), eps = s("eps"), weight_decay = s("weight_decay");
        decoupled = s("decoupled_weight_decay"), maximize = s("maximize"), step = s("step");
        exp_avg = s("exp_avg"), exp_avg_sq = s("exp_avg_sq"), master = s("master");
    }
};

bool same_layout(const at::Tensor &a, const at::Tensor &b) {
    return a.sizes() == b.sizes() && ((a.is_contiguous() && b.is_contiguous()) || a.strides() == b.strides());
}

float *moment(PyObject *slot, PyObject *key, const at::Tensor &p, int &device) {
    const at::Tensor &t = tensor_of(item(slot, key));
    plain(t, device);
    if (t.scalar_type() != at::kFloat || !same_layout(t, p)) throw NotPlain();
    return t.numel() ? t.data_ptr<float>() : nullptr;
}

}  // namespace

extern "C" {

// the torch whose headers this was built with: another one's tensors may be laid out in another way
const char *cista_torch_version() { return TORCH_VERSION; }

// the norm of the list's tensors
PyObject *cista_torch_grad_norm(PyObject *tensors, int norm_kind) {
    return guarded([&] {
        int device = -1;
        const auto t = read(tensors, false, device);
        Call c(device, t.size(), true);
        must(cista_grad_norm(t.data(), (int)t.size(), norm_kind, c.norm_at(), c.workspace.data_ptr(), c.workspace.numel(),
                             c.stream));
        return c.result();
    });
}

// clips the gradients of the list's parameters; the norm that they had
PyObject *cista_torch_clip_grads(PyObject *parameters, int norm_kind, double max_norm) {
    return guarded([&] {
        int device = -1;
        const auto t = read(parameters, true, device);
        Call c(device, t.size(), true);
        must(cista_clip_grads(t.data(), (int)t.size(), norm_kind, max_norm, c.norm_at(), c.workspace.data_ptr(),
                              c.workspace.numel(), c.stream));
        changed(parameters);
        return c.result();
    });
}

// one Adam step over an optimizer's param_groups (a list of dicts) with its state (a dict); None, or the norm
PyObject *cista_torch_adam_step(PyObject *param_groups, PyObject *state, int norm_kind, double max_norm) {
    return guarded([&] {
        static const Keys key;
        const List list(param_groups);
        if (!PyDict_Check(state)) throw NotPlain();
        int device = -1;
        std::vector<cista_adam_tensor> rows;
        std::vector<cista_adam_group> groups;
        std::vector<c10::TensorImpl *> written;
        for (Py_ssize_t k = 0; k < list.n; ++k) {
            PyObject *g = list.items[k];
            if (!PyDict_Check(g)) throw NotPlain();
            const List params(item(g, key.params));
            const size_t before = rows.size();
            for (Py_ssize_t i = 0; i < params.n; ++i) {
                const at::Tensor &p = tensor_of(params.items[i]);
                if (!p.is_leaf()) throw NotPlain();
                const at::Tensor &grad = p.grad();
                if (!grad.defined()) continue;
                plain(p, device);
                plain(grad, device);
                if (grad.scalar_type() != p.scalar_type() || !same_layout(grad, p)) throw NotPlain();
                PyObject *slot = item(state, params.items[i]);
                if (!PyDict_Check(slot)) throw NotPlain();
                const at::Tensor &step = tensor_of(item(slot, key.step));
                plain(step, device);
                if (step.scalar_type() != at::kFloat || step.numel() != 1) throw NotPlain();
                cista_adam_tensor r;
                r.type = type_of(p);
                r.numel = p.numel();
                r.param = r.numel ? p.data_ptr() : nullptr;
                r.grad = r.numel ? grad.data_ptr() : nullptr;
                r.exp_avg = moment(slot, key.exp_avg, p, device);
                r.exp_avg_sq = moment(slot, key.exp_avg_sq, p, device);
                // a float32 parameter has no master copy; one left from 16-bit steps is dropped in Python
                if (r.type == CISTA_F32 && has(slot, key.master)) throw NotPlain();
                r.master = r.type == CISTA_F32 ? nullptr : moment(slot, key.master, p, device);
                r.step = step.data_ptr<float>();
                rows.push_back(r);
                written.push_back(p.unsafeGetTensorImpl());
            }
            cista_adam_group q = {};
            PyObject *lr = item(g, key.lr);
            if (THPVariable_Check(lr)) {
                const at::Tensor &t = THPVariable_Unpack(lr);
                plain(t, device);
                if (t.scalar_type() != at::kFloat || t.numel() != 1) throw NotPlain();
                q.lr_device = t.data_ptr<float>();
            } else {
                q.lr = number(lr);
            }
            const List betas(item(g, key.betas));
            if (betas.n != 2) throw NotPlain();
            q.beta1 = number(betas.items[0]);
            q.beta2 = number(betas.items[1]);
            q.eps = number(item(g, key.eps));
            q.weight_decay = number(item(g, key.weight_decay));
            q.decoupled = truth(item(g, key.decoupled));
            q.maximize = truth(item(g, key.maximize));
            q.n = (int)(rows.size() - before);
            groups.push_back(q);
        }
        if (rows.empty()) throw NotPlain();
        Call c(device, rows.size(), norm_kind != 0);
        must(cista_adam_step(rows.data(), groups.data(), (int)groups.size(), norm_kind, max_norm, c.norm_at(),
                             c.workspace.data_ptr(), c.workspace.numel(), c.stream));
        for (c10::TensorImpl *t : written) t->bump_version();
        return c.result();
    });
}

}  // extern "C"
