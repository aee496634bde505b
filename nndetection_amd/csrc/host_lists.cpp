// Fast path of the optimiser's host side: the tensors of a call to the NndetOptTensor structs of include/nndet_amd.h.
//
// The checks that nndetection_amd/optim.py makes of every tensor (device, type, shape, density, distinct addresses) cost it about 2 us a
// tensor, more than the GPU needs for the step of a network of 92 tensors. pack() makes the same checks here, a few ns each. It knows the
// ordinary case alone -- everything dense on one GPU, in one memory order -- and answers None for anything else: then optim.py looks itself, copies
// what lies in another order, and words the refusal.
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/core/TensorBody.h>

#include <cstring>
#include <vector>

#include "../../include/nndet_amd.h"

namespace {

struct List {                                        // a list or tuple, or nothing
    PyObject* seq = nullptr;
    Py_ssize_t n = 0;
    bool take(PyObject* o) {
        if (o == Py_None) return true;
        if (!PyList_CheckExact(o) && !PyTuple_Check(o)) return false;
        seq = o;
        n = PySequence_Fast_GET_SIZE(o);
        return true;
    }
    PyObject* operator[](Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(seq, i); }
};

// `o` as a plain dense GPU tensor on `device`, or nullptr
c10::TensorImpl* plain(const at::TensorBase& t, c10::DeviceIndex device) {
    if (!t.defined()) return nullptr;
    c10::TensorImpl* x = t.unsafeGetTensorImpl();
    if (x->layout() != c10::kStrided || x->is_python_dispatch() || x->device() != c10::Device(c10::kCUDA, device)) return nullptr;
    if (x->key_set().has(c10::DispatchKey::Negative)) return nullptr;     // (the sign is still to be changed)
    if (!(x->is_contiguous() || x->is_non_overlapping_and_dense())) return nullptr;
    return x;
}
c10::TensorImpl* plain(PyObject* o, c10::DeviceIndex device) {
    return THPVariable_Check(o) ? plain(THPVariable_Unpack(o), device) : nullptr;
}

// of one shape, and in one memory order
bool same(const c10::TensorImpl* a, const c10::TensorImpl* b) {
    return a->sizes().equals(b->sizes()) && ((a->is_contiguous() && b->is_contiguous()) || a->strides().equals(b->strides()));
}

int type_of(const c10::TensorImpl* x) {
    switch (c10::typeMetaToScalarType(x->dtype())) {
        case c10::ScalarType::Float: return NNDET_F32;
        case c10::ScalarType::BFloat16: return NNDET_BF16;
        case c10::ScalarType::Half: return NNDET_F16;
        default: return -1;
    }
}
bool is(const c10::TensorImpl* x, c10::ScalarType t) { return c10::typeMetaToScalarType(x->dtype()) == t; }

struct Addresses {                                   // a set of addresses: open addressing, at most half full
    std::vector<const void*> slot;
    size_t mask;
    explicit Addresses(size_t n) {
        size_t size = 16;
        while (size < 2 * n) size *= 2;
        slot.assign(size, nullptr);
        mask = size - 1;
    }
    bool add(const void* p) {                        // false if it is there already
        for (size_t i = ((uintptr_t)p >> 4) * 0x9E3779B97F4A7C15ull >> 32 & mask;; i = (i + 1) & mask) {
            if (slot[i] == p) return false;
            if (!slot[i]) { slot[i] = p; return true; }
        }
    }
    bool has(const void* p) const {
        for (size_t i = ((uintptr_t)p >> 4) * 0x9E3779B97F4A7C15ull >> 32 & mask;; i = (i + 1) & mask) {
            if (slot[i] == p) return true;
            if (!slot[i]) return false;
        }
    }
};

// pack(params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, root_scales, weight_decay, bits, device, both)
//   -> (structs, n) or None
//   params None: grads alone. grads None: params[i].grad. A gradient that is None leaves its tensor out (slot = place in the list).
//   exp_avgs None: no moments. bits: 32, 8, or 0 for either, by the type of exp_avgs[i]. weight_decay: a number or a list.
//   both: grads are written too. What is written is taken by its mutable address, which gives a lazily cloned tensor memory of its own first.
PyObject* pack(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 10) {
        PyErr_SetString(PyExc_TypeError, "pack() takes 10 arguments");
        return nullptr;
    }
    PyObject* out = nullptr;
    try {
        List p, g, m, v, ms, rs, wd;
        const bool listed = PyList_CheckExact(args[6]) || PyTuple_Check(args[6]);
        if (!p.take(args[0]) || !g.take(args[1]) || !m.take(args[2]) || !v.take(args[3]) || !ms.take(args[4]) || !rs.take(args[5]) || (listed && !wd.take(args[6])))
            Py_RETURN_NONE;
        const double one_wd = listed ? 0.0 : PyFloat_AsDouble(args[6]);
        const long bits = PyLong_AsLong(args[7]), device = PyLong_AsLong(args[8]), both = PyLong_AsLong(args[9]);
        if (PyErr_Occurred()) return nullptr;
        const Py_ssize_t n = p.seq ? p.n : g.n;
        if ((!p.seq && !g.seq) || n >= (1 << 24) || (g.seq && g.n != n) || (m.seq && (!v.seq || m.n != n || v.n != n)) || (listed && wd.n != n)) Py_RETURN_NONE;
        if (ms.seq && (!rs.seq || ms.n != n || rs.n != n)) Py_RETURN_NONE;
        out = PyBytes_FromStringAndSize(nullptr, n * (Py_ssize_t)sizeof(NndetOptTensor));
        if (!out) return nullptr;
        NndetOptTensor* t = reinterpret_cast<NndetOptTensor*>(PyBytes_AS_STRING(out));
        Addresses seen((p.seq ? 1 + (both != 0) : 1) * n + (m.seq ? 2 * n : 0) + (ms.seq ? 2 * n : 0));
        Py_ssize_t k = 0;
        for (Py_ssize_t i = 0; i < n; ++i) {
            c10::TensorImpl *px = nullptr, *gx = nullptr;
            if (g.seq && g[i] == Py_None) continue;
            if (p.seq) {
                px = plain(p[i], device);
                if (!px) goto other;
            }
            if (g.seq) {
                gx = plain(g[i], device);
            } else {
                const at::Tensor& grad = THPVariable_Unpack(p[i]).grad();
                if (!grad.defined()) continue;
                gx = plain(grad, device);
            }
            if (!gx) goto other;
            NndetOptTensor& e = t[k];
            memset(&e, 0, sizeof(e));
            const c10::TensorImpl* x = px ? px : gx;
            const int type = type_of(x);
            if (type < 0 || (px && (px->dtype() != gx->dtype() || !same(px, gx)))) goto other;
            e.param = px ? px->mutable_data() : nullptr;
            e.grad = both ? gx->mutable_data() : const_cast<void*>(gx->data());
            e.numel = x->numel();
            e.slot = (int32_t)i;
            e.dtype = (int16_t)type;
            e.state_bits = 32;
            if (listed) {
                if (!PyFloat_Check(wd[i])) goto other;   // (no Python code runs here that could change the lists)
                e.weight_decay = PyFloat_AS_DOUBLE(wd[i]);
            } else {
                e.weight_decay = one_wd;
            }
            if (m.seq) {
                c10::TensorImpl *mx = plain(m[i], device), *vx = plain(v[i], device);
                if (!mx || !vx || !same(mx, x) || !same(vx, x) || mx->dtype() != vx->dtype()) goto other;
                e.exp_avg = mx->mutable_data();
                e.exp_avg_sq = vx->mutable_data();
                if (is(mx, c10::ScalarType::Float8_e4m3fn) && bits != 32 && ms.seq) {
                    c10::TensorImpl *sx = plain(ms[i], device), *rx = plain(rs[i], device);
                    const int64_t blocks = (e.numel + 255) / 256;
                    if (!sx || !rx || !is(sx, c10::ScalarType::Float) || !is(rx, c10::ScalarType::Float) || sx->numel() != blocks || rx->numel() != blocks) goto other;
                    e.exp_avg_scale = (float*)sx->mutable_data();
                    e.root_scale = (float*)rx->mutable_data();
                    e.state_bits = 8;
                } else if (!is(mx, c10::ScalarType::Float) || bits == 8) {
                    goto other;
                }
            }
            if (e.numel) {                           // what a call writes: no address twice
                if (!seen.add(px ? e.param : e.grad) || (px && both && !seen.add(e.grad))) goto other;
                if (m.seq && (!seen.add(e.exp_avg) || !seen.add(e.exp_avg_sq))) goto other;
                if (e.state_bits == 8 && (!seen.add(e.exp_avg_scale) || !seen.add(e.root_scale))) goto other;
            }
            ++k;
        }
        if (p.seq && !both)                          // what it reads: a gradient may be its own tensor's memory, but no other's
            for (Py_ssize_t i = 0; i < k; ++i)
                if (t[i].numel && seen.has(t[i].grad) && t[i].grad != t[i].param && t[i].grad != t[i].exp_avg && t[i].grad != t[i].exp_avg_sq) goto other;
        if (k != n && _PyBytes_Resize(&out, k * (Py_ssize_t)sizeof(NndetOptTensor)) < 0) return nullptr;
        return Py_BuildValue("Nn", out, k);
    other:
        Py_DECREF(out);
        Py_RETURN_NONE;
    } catch (const std::exception& e) {              // (a tensor without storage, as torch.func's wrappers are)
        Py_XDECREF(out);
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// written(tensors, grads): advance the version counters of the tensors (of those with a gradient, unless grads is None)
PyObject* written(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    List t, g;
    if (nargs != 2 || !t.take(args[0]) || !g.take(args[1]) || (g.seq && g.n != t.n)) {
        PyErr_SetString(PyExc_TypeError, "written(tensors, grads) takes two lists of one length");
        return nullptr;
    }
    try {
        for (Py_ssize_t i = 0; i < t.n; ++i) {
            if ((g.seq && g[i] == Py_None) || !THPVariable_Check(t[i])) continue;
            const at::Tensor& x = THPVariable_Unpack(t[i]);
            if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
        }
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"pack", (PyCFunction)(void (*)(void))pack, METH_FASTCALL, nullptr},
    {"written", (PyCFunction)(void (*)(void))written, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "nndet_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// built_for: the torch and the Python whose headers this was compiled with (build.sh), which the loader compares with those that run
PyMODINIT_FUNC PyInit_nndet_host() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "built_for", NNDET_BUILT_FOR) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
