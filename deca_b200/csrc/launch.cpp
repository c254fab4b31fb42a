// Host side of the serving operators: a small CPython extension (deca_b200/_launch.so) that checks the
// tensors of a call, allocates its outputs and workspace and calls the C ABI of libdeca_b200.so.
//
// A decoding step makes a handful of launches per layer that run for a few microseconds each, so what the
// host spends on a call is its cost.  The same checks, allocations and foreign call take 22 - 33 us a call
// in Python (measured on the kernels' first version) and 4 - 6 here.  Nothing is computed in this file.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>
#include <vector>

#include "deca_b200.h"

namespace {

struct PyFailure {};  // a Python exception is set

[[noreturn]] void refuse(const std::string &text) {
    PyErr_SetString(PyExc_ValueError, text.c_str());
    throw PyFailure();
}

// DecaError(status, what) of deca_b200.native
void check_status(int status, const char *what) {
    if (status == DECA_OK) return;
    PyObject *mod = PyImport_ImportModule("deca_b200.native");
    if (mod) {
        PyObject *cls = PyObject_GetAttrString(mod, "DecaError");
        if (cls) {
            PyObject *err = PyObject_CallFunction(cls, "is", status, what);
            if (err) {
                PyErr_SetObject(cls, err);
                Py_DECREF(err);
            }
            Py_DECREF(cls);
        }
        Py_DECREF(mod);
    }
    throw PyFailure();
}

at::ScalarType type_of(int dtype) { return dtype == DECA_F16 ? at::kHalf : at::kBFloat16; }

constexpr int64_t ANY = -1;

std::string text_of(at::IntArrayRef v) {
    std::string s = "(";
    for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + (v[i] == ANY ? std::string("any") : std::to_string(v[i]));
    return s + ")";
}

// A CUDA tensor on the current device with this type and shape whose last dimension is contiguous.  Kernels are
// launched on the current device's current stream and record no gradient, so what lives elsewhere, asks for
// one or carries a tangent is refused.
const at::Tensor &view(PyObject *o, const char *name, at::ScalarType dtype, at::IntArrayRef shape, int device) {
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s: expected a tensor, got %s", name, Py_TYPE(o)->tp_name);
        throw PyFailure();
    }
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda()) refuse(std::string(name) + ": expected a CUDA tensor");
    bool ok = t.scalar_type() == dtype && t.dim() == (int64_t)shape.size() && t.layout() == at::kStrided;
    for (size_t i = 0; ok && i < shape.size(); ++i) ok = shape[i] == ANY || t.size(i) == shape[i];
    if (!ok)
        refuse(std::string(name) + ": expected " + c10::toString(dtype) + " of shape " + text_of(shape) + ", got " +
               c10::toString(t.scalar_type()) + " of shape " + text_of(t.sizes()));
    const int64_t last = t.dim() - 1;
    if (last >= 0 && t.size(last) > 1 && t.stride(last) != 1) refuse(std::string(name) + ": the last dimension must be contiguous");
    if (t.get_device() != device)
        refuse(std::string(name) + ": on cuda:" + std::to_string(t.get_device()) + ", but the current device is cuda:" + std::to_string(device));
    if (t.requires_grad() && c10::GradMode::is_enabled())
        refuse(std::string(name) + ": requires grad, but this operator records no gradient; call it under torch.no_grad()");
    if (t.is_neg()) refuse(std::string(name) + ": a view with pending negation; call it on tensor.resolve_neg()");
    if (t._fw_grad(0).defined()) refuse(std::string(name) + ": carries a forward-mode tangent, but this operator computes none");
    return t;
}

// The current device, once the call's first tensor is known to live on a GPU.
int launch_device(PyObject *first, const char *name) {
    if (!THPVariable_Check(first)) {
        PyErr_Format(PyExc_TypeError, "%s: expected a tensor, got %s", name, Py_TYPE(first)->tp_name);
        throw PyFailure();
    }
    if (!THPVariable_Unpack(first).is_cuda()) refuse(std::string(name) + ": expected a CUDA tensor");
    return c10::cuda::current_device();
}

bool given(PyObject *const *args, Py_ssize_t n, Py_ssize_t i) { return i < n && args[i] != Py_None; }

at::Tensor fresh(at::IntArrayRef shape, at::ScalarType dtype, int device) {
    return at::detail::empty_cuda(shape, dtype, c10::Device(c10::kCUDA, (c10::DeviceIndex)device), std::nullopt);
}

// Several one-dimensional tensors in one allocation, each on a boundary of 256 bytes: an allocation costs the host
// about as much as a launch.
struct Shared {
    int64_t bytes = 0;
    at::Tensor buffer;
    int64_t reserve(int64_t count, int64_t size) {
        const int64_t at = bytes;
        bytes += (count * size + 255) / 256 * 256;
        return at;
    }
    at::Tensor tensor(int64_t at, int64_t count, at::ScalarType dtype) const {
        at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buffer.storage()), buffer.key_set(), c10::scalarTypeToTypeMeta(dtype));
        c10::TensorImpl *impl = t.unsafeGetTensorImpl();
        impl->set_sizes_contiguous({count});
        impl->set_storage_offset(at / (int64_t)c10::elementSize(dtype));
        return t;
    }
};

// An output: the caller's tensor, or a new contiguous one.
at::Tensor output(PyObject *const *args, Py_ssize_t n, Py_ssize_t i, const char *name, at::ScalarType dtype, at::IntArrayRef shape, int device) {
    if (given(args, n, i)) return view(args[i], name, dtype, shape, device);
    return fresh(shape, dtype, device);
}

void *stream_of(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

PyObject *tuple_of(std::initializer_list<at::Tensor> ts) {
    PyObject *out = PyTuple_New((Py_ssize_t)ts.size());
    if (!out) return nullptr;
    Py_ssize_t i = 0;
    for (const at::Tensor &t : ts) PyTuple_SET_ITEM(out, i++, THPVariable_Wrap(t));
    return out;
}

// Runs `body` and turns C++ exceptions into Python ones.
template <typename F>
PyObject *guarded(F body) {
    try {
        return body();
    } catch (const PyFailure &) {
    } catch (const c10::OutOfMemoryError &e) {
        PyObject *mod = PyImport_ImportModule("torch");
        PyObject *cls = mod ? PyObject_GetAttrString(mod, "OutOfMemoryError") : nullptr;
        PyErr_SetString(cls ? cls : PyExc_MemoryError, e.what_without_backtrace());
        Py_XDECREF(cls);
        Py_XDECREF(mod);
    } catch (const c10::Error &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "deca_b200: unknown C++ exception");
    }
    return nullptr;
}

template <typename T>
void destroy(PyObject *capsule) {
    delete static_cast<T *>(PyCapsule_GetPointer(capsule, T::kName));
}
template <typename T>
const T &plan_of(PyObject *const *args, Py_ssize_t n, Py_ssize_t least) {
    if (n < least) {
        PyErr_SetString(PyExc_TypeError, "too few arguments");
        throw PyFailure();
    }
    void *p = PyCapsule_GetPointer(args[0], T::kName);
    if (!p) throw PyFailure();
    return *static_cast<T *>(p);
}
template <typename T>
PyObject *capsule_of(T *plan) {
    PyObject *c = PyCapsule_New(plan, T::kName, destroy<T>);
    if (!c) delete plan;
    return c;
}

// ------------------------------------------------------------------------------- residual RMSNorm
struct AddNormPlan {
    static constexpr const char *kName = "deca_b200.add_rmsnorm";
    int dtype;
    long long M, N, groups;
    float eps;
    int out, group;
};

PyObject *add_rmsnorm_plan(PyObject *, PyObject *args) {
    AddNormPlan p;
    if (!PyArg_ParseTuple(args, "iLLLfii", &p.dtype, &p.M, &p.N, &p.groups, &p.eps, &p.out, &p.group)) return nullptr;
    return capsule_of(new AddNormPlan(p));
}

// (plan, x, res, w[, h, y, scales]) -> (h, y) or (h, y, scales)
PyObject *add_rmsnorm(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const AddNormPlan &p = plan_of<AddNormPlan>(args, n, 4);
        const at::ScalarType dt = type_of(p.dtype);
        const int64_t mn[2] = {p.M, p.N};
        const int dev = launch_device(args[1], "x");
        auto rows = [&](const at::Tensor &t, const char *name) {
            if (p.M > 1 && t.stride(0) < p.N)
                refuse(std::string(name) + ": rows overlap (row stride " + std::to_string(t.stride(0)) + " for " + std::to_string(p.N) + " columns)");
            return t.stride(0);
        };
        const at::Tensor &x = view(args[1], "x", dt, mn, dev), &r = view(args[2], "res", dt, mn, dev);
        const at::Tensor &w = view(args[3], "w", dt, {p.N}, dev);
        const bool eight = p.out == DECA_OUT_E4M3;
        const int64_t sx = rows(x, "x"), sr = rows(r, "res");
        at::Tensor h = output(args, n, 4, "res_out", dt, mn, dev);
        at::Tensor y = output(args, n, 5, "out", eight ? at::kFloat8_e4m3fn : dt, mn, dev);
        at::Tensor s;
        if (eight) {
            s = output(args, n, 6, "scales", at::kFloat, {p.M, p.groups}, dev);
            if (!s.is_contiguous()) refuse("scales: expected a contiguous tensor");
        }
        check_status(deca_add_rmsnorm(p.dtype, x.data_ptr(), sx, r.data_ptr(), sr, w.data_ptr(), h.data_ptr(), rows(h, "res_out"),
                                      y.data_ptr(), rows(y, "out"), eight ? s.data_ptr<float>() : nullptr, p.M, p.N, p.eps, p.out,
                                      p.group, stream_of(dev)),
                     "deca_add_rmsnorm");
        return eight ? tuple_of({h, y, s}) : tuple_of({h, y});
    });
}

// ---------------------------------------------------------------------------------------- rotary
struct RotaryPlan {
    static constexpr const char *kName = "deca_b200.rotary";
    int dtype, D, rot, layout, Hq, Hkv, page_size;  // the last three: of the append
    float amplitude;
    std::vector<uint64_t> turns;
};

PyObject *rotary_plan(PyObject *, PyObject *args) {
    RotaryPlan p;
    PyObject *turns;
    if (!PyArg_ParseTuple(args, "iiiiiiifO!", &p.dtype, &p.D, &p.rot, &p.layout, &p.Hq, &p.Hkv, &p.page_size, &p.amplitude, &PyList_Type, &turns))
        return nullptr;
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(turns); ++i) {
        p.turns.push_back(PyLong_AsUnsignedLongLong(PyList_GET_ITEM(turns, i)));
        if (PyErr_Occurred()) return nullptr;
    }
    if ((int)p.turns.size() != p.rot / 2) {
        PyErr_SetString(PyExc_ValueError, "turns: one for each pair");
        return nullptr;
    }
    return capsule_of(new RotaryPlan(p));
}

deca_rotation rotation_of(const RotaryPlan &p, bool inverse) {
    return deca_rotation{p.D, p.rot, p.layout, inverse ? 1 : 0, p.amplitude, p.turns.data()};
}
deca_tokens tokens_of(const at::Tensor &t) { return deca_tokens{t.data_ptr(), t.stride(0), t.stride(1)}; }
deca_cache cache_of(const at::Tensor &t) { return deca_cache{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)}; }

// A written [tokens, heads, D] tensor may not hold an element twice.
void no_overlap(const at::Tensor &t, const char *name) {
    const int64_t T = t.size(0), H = t.size(1), D = t.size(2), st = t.stride(0), sh = t.stride(1);
    const bool heads_inside = (H <= 1 || sh >= D) && (T <= 1 || st >= (H - 1) * sh + D);
    const bool tokens_inside = (T <= 1 || st >= D) && (H <= 1 || sh >= (T - 1) * st + D);
    if (T > 0 && H > 0 && !heads_inside && !tokens_inside) refuse(std::string(name) + ": elements overlap (strides " + text_of(t.strides()) + ")");
}
// Nor may a cache: its three outer dimensions, taken from the closest one outwards, must each clear the last.
void no_overlap_cache(const at::Tensor &t, const char *name) {
    int64_t end = t.size(3);
    bool done[3] = {false, false, false};
    for (int k = 0; k < 3; ++k) {
        int at = -1;
        for (int i = 0; i < 3; ++i)
            if (!done[i] && (at < 0 || t.stride(i) < t.stride(at))) at = i;
        done[at] = true;
        if (t.size(at) <= 1) continue;
        if (t.stride(at) < end) refuse(std::string(name) + ": elements overlap (strides " + text_of(t.strides()) + ")");
        end += (t.size(at) - 1) * t.stride(at);
    }
}

// (plan, x, positions[, y, inverse]) -> y
PyObject *rotary(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const RotaryPlan &p = plan_of<RotaryPlan>(args, n, 3);
        const at::ScalarType dt = type_of(p.dtype);
        const int dev = launch_device(args[1], "x");
        const at::Tensor &x = view(args[1], "x", dt, {ANY, ANY, p.D}, dev);
        const int64_t T = x.size(0), H = x.size(1);
        if (H > 65536) refuse("x: more than 65536 heads");  // the entry counts them in 32 bits
        const at::Tensor &pos = view(args[2], "positions", at::kInt, {T}, dev);
        at::Tensor y = output(args, n, 3, "out", dt, {T, H, p.D}, dev);
        no_overlap(y, "out");
        const int inverse = given(args, n, 4) ? PyObject_IsTrue(args[4]) : 0;
        if (inverse < 0) throw PyFailure();
        if (T > 0 && H > 0) {
            const deca_rotation rot = rotation_of(p, inverse != 0);
            const deca_tokens xs = tokens_of(x), ys = tokens_of(y);
            check_status(deca_rotary(p.dtype, &xs, &ys, pos.data_ptr<int32_t>(), T, (int)H, &rot, stream_of(dev)), "deca_rotary");
        }
        return THPVariable_Wrap(y);
    });
}

// (plan, q, k, v, positions, slots, k_cache, v_cache[, q_out]) -> q_out
PyObject *rotary_append(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const RotaryPlan &p = plan_of<RotaryPlan>(args, n, 8);
        const at::ScalarType dt = type_of(p.dtype);
        const int dev = launch_device(args[1], "q");
        const at::Tensor &q = view(args[1], "q", dt, {ANY, p.Hq, p.D}, dev);
        const int64_t T = q.size(0);
        const at::Tensor &k = view(args[2], "k", dt, {T, p.Hkv, p.D}, dev), &v = view(args[3], "v", dt, {T, p.Hkv, p.D}, dev);
        const at::Tensor &pos = view(args[4], "positions", at::kInt, {T}, dev), &slots = view(args[5], "slots", at::kLong, {T}, dev);
        const at::Tensor &kc = view(args[6], "k_cache", dt, {ANY, p.page_size, p.Hkv, p.D}, dev);
        const int64_t pages = kc.size(0);
        const at::Tensor &vc = view(args[7], "v_cache", dt, {pages, p.page_size, p.Hkv, p.D}, dev);
        at::Tensor out = output(args, n, 8, "out", dt, {T, p.Hq, p.D}, dev);
        no_overlap(out, "out");
        no_overlap_cache(kc, "k_cache");
        no_overlap_cache(vc, "v_cache");
        if (T > 0) {
            const deca_rotation rot = rotation_of(p, false);
            const deca_tokens qs = tokens_of(q), ks = tokens_of(k), vs = tokens_of(v), os = tokens_of(out);
            const deca_cache kcs = cache_of(kc), vcs = cache_of(vc);
            check_status(deca_rotary_append(p.dtype, &qs, &ks, &vs, &os, &kcs, &vcs, pos.data_ptr<int32_t>(), slots.data_ptr<int64_t>(), T,
                                            p.Hq, p.Hkv, pages, p.page_size, &rot, stream_of(dev)),
                         "deca_rotary_append");
        }
        return THPVariable_Wrap(out);
    });
}

// ------------------------------------------------------------------------------------ paged step
struct StepPlan {
    static constexpr const char *kName = "deca_b200.paged_step";
    int B, page_size, W;
    long long T;
};

PyObject *paged_step_plan(PyObject *, PyObject *args) {
    StepPlan p;
    if (!PyArg_ParseTuple(args, "iiiL", &p.B, &p.page_size, &p.W, &p.T)) return nullptr;
    return capsule_of(new StepPlan(p));
}

// (plan, ctx_lens, new_lens, block_table, free_pages, n_free[, cu_q, kv_lens, positions, slots, n_free_out, short])
// -> the six outputs
PyObject *paged_step(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const StepPlan &p = plan_of<StepPlan>(args, n, 6);
        const int dev = launch_device(args[1], "ctx_lens");
        const at::Tensor &ctx = view(args[1], "ctx_lens", at::kInt, {p.B}, dev), &add = view(args[2], "new_lens", at::kInt, {p.B}, dev);
        const at::Tensor &table = view(args[3], "block_table", at::kInt, {p.B, p.W}, dev);
        const at::Tensor &pages = view(args[4], "free_pages", at::kInt, {ANY}, dev), &n_free = view(args[5], "n_free", at::kInt, {1}, dev);
        const int64_t stride = p.B > 1 ? table.stride(0) : p.W;
        if (stride < p.W) refuse("block_table: rows overlap");
        if (pages.size(0) > 2147483647ll) refuse("free_pages: more than 2^31 - 1 entries");
        at::Tensor cu, kv, pos, slots, left, missing;
        if (n <= 6) {
            Shared all;
            const int64_t a = all.reserve(p.B + 1, 4), b = all.reserve(p.B, 4), c = all.reserve(p.T, 4), d = all.reserve(p.T, 8),
                          e = all.reserve(1, 4), f = all.reserve(1, 4);
            all.buffer = fresh({all.bytes}, at::kByte, dev);
            cu = all.tensor(a, p.B + 1, at::kInt), kv = all.tensor(b, p.B, at::kInt), pos = all.tensor(c, p.T, at::kInt);
            slots = all.tensor(d, p.T, at::kLong), left = all.tensor(e, 1, at::kInt), missing = all.tensor(f, 1, at::kInt);
        } else {
            cu = output(args, n, 6, "cu_q", at::kInt, {p.B + 1}, dev), kv = output(args, n, 7, "kv_lens", at::kInt, {p.B}, dev);
            pos = output(args, n, 8, "positions", at::kInt, {p.T}, dev), slots = output(args, n, 9, "slots", at::kLong, {p.T}, dev);
            left = output(args, n, 10, "n_free_out", at::kInt, {1}, dev), missing = output(args, n, 11, "short", at::kInt, {1}, dev);
        }
        check_status(deca_paged_step(ctx.data_ptr<int32_t>(), add.data_ptr<int32_t>(), p.B, table.data_ptr<int32_t>(), stride, p.W,
                                     pages.data_ptr<int32_t>(), (int)pages.size(0), n_free.data_ptr<int32_t>(), p.page_size, p.T,
                                     cu.data_ptr<int32_t>(), kv.data_ptr<int32_t>(), pos.data_ptr<int32_t>(), slots.data_ptr<int64_t>(),
                                     left.data_ptr<int32_t>(), missing.data_ptr<int32_t>(), stream_of(dev)),
                     "deca_paged_step");
        return tuple_of({cu, kv, pos, slots, left, missing});
    });
}

// ------------------------------------------------------------------------------- paged attention
struct AttnPlan {
    static constexpr const char *kName = "deca_b200.paged_attn";
    deca_paged_attn_args a;
};

PyObject *paged_attn_plan(PyObject *, PyObject *args) {
    AttnPlan p = {};
    deca_paged_attn_args &a = p.a;
    if (!PyArg_ParseTuple(args, "iiiiiiifii", &a.dtype, &a.B, &a.H_q, &a.H_kv, &a.D, &a.page_size, &a.causal, &a.scale, &a.max_q, &a.max_kv))
        return nullptr;
    return capsule_of(new AttnPlan(p));
}

// (plan, q, k_cache, v_cache, block_table, cu_q, kv_lens[, out]) -> out.  The workspace comes from the caching
// allocator for each call, on the call's stream, so calls that overlap (captured ones too) never share one.
PyObject *paged_attn(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        deca_paged_attn_args a = plan_of<AttnPlan>(args, n, 7).a;
        const at::ScalarType dt = type_of(a.dtype);
        const int dev = launch_device(args[1], "q");
        const at::Tensor &q = view(args[1], "q", dt, {ANY, a.H_q, a.D}, dev);
        a.T = q.size(0);
        const at::Tensor &kc = view(args[2], "k_cache", dt, {ANY, a.page_size, a.H_kv, a.D}, dev);
        a.num_pages = kc.size(0);
        const at::Tensor &vc = view(args[3], "v_cache", dt, {a.num_pages, a.page_size, a.H_kv, a.D}, dev);
        const at::Tensor &table = view(args[4], "block_table", at::kInt, {a.B, ANY}, dev);
        const at::Tensor &cu = view(args[5], "cu_q", at::kInt, {a.B + 1}, dev), &kv = view(args[6], "kv_lens", at::kInt, {a.B}, dev);
        at::Tensor out = output(args, n, 7, "out", dt, {a.T, a.H_q, a.D}, dev);
        no_overlap(out, "out");
        if (table.size(1) > 2147483647ll) refuse("block_table: more than 2^31 - 1 entries a request");
        if (a.T > 0) {
            a.table_width = (int)table.size(1);
            a.table_stride = a.B > 1 ? table.stride(0) : table.size(1);
            a.Q = tokens_of(q), a.O = tokens_of(out);
            a.K = cache_of(kc), a.V = cache_of(vc);
            a.block_table = table.data_ptr<int32_t>(), a.cu_q = cu.data_ptr<int32_t>(), a.kv_lens = kv.data_ptr<int32_t>();
            size_t bytes = 0;
            check_status(deca_paged_attn_workspace_bytes(&a, &bytes), "deca_paged_attn_workspace_bytes");
            at::Tensor ws;
            if (bytes > 0) {
                ws = fresh({(int64_t)bytes}, at::kByte, dev);
                a.workspace = ws.data_ptr(), a.workspace_bytes = bytes;
            }
            check_status(deca_paged_attn(&a, stream_of(dev)), "deca_paged_attn");
        }
        return THPVariable_Wrap(out);
    });
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
#define PLAN(name) {#name, name, METH_VARARGS, nullptr}
PyMethodDef methods[] = {PLAN(add_rmsnorm_plan), FAST(add_rmsnorm), PLAN(rotary_plan), FAST(rotary), FAST(rotary_append),
                         PLAN(paged_step_plan), FAST(paged_step), PLAN(paged_attn_plan), FAST(paged_attn), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_launch", "Checked launches of the serving operators", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__launch(void) { return PyModule_Create(&module); }
