// The calls of KvCache and residual_norm from Python: checks of their tensors, results, and the C entry point, without an interpreter's steps between.
// For a few rows such a call is bound by the host: one new row of one sequence took 10.2 us through ctypes, of which the library and the launch are 3.9.
// The entry points come as addresses from the loaded library (setup); nothing of it is linked here, and the library knows nothing of torch.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <vector>

#include "../../include/o1_b200.h"

namespace {

constexpr int64_t D = 128;
decltype(&o1_kv_write) f_write;
decltype(&o1_kv_read) f_read;
decltype(&o1_kv_attention) f_attend;
decltype(&o1_residual_norm) f_norm;
decltype(&o1_get_stream) f_stream;
decltype(&o1_capture_id) f_capture;
PyObject *O1Error, *check;

struct Handle {
    const o1_kv_cache* cache;
    int64_t heads;
    int device;
    struct Work { void* stream; uint64_t capture; int64_t heads; void* p; int64_t bytes; };
    std::vector<Work> work;
};

PyObject* fail(const char* text) {
    PyErr_SetString(O1Error, text);
    return nullptr;
}
PyObject* fail(const char* who, const char* text) {
    PyErr_Format(O1Error, "%s: %s", who, text);
    return nullptr;
}
bool status(hd_status rc, const char* what) {        // Python's check() takes the library's texts and raises
    if (rc == HD_OK) return true;
    PyObject* r = PyObject_CallFunction(check, "is", (int)rc, what);
    Py_XDECREF(r);
    if (r) PyErr_Format(O1Error, "%s failed", what);
    return false;
}

// The library's current stream as torch's, where they differ: what torch allocates, copies and frees on a call's behalf is in the order of the call's kernels.
struct OnLibrary {
    c10::cuda::OptionalCUDAStreamGuard guard;
    explicit OnLibrary(int device) {
        const auto at = (c10::DeviceIndex)device;
        const auto stream = (cudaStream_t)f_stream();
        if (c10::cuda::getCurrentCUDAStream(at).stream() != stream)
            guard.reset_stream(stream ? c10::cuda::getStreamFromExternal(stream, at) : c10::cuda::getDefaultCUDAStream(at));
    }
};

// As torch.empty() makes it, without the dispatcher's steps (0.3 us of a call).
at::Tensor empty_on(at::IntArrayRef size, at::ScalarType type, int device) {
    return at::Tensor(at::detail::empty_cuda(size, type, c10::Device(c10::kCUDA, (c10::DeviceIndex)device), c10::nullopt));
}
bool bf16_on(const at::Tensor& t, int device) { return t.scalar_type() == at::kBFloat16 && t.is_cuda() && t.device().index() == device; }

// bf16 rows [n, heads, 128] whose heads lie side by side; n < 0: any number
bool rows_ok(const at::Tensor& t, int64_t n, int64_t heads, int device, int64_t& ld, const char* who) {
    if (t.dim() != 3 || !bf16_on(t, device) || t.size(1) != heads || t.size(2) != D) {
        PyErr_Format(O1Error, "%s: bf16 [rows, %lld, %lld] on the cache's GPU wanted", who, (long long)heads, (long long)D);
        return false;
    }
    if (t.stride(2) != 1 || (t.stride(1) != D && heads > 1)) { fail(who, "a row's heads must lie side by side"); return false; }
    if (n >= 0 && t.size(0) != n) { fail(who, "another number of rows than the others"); return false; }
    if (t.size(0) > INT32_MAX) { fail(who, "too many rows"); return false; }
    ld = t.size(0) > 1 ? t.stride(0) : heads * D;
    return true;
}
const at::Tensor* tensor(PyObject* o, const char* who) {
    if (!THPVariable_Check(o)) { fail(who, "a tensor wanted"); return nullptr; }
    return &THPVariable_Unpack(o);
}
Handle* handle(PyObject* o) { return (Handle*)PyCapsule_GetPointer(o, "o1_kv_cache"); }
bool arguments(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return n == want;
}
// the int64 slots of a write or read; -1 on error
int64_t slots_of(const at::Tensor& t, const Handle* h, const char* who) {
    if (t.scalar_type() != at::kLong || t.dim() != 1 || !t.is_contiguous() || !t.is_cuda() || t.device().index() != h->device) {
        fail(who, "slots int64 [rows], contiguous, on the cache's GPU wanted");
        return -1;
    }
    return t.size(0);
}

// handle(address of an o1_kv_cache, kv_heads, device index)
PyObject* py_handle(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!arguments(n, 3)) return nullptr;
    const auto address = PyLong_AsUnsignedLongLong(a[0]);
    const auto heads = PyLong_AsLongLong(a[1]), device = PyLong_AsLongLong(a[2]);
    if (PyErr_Occurred()) return nullptr;
    Handle* h = new (std::nothrow) Handle{(const o1_kv_cache*)address, heads, (int)device, {}};
    if (!h) return PyErr_NoMemory();
    return PyCapsule_New(h, "o1_kv_cache", [](PyObject* o) { delete handle(o); });
}

// write(handle, k, v, slots)
PyObject* py_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    static const char* who = "KvCache.write";
    if (!arguments(n, 4)) return nullptr;
    Handle* h = handle(a[0]);
    const at::Tensor *k = tensor(a[1], who), *v = k ? tensor(a[2], who) : nullptr, *slots = v ? tensor(a[3], who) : nullptr;
    if (!h || !slots) return nullptr;
    int64_t ldk, ldv;
    const int64_t rows = slots_of(*slots, h, who);
    if (rows < 0 || !rows_ok(*k, rows, h->heads, h->device, ldk, "KvCache.write: k") || !rows_ok(*v, rows, h->heads, h->device, ldv, "KvCache.write: v")) return nullptr;
    if (!status(f_write(h->cache, k->data_ptr(), ldk, v->data_ptr(), ldv, (const int64_t*)slots->data_ptr(), (int)rows), "o1_kv_write")) return nullptr;
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// read(handle, slots, k or None, v or None) -> (k, v)
PyObject* py_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    static const char* who = "KvCache.read";
    if (!arguments(n, 4)) return nullptr;
    Handle* h = handle(a[0]);
    const at::Tensor* slots = tensor(a[1], who);
    if (!h || !slots) return nullptr;
    const int64_t rows = slots_of(*slots, h, who);
    if (rows < 0) return nullptr;
    const OnLibrary on(h->device);
    at::Tensor out[2];
    int64_t ld[2] = {h->heads * D, h->heads * D};
    for (int i = 0; i < 2; ++i) {
        if (a[2 + i] == Py_None) {
            out[i] = empty_on({rows, h->heads, D}, at::kBFloat16, h->device);
            continue;
        }
        const at::Tensor* t = tensor(a[2 + i], who);
        if (!t || !rows_ok(*t, rows, h->heads, h->device, ld[i], i ? "KvCache.read: v" : "KvCache.read: k")) return nullptr;
        out[i] = *t;
    }
    if (!status(f_read(h->cache, out[0].data_ptr(), ld[0], out[1].data_ptr(), ld[1], (const int64_t*)slots->data_ptr(), (int)rows), "o1_kv_read")) return nullptr;
    PyObject *k = THPVariable_Wrap(out[0]), *v = THPVariable_Wrap(out[1]), *both = k && v ? PyTuple_Pack(2, k, v) : nullptr;
    Py_XDECREF(k);
    Py_XDECREF(v);
    return both;
    END_HANDLE_TH_ERRORS
}

// attend(handle, cache object, q, pages, lens, k or None, v or None, out or None, lse: tensor, True, False or None, scale)
PyObject* py_attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    static const char* who = "KvCache.attend";
    if (!arguments(n, 10)) return nullptr;
    Handle* h = handle(a[0]);
    const at::Tensor *q = tensor(a[2], who), *pages = q ? tensor(a[3], who) : nullptr, *lens = pages ? tensor(a[4], who) : nullptr;
    if (!h || !lens) return nullptr;
    if (q->dim() != 3) return fail(who, "q [batch, heads, 128] wanted");
    const int64_t batch = q->size(0), heads = q->size(1);
    int64_t ldq, ldk = 0, ldv = 0, ldo;
    if (!rows_ok(*q, -1, heads, h->device, ldq, "KvCache.attend: q")) return nullptr;
    auto on_gpu = [&](const at::Tensor& t) { return t.is_cuda() && t.device().index() == h->device; };
    if (pages->scalar_type() != at::kInt || pages->dim() != 2 || pages->size(0) != batch || !on_gpu(*pages)) return fail(who, "pages int32 [batch, width] on the cache's GPU wanted");
    const int64_t width = pages->size(1), ldp = batch > 1 ? pages->stride(0) : width;
    if (width > INT32_MAX) return fail(who, "a table of too many pages");
    if (width > 1 && pages->stride(1) != 1) return fail(who, "the pages of a sequence must lie side by side");
    if (lens->scalar_type() != at::kInt || lens->dim() != 1 || lens->size(0) != batch || !lens->is_contiguous() || !on_gpu(*lens)) return fail(who, "lens int32 [batch] on the cache's GPU wanted");
    if ((a[5] == Py_None) != (a[6] == Py_None)) return fail(who, "k and v [batch, kv_heads, 128], both or neither");
    void *pk = nullptr, *pv = nullptr, *pl = nullptr;
    if (a[5] != Py_None) {
        const at::Tensor *k = tensor(a[5], who), *v = k ? tensor(a[6], who) : nullptr;
        if (!v || !rows_ok(*k, batch, h->heads, h->device, ldk, "KvCache.attend: k") || !rows_ok(*v, batch, h->heads, h->device, ldv, "KvCache.attend: v")) return nullptr;
        pk = k->data_ptr();
        pv = v->data_ptr();
    }
    const OnLibrary on(h->device);
    at::Tensor out, lse;
    if (a[7] == Py_None) {
        out = empty_on({batch, heads, D}, at::kBFloat16, h->device);
        ldo = heads * D;
    } else {
        const at::Tensor* t = tensor(a[7], who);
        if (!t || !rows_ok(*t, batch, heads, h->device, ldo, "KvCache.attend: out")) return nullptr;
        out = *t;
    }
    if (a[8] == Py_True) lse = empty_on({batch, heads}, at::kFloat, h->device);
    else if (a[8] != Py_None && a[8] != Py_False) {
        const at::Tensor* t = tensor(a[8], who);
        if (!t) return nullptr;
        if (t->scalar_type() != at::kFloat || t->dim() != 2 || t->size(0) != batch || t->size(1) != heads || !t->is_contiguous() || !on_gpu(*t)) return fail(who, "lse fp32 [batch, heads] wanted");
        lse = *t;
    }
    if (lse.defined()) pl = lse.data_ptr();
    const double scale = a[9] == Py_None ? 0.08838834764831845 : PyFloat_AsDouble(a[9]);
    if (PyErr_Occurred()) return nullptr;
    void* const stream = f_stream();
    const uint64_t capture = f_capture();
    Handle::Work* work = nullptr;
    for (auto& w : h->work)
        if (w.stream == stream && w.heads == heads) work = &w;
    if (!work || work->capture != capture) {       // the cache object has it
        PyObject* made = PyObject_CallMethod(a[1], "_workspace", "L", (long long)heads);
        if (!made) return nullptr;
        Handle::Work w = {stream, capture, heads, nullptr, 0};
        unsigned long long p = 0;
        long long bytes = 0;
        const int got = PyArg_ParseTuple(made, "KL", &p, &bytes);
        Py_DECREF(made);
        if (!got) return nullptr;
        w.p = (void*)p;
        w.bytes = bytes;
        if (work) *work = w;       // (a stream is in one capture at a time)
        else {
            h->work.push_back(w);
            work = &h->work.back();
        }
    }
    if (!status(f_attend(h->cache, q->data_ptr(), ldq, pk, ldk, pv, ldv, (const int32_t*)pages->data_ptr(), ldp, (int)width, (const int32_t*)lens->data_ptr(), out.data_ptr(), ldo,
                         (float*)pl, (int)batch, (int)heads, (float)scale, work->p, work->bytes), "o1_kv_attention"))
        return nullptr;
    PyObject* o = THPVariable_Wrap(out);
    if (!lse.defined()) return o;
    PyObject *l = THPVariable_Wrap(lse), *both = o && l ? PyTuple_Pack(2, o, l) : nullptr;
    Py_XDECREF(o);
    Py_XDECREF(l);
    return both;
    END_HANDLE_TH_ERRORS
}

// The vectors [cols] or (many) [groups, cols] in o; 0: none, -1: wrong.
int64_t vectors(PyObject* o, int64_t cols, int device, bool many, const char* name, const at::Tensor*& t) {
    t = nullptr;
    if (o == Py_None) return 0;
    if (!(t = tensor(o, "residual_norm"))) return -1;
    const int64_t dim = t->dim();
    if (!bf16_on(*t, device) || dim < 1 || dim > (many ? 2 : 1) || t->size(-1) != cols || !t->is_contiguous() || t->size(0) == 0) {
        PyErr_Format(O1Error, "residual_norm: %s bf16 [%s%lld] wanted", name, many ? "groups, " : "", (long long)cols);
        return -1;
    }
    return dim == 2 ? t->size(0) : 1;
}

// residual_norm(x, branch, pre_w, post_w, gate, scale, shift, alpha, eps, y, h) -> (y, h)
PyObject* py_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    static const char* who = "residual_norm";
    if (!arguments(n, 11)) return nullptr;
    const at::Tensor *x = tensor(a[0], who), *branch = x ? tensor(a[1], who) : nullptr;
    if (!branch) return nullptr;
    if (x->dim() != 2 || branch->dim() != 2 || !x->is_cuda()) return fail(who, "x and branch bf16 [rows, cols] on the GPU wanted");
    const int device = x->device().index();
    const int64_t rows = x->size(0), cols = x->size(1);
    if (rows > INT32_MAX || cols > INT32_MAX) return fail(who, "too many rows or columns");
    auto like_x = [&](const at::Tensor& t) { return t.dim() == 2 && bf16_on(t, device) && t.size(0) == rows && t.size(1) == cols; };
    if (!like_x(*x) || !like_x(*branch)) return fail(who, "x and branch bf16 [rows, cols] on the GPU wanted");
    const at::Tensor *pre, *post, *mod[3];
    const int64_t n_pre = vectors(a[2], cols, device, false, "pre_w", pre), n_post = n_pre < 0 ? -1 : vectors(a[3], cols, device, false, "post_w", post);
    if (n_post < 0) return nullptr;
    static const char* const names[3] = {"gate", "scale", "shift"};
    int64_t groups = 1, each[3];
    for (int i = 0; i < 3; ++i) {
        each[i] = vectors(a[4 + i], cols, device, true, names[i], mod[i]);
        if (each[i] < 0) return nullptr;
        if (each[i] > 1 && groups > 1 && each[i] != groups) return fail(who, "gate, scale and shift differ in groups");
        if (each[i] > groups) groups = each[i];
    }
    if ((mod[1] == nullptr) != (mod[2] == nullptr)) return fail(who, "scale and shift, both or neither");
    const OnLibrary on(device);
    at::Tensor spread[3];
    void* pm[3];
    for (int i = 0; i < 3; ++i) {
        if (mod[i] && groups > 1 && each[i] == 1) {       // one vector for all groups
            spread[i] = mod[i]->reshape({1, cols}).expand({groups, cols}).contiguous();
            mod[i] = &spread[i];
        }
        pm[i] = mod[i] ? mod[i]->data_ptr() : nullptr;
    }
    const double alpha = PyFloat_AsDouble(a[7]), eps = PyFloat_AsDouble(a[8]);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor y, h;
    auto result = [&](PyObject* o, at::Tensor& t) {
        if (o == Py_None) { t = empty_on({rows, cols}, at::kBFloat16, device); return true; }
        const at::Tensor* given = tensor(o, who);
        if (!given) return false;
        if (!like_x(*given)) { fail(who, "y and h bf16 [rows, cols] wanted"); return false; }
        t = *given;
        return true;
    };
    if (!result(a[9], y)) return nullptr;
    if (n_pre) {
        if (!result(a[10], h)) return nullptr;
    } else if (a[10] != Py_None) return fail(who, "h without pre_w");
    int64_t ld[4] = {0, 0, 0, 0};
    const at::Tensor* all[4] = {x, branch, &y, h.defined() ? &h : nullptr};
    for (int i = 0; i < 4; ++i) {
        if (!all[i]) continue;
        if (cols > 1 && all[i]->stride(1) != 1) return fail(who, "the values of a row must lie side by side");
        ld[i] = rows > 1 ? all[i]->stride(0) : cols;
    }
    if (!status(f_norm(x->data_ptr(), ld[0], branch->data_ptr(), ld[1], post ? post->data_ptr() : nullptr, pm[0], (float)alpha, pre ? pre->data_ptr() : nullptr, pm[1], pm[2], (int)groups,
                       y.data_ptr(), ld[2], h.defined() ? h.data_ptr() : nullptr, ld[3], (int)rows, (int)cols, (float)eps), "o1_residual_norm"))
        return nullptr;
    PyObject* py = THPVariable_Wrap(y);
    PyObject* ph = h.defined() ? THPVariable_Wrap(h) : Py_NewRef(Py_None);
    PyObject* both = py && ph ? PyTuple_Pack(2, py, ph) : nullptr;
    Py_XDECREF(py);
    Py_XDECREF(ph);
    return both;
    END_HANDLE_TH_ERRORS
}

// setup(addresses of o1_kv_write, o1_kv_read, o1_kv_attention, o1_residual_norm, o1_get_stream, o1_capture_id; O1Error; check)
PyObject* py_setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!arguments(n, 8)) return nullptr;
    unsigned long long p[6];
    for (int i = 0; i < 6; ++i) p[i] = PyLong_AsUnsignedLongLong(a[i]);
    if (PyErr_Occurred()) return nullptr;
    f_write = (decltype(f_write))p[0];
    f_read = (decltype(f_read))p[1];
    f_attend = (decltype(f_attend))p[2];
    f_norm = (decltype(f_norm))p[3];
    f_stream = (decltype(f_stream))p[4];
    f_capture = (decltype(f_capture))p[5];
    O1Error = Py_NewRef(a[6]);
    check = Py_NewRef(a[7]);
    Py_RETURN_NONE;
}

#define FAST(name, f) {name, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST("setup", py_setup), FAST("handle", py_handle), FAST("write", py_write), FAST("read", py_read), FAST("attend", py_attend),
                         FAST("residual_norm", py_norm), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", "Calls of KvCache and residual_norm.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) != 0) { Py_DECREF(m); return nullptr; }
    return m;
}
