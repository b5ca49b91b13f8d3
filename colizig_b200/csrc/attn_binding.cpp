// Python side of the attention entry points (include/colizig_cuda.h, Part 3) for
// colizig_b200/attn.py: checks a call's tensors, makes the outputs that were not given and
// calls the library, which only sees raw pointers.  A decode step is a few microseconds
// on the device; the same checks through tensor attributes and ctypes took 8 (decode) to
// 13 us (cache write) of host time a call.
//
// Every function returns its outputs, or the library's return code when that is not 0, and
// raises ValueError for tensors that do not fit.  No C++ exception leaves it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ATen.h>
#include <torch/csrc/autograd/python_variable.h>

#include <sstream>
#include <string>

#include "../../include/colizig_cuda.h"

namespace {

decltype(&colizig_cuda_attn_append) lib_append = nullptr;
decltype(&colizig_cuda_attn_decode) lib_decode = nullptr;
decltype(&colizig_cuda_attn_prefill) lib_prefill = nullptr;

struct Refused {
    std::string why;
};

std::string shown(const at::Tensor& t) {
    std::ostringstream s;
    s << t.scalar_type() << " " << t.sizes() << " (strides " << t.strides() << ") on " << t.device();
    return s.str();
}

const at::Tensor& tensor(const char* name, PyObject* o) {
    if (!THPVariable_Check(o)) throw Refused{std::string(name) + " must be a tensor"};
    return THPVariable_Unpack(o);
}

bool on(const at::Tensor& t, int index) { return t.is_cuda() && t.device().index() == index; }

struct Rows {
    int64_t n, heads, stride;
    const void* at;
};

// [rows, heads, dim] with packed heads and any 16-byte aligned row stride (heads < 0: any number).
Rows rows(const char* name, const at::Tensor& t, int64_t heads, int64_t dim, at::ScalarType dtype, int index) {
    if (t.dim() == 3 && t.scalar_type() == dtype && on(t, index)) {
        const int64_t n = t.size(0), h = t.size(1);
        if (t.size(2) == dim && (heads < 0 || h == heads) && t.stride(2) == 1 && (t.stride(1) == dim || h <= 1)) {
            const int64_t stride = n <= 1 ? h * dim : t.stride(0);  // one row (or none): its stride is never used
            const int64_t elt = (int64_t)t.element_size();
            const void* at = t.const_data_ptr();
            if (stride >= h * dim && ((stride * elt) & 15) == 0 && (reinterpret_cast<uintptr_t>(at) & 15) == 0)
                return {n, h, stride, at};
            throw Refused{std::string(name) + ": rows must be 16-byte aligned and must not overlap, got " + shown(t)};
        }
    }
    std::ostringstream s;
    s << name << " must be " << dtype << " [rows, ";
    heads < 0 ? s << "heads" : s << heads;
    s << ", " << dim << "] with packed heads on cuda:" << index << ", got " << shown(t);
    throw Refused{s.str()};
}

const void* vector(const char* name, const at::Tensor& t, int64_t n, at::ScalarType dtype, int index, bool aligned) {
    if (t.dim() == 1 && t.size(0) == n && t.scalar_type() == dtype && on(t, index) && (n <= 1 || t.stride(0) == 1)) {
        const void* at = t.const_data_ptr();
        if (!aligned || (reinterpret_cast<uintptr_t>(at) & 15) == 0) return at;
    }
    std::ostringstream s;
    s << name << " must be a packed" << (aligned ? ", 16-byte aligned " : " ") << dtype << " tensor [" << n << "] on cuda:"
      << index << ", got " << shown(t);
    throw Refused{s.str()};
}

// The given output, checked, or a new one (`made` keeps it; o None).
void* output(const char* name, PyObject* o, int64_t n, int64_t heads, int64_t dim, const at::Tensor& like, int index,
             at::Tensor& made) {
    if (o == Py_None) {
        made = at::empty({n, heads, dim}, like.options().dtype(at::kBFloat16).requires_grad(false));
        return made.data_ptr();
    }
    made = tensor(name, o);
    if (made.scalar_type() != at::kBFloat16 || made.dim() != 3 || made.size(0) != n || made.size(1) != heads ||
        made.size(2) != dim || !on(made, index) || !made.is_contiguous() ||
        (reinterpret_cast<uintptr_t>(made.data_ptr()) & 15)) {
        std::ostringstream s;
        s << name << " must be a contiguous, 16-byte aligned bf16 tensor [" << n << ", " << heads << ", " << dim
          << "] on cuda:" << index << ", got " << shown(made);
        throw Refused{s.str()};
    }
    return made.data_ptr();
}

PyObject* wrapped(PyObject* given, const at::Tensor& made) {
    if (!made.defined()) Py_RETURN_NONE;
    if (given != Py_None) {
        Py_INCREF(given);
        return given;
    }
    return THPVariable_Wrap(made);
}

int64_t integer(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused{""};
    return v;
}
void* address(PyObject* o) {
    void* p = PyLong_AsVoidPtr(o);
    if (!p && PyErr_Occurred()) throw Refused{""};
    return p;
}
double real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refused{""};
    return v;
}
std::string number(int64_t v) { return std::to_string(v); }

// The library's calls run without the interpreter lock: they wait for the library's mutex, which another thread's
// host-pointer call holds until its stream has finished.
template <class F>
int unlocked(F call) {
    PyThreadState* state = PyEval_SaveThread();
    const int rc = call();
    PyEval_RestoreThread(state);
    return rc;
}

template <class F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F body) {
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, %zd wanted", n, want);
        return nullptr;
    }
    try {
        return body();
    } catch (const Refused& r) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, r.why.c_str());
    } catch (const std::exception& e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 3, [&]() -> PyObject* {
        lib_append = reinterpret_cast<decltype(lib_append)>(address(a[0]));
        lib_decode = reinterpret_cast<decltype(lib_decode)>(address(a[1]));
        lib_prefill = reinterpret_cast<decltype(lib_prefill)>(address(a[2]));
        Py_RETURN_NONE;
    });
}

// append(cache, index, q, k, v, positions, slots, rope, q_norm, k_norm, eps, packed, q_out, k_out, v_out, stream)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 16, [&]() -> PyObject* {
        const auto* cache = reinterpret_cast<const colizig_kv_cache*>(address(a[0]));
        const int index = (int)integer(a[1]);
        const int64_t d = cache->head_dim, hk = cache->kv_heads;
        const at::Tensor& tq = tensor("q", a[2]);
        const at::ScalarType dt = tq.scalar_type() == at::kFloat ? at::kFloat : at::kBFloat16;
        const Rows q = rows("q", tq, -1, d, dt, index);
        if (q.heads < 1 || q.heads % hk)
            throw Refused{number(q.heads) + " query heads are not a multiple of " + number(hk) + " key/value heads"};
        const at::Tensor& tk = tensor("k", a[3]);
        const Rows k = rows("k", tk, hk, d, dt, index);
        const Rows v = rows("v", tensor("v", a[4]), hk, d, dt, index);
        if (k.n != q.n || v.n != q.n) throw Refused{"q, k and v must hold the same tokens"};
        if (q.n > 0x7fffffff) throw Refused{"too many tokens"};
        const void* slots = vector("slots", tensor("slots", a[6]), q.n, at::kLong, index, false);
        const void *rope = nullptr, *positions = nullptr;
        int64_t rope_len = 0, rot = 0;
        if (a[7] != Py_None) {
            const at::Tensor& r = tensor("rope", a[7]);
            if (r.dim() != 2 || r.scalar_type() != at::kFloat || !on(r, index) || !r.is_contiguous() ||
                (reinterpret_cast<uintptr_t>(r.const_data_ptr()) & 15) || r.size(1) % 16 || r.size(1) < 1 ||
                r.size(1) > d || r.size(0) < 1 || r.size(0) > 0x7fffffff)
                throw Refused{"rope must be a contiguous f32 [positions, rot_dim] table on cuda:" + number(index) +
                              ", rot_dim a multiple of 16 up to " + number(d) + ", got " + shown(r)};
            rope = r.const_data_ptr();
            rope_len = r.size(0);
            rot = r.size(1);
            positions = vector("positions", tensor("positions", a[5]), q.n, at::kInt, index, false);
        }
        const void* qn = a[8] == Py_None ? nullptr : vector("q_norm", tensor("q_norm", a[8]), d, at::kFloat, index, true);
        const void* kn = a[9] == Py_None ? nullptr : vector("k_norm", tensor("k_norm", a[9]), d, at::kFloat, index, true);
        const float eps = (float)real(a[10]);
        const int packed = PyObject_IsTrue(a[11]);
        if (packed < 0) return nullptr;
        at::Tensor qo, ko, vo;
        void* qp = output("q_out", a[12], q.n, q.heads, d, tq, index, qo);
        void* kp = packed || a[13] != Py_None ? output("k_out", a[13], q.n, hk, d, tk, index, ko) : nullptr;
        void* vp = packed || a[14] != Py_None ? output("v_out", a[14], q.n, hk, d, tk, index, vo) : nullptr;
        void* stream = address(a[15]);
        const int rc = unlocked([&] {
            return lib_append(cache, q.at, k.at, v.at, dt == at::kFloat ? COLIZIG_X_F32 : COLIZIG_X_BF16, (int)q.n,
                              (uint32_t)q.heads, q.stride, k.stride, v.stride, static_cast<const int32_t*>(positions),
                              static_cast<const int64_t*>(slots), static_cast<const float*>(rope), (uint32_t)rope_len,
                              (uint32_t)rot, static_cast<const float*>(qn), static_cast<const float*>(kn), eps, qp, kp, vp,
                              stream);
        });
        if (rc) return PyLong_FromLong(rc);
        PyObject* out[3] = {wrapped(a[12], qo), wrapped(a[13], ko), wrapped(a[14], vo)};
        PyObject* t = out[0] && out[1] && out[2] ? PyTuple_Pack(3, out[0], out[1], out[2]) : nullptr;
        for (PyObject* o : out) Py_XDECREF(o);
        return t;
    });
}

// decode(cache, index, q_heads, max_batch, scale, workspace, q, table, lens, out, stream)
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 11, [&]() -> PyObject* {
        const auto* cache = reinterpret_cast<const colizig_kv_cache*>(address(a[0]));
        const int index = (int)integer(a[1]);
        const int64_t hq = integer(a[2]), most = integer(a[3]), d = cache->head_dim;
        const at::Tensor& tq = tensor("q", a[6]);
        const Rows q = rows("q", tq, hq, d, at::kBFloat16, index);
        if (q.n > most) throw Refused{number(q.n) + " sequences, the plan holds " + number(most)};
        const at::Tensor& t = tensor("table", a[7]);
        if (t.dim() != 2 || t.size(0) != q.n || t.size(1) < 1 || t.size(1) > 0x7fffffff || t.scalar_type() != at::kInt ||
            !on(t, index) || (t.stride(1) != 1 && t.size(1) > 1) || (q.n > 1 && t.stride(0) < t.size(1)))
            throw Refused{"table must be an int32 tensor [" + number(q.n) + ", width] on cuda:" + number(index) +
                          " whose rows are packed and do not overlap, got " + shown(t)};
        const void* lens = vector("lens", tensor("lens", a[8]), q.n, at::kInt, index, false);
        at::Tensor o;
        void* op = output("out", a[9], q.n, hq, d, tq, index, o);
        const void* table = t.const_data_ptr();
        const int64_t width = t.size(1), row = q.n > 1 ? t.stride(0) : width;
        const float scale = (float)real(a[4]);
        void *workspace = address(a[5]), *stream = address(a[10]);
        const int rc = unlocked([&] {
            return lib_decode(cache, q.at, q.stride, (int)q.n, (uint32_t)hq, static_cast<const int32_t*>(table),
                              (uint32_t)width, row, static_cast<const int32_t*>(lens), scale, op, workspace, stream);
        });
        return rc ? PyLong_FromLong(rc) : wrapped(a[9], o);
    });
}

// prefill(index, q, k, v, cu_q, cu_k, scale, out, stream)
PyObject* prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 9, [&]() -> PyObject* {
        const int index = (int)integer(a[0]);
        const at::Tensor& tq = tensor("q", a[1]);
        const int64_t d = tq.dim() == 3 ? tq.size(2) : 0;
        if (d != 64 && d != 128) throw Refused{"q must be [rows, heads, 64 or 128], got " + shown(tq)};
        const Rows q = rows("q", tq, -1, d, at::kBFloat16, index);
        const Rows k = rows("k", tensor("k", a[2]), -1, d, at::kBFloat16, index);
        const Rows v = rows("v", tensor("v", a[3]), k.heads, d, at::kBFloat16, index);
        if (k.heads < 1 || q.heads < 1 || q.heads % k.heads || v.n != k.n)
            throw Refused{"q, k and v do not belong together: " + number(q.heads) + " query heads, " + number(k.heads) +
                          " key/value heads, " + number(k.n) + " and " + number(v.n) + " rows of k and v"};
        if (q.n > 0x7fffffff || k.n > 0x7fffffff) throw Refused{"too many tokens"};
        const at::Tensor& cq = tensor("cu_q", a[4]);
        const int64_t m = cq.dim() == 1 ? cq.size(0) : 0;
        if (m < 1) throw Refused{"cu_q must hold at least the leading 0"};
        const bool same = a[5] == Py_None;
        if (same && q.n != k.n) throw Refused{"without cu_k, q and k must hold the same tokens"};
        const void* cqp = vector("cu_q", cq, m, at::kInt, index, false);
        const void* ckp = same ? cqp : vector("cu_k", tensor("cu_k", a[5]), m, at::kInt, index, false);
        at::Tensor o;
        void* op = output("out", a[7], q.n, q.heads, d, tq, index, o);
        const float scale = (float)real(a[6]);
        void* stream = address(a[8]);
        const int rc = unlocked([&] {
            return lib_prefill(q.at, k.at, v.at, q.stride, k.stride, v.stride, (int)q.n, (int)k.n, (int)(m - 1),
                               (uint32_t)q.heads, (uint32_t)k.heads, (uint32_t)d, static_cast<const int32_t*>(cqp),
                               static_cast<const int32_t*>(ckp), scale, op, stream);
        });
        return rc ? PyLong_FromLong(rc) : wrapped(a[7], o);
    });
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f))
PyMethodDef methods[] = {{"bind", FAST(bind), METH_FASTCALL, "addresses of the library's append, decode, prefill"},
                         {"append", FAST(append), METH_FASTCALL, nullptr},
                         {"decode", FAST(decode), METH_FASTCALL, nullptr},
                         {"prefill", FAST(prefill), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_attn_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__attn_native(void) { return PyModule_Create(&module); }
