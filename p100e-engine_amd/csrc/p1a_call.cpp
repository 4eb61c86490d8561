// The Python side of a call in native code: arguments -> the C ABI of include/p1a_attn.h. A one-row step of a small model is
// bound by what the host does around its three launches, and half of what was not the launches was the ctypes call: 19
// arguments converted one by one, a descriptor built field by field, a stream looked up from Python. The calls a step is made of
// come here instead; arguments are taken as ctypes takes them (whole numbers cut to 32 bits, floats, ctypes numbers of the parameter's
// type, what _as_parameter_ stands for, None for a null pointer, anything with data_ptr() as a device pointer), and the GIL is released around the call. One token of 4 heads of 64, prep and decode from Python:
// 18.1 us with ctypes, 15.6 so (7.7 of them the C calls, 3.5 the caller's own indexing); two layers of 24 / 4 heads of 96 34.4 -> 29.2.
// The small calls around a drafted tree, a launch of 2 ... 5 us each, come here too, with their checks of tensors: masks of
// a tree's nodes 6.8 -> 6.2 us, an accepted path moved 7.3 -> 6.8 (2.7 of them the launch, 1.3 the caller's Rows).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>
#include <cstring>

#include "p1a_attn.h"

namespace {

PyObject * s_data_ptr, * s_struct, * s_value, * s_as_parameter, * s_field[11], * s_dtype, * s_numel, * s_is_contiguous, * s_size, * s_T, * s_n_seq, * s_st, * last_dim;
const char * const FIELDS[11] = {"type", "n_ctx", "Hkv", "D", "k", "v", "pt", "rtab", "psh", "pstride", "_pt_off"};
enum { INT, UINT, SIZE, FLOAT, POINTER, DESC, NCLASS };

// A module's state (a process may load the binding more than once), set by bind()
struct calls {
    // the library's entry points, the class whose fields are read directly, and how the current stream is found
    decltype(&p1a_attn_prep) f_prep;
    decltype(&p1a_attn_decode_a16) f_decode;
    decltype(&p1a_attn_prefill) f_prefill;
    decltype(&p1a_kv_append) f_append;
    PyObject * kv_class, * stream_of;
    // the same of drafted trees, set by bind_trees(): what checks a tensor and says what is wrong with it, and torch's int32
    decltype(&p1a_tree_rows) f_rows;
    decltype(&p1a_tree_commit) f_commit;
    PyObject * check, * int32;
    PyObject * classes[NCLASS];   // ctypes' c_int, c_uint32, c_size_t, c_float, c_void_p, and the descriptor's Structure

    // (each reader does nothing once an error is set, so that the callers test for one at the end)
    // The value of a ctypes number, for a parameter of just that type; else null. of: its class (c_int, c_float, ...)
    PyObject * plain(PyObject * o, int of) {
        if (PyErr_Occurred()) return nullptr;
        const int is = PyObject_IsInstance(o, classes[of]);
        return is == 1 ? PyObject_GetAttr(o, s_value) : nullptr;
    }
    // what an argument says it stands for, or null (and the error there was stays)
    PyObject * stand_in(PyObject * o, bool argument) {
        if (!argument || !PyErr_ExceptionMatches(PyExc_TypeError)) return nullptr;
        PyObject * t, * v, * tb;
        PyErr_Fetch(&t, &v, &tb);
        PyObject * r = PyObject_GetAttr(o, s_as_parameter);
        if (!r) { PyErr_Clear(); PyErr_Restore(t, v, tb); return nullptr; }
        Py_XDECREF(t); Py_XDECREF(v); Py_XDECREF(tb);
        return r;
    }
    uint64_t whole(PyObject * o, int of, bool argument = true) {
        if (PyErr_Occurred()) return 0;
        if (PyLong_CheckExact(o)) return (uint64_t) PyLong_AsUnsignedLongMask(o);
        uint64_t r = 0;
        if (PyObject * v = plain(o, of)) { r = whole(v, of, false); Py_DECREF(v); return r; }
        if (PyErr_Occurred()) return 0;
        if (PyFloat_Check(o)) PyErr_SetString(PyExc_TypeError, "int expected instead of float instance");
        else r = (uint64_t) PyLong_AsUnsignedLongMask(o);
        if (PyErr_Occurred())
            if (PyObject * v = stand_in(o, argument)) { r = Py_EnterRecursiveCall(" in a call's argument") ? 0 : (r = whole(v, of), Py_LeaveRecursiveCall(), r); Py_DECREF(v); }
        return r;
    }
    int as_int(PyObject * o) { return (int) (uint32_t) whole(o, INT); }
    size_t as_size(PyObject * o) { return (size_t) whole(o, SIZE); }
    float as_float(PyObject * o) {
        if (PyErr_Occurred()) return 0.f;
        if (PyFloat_CheckExact(o)) return (float) PyFloat_AS_DOUBLE(o);
        float r = 0.f;
        if (PyObject * v = plain(o, FLOAT)) { r = as_float(v); Py_DECREF(v); return r; }
        if (PyErr_Occurred()) return 0.f;
        r = (float) PyFloat_AsDouble(o);
        if (PyErr_Occurred())
            if (PyObject * v = stand_in(o, true)) { r = Py_EnterRecursiveCall(" in a call's argument") ? 0.f : (r = as_float(v), Py_LeaveRecursiveCall(), r); Py_DECREF(v); }
        return r;
    }
    // a pointer: None, a Python int, a c_void_p
    void * address(PyObject * o) {
        if (PyErr_Occurred() || o == Py_None) return nullptr;
        if (PyLong_Check(o)) return (void *) (uintptr_t) PyLong_AsUnsignedLongMask(o);
        void * r = nullptr;
        if (PyObject * v = plain(o, POINTER)) { r = address(v); Py_DECREF(v); }
        else if (!PyErr_Occurred()) PyErr_Format(PyExc_TypeError, "address expected instead of %s instance", Py_TYPE(o)->tp_name);
        return r;
    }
    PyObject * data_ptr_of(PyObject * t) { return PyErr_Occurred() ? nullptr : PyObject_CallMethodNoArgs(t, s_data_ptr); }
    void * data_ptr(PyObject * t) {
        if (PyErr_Occurred() || t == Py_None) return nullptr;
        PyObject * r = data_ptr_of(t);
        if (!r) return nullptr;
        void * p = address(r);
        Py_DECREF(r);
        return p;
    }
    template <typename T> T * ptr(PyObject * t) { return (T *) data_ptr(t); }
    // the page table from its entry `off` on
    const int32_t * table(PyObject * t, PyObject * off) {
        if (PyErr_Occurred() || t == Py_None) return nullptr;
        PyObject * r = data_ptr_of(t);
        if (!r) return nullptr;
        const char * p = nullptr;
        if (PyLong_Check(r) && PyLong_Check(off)) p = (const char *) (uintptr_t) PyLong_AsUnsignedLongMask(r) + 4 * (ptrdiff_t) PyLong_AsUnsignedLongMask(off);
        else PyErr_SetString(PyExc_TypeError, "the page table's address and offset are whole numbers");
        Py_DECREF(r);
        return (const int32_t *) p;
    }

    // the cache's descriptor as it is now: a KVCache's fields, or what its struct() gives
    bool describe(PyObject * c, p1a_kv & kv) {
        if (PyErr_Occurred()) return false;
        if ((PyObject *) Py_TYPE(c) != kv_class) {
            PyObject * st = PyObject_CallMethodNoArgs(c, s_struct);
            if (!st) return false;
            Py_buffer b;
            const int is = PyObject_IsInstance(st, classes[DESC]);
            if (is == 0) PyErr_SetString(PyExc_TypeError, "struct() gave no p1a_kv");
            if (is == 1 && PyObject_GetBuffer(st, &b, PyBUF_SIMPLE) == 0) {
                memcpy(&kv, b.buf, sizeof kv);
                PyBuffer_Release(&b);
            }
            Py_DECREF(st);
            return !PyErr_Occurred();
        }
        PyObject * f[11] = {};
        for (int i = 0; i < 11 && !PyErr_Occurred(); ++i) f[i] = PyObject_GetAttr(c, s_field[i]);
        if (!PyErr_Occurred()) {
            kv.type = (uint32_t) whole(f[0], UINT, false);
            kv.n_ctx = (int) whole(f[1], INT, false); kv.Hkv = (int) whole(f[2], INT, false); kv.D = (int) whole(f[3], INT, false);
            kv.k = address(f[4]); kv.v = address(f[5]);
            kv.pt = table(f[6], f[10]);
            kv.rtab = ptr<int32_t>(f[7]);
            kv.psh = (int) whole(f[8], INT, false);
            kv.pstride = (size_t) whole(f[9], SIZE, false);
        }
        for (PyObject * x : f) Py_XDECREF(x);
        return !PyErr_Occurred();
    }
    long long number(PyObject * r) {                          // of a call or an attribute, which it takes
        const long long n = r ? PyLong_AsLongLong(r) : 0;
        Py_XDECREF(r);
        return n;
    }
    long long attribute(PyObject * o, PyObject * name) { return PyErr_Occurred() ? 0 : number(PyObject_GetAttr(o, name)); }
    // the p1a_rows of a Rows
    void rows_of(PyObject * o, p1a_rows & rows) {
        PyObject * st = PyErr_Occurred() ? nullptr : PyObject_GetAttr(o, s_st);
        if (!st) return;
        Py_buffer b;
        if (PyObject_GetBuffer(st, &b, PyBUF_SIMPLE) == 0) {
            if (b.len == (Py_ssize_t) sizeof rows) memcpy(&rows, b.buf, sizeof rows);
            else PyErr_SetString(PyExc_TypeError, "no p1a_rows");
            PyBuffer_Release(&b);
        }
        Py_DECREF(st);
    }
    long long last_size(PyObject * t) { return PyErr_Occurred() ? 0 : number(PyObject_CallMethodOneArg(t, s_size, last_dim)); }
    // the address of a tensor of at least `least` numbers on end, of torch's int32; None: null. What is not right about one the binding says
    void * ints(PyObject * t, long long least, const char * what) {
        if (PyErr_Occurred() || t == Py_None) return nullptr;
        PyObject * type = PyObject_GetAttr(t, s_dtype);
        if (!type) return nullptr;
        bool right = type == int32;
        Py_DECREF(type);
        if (right) right = number(PyObject_CallMethodNoArgs(t, s_numel)) >= least && !PyErr_Occurred();
        if (right) {
            PyObject * r = PyObject_CallMethodNoArgs(t, s_is_contiguous);
            right = r == Py_True;
            Py_XDECREF(r);
        }
        if (PyErr_Occurred()) return nullptr;
        if (right) return data_ptr(t);
        PyObject * r = PyObject_CallFunction(check, "OOLs", t, Py_False, least, what);
        if (!r) return nullptr;
        void * p = address(r);
        Py_DECREF(r);
        return p;
    }
    void * stream() {
        if (PyErr_Occurred()) return nullptr;
        PyObject * r = PyObject_CallNoArgs(stream_of);
        if (!r) return nullptr;
        void * p = address(r);
        Py_DECREF(r);
        return p;
    }
};

bool takes(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) PyErr_Format(PyExc_TypeError, "%zd arguments expected, %zd given", want, n);
    return n == want;
}
bool bound(const calls & C, bool too = true) {
    if (!C.f_append || !too) PyErr_SetString(PyExc_RuntimeError, "bind() comes first");
    return C.f_append && too;
}
#define P1A_CALL(expr) do { if (PyErr_Occurred()) return nullptr; int rc_; Py_BEGIN_ALLOW_THREADS rc_ = (expr); Py_END_ALLOW_THREADS return PyLong_FromLong(rc_); } while (0)

// (qg, k, v, q_norm, k_norm, pos, q, gate, cache, p0, T, Hq, n_rot, freq_base, eps, ldq, ldk, ldv)
PyObject * prep(PyObject * self, PyObject * const * a, Py_ssize_t n) {
    calls & C = *(calls *) PyModule_GetState(self);
    if (!takes(n, 18) || !bound(C)) return nullptr;
    p1a_kv kv;
    float * p[8];
    for (int i = 0; i < 8; ++i) p[i] = C.ptr<float>(a[i]);
    C.describe(a[8], kv);
    const int p0 = C.as_int(a[9]), T = C.as_int(a[10]), Hq = C.as_int(a[11]), nr = C.as_int(a[12]);
    const float base = C.as_float(a[13]), eps = C.as_float(a[14]);
    const int lq = C.as_int(a[15]), lk = C.as_int(a[16]), lv = C.as_int(a[17]);
    void * s = C.stream();
    P1A_CALL(C.f_prep(p[0], p[1], p[2], p[3], p[4], (const int32_t *) p[5], p[6], p[7], &kv, p0, T, Hq, nr, base, eps, lq, lk, lv, s));
}
// (q, cache, out, gate, qbuf, T, p0, p0_dev, pos, rows_per_seq, Hq, scale)
PyObject * decode(PyObject * self, PyObject * const * a, Py_ssize_t n) {
    calls & C = *(calls *) PyModule_GetState(self);
    if (!takes(n, 12) || !bound(C)) return nullptr;
    p1a_kv kv;
    const float * q = C.ptr<float>(a[0]);
    C.describe(a[1], kv);
    float * out = C.ptr<float>(a[2]);
    const float * gate = C.ptr<float>(a[3]);
    void * qbuf = C.data_ptr(a[4]);
    const int T = C.as_int(a[5]), p0 = C.as_int(a[6]);
    const int32_t * p0_dev = C.ptr<int32_t>(a[7]), * pos = C.ptr<int32_t>(a[8]);
    const int rps = C.as_int(a[9]), Hq = C.as_int(a[10]);
    const float scale = C.as_float(a[11]);
    void * s = C.stream();
    P1A_CALL(C.f_decode(q, &kv, out, gate, qbuf, T, p0, p0_dev, pos, rps, Hq, scale, s));
}
// (q, cache, out, gate, T, p0, Hq, scale, scratch, scratch_bytes)
PyObject * prefill(PyObject * self, PyObject * const * a, Py_ssize_t n) {
    calls & C = *(calls *) PyModule_GetState(self);
    if (!takes(n, 10) || !bound(C)) return nullptr;
    p1a_kv kv;
    const float * q = C.ptr<float>(a[0]);
    C.describe(a[1], kv);
    float * out = C.ptr<float>(a[2]);
    const float * gate = C.ptr<float>(a[3]);
    const int T = C.as_int(a[4]), p0 = C.as_int(a[5]), Hq = C.as_int(a[6]);
    const float scale = C.as_float(a[7]);
    void * scratch = C.data_ptr(a[8]);
    const size_t bytes = C.as_size(a[9]);
    void * s = C.stream();
    P1A_CALL(C.f_prefill(q, &kv, out, gate, T, p0, Hq, scale, scratch, bytes, s));
}
// (cache, k, v, p0, p0_dev, pos, T)
PyObject * append(PyObject * self, PyObject * const * a, Py_ssize_t n) {
    calls & C = *(calls *) PyModule_GetState(self);
    if (!takes(n, 7) || !bound(C)) return nullptr;
    p1a_kv kv;
    C.describe(a[0], kv);
    const float * k = C.ptr<float>(a[1]), * v = C.ptr<float>(a[2]);
    const int p0 = C.as_int(a[3]);
    const int32_t * p0_dev = C.ptr<int32_t>(a[4]), * pos = C.ptr<int32_t>(a[5]);
    const int T = C.as_int(a[6]);
    void * s = C.stream();
    P1A_CALL(C.f_append(&kv, k, v, p0, p0_dev, pos, T, s));
}
// (parent, rows, mask, pos, slot)
PyObject * tree_rows(PyObject * self, PyObject * const * a, Py_ssize_t n) {
    calls & C = *(calls *) PyModule_GetState(self);
    if (!takes(n, 5) || !bound(C, C.f_rows)) return nullptr;
    const long long T = C.attribute(a[1], s_T), words = C.last_size(a[2]);
    int32_t * pos = (int32_t *) C.ints(a[3], T, "pos"), * slot = (int32_t *) C.ints(a[4], T, "slot"), * parent = (int32_t *) C.ints(a[0], T, "parent");
    p1a_rows rows;
    C.rows_of(a[1], rows);
    uint32_t * mask = (uint32_t *) C.ints(a[2], T * words, "mask");
    void * s = C.stream();
    P1A_CALL(C.f_rows(parent, &rows, mask, (int) words, pos, slot, s));
}
// (the layers' descriptors, how many they are, rows, n_accept, path)
PyObject * tree_commit(PyObject * self, PyObject * const * a, Py_ssize_t n) {
    calls & C = *(calls *) PyModule_GetState(self);
    if (!takes(n, 5) || !bound(C, C.f_commit)) return nullptr;
    const p1a_kv * layers = (const p1a_kv *) C.address(a[0]);
    const int count = C.as_int(a[1]);
    const long long n_seq = C.attribute(a[2], s_n_seq), width = C.last_size(a[4]);
    p1a_rows rows;
    C.rows_of(a[2], rows);
    const int32_t * n_accept = (const int32_t *) C.ints(a[3], n_seq, "n_accept"), * path = (const int32_t *) C.ints(a[4], n_seq * width, "path");
    void * s = C.stream();
    P1A_CALL(C.f_commit(layers, count, &rows, n_accept, path, (int) width, s));
}
// (addresses of p1a_tree_rows, p1a_tree_commit; the binding's check of a tensor; torch.int32)
PyObject * bind_trees(PyObject * self, PyObject * const * a, Py_ssize_t n) {
    calls & C = *(calls *) PyModule_GetState(self);
    if (!takes(n, 4)) return nullptr;
    C.f_rows = (decltype(C.f_rows)) C.address(a[0]);
    C.f_commit = (decltype(C.f_commit)) C.address(a[1]);
    if (PyErr_Occurred()) return nullptr;
    Py_INCREF(a[2]); Py_XSETREF(C.check, a[2]);
    Py_INCREF(a[3]); Py_XSETREF(C.int32, a[3]);
    Py_RETURN_NONE;
}
// (addresses of p1a_attn_prep, p1a_attn_decode_a16, p1a_attn_prefill, p1a_kv_append; the cache class; the current stream's handle; the
// ctypes classes)
PyObject * bind(PyObject * self, PyObject * const * a, Py_ssize_t n) {
    calls & C = *(calls *) PyModule_GetState(self);
    if (!takes(n, 6 + NCLASS)) return nullptr;
    C.f_prep = (decltype(C.f_prep)) C.address(a[0]);
    C.f_decode = (decltype(C.f_decode)) C.address(a[1]);
    C.f_prefill = (decltype(C.f_prefill)) C.address(a[2]);
    C.f_append = (decltype(C.f_append)) C.address(a[3]);
    if (PyErr_Occurred()) return nullptr;
    Py_INCREF(a[4]); Py_XSETREF(C.kv_class, a[4]);
    Py_INCREF(a[5]); Py_XSETREF(C.stream_of, a[5]);
    for (int i = 0; i < NCLASS; ++i) { Py_INCREF(a[6 + i]); Py_XSETREF(C.classes[i], a[6 + i]); }
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction) (void (*)(void)) bind, METH_FASTCALL, nullptr}, {"prep", (PyCFunction) (void (*)(void)) prep, METH_FASTCALL, nullptr},
    {"decode", (PyCFunction) (void (*)(void)) decode, METH_FASTCALL, nullptr}, {"prefill", (PyCFunction) (void (*)(void)) prefill, METH_FASTCALL, nullptr},
    {"append", (PyCFunction) (void (*)(void)) append, METH_FASTCALL, nullptr}, {"bind_trees", (PyCFunction) (void (*)(void)) bind_trees, METH_FASTCALL, nullptr},
    {"tree_rows", (PyCFunction) (void (*)(void)) tree_rows, METH_FASTCALL, nullptr}, {"tree_commit", (PyCFunction) (void (*)(void)) tree_commit, METH_FASTCALL, nullptr}, {nullptr, nullptr, 0, nullptr}};
int setup(PyObject *) {
    if (s_data_ptr) return 0;
    s_struct = PyUnicode_InternFromString("struct");
    s_value = PyUnicode_InternFromString("value");
    s_as_parameter = PyUnicode_InternFromString("_as_parameter_");
    for (int i = 0; i < 11; ++i) s_field[i] = PyUnicode_InternFromString(FIELDS[i]);
    s_dtype = PyUnicode_InternFromString("dtype"); s_numel = PyUnicode_InternFromString("numel"); s_is_contiguous = PyUnicode_InternFromString("is_contiguous");
    s_size = PyUnicode_InternFromString("size"); s_T = PyUnicode_InternFromString("T"); s_n_seq = PyUnicode_InternFromString("n_seq"); s_st = PyUnicode_InternFromString("_st");
    last_dim = PyLong_FromLong(-1);
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    return PyErr_Occurred() ? -1 : 0;
}
int traverse(PyObject * self, visitproc visit, void * arg) {
    if (calls * C = (calls *) PyModule_GetState(self)) {
        Py_VISIT(C->kv_class); Py_VISIT(C->stream_of); Py_VISIT(C->check); Py_VISIT(C->int32);
        for (PyObject * x : C->classes) Py_VISIT(x);
    }
    return 0;
}
int clear(PyObject * self) {
    if (calls * C = (calls *) PyModule_GetState(self)) {
        Py_CLEAR(C->kv_class); Py_CLEAR(C->stream_of); Py_CLEAR(C->check); Py_CLEAR(C->int32);
        for (PyObject * & x : C->classes) Py_CLEAR(x);
    }
    return 0;
}
void drop(void * self) { clear((PyObject *) self); }
PyModuleDef_Slot slots[] = {{Py_mod_exec, (void *) setup}, {0, nullptr}};
PyModuleDef module_ = {PyModuleDef_HEAD_INIT, "_p1a_call", nullptr, sizeof(calls), methods, slots, traverse, clear, drop};

}   // namespace

PyMODINIT_FUNC PyInit__p1a_call(void) { return PyModuleDef_Init(&module_); }
