// The paged cache's calls without Python in between: a CPython module,
// foveated_kv_amd/_fkv_calls.so, whose functions take the tensors of a call
// as they are, check them, allocate results and call libfkv's entry points.
//
// A decode step's kernels take 4 to 5 us and their launch 3, which the checks in
// Python more than doubled.  Host time of a call, a step of 64 sequences with 32
// query and 8 KV heads: rotation 8.1 us from Python, 4.6 so; write 10.9 and 5.1;
// attention over 512 tokens of one 9.5 and 4.6.
//
// Each function returns NotImplemented for whatever is not plain -- a wrong
// argument, a tensor to be copied first, one of another GPU than the current
// one -- and has done nothing then: paged.py goes on with its own checks, which
// raise or handle it.  So there is one place that words refusals.  An entry
// point that failed otherwise than by refusing its arguments may have started
// work, which must not be done twice (rows rotated in place): that is raised
// here, by _lib.py's check().
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../../include/fkv.h"

namespace {

// Entry points of the library that _lib.py loaded.
struct {
    decltype(&fkv_rope_apply) rope;
    decltype(&fkv_paged_write) write;
    decltype(&fkv_paged_read) read;
    decltype(&fkv_paged_attn_workspace) workspace;
    decltype(&fkv_paged_attn) attn;
} lib;
PyObject* check = nullptr;  // _lib.check(code, name), which raises

// What a call meets that paged.py has to look at.
struct NotPlain {};
// An entry point's error that is not a refusal.
struct Failed {
    int code;
    const char* name;
};
void need(bool ok) {
    if (!ok) throw NotPlain{};
}

int64_t integer(PyObject* o) {
    need(PyLong_Check(o));
    int overflow = 0;
    const int64_t v = PyLong_AsLongLongAndOverflow(o, &overflow);
    need(!overflow);
    return v;
}

int32_t int32_of(int64_t v) {
    need(v == (int32_t)v);
    return (int32_t)v;
}

// A tensor proper on GPU `index` that wants no gradient and has no tangent.
const at::Tensor& tensor(PyObject* o, int64_t index) {
    need(THPVariable_CheckExact(o));
    const at::Tensor& t = THPVariable_Unpack(o);
    need(t.is_cuda() && t.layout() == at::kStrided && t.get_device() == index && !t.requires_grad() &&
         !t._fw_grad(0).defined());
    return t;
}

int32_t dtype_code(at::ScalarType t) {
    if (t == at::kHalf) return 0;
    if (t == at::kBFloat16) return 1;
    need(t == at::kFloat);
    return 2;
}

// Rows that need no copy (strides of dimensions of one element mean nothing).
fkv_rows rows(const at::Tensor& t) {
    const auto n = t.sizes(), s = t.strides();
    auto stride = [&](int d) { return n[d] > 1 ? s[d] : 0; };
    const fkv_rows r = {t.data_ptr(), stride(0), stride(1), stride(2)};
    need(s[3] == 1 && !((uintptr_t)r.data & 15) && !((r.stride_b | r.stride_h | r.stride_l) & 7));
    return r;
}

// The caller's result tensor (None: a new one like x).
at::Tensor result(PyObject* o, int64_t index, const at::Tensor& x, bool zero) {
    if (o == Py_None) return zero ? at::zeros_like(x) : at::empty_like(x);
    const at::Tensor& t = tensor(o, index);
    need(t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type());
    for (int d = 0; d < 4; d++) need(t.size(d) <= 1 || t.stride(d) != 0);
    return t;
}

fkv_positions positions(PyObject* o, int64_t index, int64_t B, int64_t L, bool per_token_allowed) {
    fkv_positions p = {nullptr, 0, 0, 0, 0, 0};
    if (!THPVariable_Check(o)) {
        p.base = integer(o);
        return p;
    }
    const at::Tensor& t = tensor(o, index);
    need(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong);
    p.data = t.data_ptr();
    p.is64 = t.scalar_type() == at::kLong;
    if (t.dim() == 1 && t.size(0) == B) {
        p.stride_b = t.stride(0);
    } else if (t.dim() > 1 || t.numel() != 1) {
        need(per_token_allowed && t.dim() == 2 && (t.size(0) == B || t.size(0) == 1) && t.size(1) == L);
        p.stride_b = t.size(0) > 1 ? t.stride(0) : 0;
        p.stride_l = t.stride(1);
        p.per_token = 1;
    }
    return p;
}

struct Table {
    const int32_t* ids;
    int32_t B, n;
    int64_t stride;
};
Table table(PyObject* o, int64_t index) {
    const at::Tensor& t = tensor(o, index);
    need(t.scalar_type() == at::kInt && t.dim() == 2);
    const int64_t B = t.size(0), P = t.size(1);
    need((P <= 1 || t.stride(1) == 1) && (B <= 1 || t.stride(0) >= P));
    return Table{(const int32_t*)t.data_ptr(), int32_of(B), int32_of(P), B > 1 ? t.stride(0) : P};
}

const int32_t* lengths(PyObject* o, int64_t index, int64_t B) {
    const at::Tensor& t = tensor(o, index);
    need(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == B && (B <= 1 || t.stride(0) == 1));
    return (const int32_t*)t.data_ptr();
}

// The stream of a call on GPU `index`, which must be the current one.
void* stream_of(int64_t index) {
    need(c10::hip::current_device() == index);
    return (void*)c10::hip::getCurrentHIPStream((c10::DeviceIndex)index).stream();
}

// Runs f(begun), which checks a call's arguments, launches it and returns a new
// reference.
template <typename F>
PyObject* plain(Py_ssize_t n, Py_ssize_t wanted, F f) {
    bool begun = false;
    try {
        if (n == wanted) return f(begun);
    } catch (const Failed& e) {
        PyObject* none = PyObject_CallFunction(check, "is", e.code, e.name);
        Py_XDECREF(none);
        return nullptr;
    } catch (...) {
        if (begun) {  // (no memory for the result's Python object)
            if (!PyErr_Occurred()) PyErr_NoMemory();
            return nullptr;
        }
        PyErr_Clear();  // (paged.py meets the same, and words it)
    }
    Py_RETURN_NOTIMPLEMENTED;
}

template <typename F>
void launch(bool& begun, const char* name, F f) {
    struct Released {  // (other threads run while a full queue makes the launch wait)
        PyThreadState* state = PyEval_SaveThread();
        ~Released() { PyEval_RestoreThread(state); }
    };
    int rc;
    {
        Released gil;
        rc = f();
    }
    need(rc != FKV_EINVAL);  // (arguments are refused before anything is done)
    begun = true;
    if (rc != FKV_OK) throw Failed{rc, name};
}

// A rotary table's (fkv_rope's address, GPU, head dim).
struct RopeKey {
    const fkv_rope* rope;
    int64_t index, D;
    explicit RopeKey(PyObject* o) {
        need(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 3);
        rope = (const fkv_rope*)(uintptr_t)integer(PyTuple_GET_ITEM(o, 0));
        index = integer(PyTuple_GET_ITEM(o, 1));
        D = integer(PyTuple_GET_ITEM(o, 2));
    }
};
// A layer's (fkv_pages' address, GPU).
struct PagesKey {
    const fkv_pages* pages;
    int64_t index;
    explicit PagesKey(PyObject* o) {
        need(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 2);
        pages = (const fkv_pages*)(uintptr_t)integer(PyTuple_GET_ITEM(o, 0));
        index = integer(PyTuple_GET_ITEM(o, 1));
    }
};

// rope(key, x, positions, out)
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return plain(n, 4, [&](bool& begun) {
        const RopeKey key(a[0]);
        void* stream = stream_of(key.index);
        const at::Tensor& x = tensor(a[1], key.index);
        need(x.dim() == 4 && x.size(3) == key.D);
        const int32_t dt = dtype_code(x.scalar_type()), B = int32_of(x.size(0)), H = int32_of(x.size(1)),
                      L = int32_of(x.size(2));
        const fkv_positions pos = positions(a[2], key.index, B, L, true);
        const fkv_rows src = rows(x);
        at::Tensor out = result(a[3], key.index, x, false);
        const fkv_rows dst = rows(out);
        launch(begun, "fkv_rope_apply", [&] {
            return lib.rope(key.rope, &src, &dst, dt, B, H, L, (int32_t)key.D, &pos, stream);
        });
        return THPVariable_Wrap(std::move(out));
    });
}

// write(key, k, v, table, start, n_new, q, rope's key, q_out)
PyObject* write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return plain(n, 9, [&](bool& begun) -> PyObject* {
        const PagesKey key(a[0]);
        const fkv_pages* pg = key.pages;
        void* stream = stream_of(key.index);
        const at::Tensor &k = tensor(a[1], key.index), &v = tensor(a[2], key.index);
        need(k.dim() == 4 && k.size(1) == pg->H && k.size(3) == pg->D && v.sizes() == k.sizes() &&
             v.scalar_type() == k.scalar_type());
        const int32_t dt = dtype_code(k.scalar_type()), B = int32_of(k.size(0)), L = int32_of(k.size(2));
        const Table t = table(a[3], key.index);
        need(t.B == B);
        const fkv_rope* rope = nullptr;
        if (a[7] != Py_None) {
            const RopeKey r(a[7]);
            need(r.D == pg->D && r.index == key.index);
            rope = r.rope;
        }
        const fkv_positions start = positions(a[4], key.index, B, L, false);
        const int32_t* n_new = a[5] == Py_None ? nullptr : lengths(a[5], key.index, B);
        const fkv_rows rk = rows(k), rv = rows(v);
        fkv_rows rq, ro;
        at::Tensor out;
        int32_t Hq = 0;
        const bool queries = a[6] != Py_None;
        if (queries) {
            const at::Tensor& q = tensor(a[6], key.index);
            need(q.dim() == 4 && q.size(0) == B && q.size(2) == L && q.size(3) == pg->D &&
                 q.scalar_type() == k.scalar_type());
            Hq = int32_of(q.size(1));
            rq = rows(q);
            out = result(a[8], key.index, q, n_new != nullptr);
            ro = rows(out);
        } else {
            need(a[8] == Py_None);
        }
        launch(begun, "fkv_paged_write", [&] {
            return lib.write(pg, &rk, &rv, dt, B, L, t.ids, t.n, t.stride, &start, n_new, rope, queries ? &rq : nullptr,
                             queries ? &ro : nullptr, Hq, stream);
        });
        if (!queries) Py_RETURN_NONE;
        return THPVariable_Wrap(std::move(out));
    });
}

// read(key, table, lens, max_len, dtype)
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return plain(n, 5, [&](bool& begun) {
        const PagesKey key(a[0]);
        const fkv_pages* pg = key.pages;
        void* stream = stream_of(key.index);
        const Table t = table(a[1], key.index);
        const int32_t* lens = lengths(a[2], key.index, t.B);
        const int32_t S = int32_of(a[3] == Py_None ? (int64_t)t.n * pg->page_size : integer(a[3]));
        need(S >= 0);
        at::ScalarType dtype = pg->format == FKV_PAGES_BF16 ? at::kBFloat16 : at::kHalf;
        if (a[4] != Py_None) {
            need(THPDtype_Check(a[4]));
            dtype = ((THPDtype*)a[4])->scalar_type;
        }
        const int32_t dt = dtype_code(dtype);
        const auto options = THPVariable_Unpack(a[1]).options().dtype(dtype);
        at::Tensor k = at::empty({t.B, pg->H, S, pg->D}, options), v = at::empty({t.B, pg->H, S, pg->D}, options);
        launch(begun, "fkv_paged_read", [&] {
            return lib.read(pg, t.ids, t.n, t.stride, lens, t.B, S, k.data_ptr(), v.data_ptr(), dt, stream);
        });
        return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(k)), THPVariable_Wrap(std::move(v)));
    });
}

// attend(key, query, table, lens, max_len, lens_add, scale, out, return_lse)
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return plain(n, 9, [&](bool& begun) {
        const PagesKey key(a[0]);
        const fkv_pages* pg = key.pages;
        void* stream = stream_of(key.index);
        const at::Tensor& q = tensor(a[1], key.index);
        need(q.dim() == 4 && q.size(2) == 1 && q.size(3) == pg->D);
        const int32_t dt = dtype_code(q.scalar_type()), B = int32_of(q.size(0)), Hq = int32_of(q.size(1));
        const Table t = table(a[2], key.index);
        need(t.B == B);
        const int32_t* lens = lengths(a[3], key.index, B);
        int64_t most = (int64_t)t.n * pg->page_size;
        if (a[4] != Py_None) most = std::min(most, integer(a[4]));
        const int32_t lens_add = int32_of(integer(a[5]));
        double scale = 1.0 / std::sqrt((double)pg->D);
        if (a[6] != Py_None) {
            need(PyFloat_Check(a[6]) || PyLong_Check(a[6]));
            scale = PyFloat_AsDouble(a[6]);
            need(!PyErr_Occurred());
        }
        const fkv_rows rq = rows(q);
        at::Tensor out, lse, work;
        if (a[7] == Py_None) {
            out = at::empty(q.sizes(), q.options());
        } else {
            out = result(a[7], key.index, q, false);
            need(out.is_contiguous() && !((uintptr_t)out.data_ptr() & 15));
        }
        need(PyBool_Check(a[8]));
        const bool want_lse = a[8] == Py_True;
        if (want_lse) lse = at::empty({B, Hq}, q.options().dtype(at::kFloat));
        const int64_t bytes = lib.workspace(pg, Hq, B, most);
        need(bytes >= 0);
        if (bytes) work = at::empty({bytes}, q.options().dtype(at::kByte));
        launch(begun, "fkv_paged_attn", [&] {
            return lib.attn(pg, &rq, dt, Hq, B, t.ids, t.n, t.stride, lens, lens_add, most, (float)scale, out.data_ptr(),
                            want_lse && lse.numel() ? (float*)lse.data_ptr() : nullptr, bytes ? work.data_ptr() : nullptr,
                            bytes, stream);
        });
        PyObject* o = THPVariable_Wrap(std::move(out));
        return want_lse ? Py_BuildValue("(NN)", o, THPVariable_Wrap(std::move(lse))) : o;
    });
}

// bind(addresses of fkv_rope_apply, fkv_paged_write, fkv_paged_read,
// fkv_paged_attn_workspace, fkv_paged_attn; _lib.check)
PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long p[5];
    PyObject* raise;
    if (!PyArg_ParseTuple(args, "KKKKKO", p, p + 1, p + 2, p + 3, p + 4, &raise)) return nullptr;
    Py_INCREF(raise);
    Py_XSETREF(check, raise);
    lib = {(decltype(lib.rope))p[0], (decltype(lib.write))p[1], (decltype(lib.read))p[2],
           (decltype(lib.workspace))p[3], (decltype(lib.attn))p[4]};
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, "addresses of libfkv's entry points, _lib.check"},
    {"rope", (PyCFunction)(void (*)())rope, METH_FASTCALL, "Rope.__call__"},
    {"write", (PyCFunction)(void (*)())write, METH_FASTCALL, "PagedLayer.write"},
    {"read", (PyCFunction)(void (*)())read, METH_FASTCALL, "PagedLayer.read"},
    {"attend", (PyCFunction)(void (*)())attend, METH_FASTCALL, "PagedLayer.attend"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fkv_calls", "the paged cache's calls", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fkv_calls() { return PyModule_Create(&module); }
