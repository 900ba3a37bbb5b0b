// Python's way to the operators of a shared prefix (ops/__init__.py: rotate_axes, rope_axes_kv_write, attention_shared): checks torch
// tensors, takes scratch and results from torch, and calls the C interface of libfriday_engine (include/friday/capi.h) on torch's
// current stream.  A step of a few rows is over in the time of some thirty calls of the interpreter, so what the interpreter would do
// for each tensor (device, type, shape, strides, address) is done here: one call of attention over four rows took 17.2 us of host
// time when Python made the checks, 8.0 this way, a rotation 7.7 and 3.5, an append 11.0 and 3.8.
//
// The functions' addresses and the callable that raises for a non-zero return code are handed in by init(); nothing is linked to the
// engine.  The interpreter's lock is released while the library works.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/util/Exception.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <string>
#include <vector>

#include "friday/capi.h"

namespace {

decltype(&friday_ops_rotate_axes) rotate_fn = nullptr;
decltype(&friday_ops_rope_axes_kv_write) append_fn = nullptr;
decltype(&friday_ops_attention_shared) shared_fn = nullptr;
decltype(&friday_ops_attention_shared_floats) floats_fn = nullptr;
PyObject* check_code = nullptr;           // native.check
PyObject* refusal = nullptr;              // native.KernelError
PyObject* out_of_memory = nullptr;        // torch.OutOfMemoryError

struct Refused {
    std::string why;
};
struct Raised {};                         // a Python exception is set

std::string text_of(const at::Tensor& t) {
    std::string s = std::string(c10::toString(t.scalar_type())) + " [";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    s += "] with strides [";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.stride(i));
    return s + "] on " + t.device().str();
}

// The arguments of one call, in order.
struct Args {
    const char* what;
    PyObject* const* at;
    Py_ssize_t n, next = 0;
    int device = 0;

    PyObject* object() {
        if (next >= n) throw Refused{"an argument is missing"};
        return at[next++];
    }
    long long number(const char* name) {
        PyObject* o = object();
        PyObject* i = PyNumber_Index(o);
        if (i == nullptr) {
            PyErr_Clear();
            throw Refused{std::string(name) + " must be a whole number"};
        }
        const long long v = PyLong_AsLongLong(i);
        Py_DECREF(i);
        if (v == -1 && PyErr_Occurred()) {
            PyErr_Clear();
            throw Refused{std::string(name) + " is out of range"};
        }
        return v;
    }
    int small(const char* name) {
        const long long v = number(name);
        if (v < -2147483647LL || v > 2147483647LL) throw Refused{std::string(name) + " is out of range"};
        return (int)v;
    }
    bool truth() {
        const int v = PyObject_IsTrue(object());
        if (v < 0) throw Raised{};
        return v != 0;
    }
    const at::Tensor& tensor(const char* name) {
        PyObject* o = object();
        if (!THPVariable_Check(o)) throw Refused{std::string(name) + " must be a tensor"};
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.is_cuda() || t.get_device() != device)
            throw Refused{std::string(name) + " is on " + t.device().str() + ", these operations are cuda:" + std::to_string(device) + "'s"};
        return t;
    }
    // rows of float32 or bfloat16
    const at::Tensor& rows(const char* name) {
        const at::Tensor& t = tensor(name);
        const bool typed = t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16;
        if (!typed || t.dim() != 2 || (t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1)))
            throw Refused{std::string(name) + " must be rows of float32 or bfloat16 with unit inner stride, got " + text_of(t)};
        return t;
    }
    // what kernels index as a plain int32 array
    const at::Tensor& numbers(const char* name, long long at_least) {
        const at::Tensor& t = tensor(name);
        if (t.scalar_type() != at::kInt || !t.is_contiguous() || t.numel() < at_least)
            throw Refused{std::string(name) + " must be at least " + std::to_string(at_least) + " contiguous int32 numbers, got " + text_of(t)};
        return t;
    }
};

int code_of(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? 0 : 1; }
const int* ints(const at::Tensor& t) { return (const int*)t.data_ptr(); }
int64_t row_length(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

struct Axes {
    int sections[4], n = 0;
    const int* positions = nullptr;
    const float* denominators = nullptr;
    bool interleaved = false, neighbours = false;
};
// positions, denominators, sections
Axes axes_of(Args& a, int64_t rows) {
    Axes x;
    const at::Tensor& positions = a.numbers("positions", 0);
    const at::Tensor& denom = a.tensor("denom");
    PyObject* list = PySequence_Fast(a.object(), "");
    long long pairs = 0;
    bool fine = list != nullptr;
    if (fine) {
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(list);
        fine = n >= 1 && n <= 4;
        for (Py_ssize_t i = 0; fine && i < n; ++i) {
            PyObject* index = PyNumber_Index(PySequence_Fast_GET_ITEM(list, i));
            const long long v = index ? PyLong_AsLongLong(index) : -1;
            Py_XDECREF(index);
            fine = v >= 0 && v < 65536;
            x.sections[i] = (int)v;
            pairs += v;
        }
        x.n = (int)n;
        Py_DECREF(list);
    }
    PyErr_Clear();
    if (!fine || pairs < 1) throw Refused{"sections are 1 to 4 numbers of pairs, one per axis, with at least one pair between them"};
    if (positions.dim() != 2 || positions.size(0) != rows || positions.size(1) != x.n)
        throw Refused{"positions must be [" + std::to_string(rows) + " rows, " + std::to_string(x.n) + " axes], got " + text_of(positions)};
    if (denom.scalar_type() != at::kFloat || !denom.is_contiguous() || denom.numel() != pairs)
        throw Refused{"denom must be " + std::to_string(pairs) + " contiguous float32 numbers, one per pair, got " + text_of(denom)};
    x.positions = ints(positions);
    x.denominators = (const float*)denom.data_ptr();
    return x;
}

struct Cache {
    void *k = nullptr, *v = nullptr;
    int pages = 0, page = 0, seqs = 0, width = 0;
    const int* table = nullptr;
};
// k_pool, v_pool, block_table, page_size
Cache cache_of(Args& a, at::ScalarType type, int n_kv_heads, int head_dim) {
    Cache c;
    const at::Tensor &k = a.tensor("k_pool"), &v = a.tensor("v_pool"), &table = a.numbers("block_table", 0);
    c.page = a.small("page_size");
    const bool shaped = k.dim() == 4 && k.sizes() == v.sizes() && k.size(0) > 0 && k.size(0) <= 2147483647LL && k.size(1) == c.page && k.size(2) == n_kv_heads &&
                        k.size(3) == head_dim;
    if (!shaped || k.scalar_type() != type || v.scalar_type() != type || !k.is_contiguous() || !v.is_contiguous() || k.data_ptr() == v.data_ptr())
        throw Refused{"keys and values need contiguous pools of their own, [pages, " + std::to_string(c.page) + ", " + std::to_string(n_kv_heads) + ", " +
                      std::to_string(head_dim) + "] of the rows' type, got " + text_of(k) + " and " + text_of(v)};
    if (table.dim() != 2 || table.size(0) > 2147483647LL || table.size(1) > 2147483647LL)
        throw Refused{"the block table is [sequences, pages], got " + text_of(table)};
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    c.pages = (int)k.size(0);
    c.table = ints(table);
    c.seqs = (int)table.size(0);
    c.width = (int)table.size(1);
    return c;
}

PyObject* raise_code(int code) {
    PyObject* r = PyObject_CallFunction(check_code, "i", code);
    Py_XDECREF(r);
    if (r != nullptr) PyErr_Format(PyExc_RuntimeError, "the library returned %d", code);
    return nullptr;
}

// Runs `body` (which returns a new reference) and turns what it throws into Python's exceptions.
template <class F>
PyObject* guarded(const char* what, F body) {
    try {
        return body();
    } catch (const Raised&) {
        return nullptr;
    } catch (const Refused& r) {
        PyErr_SetString(refusal, (std::string(what) + ": " + r.why).c_str());
        return nullptr;
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_SetString(out_of_memory, e.what_without_backtrace());
        return nullptr;
    } catch (const std::exception& e) {      // torch's other errors
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// (handle, device, x, heads, head_dim, positions, denom, sections, interleaved, neighbours, out or None) -> out
PyObject* rotate_axes(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    return guarded("rotate_axes", [&]() -> PyObject* {
        Args a{"rotate_axes", argv, n};
        void* handle = (void*)(intptr_t)a.number("handle");
        a.device = a.small("device");
        const at::Tensor& x = a.rows("x");
        const int heads = a.small("heads"), hd = a.small("head_dim");
        const int64_t rows = x.size(0);
        Axes axes = axes_of(a, rows);
        axes.interleaved = a.truth();
        axes.neighbours = a.truth();
        if (heads < 1 || hd < 1) throw Refused{"heads and head_dim must be positive"};
        at::Tensor out;
        if (n > a.next && argv[a.next] == Py_None) out = at::empty({rows, (int64_t)heads * hd}, x.options());
        else out = a.rows("out");
        if (out.scalar_type() != x.scalar_type()) throw Refused{"x and out are of one type, got " + text_of(x) + " and " + text_of(out)};
        if (rows > 0) {
            void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)a.device).stream();
            int rc;
            Py_BEGIN_ALLOW_THREADS
            rc = rotate_fn(handle, x.data_ptr(), rows, x.size(1), row_length(x), out.data_ptr(), out.size(0), out.size(1), row_length(out), code_of(x),
                           axes.positions, axes.denominators, axes.sections, axes.n, axes.interleaved, axes.neighbours, heads, hd, stream);
            Py_END_ALLOW_THREADS
            if (rc != 0) return raise_code(rc);
        }
        return THPVariable_Wrap(out);
    });
}

// (handle, device, qkv, n_heads, n_kv_heads, head_dim, positions, denom, sections, interleaved, neighbours, row_seq, row_pos, k_pool,
// v_pool, block_table, page_size, q_out or None) -> q_out
PyObject* rope_axes_kv_write(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    return guarded("rope_axes_kv_write", [&]() -> PyObject* {
        Args a{"rope_axes_kv_write", argv, n};
        void* handle = (void*)(intptr_t)a.number("handle");
        a.device = a.small("device");
        const at::Tensor& qkv = a.rows("qkv");
        const int nq = a.small("n_heads"), nkv = a.small("n_kv_heads"), hd = a.small("head_dim");
        const int64_t rows = qkv.size(0);
        Axes axes = axes_of(a, rows);
        axes.interleaved = a.truth();
        axes.neighbours = a.truth();
        const at::Tensor &row_seq = a.numbers("row_seq", rows), &row_pos = a.numbers("row_pos", rows);
        if (nq < 0 || nkv < 1 || hd < 1) throw Refused{"n_heads, n_kv_heads and head_dim must be positive (n_heads may be 0)"};
        const Cache c = cache_of(a, qkv.scalar_type(), nkv, hd);
        at::Tensor out;
        if (n > a.next && argv[a.next] == Py_None) out = at::empty({rows, (int64_t)nq * hd}, qkv.options());
        else out = a.rows("q_out");
        if (out.scalar_type() != qkv.scalar_type()) throw Refused{"qkv and q_out are of one type, got " + text_of(qkv) + " and " + text_of(out)};
        if (rows > 0) {
            if (c.seqs == 0 || c.width == 0) throw Refused{"the block table is empty"};
            void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)a.device).stream();
            int rc;
            Py_BEGIN_ALLOW_THREADS
            rc = append_fn(handle, qkv.data_ptr(), rows, qkv.size(1), row_length(qkv), nq > 0 ? out.data_ptr() : nullptr, out.size(0), out.size(1),
                           row_length(out), code_of(qkv), ints(row_seq), ints(row_pos), axes.positions, axes.denominators, axes.sections, axes.n,
                           axes.interleaved, axes.neighbours, nq, nkv, hd, c.k, c.v, c.pages, c.page, c.table, c.seqs, c.width, stream);
            Py_END_ALLOW_THREADS
            if (rc != 0) return raise_code(rc);
        }
        return THPVariable_Wrap(out);
    });
}

// (handle, device, q, q_stride, out, n_heads, n_kv_heads, head_dim, k_pool, v_pool, block_table, page_size, prefix_table or None,
// prefix_len, row_seq, row_pos, window or None, scale, n_seqs, max_q_len, max_kv_len, seq_start, seq_qlen)
PyObject* attention_shared(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    return guarded("attention_shared", [&]() -> PyObject* {
        Args a{"attention_shared", argv, n};
        void* handle = (void*)(intptr_t)a.number("handle");
        a.device = a.small("device");
        const at::Tensor& q = a.rows("q");
        const long long q_stride = a.number("q_stride");
        const at::Tensor& out = a.rows("out");
        const int nq = a.small("n_heads"), nkv = a.small("n_kv_heads"), hd = a.small("head_dim");
        const int64_t rows = out.size(0);
        if (out.scalar_type() != q.scalar_type() || (rows > 1 && out.stride(0) != out.size(1)) || (rows > 1 && q.stride(0) != q_stride) || rows > 2147483647LL)
            throw Refused{"queries q_stride apart and contiguous results of one type are wanted, got q_stride " + std::to_string(q_stride) + ", " + text_of(q) +
                          " and " + text_of(out)};
        if (nq < 1 || nkv < 1 || hd < 1) throw Refused{"n_heads, n_kv_heads and head_dim must be positive"};
        const Cache c = cache_of(a, q.scalar_type(), nkv, hd);
        PyObject* prefix_object = a.object();
        const int prefix = a.small("prefix_len");
        const int* prefix_table = nullptr;
        if (prefix > 0) {
            if (prefix_object == Py_None) throw Refused{"a prefix of " + std::to_string(prefix) + " needs its pages"};
            if (c.page < 1) throw Refused{"pages of " + std::to_string(c.page) + " rows"};
            Args one{a.what, &prefix_object, 1, 0, a.device};
            prefix_table = ints(one.numbers("prefix_table", ((long long)prefix + c.page - 1) / c.page));
        }
        const at::Tensor &row_seq = a.numbers("row_seq", rows), &row_pos = a.numbers("row_pos", rows);
        int window = 0;
        if (a.next < n && argv[a.next] == Py_None) ++a.next;
        else window = a.small("window");
        const double scale = PyFloat_AsDouble(a.object());
        if (scale == -1.0 && PyErr_Occurred()) throw Raised{};
        const int n_seqs = a.small("n_seqs"), max_q = a.small("max_q_len"), max_kv = a.small("max_kv_len");
        const at::Tensor &starts = a.numbers("seq_start", n_seqs), &lens = a.numbers("seq_qlen", n_seqs);
        if (c.seqs < n_seqs) throw Refused{std::to_string(n_seqs) + " sequences, a block table of " + std::to_string(c.seqs)};
        if (rows == 0 || n_seqs <= 0) Py_RETURN_NONE;
        int64_t floats = 0;
        void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)a.device).stream();
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = floats_fn(handle, (int)rows, n_seqs, max_q, max_kv, prefix, nq, nkv, hd, c.page, window, code_of(q), &floats);
        Py_END_ALLOW_THREADS
        if (rc != 0) return raise_code(rc);
        at::Tensor scratch;
        if (floats > 0) scratch = at::empty({floats}, q.options().dtype(at::kFloat));
        Py_BEGIN_ALLOW_THREADS
        rc = shared_fn(handle, q.data_ptr(), q.size(0), q.size(1), q_stride, out.data_ptr(), rows, out.size(1), code_of(q), c.k, c.v, c.pages, c.page, prefix_table,
                       prefix, c.table, n_seqs, c.width, ints(row_seq), ints(row_pos), ints(starts), ints(lens), max_q, max_kv, nq, nkv, hd, window, (float)scale,
                       floats > 0 ? (float*)scratch.data_ptr() : nullptr, floats, stream);
        Py_END_ALLOW_THREADS
        if (rc != 0) return raise_code(rc);
        Py_RETURN_NONE;
    });
}

// (addresses of the four C functions, native.check, native.KernelError, torch.OutOfMemoryError)
PyObject* init(PyObject*, PyObject* args) {
    unsigned long long rotate = 0, append = 0, shared = 0, floats = 0;
    PyObject *check = nullptr, *error = nullptr, *memory = nullptr;
    if (!PyArg_ParseTuple(args, "KKKKOOO", &rotate, &append, &shared, &floats, &check, &error, &memory)) return nullptr;
    rotate_fn = (decltype(rotate_fn))rotate;
    append_fn = (decltype(append_fn))append;
    shared_fn = (decltype(shared_fn))shared;
    floats_fn = (decltype(floats_fn))floats;
    Py_INCREF(check);
    Py_INCREF(error);
    Py_INCREF(memory);
    check_code = check;
    refusal = error;
    out_of_memory = memory;
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"init", init, METH_VARARGS, nullptr},
                         {"rotate_axes", (PyCFunction)(void (*)(void))rotate_axes, METH_FASTCALL, nullptr},
                         {"rope_axes_kv_write", (PyCFunction)(void (*)(void))rope_axes_kv_write, METH_FASTCALL, nullptr},
                         {"attention_shared", (PyCFunction)(void (*)(void))attention_shared, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "friday_torch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_friday_torch_ops(void) { return PyModule_Create(&module); }
