// The argument blocks of the 4-bit caches' calls (include/fav4_mx4.h) from torch tensors,
// for the ctypes binding: dtypes, shapes, strides and devices checked, pointers and sizes
// packed.  In Python a small call's checks (some 60 attribute reads) take as long as its
// launch: append 4.8 us, 0.3 here (a call of 4 tokens 9.1 and 4.7).
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>
#include <cstring>
#include <string>

#include "fav4_mx4.h"

namespace {

constexpr int64_t D = 128;
constexpr const char* ONE_DEVICE = "all tensors on one device";

struct Refused {
    PyObject* type;
    std::string what;
};
void check(bool ok, const char* what) {
    if (!ok) throw Refused{PyExc_AssertionError, what};
}
int fit(int64_t v, const char* what) {
    if (v < INT_MIN || v > INT_MAX) throw Refused{PyExc_OverflowError, std::string(what) + " does not fit an int"};
    return int(v);
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) throw Refused{PyExc_TypeError, std::string(name) + " is not a tensor"};
    return THPVariable_Unpack(o);
}
int integer(PyObject* o, const char* name) {
    PyObject* n = PyNumber_Long(o);
    if (!n) throw Refused{nullptr, {}};
    int overflow = 0;
    const long long v = PyLong_AsLongLongAndOverflow(n, &overflow);
    Py_DECREF(n);
    return fit(overflow ? LLONG_MAX : v, name);
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1 && PyErr_Occurred()) throw Refused{nullptr, {}};
    return v;
}

// A contiguous tensor of this type and shape on device dev; its address.
template <class T = void>
T* whole(const at::Tensor& t, at::ScalarType type, at::IntArrayRef shape, int64_t dev, const char* what) {
    check(t.scalar_type() == type && t.sizes() == shape && t.is_contiguous(), what);
    check(t.get_device() == dev, ONE_DEVICE);
    return static_cast<T*>(t.data_ptr());
}

struct Caches {
    int64_t pages, kv_heads, page_size;
    void *k, *ks, *v, *vs;
};
Caches caches(PyObject* const* a, int64_t dev) {
    const at::Tensor &k = tensor(a[0], "k_cache"), &ks = tensor(a[1], "k_scales"), &v = tensor(a[2], "v_cache"),
                     &vs = tensor(a[3], "v_scales");
    const char* what = "caches: contiguous uint8 [num_pages, kv_heads, page_size, 64] (scales: 4)";
    check(k.dim() == 4, what);
    const int64_t n = k.size(0), h = k.size(1), p = k.size(2);
    const int64_t codes[] = {n, h, p, D / 2}, scales[] = {n, h, p, D / 32};
    return {n, h, p, whole(k, at::kByte, codes, dev, what), whole(ks, at::kByte, scales, dev, what),
            whole(v, at::kByte, codes, dev, what), whole(vs, at::kByte, scales, dev, what)};
}

int* ints(PyObject* o, int64_t n, int64_t dev, const char* what) {
    return whole<int>(tensor(o, what), at::kInt, {n}, dev, what);
}
int* block_table(PyObject* o, int64_t dev, int64_t& batch, int64_t& pages) {
    const at::Tensor& t = tensor(o, "block_table");
    check(t.dim() == 2, "block_table: int32 [batch, max_pages]");
    batch = t.size(0), pages = t.size(1);
    return whole<int>(t, at::kInt, t.sizes(), dev, "block_table: contiguous int32 [batch, max_pages]");
}

// BF16 rows [tokens, heads, 128] of any stride between tokens, heads and dims contiguous; the
// stride (a single token has none that counts).
void* rows(const at::Tensor& t, int64_t tokens, int64_t heads, int64_t dev, const char* what, long long& stride) {
    const int64_t shape[] = {tokens, heads, D};
    check(t.scalar_type() == at::kBFloat16 && t.sizes() == at::IntArrayRef(shape), what);
    check(t.stride(2) == 1 && (heads == 1 || t.stride(1) == D), what);
    check(t.get_device() == dev, ONE_DEVICE);
    stride = tokens == 1 ? heads * D : t.stride(0);
    return t.data_ptr();
}

template <class Args>
PyObject* bytes(const Args& a) {
    return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(&a), sizeof a);
}

// q, k, v, q_out, k_cache, k_scales, v_cache, v_scales, cu_q, seqlens_k, block_table, cos, sin, interleaved, positions
PyObject* append(PyObject* const* o) {
    Fav4Mx4AppendArgs args;
    std::memset(&args, 0, sizeof args);
    Fav4AppendArgs& a = args.append;
    const at::Tensor& k = tensor(o[1], "k");
    const int64_t dev = k.get_device();
    const Caches c = caches(o + 4, dev);
    a.k_cache = c.k, a.v_cache = c.v, args.k_scales = c.ks, args.v_scales = c.vs;
    int64_t batch, pages;
    a.block_table = block_table(o[10], dev, batch, pages);
    a.cu_seqlens_q = ints(o[8], batch + 1, dev, "cu_q: contiguous int32 [batch + 1]");
    a.seqlens_k = ints(o[9], batch, dev, "seqlens_k: contiguous int32 [batch]");
    check(k.dim() == 3, "k: BF16 [tokens, kv_heads, 128]");
    const int64_t tokens = k.size(0);
    a.k = rows(k, tokens, c.kv_heads, dev, "k: BF16 [tokens, kv_heads, 128], heads and dims contiguous", a.k_stride);
    a.v = rows(tensor(o[2], "v"), tokens, c.kv_heads, dev, "v: BF16 [tokens, kv_heads, 128], heads and dims contiguous",
               a.v_stride);
    check((o[0] == Py_None) == (o[3] == Py_None), "q and q_out: both or neither");
    int64_t heads = 1;
    if (o[0] != Py_None) {
        const at::Tensor& q = tensor(o[0], "q");
        check(q.dim() == 3, "q: BF16 [tokens, heads, 128]");
        heads = q.size(1);
        a.q = rows(q, tokens, heads, dev, "q: BF16 [tokens, heads, 128], heads and dims contiguous", a.q_stride);
        a.q_out = rows(tensor(o[3], "q_out"), tokens, heads, dev, "q_out: as q", a.q_out_stride);
    }
    check((o[11] == Py_None) == (o[12] == Py_None), "cos and sin: both or neither");
    if (o[11] != Py_None) {
        const at::Tensor& cos = tensor(o[11], "cos");
        check(cos.dim() == 2, "cos: FP32 [rows, rotary_dim / 2]");
        a.cos = whole<float>(cos, at::kFloat, cos.sizes(), dev, "cos: contiguous FP32 [rows, rotary_dim / 2]");
        a.sin = whole<float>(tensor(o[12], "sin"), at::kFloat, cos.sizes(), dev, "sin: as cos");
        a.rotary_rows = fit(cos.size(0), "rotary rows");
        a.rotary_dim = fit(2 * cos.size(1), "rotary_dim");
    }
    const int interleaved = PyObject_IsTrue(o[13]);
    if (interleaved < 0) throw Refused{nullptr, {}};
    if (o[14] != Py_None) a.positions = ints(o[14], tokens, dev, "positions: contiguous int32 [tokens]");
    a.interleaved = interleaved;
    a.batch = fit(batch, "batch"), a.heads = fit(heads, "heads"), a.kv_heads = fit(c.kv_heads, "kv_heads");
    a.total_q = fit(tokens, "tokens"), a.num_pages = fit(c.pages, "num_pages");
    a.page_size = fit(c.page_size, "page_size"), a.max_pages_per_seq = fit(pages, "max_pages");
    return bytes(args);
}

// k_cache, k_scales, v_cache, v_scales, k, v, cu_k, block_table, starts
PyObject* gather(PyObject* const* o) {
    Fav4Mx4GatherArgs a;
    std::memset(&a, 0, sizeof a);
    const at::Tensor& k = tensor(o[4], "k");
    const int64_t dev = k.get_device();
    const Caches c = caches(o, dev);
    a.k_cache = c.k, a.k_scales = c.ks, a.v_cache = c.v, a.v_scales = c.vs;
    int64_t batch, pages;
    a.block_table = block_table(o[7], dev, batch, pages);
    a.cu_seqlens_k = ints(o[6], batch + 1, dev, "cu_k: contiguous int32 [batch + 1]");
    check(k.dim() == 3, "k: BF16 [total_k, kv_heads, 128]");
    const int64_t total = k.size(0);
    a.k = rows(k, total, c.kv_heads, dev, "k: BF16 [total_k, kv_heads, 128], heads and dims contiguous", a.k_stride);
    a.v = rows(tensor(o[5], "v"), total, c.kv_heads, dev, "v: BF16 [total_k, kv_heads, 128], heads and dims contiguous",
               a.v_stride);
    if (o[8] != Py_None) a.starts = ints(o[8], batch, dev, "starts: contiguous int32 [batch]");
    a.batch = fit(batch, "batch"), a.kv_heads = fit(c.kv_heads, "kv_heads"), a.total_k = fit(total, "total_k");
    a.num_pages = fit(c.pages, "num_pages"), a.page_size = fit(c.page_size, "page_size");
    a.max_pages_per_seq = fit(pages, "max_pages");
    return bytes(a);
}

// q, k_cache, k_scales, v_cache, v_scales, o, lse, cu_q, seqlens_k, block_table, max_q, max_k, total_k, scale
PyObject* paged(PyObject* const* o) {
    Fav4Mx4PagedArgs args;
    std::memset(&args, 0, sizeof args);
    Fav4PagedArgs& a = args.paged;
    const at::Tensor& q = tensor(o[0], "q");
    const int64_t dev = q.get_device();
    const Caches c = caches(o + 1, dev);
    a.k_cache = c.k, a.v_cache = c.v, args.k_scales = c.ks, args.v_scales = c.vs;
    int64_t batch, pages;
    a.block_table = block_table(o[9], dev, batch, pages);
    a.cu_seqlens_q = ints(o[7], batch + 1, dev, "cu_q: contiguous int32 [batch + 1]");
    a.seqlens_k = ints(o[8], batch, dev, "seqlens_k: contiguous int32 [batch]");
    check(q.dim() == 3 && q.size(2) == D, "q: BF16 [tokens, heads, 128]");
    const int64_t tokens = q.size(0), heads = q.size(1);
    a.q = whole(q, at::kBFloat16, q.sizes(), dev, "q: contiguous BF16 [tokens, heads, 128]");
    a.o = whole(tensor(o[5], "o"), at::kBFloat16, q.sizes(), dev, "o: as q");
    if (o[6] != Py_None)
        a.lse = whole<float>(tensor(o[6], "lse"), at::kFloat, {heads, tokens}, dev, "lse: contiguous FP32 [heads, tokens]");
    a.max_seqlen_q = integer(o[10], "max_q"), a.max_seqlen_k = integer(o[11], "max_k");
    a.total_k = o[12] == Py_None ? 0 : integer(o[12], "total_k");
    a.scale = float(o[13] == Py_None ? 1 / std::sqrt(double(D)) : number(o[13]));
    a.batch = fit(batch, "batch"), a.heads = fit(heads, "heads"), a.kv_heads = fit(c.kv_heads, "kv_heads");
    a.total_q = fit(tokens, "tokens"), a.num_pages = fit(c.pages, "num_pages");
    a.page_size = fit(c.page_size, "page_size"), a.max_pages_per_seq = fit(pages, "max_pages");
    return bytes(args);
}

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "%d arguments expected, %zd given", N, n);
        return nullptr;
    }
    try {
        return F(args);
    } catch (const Refused& r) {
        if (r.type) PyErr_SetString(r.type, r.what.c_str());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

template <PyObject* (*F)(PyObject* const*), int N>
PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<F, N>)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<append, 15>("append"), method<gather, 9>("gather"), method<paged, 14>("paged"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "fav4_mx4_blocks", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch_version: of the torch that this file was compiled against.  Its tensors' C++ layout
// is no stable interface, so the loader compares it with the one in the process.
PyMODINIT_FUNC PyInit_fav4_mx4_blocks() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", FAV4_TORCH) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
