// serve_torch.cpp — the host side of booster_b200/serve.py: tensors in, checks, struct b200_kv4 / b200_pages, one call of the library (include/booster_b200.h). In C++, because a call of
// these operators on a few rows takes the device 5 to 10 us, and the same checks in Python take the host longer: attention of a token of 48 sequences 19.3 us a call, 9.6 from here (two
// launches), 48 rows written and read 25.8 and 11, a row drawn 12.4 and 6.3.
//
// The library's functions come by address (bind), so that this module works with whichever build of it serve.py has loaded. ValueError: an argument that cannot be; the class that bind
// was given: what the library refused.
#include <Python.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <stdexcept>
#include <string>

#include "../../include/booster_b200.h"

namespace {

struct Api {
    decltype(&b200_last_error) last_error;
    decltype(&b200_kv4_append) kv4_append;
    decltype(&b200_kv4_read) kv4_read;
    decltype(&b200_kv4_attention_workspace) kv4_attention_workspace;
    decltype(&b200_kv4_attention) kv4_attention;
    decltype(&b200_pages_workspace) pages_workspace;
    decltype(&b200_pages_reserve) pages_reserve;
    decltype(&b200_pages_fork) pages_fork;
    decltype(&b200_pages_free) pages_free;
    decltype(&b200_pages_compact) pages_compact;
    decltype(&b200_pages_copy) pages_copy;
    decltype(&b200_sample) sample;
} api;
PyObject * library_error;

struct Refused : std::runtime_error { using std::runtime_error::runtime_error; };        // ValueError
struct Failed : std::runtime_error { using std::runtime_error::runtime_error; };         // the library's error
inline void need(bool ok, const char * what) { if (__builtin_expect(!ok, 0)) throw Refused(what); }
inline void done(bool ok, const char * what) { if (__builtin_expect(!ok, 0)) throw Failed(std::string(what) + ": " + api.last_error()); }

inline const at::Tensor & tensor(PyObject * o, const char * name) {
    if (!THPVariable_Check(o)) throw Refused(std::string(name) + " is a tensor");
    return THPVariable_Unpack(o);
}
inline int number(PyObject * o, const char * name) {
    const long x = PyLong_AsLong(o);
    if (x == -1 && PyErr_Occurred()) { PyErr_Clear(); throw Refused(std::string(name) + " is a whole number"); }
    if (x < INT_MIN || x > INT_MAX) throw Refused(std::string(name) + " is a whole number of 32 bits");
    return (int) x;
}
inline int type_of(const at::Tensor & t) {
    switch (t.scalar_type()) {
        case at::kFloat: return B200_DTYPE_F32;
        case at::kBFloat16: return B200_DTYPE_BF16;
        case at::kHalf: return B200_DTYPE_F16;
        default: return -1;
    }
}
inline int on(const at::Tensor & t) {
    need(t.is_cuda(), "tensors are on a CUDA device: booster_b200 has no CPU fallback");
    return t.get_device();
}
inline bool there(const at::Tensor & t, int index) { return t.is_cuda() && t.get_device() == index; }
inline void * stream_of(int index) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex) index).stream(); }
inline int small(int64_t n, const char * what) { need(n <= INT_MAX, what); return (int) n; }

// a contiguous int32 vector (of n entries) on device `index`
int32_t * ints(const char * name, PyObject * o, int index, int64_t n = -1) {
    const at::Tensor & t = tensor(o, name);
    if (t.scalar_type() != at::kInt || !there(t, index) || t.dim() != 1 || !t.is_contiguous() || (n >= 0 && t.numel() != n))
        throw Refused(std::string(name) + " is a contiguous int32 tensor of 1 dimension" + (n >= 0 ? " and " + std::to_string(n) + " entries" : "") + " on the device of the others");
    return static_cast<int32_t *>(t.data_ptr());
}
struct Table { int32_t * at; int slots, most; int64_t stride; };
Table table_of(PyObject * o, int index) {
    const at::Tensor & t = tensor(o, "table");
    need(t.scalar_type() == at::kInt && there(t, index) && t.dim() == 2 && (t.stride(1) == 1 || t.size(1) == 1), "table is an int32 tensor [n_slots, max_pages] of contiguous rows on the device of the others");
    return {static_cast<int32_t *>(t.data_ptr()), small(t.size(0), "table: too many slots"), small(t.size(1), "table: too many pages"), t.size(0) > 1 ? t.stride(0) : t.size(1)};
}
// pool [..., n_pages, n_head_kv, page_tokens / 16, 18 * head_dim]
int64_t page_stride(const at::Tensor & pool) {
    const int64_t d = pool.dim(), size = pool.size(d - 1), tiles = pool.size(d - 2), kv = pool.size(d - 3);
    need(pool.scalar_type() == at::kByte && size % 18 == 0 && pool.stride(d - 1) == 1 && (tiles == 1 || pool.stride(d - 2) == size) && (kv == 1 || pool.stride(d - 3) == tiles * size),
         "pool is a uint8 tensor [..., n_pages, n_head_kv, page_tokens / 16, 18 * head_dim] of contiguous pages");
    return pool.size(d - 4) > 1 ? pool.stride(d - 4) : std::max(pool.stride(d - 4), kv * tiles * size);
}
// one layer's cache and a step
b200_kv4 step_of(const at::Tensor & pool, PyObject * table, PyObject * held, PyObject * first, PyObject * slots, int64_t n_rows) {
    const int index = on(pool);
    need(pool.dim() == 4, "pool is one layer's [n_pages, n_head_kv, page_tokens / 16, 18 * head_dim]");
    const int64_t n_seq = tensor(first, "first").numel() - 1;
    need(n_seq >= 0, "first has one entry more than there are sequences");
    const Table t = table_of(table, index);
    b200_kv4 c;
    c.device = index;
    c.page_stride = page_stride(pool);
    c.n_pages = small(pool.size(0), "pool: too many pages");
    c.n_head_kv = small(pool.size(1), "pool: too many heads");
    c.page_tokens = small(16 * pool.size(2), "pool: pages too long");
    c.head_dim = small(pool.size(3) / 18, "pool: heads too wide");
    c.n_slots = t.slots; c.max_pages = t.most;
    c.n_seq = small(n_seq, "first: too many sequences");
    c.n_rows = small(n_rows, "too many rows");
    c.stream = stream_of(index);
    c.pool = pool.data_ptr();
    c.table_stride = t.stride;
    c.table = t.at;
    c.held = ints("held", held, index, t.slots);
    c.first = ints("first", first, index);
    if (slots == Py_None) { need(n_seq <= t.slots, "without slots, sequence i is slot i: more sequences than slots"); c.slots = nullptr; }
    else c.slots = ints("slots", slots, index, n_seq);
    return c;
}
struct Rows { int64_t row, head; };
Rows rows_of(const char * name, const at::Tensor & x, const at::Tensor & pool, int64_t heads = -1) {
    if (x.dim() != 3 || x.device() != pool.device() || pool.dim() < 1 || x.size(2) * 18 != pool.size(pool.dim() - 1) || (heads >= 0 && x.size(1) != heads))
        throw Refused(std::string(name) + " is a tensor [rows, heads, head_dim] that fits the pool, on its device");
    if (x.stride(2) != 1) throw Refused(std::string(name) + ": the entries of a head are contiguous");
    return {x.stride(0), x.stride(1)};
}

PyObject * kv4_append(PyObject * const * a) {                            // pool, table, held, first, k, v, slots
    const at::Tensor & pool = tensor(a[0], "pool"), & k = tensor(a[4], "k"), & v = tensor(a[5], "v");
    const int64_t kv = pool.dim() == 4 ? pool.size(1) : -1;
    const Rows rk = rows_of("k", k, pool, kv), rv = rows_of("v", v, pool, kv);
    const int type = type_of(k);
    need(type >= 0 && k.scalar_type() == v.scalar_type() && k.sizes() == v.sizes(), "k and v are float32, bfloat16 or float16, and alike");
    const b200_kv4 c = step_of(pool, a[1], a[2], a[3], a[6], k.size(0));
    done(api.kv4_append(&c, type, k.data_ptr(), rk.row, rk.head, v.data_ptr(), rv.row, rv.head) == 0, "kv4_append");
    Py_RETURN_NONE;
}
PyObject * kv4_read(PyObject * const * a) {                              // pool, table, held, first, rows, dtype, slots, out
    const at::Tensor & pool = tensor(a[0], "pool");
    need(THPDtype_Check(a[5]), "dtype is float32, bfloat16 or float16");
    const at::ScalarType type = reinterpret_cast<THPDtype *>(a[5])->scalar_type;
    need(type == at::kFloat || type == at::kBFloat16 || type == at::kHalf, "dtype is float32, bfloat16 or float16");
    const int rows = number(a[4], "rows");
    const b200_kv4 c = step_of(pool, a[1], a[2], a[3], a[6], rows);
    need(rows >= 0, "rows is the number of rows of the step");
    const int64_t shape[3] = {rows, c.n_head_kv, c.head_dim};
    at::Tensor k, v;
    if (a[7] == Py_None) {
        k = at::empty(shape, pool.options().dtype(type));
        v = at::empty(shape, pool.options().dtype(type));
    } else {
        const char * what = "out is a pair of contiguous tensors [rows, n_head_kv, head_dim] of dtype";
        need(PySequence_Check(a[7]) && PySequence_Size(a[7]) == 2, what);
        for (int i = 0; i < 2; i++) {
            PyObject * o = PySequence_GetItem(a[7], i);
            at::Tensor & x = i ? v : k;
            const bool is = o && THPVariable_Check(o);
            if (is) x = THPVariable_Unpack(o);
            Py_XDECREF(o);
            need(is && x.sizes() == at::IntArrayRef(shape, 3) && x.scalar_type() == type && x.device() == pool.device() && x.is_contiguous(), what);
        }
    }
    done(api.kv4_read(&c, type_of(k), k.data_ptr(), v.data_ptr()) == 0, "kv4_read");
    PyObject * pk = THPVariable_Wrap(k), * pv = THPVariable_Wrap(v), * r = pk && pv ? PyTuple_Pack(2, pk, pv) : nullptr;
    Py_XDECREF(pk); Py_XDECREF(pv);
    return r;
}
PyObject * kv4_attention(PyObject * const * a) {                         // q, pool, table, held, first, slots, scale, window, max_rows, out
    const at::Tensor & q = tensor(a[0], "q"), & pool = tensor(a[1], "pool");
    const Rows r = rows_of("q", q, pool);
    const int type = type_of(q);
    need(type == B200_DTYPE_BF16 || type == B200_DTYPE_F16, "q is bfloat16 or float16");
    const int64_t rows = q.size(0);
    const b200_kv4 c = step_of(pool, a[2], a[3], a[4], a[5], rows);
    const int heads = small(q.size(1), "q: too many heads"), window = number(a[7], "window");
    double scale = 1.0 / std::sqrt((double) c.head_dim);
    if (a[6] != Py_None) {
        scale = PyFloat_AsDouble(a[6]);
        if (scale == -1.0 && PyErr_Occurred()) { PyErr_Clear(); throw Refused("scale is a number"); }
    }
    const int most = a[8] != Py_None ? std::max(1, number(a[8], "max_rows")) : std::max<int>(1, (int) ((rows + c.n_seq - 1) / std::max(1, c.n_seq)));
    at::Tensor out;
    if (a[9] == Py_None) out = at::empty(q.sizes(), q.options());
    else {
        out = tensor(a[9], "out");
        need(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.device() == q.device() && out.is_contiguous(), "out is a contiguous tensor like q");
    }
    const int64_t size = api.kv4_attention_workspace(&c, heads, most);
    done(size >= 0, "kv4_attention");
    const at::Tensor work = at::empty({size}, pool.options());
    done(api.kv4_attention(&c, type, q.data_ptr(), r.row, r.head, heads, (float) scale, window, most, out.data_ptr(), work.data_ptr(), size) == 0, "kv4_attention");
    return THPVariable_Wrap(out);
}

b200_pages pages_of(PyObject * table, PyObject * held, PyObject * refs_o, int page_tokens, PyObject * pool_o) {
    const at::Tensor & refs = tensor(refs_o, "refs");
    const int index = on(refs);
    const Table t = table_of(table, index);
    b200_pages p;
    p.device = index;
    p.n_pages = small(refs.numel(), "refs: too many pages");
    p.page_tokens = page_tokens;
    p.n_head_kv = 1; p.head_dim = 64; p.n_layer = 1;
    p.n_slots = t.slots; p.max_pages = t.most;
    p.stream = stream_of(index);
    p.pool = nullptr;
    p.layer_stride = p.page_stride = 0;
    p.table_stride = t.stride;
    p.table = t.at;
    p.held = held ? ints("held", held, index, t.slots) : t.at;
    p.refs = ints("refs", refs_o, index);
    if (pool_o) {
        const at::Tensor & pool = tensor(pool_o, "pool");
        need(pool.dim() == 5 && there(pool, index) && pool.size(1) == p.n_pages, "pool is [n_layer, n_pages, n_head_kv, page_tokens / 16, 18 * head_dim], refs has an entry a page");
        p.page_stride = page_stride(pool);
        p.n_layer = small(pool.size(0), "pool: too many layers");
        p.n_head_kv = small(pool.size(2), "pool: too many heads");
        p.page_tokens = small(16 * pool.size(3), "pool: pages too long");
        p.head_dim = small(pool.size(4) / 18, "pool: heads too wide");
        p.pool = pool.data_ptr();
        p.layer_stride = pool.stride(0);
    }
    return p;
}
// one number on the device of refs, and a workspace
at::Tensor word_beside(PyObject * refs) { return at::empty({1}, THPVariable_Unpack(refs).options()); }
at::Tensor work_for(const b200_pages & p, int n, const at::Tensor & pool) {
    const int64_t size = api.pages_workspace(&p, n);
    done(size >= 0, "pages_workspace");
    return at::empty({size}, pool.options());
}
PyObject * pages_reserve(PyObject * const * a) {                         // table, held, refs, first, page_tokens, slots
    const int64_t n64 = tensor(a[3], "first").numel() - 1;
    need(n64 >= 0, "first has one entry more than there are sequences");
    const int n = small(n64, "first: too many sequences");
    const b200_pages p = pages_of(a[0], a[1], a[2], number(a[4], "page_tokens"), nullptr);
    need(a[5] != Py_None || n <= p.n_slots, "without slots, sequence i is slot i: more sequences than slots");
    const int32_t * slots = a[5] != Py_None ? ints("slots", a[5], p.device, n) : nullptr, * first = ints("first", a[3], p.device);
    const at::Tensor status = word_beside(a[2]);
    done(api.pages_reserve(&p, slots, first, n, static_cast<int32_t *>(status.data_ptr())) == 0, "pages_reserve");
    return THPVariable_Wrap(status);
}
PyObject * pages_fork(PyObject * const * a) {                            // pool, table, held, refs, parents, children
    const b200_pages p = pages_of(a[1], a[2], a[3], 0, a[0]);
    const int n = small(tensor(a[4], "parents").numel(), "parents: too many");
    const int32_t * parents = ints("parents", a[4], p.device), * children = ints("children", a[5], p.device, n);
    const at::Tensor work = work_for(p, n, THPVariable_Unpack(a[0])), status = word_beside(a[3]);
    done(api.pages_fork(&p, parents, children, n, static_cast<int32_t *>(status.data_ptr()), work.data_ptr(), work.numel()) == 0, "pages_fork");
    return THPVariable_Wrap(status);
}
PyObject * pages_free(PyObject * const * a) {                            // table, held, refs, slots
    const b200_pages p = pages_of(a[0], a[1], a[2], 16, nullptr);
    const int32_t * slots = ints("slots", a[3], p.device);
    done(api.pages_free(&p, slots, small(THPVariable_Unpack(a[3]).numel(), "slots: too many")) == 0, "pages_free");
    Py_RETURN_NONE;
}
PyObject * pages_compact(PyObject * const * a) {                         // pool, table, refs
    const b200_pages p = pages_of(a[1], nullptr, a[2], 0, a[0]);
    const at::Tensor work = work_for(p, p.n_pages, THPVariable_Unpack(a[0])), live = word_beside(a[2]);
    done(api.pages_compact(&p, static_cast<int32_t *>(live.data_ptr()), work.data_ptr(), work.numel()) == 0, "pages_compact");
    return THPVariable_Wrap(live);
}
PyObject * pages_copy(PyObject * const * a) {                            // pool, table, refs, src, dst
    const b200_pages p = pages_of(a[1], nullptr, a[2], 0, a[0]);
    const int n = small(tensor(a[3], "src").numel(), "src: too many");
    const int32_t * src = ints("src", a[3], p.device), * dst = ints("dst", a[4], p.device, n);
    const at::Tensor work = work_for(p, n, THPVariable_Unpack(a[0])), status = word_beside(a[2]);
    done(api.pages_copy(&p, src, dst, n, static_cast<int32_t *>(status.data_ptr()), work.data_ptr(), work.numel()) == 0, "pages_copy");
    return THPVariable_Wrap(status);
}
const void * per_row(const char * name, PyObject * o, at::ScalarType type, int64_t rows, int index) {
    if (o == Py_None) return nullptr;
    const at::Tensor & t = tensor(o, name);
    if (t.scalar_type() != type || t.dim() != 1 || t.numel() != rows || !there(t, index) || !t.is_contiguous())
        throw Refused(std::string(name) + " is a contiguous " + (type == at::kInt ? "int32" : "float32") + " tensor of " + std::to_string(rows) + " entries on the logits' device");
    return t.data_ptr();
}
PyObject * sample(PyObject * const * a) {                                // logits, u, temperature, top_k, top_p, min_p
    const at::Tensor & logits = tensor(a[0], "logits");
    const int index = on(logits), type = type_of(logits);
    need(logits.dim() == 2 && type >= 0 && (logits.stride(1) == 1 || logits.size(1) == 1), "logits is a float32, bfloat16 or float16 tensor [rows, n_vocab] of contiguous rows");
    const int rows = small(logits.size(0), "logits: too many rows"), vocab = small(logits.size(1), "logits: too many a row");
    const float * u = static_cast<const float *>(per_row("u", a[1], at::kFloat, rows, index)), * temperature = static_cast<const float *>(per_row("temperature", a[2], at::kFloat, rows, index));
    const int32_t * top_k = static_cast<const int32_t *>(per_row("top_k", a[3], at::kInt, rows, index));
    const float * top_p = static_cast<const float *>(per_row("top_p", a[4], at::kFloat, rows, index)), * min_p = static_cast<const float *>(per_row("min_p", a[5], at::kFloat, rows, index));
    const at::Tensor ids = at::empty({rows}, logits.options().dtype(at::kInt)), logprobs = at::empty({rows}, logits.options().dtype(at::kFloat));
    done(api.sample(index, stream_of(index), type, logits.data_ptr(), rows > 1 ? logits.stride(0) : vocab, rows, vocab, u, temperature, top_k, top_p, min_p,
                    static_cast<int32_t *>(ids.data_ptr()), static_cast<float *>(logprobs.data_ptr())) == 0, "sample");
    PyObject * pi = THPVariable_Wrap(ids), * pl = THPVariable_Wrap(logprobs), * r = pi && pl ? PyTuple_Pack(2, pi, pl) : nullptr;
    Py_XDECREF(pi); Py_XDECREF(pl);
    return r;
}

template <PyObject * (*F)(PyObject * const *), int N> PyObject * call(PyObject *, PyObject * const * args, Py_ssize_t n) {
    if (n != N) { PyErr_SetString(PyExc_TypeError, "wrong number of arguments"); return nullptr; }
    if (!library_error) { PyErr_SetString(PyExc_RuntimeError, "bind() comes first"); return nullptr; }
    try { return F(args); }
    catch (const Refused & e) { PyErr_SetString(PyExc_ValueError, e.what()); }
    catch (const Failed & e) { PyErr_SetString(library_error, e.what()); }
    catch (...) { if (!PyErr_Occurred()) torch::translate_exception_to_python(std::current_exception()); }
    return nullptr;
}
// bind(class of the library's errors, addresses of its functions in the order of Api)
PyObject * bind(PyObject *, PyObject * const * args, Py_ssize_t n) {
    constexpr int N = sizeof(Api) / sizeof(void *);
    if (n != N + 1) { PyErr_SetString(PyExc_TypeError, "a class and the addresses of the library's functions"); return nullptr; }
    void * at[N];
    for (int i = 0; i < N; i++) {
        at[i] = PyLong_AsVoidPtr(args[1 + i]);
        if (!at[i]) { if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a function has no address"); return nullptr; }
    }
    __builtin_memcpy(&api, at, sizeof at);
    Py_INCREF(args[0]);
    Py_XSETREF(library_error, args[0]);
    Py_RETURN_NONE;
}

#define FAST(name, n) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&call<name, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&bind)), METH_FASTCALL, nullptr},
    FAST(kv4_append, 7), FAST(kv4_read, 8), FAST(kv4_attention, 10), FAST(pages_reserve, 6), FAST(pages_fork, 6), FAST(pages_free, 4), FAST(pages_compact, 3), FAST(pages_copy, 5), FAST(sample, 6),
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serve", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serve() { return PyModule_Create(&module); }
