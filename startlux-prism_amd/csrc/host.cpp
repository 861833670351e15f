// The host path of prism_amd.kv and prism_amd.delta: checks a call's tensors, fills the C entry's struct and calls it.  A
// decode-size call is bound by the host, and a dozen tensors' shapes, strides, types and pointers cost Python some 10 us;
// here they cost a few hundred ns.  A CPython extension over torch's tensors (prism_amd/_host.so); the C entries' addresses
// come from the loaded library (bind), so nothing is linked to it.
//
// The functions return the C entry's status.  TypeError: a wrong type, ValueError: a wrong shape, stride, device or
// argument.  Calls are made with the interpreter lock held, so a call's launches stay together on their stream.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/core/Tensor.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "../../include/prism_amd.h"

namespace {

struct Raised {};                                             // a Python error is set

int (*g_append)(const prism_kv_append_args*, void*);
int (*g_attend)(const prism_kv_attend_args*, void*);
int64_t (*g_attend_ws)(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t);
int (*g_step)(const prism_delta_args*, void*);
int (*g_prefill)(const prism_delta_args*, void*);
int64_t (*g_prefill_ws)(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t);
PyObject* g_stream_of;                                        // tensor -> stream handle (raises off the GPU)
PyObject* g_workspace;                                        // (tensor, bytes, stream handle) -> tensor

[[noreturn]] void raise(PyObject* kind, const std::string& what) {
    PyErr_SetString(kind, what.c_str());
    throw Raised{};
}

std::string list(at::IntArrayRef v) {
    std::string s = "[";
    for (size_t i = 0; i < v.size(); i++) s += (i ? ", " : "") + std::to_string(v[i]);
    return s + "]";
}

int64_t integer(PyObject* o, const char* name) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        raise(PyExc_TypeError, std::string(name) + " must be an integer");
    }
    return v;
}

double number(PyObject* o, const char* name) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        raise(PyExc_TypeError, std::string(name) + " must be a number");
    }
    return v;
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}

int device(const at::Tensor& t) { return t.is_cuda() ? (int)t.get_device() : -1; }

const char* type_name(at::ScalarType t) {
    return t == at::kBFloat16 ? "bf16" : t == at::kFloat ? "fp32" : t == at::kInt ? "int32" : "of another type";
}

[[noreturn]] void refuse(const char* name, const at::Tensor& t, at::ScalarType type, const std::string& want, int dev) {
    if (t.scalar_type() != type) raise(PyExc_TypeError, std::string(name) + " must be " + type_name(type));
    if (device(t) != dev) raise(PyExc_ValueError, std::string(name) + " must be on the other tensors' device");
    raise(PyExc_ValueError, std::string(name) + " must be " + want + ", unit stride in its last dim; got " + list(t.sizes()) +
                                ", strides " + list(t.strides()));
}

// [>= T, heads, dim]; the strides of rows and heads (0 where there is one).
const at::Tensor& rows_of(PyObject* o, const char* name, int64_t T, int64_t n, int64_t dim, int dev, int64_t* ld, int64_t* hs,
                          at::ScalarType type) {
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != type || t.dim() != 3 || t.size(0) < T || t.size(1) != n || t.size(2) != dim ||
        t.stride(2) != 1 || device(t) != dev)
        refuse(name, t, type, "[>= " + std::to_string(T) + ", " + std::to_string(n) + ", " + std::to_string(dim) + "]", dev);
    *ld = t.size(0) > 1 ? t.stride(0) : 0;
    *hs = n > 1 ? t.stride(1) : 0;
    return t;
}

const uint16_t* heads(PyObject* o, const char* name, int64_t T, int64_t n, int64_t dim, int dev, int64_t* ld, int64_t* hs) {
    return static_cast<const uint16_t*>(rows_of(o, name, T, n, dim, dev, ld, hs, at::kBFloat16).const_data_ptr());
}

// An output's memory, its own: a copy-on-write clone gets it here.  Taken before the inputs' pointers, which may lie in the
// same storage.  An output expanded over rows or heads is refused, as torch does where it writes in place: all of them
// would be written to one place.
void* written(const at::Tensor& t, const char* name) {
    if (at::has_internal_overlap(t) == at::MemOverlap::Yes)
        raise(PyExc_ValueError, std::string(name) + " is written and must not be expanded; got " + list(t.sizes()) +
                                    ", strides " + list(t.strides()));
    return t.mutable_data_ptr();
}

template <typename E>
E* out_heads(PyObject* o, const char* name, int64_t T, int64_t n, int64_t dim, int dev, int64_t* ld, int64_t* hs,
             at::ScalarType type) {
    return static_cast<E*>(written(rows_of(o, name, T, n, dim, dev, ld, hs, type), name));
}

const int32_t* ints(PyObject* o, const char* name, int64_t least, int dev) {
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) < least || (least > 1 && t.stride(0) != 1) ||
        device(t) != dev)
        refuse(name, t, at::kInt, "[>= " + std::to_string(least) + "]", dev);
    return static_cast<const int32_t*>(t.const_data_ptr());
}

// The live row count (every producer's `n`).
const int32_t* live(PyObject* o, int dev) {
    const at::Tensor& t = tensor(o, "n");
    if (t.scalar_type() != at::kInt || t.numel() < 1 || device(t) != dev)
        raise(PyExc_ValueError, "n must be a device int32 tensor on the tensors' device");
    return static_cast<const int32_t*>(t.const_data_ptr());
}

const float* gates(PyObject* o, const char* name, int64_t T, int64_t hv, int dev, int64_t* ld) {
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != at::kFloat || t.dim() != 2 || t.size(0) < T || t.size(1) != hv || (hv > 1 && t.stride(1) != 1) ||
        device(t) != dev)
        refuse(name, t, at::kFloat, "[>= " + std::to_string(T) + ", " + std::to_string(hv) + "]", dev);
    *ld = t.stride(0);
    return static_cast<const float*>(t.const_data_ptr());
}

const float* scales(PyObject* o, const char* name, int64_t n, bool e4m3, int dev) {
    if (o == Py_None) return nullptr;
    if (!e4m3) raise(PyExc_ValueError, std::string(name) + ": a bf16 cache has no scales");
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != at::kFloat || t.numel() != n || !t.is_contiguous() || device(t) != dev)
        raise(PyExc_ValueError, std::string(name) + " must be contiguous fp32 [" + std::to_string(n) + "] on the cache's device");
    return static_cast<const float*>(t.const_data_ptr());
}

// The caches (WRITE: outputs), their scales and the page table of at least `rows` rows.
template <bool WRITE>
void cache(prism_kv_cache& c, PyObject* ko, PyObject* vo, PyObject* kso, PyObject* vso, PyObject* to, int64_t rows, int dev) {
    const at::Tensor &k = tensor(ko, "k_cache"), &v = tensor(vo, "v_cache"), &t = tensor(to, "table");
    const at::ScalarType ty = k.scalar_type();
    if ((ty != at::kBFloat16 && ty != at::kFloat8_e4m3fn) || v.scalar_type() != ty)
        raise(PyExc_TypeError, "the caches must both be bf16 or both float8_e4m3fn");
    if (k.dim() != 4 || v.dim() != 4 || k.sizes() != v.sizes() || k.stride(3) != 1 || v.stride(3) != 1 || device(k) != dev ||
        device(v) != dev)
        raise(PyExc_ValueError, "the caches must be [pages, page, heads, dim] on the tensors' device, unit stride in dim");
    c.pages = k.size(0), c.page = k.size(1), c.heads = k.size(2), c.dim = k.size(3);
    if (c.dim != 64 && c.dim != 128 && c.dim != 256) raise(PyExc_ValueError, "the heads' dim must be 64, 128 or 256");
    if (c.page < 16 || (c.page & (c.page - 1)))
        raise(PyExc_ValueError, "a page must hold a power of two of tokens, at least 16");
    if (c.pages < 1 || c.heads < 1) raise(PyExc_ValueError, "the caches must not be empty");
    const bool many = c.pages > 1, heads = c.heads > 1;       // (the stride of a single page or head is not used)
    c.k = WRITE ? written(k, "k_cache") : const_cast<void*>(k.const_data_ptr());
    c.v = WRITE ? written(v, "v_cache") : const_cast<void*>(v.const_data_ptr());
    c.k_page = many ? k.stride(0) : 0, c.k_tok = k.stride(1), c.k_head = heads ? k.stride(2) : 0;
    c.v_page = many ? v.stride(0) : 0, c.v_tok = v.stride(1), c.v_head = heads ? v.stride(2) : 0;
    c.e4m3 = ty == at::kFloat8_e4m3fn;
    c.k_scale = scales(kso, "k_scale", c.heads, c.e4m3, dev), c.v_scale = scales(vso, "v_scale", c.heads, c.e4m3, dev);
    if (t.scalar_type() != at::kInt || t.dim() != 2 || t.size(0) < rows || t.size(1) < 1 ||
        (t.size(1) > 1 && t.stride(1) != 1) || device(t) != dev)
        refuse("table", t, at::kInt, "[>= " + std::to_string(rows) + ", >= 1]", dev);
    c.table = static_cast<const int32_t*>(t.const_data_ptr());
    c.seqs = t.size(0), c.cols = t.size(1), c.table_ld = t.size(0) > 1 ? t.stride(0) : c.cols;
}

// torch's current stream on the tensors' device; raises if that is no GPU of this library.
void* stream_of(PyObject* like) {
    PyObject* s = PyObject_CallFunctionObjArgs(g_stream_of, like, nullptr);
    if (!s) throw Raised{};
    void* p = PyLong_AsVoidPtr(s);
    Py_DECREF(s);
    if (!p && PyErr_Occurred()) throw Raised{};
    return p;
}

// `bytes` of workspace for a call on this stream; the reference keeps it until the launches are queued.
struct Workspace {
    PyObject* t = nullptr;
    void* ptr = nullptr;
    void get(PyObject* like, int64_t bytes, void* stream) {
        PyObject* n = PyLong_FromLongLong(bytes);
        PyObject* s = PyLong_FromVoidPtr(stream);
        if (n && s) t = PyObject_CallFunctionObjArgs(g_workspace, like, n, s, nullptr);
        Py_XDECREF(n);
        Py_XDECREF(s);
        if (!t) throw Raised{};
        ptr = const_cast<void*>(tensor(t, "workspace").const_data_ptr());
    }
    ~Workspace() { Py_XDECREF(t); }
};

void need_args(Py_ssize_t got, Py_ssize_t want) {
    if (got != want) raise(PyExc_TypeError, std::to_string(want) + " arguments, got " + std::to_string(got));
}

int64_t heads_of(const at::Tensor& t) {
    if (t.dim() != 3) raise(PyExc_ValueError, "q must be [rows, heads, dim]; got " + list(t.sizes()));
    return t.size(1);
}

int do_append(PyObject* const* a, Py_ssize_t n) {
    need_args(n, 15);
    enum { Q, K, V, ROPE, POS, TABLE, KC, VC, QO, N, T, SEQ, PAIRS, KS, VS };
    prism_kv_append_args h{};
    const int dev = device(tensor(a[K], "k"));
    h.T = integer(a[T], "T");
    cache<true>(h.cache, a[KC], a[VC], a[KS], a[VS], a[TABLE], 1, dev);
    if ((a[Q] == Py_None) != (a[QO] == Py_None)) raise(PyExc_ValueError, "append: q and q_out go together");
    if (a[Q] != Py_None) {
        h.hq = heads_of(tensor(a[Q], "q"));
        h.q_out = out_heads<uint16_t>(a[QO], "q_out", h.T, h.hq, h.cache.dim, dev, &h.o_ld, &h.o_hs, at::kBFloat16);
        h.q = heads(a[Q], "q", h.T, h.hq, h.cache.dim, dev, &h.q_ld, &h.q_hs);
    }
    h.k = heads(a[K], "k", h.T, h.cache.heads, h.cache.dim, dev, &h.k_ld, &h.k_hs);
    h.v = heads(a[V], "v", h.T, h.cache.heads, h.cache.dim, dev, &h.v_ld, &h.v_hs);
    if (a[ROPE] != Py_None) {
        const at::Tensor& r = tensor(a[ROPE], "rope");
        if (r.scalar_type() != at::kFloat || r.dim() != 2 || r.size(1) % 16 || r.size(1) < 1 || r.size(1) > h.cache.dim ||
            r.stride(1) != 1 || device(r) != dev)
            refuse("rope", r, at::kFloat, "[positions, R], R a multiple of 16 up to dim", dev);
        h.rope = static_cast<const float*>(r.const_data_ptr());
        h.rope_rows = r.size(0), h.rot = r.size(1), h.ldr = r.size(0) > 1 ? r.stride(0) : r.size(1);
    }
    const char* pairs = PyUnicode_Check(a[PAIRS]) ? PyUnicode_AsUTF8(a[PAIRS]) : nullptr;
    if (!pairs) PyErr_Clear();
    h.adjacent = pairs && std::string(pairs) == "adjacent";
    if (!h.adjacent && !(pairs && std::string(pairs) == "half"))
        raise(PyExc_ValueError, "append: pairs must be \"half\" or \"adjacent\"");
    h.pos = ints(a[POS], "pos", h.T, dev);
    h.seq = a[SEQ] == Py_None ? nullptr : ints(a[SEQ], "seq", h.T, dev);
    h.n_rows = live(a[N], dev);
    void* stream = stream_of(a[K]);
    return h.T == 0 ? 0 : g_append(&h, stream);              // (no rows: their tensors may have no memory)
}

int do_attend(PyObject* const* a, Py_ssize_t n) {
    need_args(n, 12);
    enum { Q, KC, VC, TABLE, LENS, OUT, N, T, SCALE, WINDOW, KS, VS };
    prism_kv_attend_args h{};
    const at::Tensor& q = tensor(a[Q], "q");
    const int dev = device(q);
    const int64_t rows = integer(a[T], "T");
    h.hq = heads_of(q);
    const at::Tensor& k = tensor(a[KC], "k_cache");
    h.out = out_heads<uint16_t>(a[OUT], "out", rows, h.hq, k.dim() == 4 ? k.size(3) : -1, dev, &h.o_ld, &h.o_hs, at::kBFloat16);
    cache<false>(h.cache, a[KC], a[VC], a[KS], a[VS], a[TABLE], rows, dev);
    h.cache.seqs = rows;
    h.q = heads(a[Q], "q", rows, h.hq, h.cache.dim, dev, &h.q_ld, &h.q_hs);
    if (h.hq < h.cache.heads || h.hq % h.cache.heads)
        raise(PyExc_ValueError, "attend: the query heads must be a multiple of the cache's heads");
    h.window = integer(a[WINDOW], "window");
    if (h.window < 0) raise(PyExc_ValueError, "attend: window must not be negative");
    h.lens = ints(a[LENS], "lens", rows, dev);
    h.n_rows = live(a[N], dev);
    h.scale = a[SCALE] == Py_None ? 1 / std::sqrt((double)h.cache.dim) : number(a[SCALE], "scale");
    void* stream = stream_of(a[Q]);
    if (rows == 0) return 0;
    Workspace ws;
    h.ws_bytes = g_attend_ws(rows, h.hq, h.cache.heads, h.cache.dim, h.cache.cols, h.cache.page);
    if (h.ws_bytes) ws.get(a[Q], h.ws_bytes, stream);
    h.ws = ws.ptr;
    return g_attend(&h, stream);
}

// Both forms: rows is the live row count of a step, the prompts' first rows of a prefill.
int do_delta(PyObject* const* a, Py_ssize_t n, bool prompts) {
    need_args(n, 13);
    enum { Q, K, V, G, BETA, STATE, OUT, ROWS, T, SLOTS, NORM, SCALE, EPS };
    prism_delta_args h{};
    const at::Tensor &q = tensor(a[Q], "q"), &v = tensor(a[V], "v"), &r = tensor(a[ROWS], prompts ? "cu" : "n");
    const int dev = device(q);
    h.T = integer(a[T], "T");
    if (q.dim() != 3 || v.dim() != 3) raise(PyExc_ValueError, "q, k and v must be [rows, heads, dim]");
    if (prompts && (r.dim() != 1 || r.size(0) < 1)) raise(PyExc_ValueError, "cu must be int32 [sequences + 1]");
    h.seqs = prompts ? r.size(0) - 1 : h.T;
    h.hk = q.size(1), h.dk = q.size(2), h.hv = v.size(1), h.dv = v.size(2);
    if ((h.dk != 64 && h.dk != 128) || (h.dv != 64 && h.dv != 128)) raise(PyExc_ValueError, "the heads' dims must be 64 or 128");
    if (h.hk < 1 || h.hv < h.hk || h.hv % h.hk) raise(PyExc_ValueError, "the value heads must be a multiple of the key heads");
    const at::Tensor& s = tensor(a[STATE], "state");
    if (s.scalar_type() != at::kFloat || s.dim() != 4 || s.size(1) != h.hv || s.size(2) != h.dk || s.size(3) != h.dv ||
        s.stride(3) != 1 || s.stride(2) != h.dv || (h.hv > 1 && s.stride(1) != h.dk * h.dv) || device(s) != dev)
        refuse("state", s, at::kFloat,
               "[slots, " + std::to_string(h.hv) + ", " + std::to_string(h.dk) + ", " + std::to_string(h.dv) +
                   "], contiguous per slot", dev);
    h.state = static_cast<float*>(written(s, "state"));
    h.nslots = s.size(0), h.slot_ld = s.size(0) > 1 ? s.stride(0) : h.hv * h.dk * h.dv;
    h.out = out_heads<float>(a[OUT], "out", h.T, h.hv, h.dv, dev, &h.o_ld, &h.o_hs, at::kFloat);
    h.q = heads(a[Q], "q", h.T, h.hk, h.dk, dev, &h.q_ld, &h.q_hs);
    h.k = heads(a[K], "k", h.T, h.hk, h.dk, dev, &h.k_ld, &h.k_hs);
    h.v = heads(a[V], "v", h.T, h.hv, h.dv, dev, &h.v_ld, &h.v_hs);
    h.g = gates(a[G], "g", h.T, h.hv, dev, &h.g_ld);
    h.beta = gates(a[BETA], "beta", h.T, h.hv, dev, &h.b_ld);
    h.slots = a[SLOTS] == Py_None ? nullptr : ints(a[SLOTS], "slots", h.seqs, dev);
    h.rows = prompts ? ints(a[ROWS], "cu", h.seqs + 1, dev) : live(a[ROWS], dev);
    h.norm = PyObject_IsTrue(a[NORM]);
    if (h.norm < 0) throw Raised{};
    h.scale = a[SCALE] == Py_None ? 1 / std::sqrt((double)h.dk) : number(a[SCALE], "scale");
    h.eps = number(a[EPS], "eps");
    void* stream = stream_of(a[Q]);
    if (h.T == 0 || h.seqs == 0 || h.nslots == 0) return 0;
    if (!prompts) return g_step(&h, stream);
    Workspace ws;
    h.ws_bytes = g_prefill_ws(h.T, h.seqs, h.hk, h.hv, h.dk, h.dv);
    if (h.ws_bytes) ws.get(a[Q], h.ws_bytes, stream);
    h.ws = ws.ptr;
    return g_prefill(&h, stream);
}

template <typename F>
PyObject* guarded(F&& f) {
    try {
        return PyLong_FromLong(f());                          // (bind runs before any other call: _lib.host)
    } catch (const Raised&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

PyObject* py_append(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded([&] { return do_append(a, n); }); }
PyObject* py_attend(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded([&] { return do_attend(a, n); }); }
PyObject* py_step(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded([&] { return do_delta(a, n, false); }); }
PyObject* py_prefill(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded([&] { return do_delta(a, n, true); }); }

// bind(addresses of the six C entries, stream_of, workspace)
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] {
        need_args(n, 8);
        void* p[6];
        for (int i = 0; i < 6; i++) {
            p[i] = PyLong_AsVoidPtr(a[i]);
            if (!p[i]) raise(PyExc_ValueError, "bind: an address is missing");
        }
        g_append = reinterpret_cast<decltype(g_append)>(p[0]);
        g_attend = reinterpret_cast<decltype(g_attend)>(p[1]);
        g_attend_ws = reinterpret_cast<decltype(g_attend_ws)>(p[2]);
        g_step = reinterpret_cast<decltype(g_step)>(p[3]);
        g_prefill = reinterpret_cast<decltype(g_prefill)>(p[4]);
        g_prefill_ws = reinterpret_cast<decltype(g_prefill_ws)>(p[5]);
        Py_INCREF(a[6]);
        Py_INCREF(a[7]);
        Py_XDECREF(g_stream_of);
        Py_XDECREF(g_workspace);
        g_stream_of = a[6], g_workspace = a[7];
        return 0;
    });
}

#define FAST(name, f, doc) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, doc}
PyMethodDef methods[] = {
    FAST("kv_append", py_append, "prism_kv_append after checks; see prism_amd.kv.append"),
    FAST("kv_attend", py_attend, "prism_kv_attend after checks; see prism_amd.kv.attend"),
    FAST("delta_step", py_step, "prism_delta_step after checks; see prism_amd.delta.step"),
    FAST("delta_prefill", py_prefill, "prism_delta_prefill after checks; see prism_amd.delta.prefill"),
    FAST("bind", py_bind, "addresses of the C entries, then stream_of and workspace"),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Host path of prism_amd.kv and prism_amd.delta.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
