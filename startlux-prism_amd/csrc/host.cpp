// The host path of prism_amd.kv, delta, fp8 and moe: checks a call's tensors, fills the C entry's struct and calls it.  A
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
int (*g_fp8_quant)(const prism_fp8_quant_args*, void*);
int (*g_fp8_gemm)(const prism_fp8_gemm_args*, void*);
int64_t (*g_fp8_gemm_ws)(int64_t, int64_t, int64_t);
int (*g_route)(const prism_moe_route_args*, void*);
int (*g_experts)(const prism_moe_experts_args*, void*);
int64_t (*g_experts_ws)(int64_t, int64_t, int64_t, int64_t);
PyObject* g_stream_of;                                        // tensor -> stream handle (raises off the GPU)
PyObject* g_stream_here;                                      // the same, refusing a device that is not the current one
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
    return t == at::kBFloat16 ? "bf16" : t == at::kFloat ? "fp32" : t == at::kInt ? "int32" :
           t == at::kFloat8_e4m3fn ? "float8_e4m3fn" : t == at::kByte ? "uint8" : "of another type";
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
void* stream_of(PyObject* like, bool here = false) {
    PyObject* s = PyObject_CallFunctionObjArgs(here ? g_stream_here : g_stream_of, like, nullptr);
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

// [>= T, cols], any stride of rows.
const at::Tensor& matrix(PyObject* o, const char* name, at::ScalarType type, int64_t T, int64_t cols, int dev, int64_t* ld) {
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != type || t.dim() != 2 || t.size(0) < T || t.size(1) != cols || (cols > 1 && t.stride(1) != 1) ||
        device(t) != dev)
        refuse(name, t, type, "[>= " + std::to_string(T) + ", " + std::to_string(cols) + "]", dev);
    *ld = t.size(0) > 1 ? t.stride(0) : cols;
    return t;
}

template <typename E>
const E* in_matrix(PyObject* o, const char* name, at::ScalarType type, int64_t T, int64_t cols, int dev, int64_t* ld) {
    return static_cast<const E*>(matrix(o, name, type, T, cols, dev, ld).const_data_ptr());
}
template <typename E>
E* out_matrix(PyObject* o, const char* name, at::ScalarType type, int64_t T, int64_t cols, int dev, int64_t* ld) {
    return static_cast<E*>(written(matrix(o, name, type, T, cols, dev, ld), name));
}

// [>= T, cols or (0) any number], fp32 or bf16; whether fp32.
const void* wide_or_bf16(PyObject* o, const char* name, int64_t T, int64_t* cols, int64_t* ld, int64_t* f32) {
    const at::Tensor& t = tensor(o, name);
    if (t.dim() != 2) raise(PyExc_ValueError, std::string(name) + " must be [rows, columns]; got " + list(t.sizes()));
    *f32 = t.scalar_type() == at::kFloat;
    *cols = t.size(1);
    return matrix(o, name, *f32 ? at::kFloat : at::kBFloat16, T, *cols, device(t), ld).const_data_ptr();
}

// An fp8.F8 (chunks, scales, n, k) of one weight (experts 0) or of so many.
struct Weight {
    const uint8_t* q;
    const float* s;
    int64_t n, k;
};
Weight weight(PyObject* o, const char* name, int64_t experts, int dev) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) raise(PyExc_TypeError, std::string(name) + " must be an fp8.F8");
    const at::Tensor &q = tensor(PyTuple_GET_ITEM(o, 0), name), &s = tensor(PyTuple_GET_ITEM(o, 1), name);
    const int64_t n = integer(PyTuple_GET_ITEM(o, 2), name), k = integer(PyTuple_GET_ITEM(o, 3), name);
    if (q.scalar_type() != at::kByte || s.scalar_type() != at::kFloat)
        raise(PyExc_TypeError, std::string(name) + " must hold uint8 chunks and fp32 scales (fp8.pack, fp8.from_rows)");
    const int64_t KB = (k + 127) / 128, d = experts ? 1 : 0;
    const bool ok = n > 0 && k > 0 && q.dim() == 3 + d && s.dim() == 2 + d && q.size(d) == (n + 15) / 16 && q.size(d + 1) == KB &&
                    q.size(d + 2) == 2048 && s.size(d) == (n + 127) / 128 && s.size(d + 1) == KB &&
                    (!experts || (q.size(0) == experts && s.size(0) == experts)) && q.is_contiguous() && s.is_contiguous() &&
                    device(q) == dev && device(s) == dev;
    if (!ok)
        raise(PyExc_ValueError, std::string(name) + " must be " + (experts ? std::to_string(experts) + " weights" : "one weight") +
                                    " as fp8.pack or fp8.from_rows leaves it, on the other tensors' device; got chunks " +
                                    list(q.sizes()) + ", scales " + list(s.sizes()) + " for n " + std::to_string(n) + ", k " +
                                    std::to_string(k));
    return {static_cast<const uint8_t*>(q.const_data_ptr()), static_cast<const float*>(s.const_data_ptr()), n, k};
}

int64_t epilogue(PyObject* o) {
    const int64_t e = integer(o, "epi");
    if (e != 0 && e != 1) raise(PyExc_ValueError, "epi must be 0 (bf16) or 1 (added into fp32)");
    return e;
}

int do_fp8_quant(PyObject* const* a, Py_ssize_t n) {
    need_args(n, 5);
    enum { X, Q, S, N, T };
    prism_fp8_quant_args h{};
    const int dev = device(tensor(a[X], "x"));
    h.T = integer(a[T], "T");
    wide_or_bf16(a[X], "x", h.T, &h.k, &h.x_ld, &h.f32);
    const int64_t KB = (h.k + 127) / 128;
    h.q = out_matrix<uint8_t>(a[Q], "q", at::kFloat8_e4m3fn, h.T, 128 * KB, dev, &h.q_ld);
    h.s = out_matrix<float>(a[S], "s", at::kFloat, h.T, KB, dev, &h.s_ld);
    h.x = tensor(a[X], "x").const_data_ptr();
    h.n_rows = live(a[N], dev);
    void* stream = stream_of(a[X], true);
    return h.T == 0 || h.k == 0 ? 0 : g_fp8_quant(&h, stream);
}

int do_fp8_gemm(PyObject* const* a, Py_ssize_t n) {
    need_args(n, 7);
    enum { A, AS, W, OUT, N, T, EPI };
    prism_fp8_gemm_args h{};
    const int dev = device(tensor(a[A], "a_q"));
    h.T = integer(a[T], "T");
    h.epi = epilogue(a[EPI]);
    const Weight w = weight(a[W], "w", 0, dev);
    h.w = w.q, h.ws = w.s, h.n = w.n, h.k = w.k;
    const int64_t KB = (h.k + 127) / 128;
    h.out = out_matrix<void>(a[OUT], "out", h.epi ? at::kFloat : at::kBFloat16, h.T, h.n, dev, &h.o_ld);
    h.a = in_matrix<uint8_t>(a[A], "a_q", at::kFloat8_e4m3fn, h.T, 128 * KB, dev, &h.a_ld);
    h.as = in_matrix<float>(a[AS], "a_s", at::kFloat, h.T, KB, dev, &h.as_ld);
    h.n_rows = live(a[N], dev);
    void* stream = stream_of(a[A], true);
    if (h.T == 0) return 0;
    Workspace ws;
    h.wsp_bytes = g_fp8_gemm_ws(h.T, h.n, h.k);
    if (h.wsp_bytes) ws.get(a[A], h.wsp_bytes, stream);
    h.wsp = ws.ptr;
    return g_fp8_gemm(&h, stream);
}

int do_route(PyObject* const* a, Py_ssize_t n) {
    need_args(n, 9);
    enum { X, IDS, W, N, T, SCORE, BIAS, RENORM, SCALE };
    prism_moe_route_args h{};
    const int dev = device(tensor(a[X], "logits"));
    h.T = integer(a[T], "T");
    wide_or_bf16(a[X], "logits", h.T, &h.E, &h.x_ld, &h.f32);
    const at::Tensor& ids = tensor(a[IDS], "ids");
    if (ids.dim() != 2) raise(PyExc_ValueError, "ids must be [rows, experts per token]; got " + list(ids.sizes()));
    h.top = ids.size(1);
    h.ids = out_matrix<int32_t>(a[IDS], "ids", at::kInt, h.T, h.top, dev, &h.ids_ld);
    h.w = out_matrix<float>(a[W], "weights", at::kFloat, h.T, h.top, dev, &h.w_ld);
    h.x = tensor(a[X], "logits").const_data_ptr();
    if (h.E < 1 || h.E > 1024) raise(PyExc_ValueError, "route: 1 to 1024 experts");
    if (h.top < 1 || h.top > 16 || h.top > h.E) raise(PyExc_ValueError, "route: 1 to 16 experts per token, no more than there are");
    const char* score = PyUnicode_Check(a[SCORE]) ? PyUnicode_AsUTF8(a[SCORE]) : nullptr;
    if (!score) PyErr_Clear();
    h.sigmoid = score && std::string(score) == "sigmoid";
    if (!h.sigmoid && !(score && std::string(score) == "softmax"))
        raise(PyExc_ValueError, "route: score must be \"softmax\" or \"sigmoid\"");
    if (a[BIAS] != Py_None) {
        const at::Tensor& b = tensor(a[BIAS], "bias");
        if (!h.sigmoid) raise(PyExc_ValueError, "route: a bias goes with score=\"sigmoid\"");
        if (b.scalar_type() != at::kFloat || b.dim() != 1 || b.size(0) != h.E || (h.E > 1 && b.stride(0) != 1) || device(b) != dev)
            refuse("bias", b, at::kFloat, "[" + std::to_string(h.E) + "]", dev);
        h.bias = static_cast<const float*>(b.const_data_ptr());
    }
    const int renorm = PyObject_IsTrue(a[RENORM]);
    if (renorm < 0) throw Raised{};
    h.renorm = renorm;
    h.scale = number(a[SCALE], "scale");
    h.n_rows = live(a[N], dev);
    void* stream = stream_of(a[X], true);
    return h.T == 0 ? 0 : g_route(&h, stream);
}

int do_experts(PyObject* const* a, Py_ssize_t n) {
    need_args(n, 10);
    enum { X, IDS, WT, GATE, UP, DOWN, OUT, N, T, EPI };
    prism_moe_experts_args h{};
    const int dev = device(tensor(a[X], "x"));
    h.T = integer(a[T], "T");
    h.epi = epilogue(a[EPI]);
    const at::Tensor& ids = tensor(a[IDS], "ids");
    if (ids.dim() != 2) raise(PyExc_ValueError, "ids must be [rows, experts per token]; got " + list(ids.sizes()));
    h.top = ids.size(1);
    if (h.top < 1 || h.top > 16) raise(PyExc_ValueError, "experts: 1 to 16 experts per token");
    if (!PyTuple_Check(a[GATE]) || PyTuple_GET_SIZE(a[GATE]) != 4) raise(PyExc_TypeError, "gate must be an fp8.F8");
    const at::Tensor& gq = tensor(PyTuple_GET_ITEM(a[GATE], 0), "gate");
    h.E = gq.dim() == 4 ? gq.size(0) : 0;
    if (h.E < 1) raise(PyExc_ValueError, "gate must hold the weights of every expert: chunks [experts, ...]");
    const Weight g = weight(a[GATE], "gate", h.E, dev), u = weight(a[UP], "up", h.E, dev), d = weight(a[DOWN], "down", h.E, dev);
    h.I = g.n, h.H = g.k;
    if (u.n != h.I || u.k != h.H || d.n != h.H || d.k != h.I)
        raise(PyExc_ValueError, "experts: gate and up must be [I, H] weights, down [H, I]; got gate [" + std::to_string(g.n) + ", " +
                                    std::to_string(g.k) + "], up [" + std::to_string(u.n) + ", " + std::to_string(u.k) +
                                    "], down [" + std::to_string(d.n) + ", " + std::to_string(d.k) + "]");
    if (h.H % 16 || h.I % 16) raise(PyExc_ValueError, "experts: H and I must be multiples of 16");
    h.gate = g.q, h.gate_s = g.s, h.up = u.q, h.up_s = u.s, h.down = d.q, h.down_s = d.s;
    h.out = out_matrix<void>(a[OUT], "out", h.epi ? at::kFloat : at::kBFloat16, h.T, h.H, dev, &h.o_ld);
    h.x = in_matrix<uint16_t>(a[X], "x", at::kBFloat16, h.T, h.H, dev, &h.x_ld);
    h.ids = in_matrix<int32_t>(a[IDS], "ids", at::kInt, h.T, h.top, dev, &h.ids_ld);
    h.w = in_matrix<float>(a[WT], "weights", at::kFloat, h.T, h.top, dev, &h.w_ld);
    h.n_rows = live(a[N], dev);
    void* stream = stream_of(a[X], true);
    if (h.T == 0) return 0;
    Workspace ws;
    h.wsp_bytes = g_experts_ws(h.T, h.top, h.H, h.I);
    ws.get(a[X], h.wsp_bytes, stream);
    h.wsp = ws.ptr;
    return g_experts(&h, stream);
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

PyObject* py_fp8_quant(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded([&] { return do_fp8_quant(a, n); }); }
PyObject* py_fp8_gemm(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded([&] { return do_fp8_gemm(a, n); }); }
PyObject* py_route(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded([&] { return do_route(a, n); }); }
PyObject* py_experts(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded([&] { return do_experts(a, n); }); }

// bind(addresses of the twelve C entries, stream_of, stream_here, workspace)
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] {
        need_args(n, 15);
        void* p[12];
        for (int i = 0; i < 12; i++) {
            p[i] = PyLong_AsVoidPtr(a[i]);
            if (!p[i]) raise(PyExc_ValueError, "bind: an address is missing");
        }
        g_append = reinterpret_cast<decltype(g_append)>(p[0]);
        g_attend = reinterpret_cast<decltype(g_attend)>(p[1]);
        g_attend_ws = reinterpret_cast<decltype(g_attend_ws)>(p[2]);
        g_step = reinterpret_cast<decltype(g_step)>(p[3]);
        g_prefill = reinterpret_cast<decltype(g_prefill)>(p[4]);
        g_prefill_ws = reinterpret_cast<decltype(g_prefill_ws)>(p[5]);
        g_fp8_quant = reinterpret_cast<decltype(g_fp8_quant)>(p[6]);
        g_fp8_gemm = reinterpret_cast<decltype(g_fp8_gemm)>(p[7]);
        g_fp8_gemm_ws = reinterpret_cast<decltype(g_fp8_gemm_ws)>(p[8]);
        g_route = reinterpret_cast<decltype(g_route)>(p[9]);
        g_experts = reinterpret_cast<decltype(g_experts)>(p[10]);
        g_experts_ws = reinterpret_cast<decltype(g_experts_ws)>(p[11]);
        for (int i = 12; i < 15; i++) Py_INCREF(a[i]);
        Py_XDECREF(g_stream_of);
        Py_XDECREF(g_stream_here);
        Py_XDECREF(g_workspace);
        g_stream_of = a[12], g_stream_here = a[13], g_workspace = a[14];
        return 0;
    });
}

#define FAST(name, f, doc) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, doc}
PyMethodDef methods[] = {
    FAST("kv_append", py_append, "prism_kv_append after checks; see prism_amd.kv.append"),
    FAST("kv_attend", py_attend, "prism_kv_attend after checks; see prism_amd.kv.attend"),
    FAST("delta_step", py_step, "prism_delta_step after checks; see prism_amd.delta.step"),
    FAST("delta_prefill", py_prefill, "prism_delta_prefill after checks; see prism_amd.delta.prefill"),
    FAST("fp8_quant", py_fp8_quant, "prism_fp8_quant after checks; see prism_amd.fp8.quantize_act"),
    FAST("fp8_gemm", py_fp8_gemm, "prism_fp8_gemm after checks; see prism_amd.fp8.gemm"),
    FAST("moe_route", py_route, "prism_moe_route after checks; see prism_amd.moe.route"),
    FAST("moe_experts", py_experts, "prism_moe_experts after checks; see prism_amd.moe.experts"),
    FAST("bind", py_bind, "addresses of the C entries, then stream_of, stream_here and workspace"),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Host path of prism_amd.kv, delta, fp8 and moe.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
