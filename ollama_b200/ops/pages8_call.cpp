// Calls of the 8-bit paged cache from Python: the checks of their arguments, the argument blocks, workspaces, and the entry points of the kernel library.  A call from Python takes
// about as long on the host as a small step's kernels take on the device (21 us for a decode step with the checks in Python); these take 2 to 3.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstring>
#include <limits>
#include <stdexcept>
#include <string>

#include "../kernels/pages8_args.h"

namespace {

constexpr int PAGE = 64, MAX_UNITS = 256;

// entry points of the kernel library, set by bind()
int (*f_append)(const Append8Args*, int, cudaStream_t);
int (*f_attn)(const Attn8Args*, int, cudaStream_t);
int (*f_decode)(const Append8Args*, const Attn8Args*, int, cudaStream_t);
int (*f_read)(const Pages8*, const PageTable*, const void*, int, void*, void*, int, int, cudaStream_t);
PyObject* kernel_error;          // exception of a launch that fails
PyObject *s_codes, *s_unit, *s_segs, *s_rows, *s_per, *s_longest, *s_masks, *s_table, *s_sizes;

struct Refused : std::invalid_argument {
    using std::invalid_argument::invalid_argument;
};
struct Raised {};                // a Python exception is set

// ---- arguments ------------------------------------------------------------------------------------------------------------------
constexpr int MOST = 32;
struct Signature {
    const char* name;
    int positional, n;           // the first `positional` may be given by position; all by name
    const char* names[MOST];
    PyObject* interned[MOST] = {};
    void intern() {
        for (int i = 0; i < n; i++) interned[i] = PyUnicode_InternFromString(names[i]);
    }
};

void parse(const Signature& s, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames, PyObject** out) {
    std::fill(out, out + s.n, nullptr);
    if (nargs > s.positional) {
        PyErr_Format(PyExc_TypeError, "%s() takes %d positional arguments but %zd were given", s.name, s.positional, nargs);
        throw Raised();
    }
    std::copy(args, args + nargs, out);
    const Py_ssize_t more = kwnames ? PyTuple_GET_SIZE(kwnames) : 0;
    int hint = (int)nargs;
    for (Py_ssize_t k = 0; k < more; k++) {
        PyObject* name = PyTuple_GET_ITEM(kwnames, k);
        int at = -1;
        for (int i = 0; i < s.n && at < 0; i++) {      // names come in about the signature's order
            const int j = (hint + i) % s.n;
            if (s.interned[j] == name) at = j;
        }
        for (int i = 0; i < s.n && at < 0; i++)
            if (PyUnicode_Compare(name, s.interned[i]) == 0) at = i;
        if (at < 0 || out[at]) {
            PyErr_Format(PyExc_TypeError, at < 0 ? "%s() got an unexpected keyword argument '%U'" : "%s() got multiple values for argument '%U'", s.name, name);
            throw Raised();
        }
        out[at] = args[nargs + k];
        hint = at + 1;
    }
}

PyObject* required(const Signature& s, PyObject** a, int i) {
    if (!a[i]) {
        PyErr_Format(PyExc_TypeError, "%s() missing required argument: '%s'", s.name, s.names[i]);
        throw Raised();
    }
    return a[i];
}
bool given(PyObject* o) { return o && o != Py_None; }
long as_long(PyObject* o, long other) {
    if (!o) return other;
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised();
    return std::min(std::max(v, -(1l << 31)), (1l << 31) - 1);
}
double as_double(PyObject* o, double other) {
    if (!o) return other;
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised();
    return v;
}
bool as_bool(PyObject* o, bool other) {
    if (!o) return other;
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Raised();
    return v;
}
struct Ref {                     // an attribute, held
    PyObject* o;
    Ref(PyObject* of, PyObject* name) : o(PyObject_GetAttr(of, name)) {
        if (!o) throw Raised();
    }
    ~Ref() { Py_DECREF(o); }
};
template <typename T>
T as_struct(PyObject* o) {       // a ctypes structure's bytes
    Py_buffer b;
    if (PyObject_GetBuffer(o, &b, PyBUF_SIMPLE)) throw Raised();
    const bool fits = b.len == (Py_ssize_t)sizeof(T);
    T v;
    if (fits) std::memcpy(&v, b.buf, sizeof(T));
    PyBuffer_Release(&b);
    if (!fits) {
        PyErr_SetString(PyExc_TypeError, "a structure of another size");
        throw Raised();
    }
    return v;
}

// ---- tensors --------------------------------------------------------------------------------------------------------------------
std::string told(const at::Tensor& t) {
    std::string s = "(";
    for (auto n : t.sizes()) s += std::to_string(n) + ",";
    return s + ") " + c10::toString(t.scalar_type()) + " on " + t.device().str();
}
[[noreturn]] void refuse(const Signature& s, const std::string& what) { throw Refused(std::string(s.name) + ": " + what); }

const at::Tensor& tensor(const Signature& s, PyObject* o, const char* name) {
    if (!given(o)) refuse(s, std::string(name) + " is missing");
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s(): %s must be a tensor, not %s", s.name, name, Py_TYPE(o)->tp_name);
        throw Raised();
    }
    return THPVariable_Unpack(o);
}
// A tensor of the type, on the device, in one piece.
const at::Tensor& piece(const Signature& s, PyObject* o, const char* name, at::ScalarType type, c10::Device dev) {
    const at::Tensor& t = tensor(s, o, name);
    if (t.scalar_type() != type || t.device() != dev || !t.is_contiguous()) refuse(s, std::string(name) + " " + told(t));
    return t;
}
template <typename... N>
const at::Tensor& shaped(const Signature& s, PyObject* o, const char* name, at::ScalarType type, c10::Device dev, N... sizes) {
    const at::Tensor& t = piece(s, o, name, type, dev);
    const int64_t want[] = {(int64_t)sizes...};
    if (!t.sizes().equals(want)) refuse(s, std::string(name) + " " + told(t));
    return t;
}
const at::Tensor& vector(const Signature& s, PyObject* o, const char* name, at::ScalarType type, c10::Device dev, int64_t least) {
    const at::Tensor& t = piece(s, o, name, type, dev);
    if (t.dim() != 1 || t.numel() < least) refuse(s, std::string(name) + " " + told(t));
    return t;
}
// Rows are a dimension of the merge's grid.
void few_rows(const Signature& s, long n) {
    if (n > 65535) refuse(s, std::to_string(n) + " rows");
}
// From a row to the next of rows that stand beside one another.
long row_step(const Signature& s, const at::Tensor& t, const char* name) {
    const long step = t.size(0) > 1 ? t.stride(0) : t.size(1);
    if (step < t.size(1) || step > (1l << 31) - 1) refuse(s, std::string(name) + " " + told(t) + " with rows " + std::to_string(step) + " apart");
    return step;
}
// read or written 16 bytes at a time
const at::Tensor& wide(const Signature& s, const at::Tensor& t, const char* name) {
    if ((uintptr_t)t.data_ptr() & 15) refuse(s, std::string(name) + " is not on a 16-byte boundary");
    return t;
}
constexpr at::ScalarType F32 = at::kFloat, F64 = at::kDouble, I32 = at::kInt, F16 = at::kHalf, B16 = at::kBFloat16;

struct Cache {
    Pages8 c;
    PageTable t;
};
// Pages as ops/pages8.py makes them; their tensors may have changed in place since.
Cache cache(const Signature& s, PyObject* k, PyObject* v, PyObject* table, c10::Device dev) {
    Ref kc(k, s_codes), ku(k, s_unit), vc(v, s_codes), vu(v, s_unit);
    const at::Tensor &a = wide(s, piece(s, kc.o, "k", at::kByte, dev), "k"), &b = wide(s, piece(s, vc.o, "v", at::kByte, dev), "v");
    if (a.dim() != 4 || a.size(2) != PAGE || (a.size(3) != 64 && a.size(3) != 128) || !a.sizes().equals(b.sizes())) refuse(s, "keys " + told(a) + ", values " + told(b));
    const at::Tensor &ua = shaped(s, ku.o, "k's units", F32, dev, a.size(0), a.size(1)), &ub = shaped(s, vu.o, "v's units", F32, dev, a.size(0), a.size(1));
    const at::Tensor& t = piece(s, table, "table", I32, dev);
    if (t.dim() != 2 || !t.numel()) refuse(s, "table " + told(t));
    return Cache{Pages8{(uint8_t*)a.data_ptr(), (float*)ua.data_ptr(), (uint8_t*)b.data_ptr(), (float*)ub.data_ptr(), (int)a.size(0), (int)a.size(1), (int)a.size(3)},
                 PageTable{(const int*)t.data_ptr(), (int)t.size(0), (int)t.size(1)}};
}

c10::Device on_gpu(const Signature& s, const at::Tensor& t) {
    if (!t.is_cuda()) refuse(s, "tensors on " + t.device().str());
    return t.device();
}
void launched(const Signature& s, int rc) {
    if (rc == 0) return;
    PyErr_Format(kernel_error, "%s failed with CUDA error %d", s.name, rc);
    throw Raised();
}
// Other threads run while memory is found and kernels are launched: either may have to wait, for blocks that are given back or for room in the launch queue.  What the call holds
// (its arguments, which the caller holds) stays.
struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};
template <typename F>
int unlocked(c10::Device dev, F launch) {
    const Unlocked lock;
    const c10::cuda::CUDAGuard guard(dev);
    return launch(c10::cuda::getCurrentCUDAStream(dev.index()).stream());
}
at::Tensor floats(c10::Device dev, long n) { return at::empty({n}, at::TensorOptions().dtype(F32).device(dev)); }
int sms_of(c10::Device dev) {
    static int sms[64] = {};
    int& n = sms[dev.index() & 63];
    if (!n && (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev.index()) != cudaSuccess || n < 1)) n = 148;
    return n;
}

// ---- append8 --------------------------------------------------------------------------------------------------------------------
enum { A_QKV, A_K, A_V, A_TABLE, A_QOUT, A_HEADS, A_DIM, A_VDIM, A_QN, A_KN, A_EPS, A_FREQS, A_NROT, A_POS, A_SLOTS, A_PORTIONS, A_HEADNORM, A_VOFF, A_MSCALE, A_MAPS, A_APPEND, A_PDL, A_N };
Signature append_sig = {"append8", 5, A_N, {"qkv", "k", "v", "table", "q_out", "heads", "dim", "vdim", "q_norm", "k_norm", "eps", "freqs", "n_rot", "positions", "slots", "portions", "head_norm",
                                            "v_off", "mscale", "maps", "append", "pdl"}};

// What both calls that append share.  a: the arguments in the order heads, dim, vdim, q_norm, k_norm, eps, freqs, n_rot; head_norm, v_off, mscale, maps, append.
struct Prep {
    PyObject *heads, *dim, *vdim, *qn, *kn, *eps, *freqs, *n_rot, *head_norm, *v_off, *mscale, *maps, *append;
};
void fill_append(const Signature& s, Append8Args& p, const at::Tensor& qkv, const Cache& c, const Prep& a) {
    const c10::Device dev = qkv.device();
    const long G = c.c.kv_heads, hd = c.c.hd, heads = as_long(a.heads, 0), dim = as_long(a.dim, 0), vdim = as_long(a.vdim, 0), maps = as_long(a.maps, 1), n_rot = as_long(a.n_rot, 0);
    const bool append = as_bool(a.append, true), head_norm = as_bool(a.head_norm, false);
    if (qkv.scalar_type() != F32 || qkv.dim() != 2 || (qkv.size(1) != 1 && qkv.stride(1) != 1)) refuse(s, "qkv " + told(qkv));
    const long cols = qkv.size(1), v_off = given(a.v_off) ? as_long(a.v_off, 0) : (heads + maps * G) * dim;
    if (heads < 1 || heads % G || dim < 1 || vdim < 1 || maps < 1 || maps > 2 || heads % maps || maps * dim > hd || vdim > hd || v_off < 0 || heads * dim > cols ||
        (append && std::max((heads + maps * G) * dim, v_off + G * vdim) > cols))
        refuse(s, std::to_string(heads) + " heads of " + std::to_string(dim) + ", " + std::to_string(G) + " of " + std::to_string(vdim) + " from column " + std::to_string(v_off) + " on, " +
                      std::to_string(maps) + " maps, in " + std::to_string(cols) + " columns and cache rows of " + std::to_string(hd));
    if (n_rot < 0 || n_rot > dim || n_rot % 2) refuse(s, std::to_string(n_rot) + " rotated dimensions of " + std::to_string(dim));
    const bool norm = given(a.qn);
    if (norm != given(a.kn) || (norm && (maps > 1 || !append))) refuse(s, "norms");
    p.qkv = (const float*)qkv.data_ptr();
    p.ldq = (int)row_step(s, qkv, "qkv");
    p.rows = (int)qkv.size(0);
    p.n_heads = heads;
    p.dim = dim;
    p.vdim = vdim;
    p.q_norm = norm ? (const float*)vector(s, a.qn, "q_norm", F32, dev, head_norm ? dim : heads * dim).data_ptr() : nullptr;
    p.k_norm = norm ? (const float*)vector(s, a.kn, "k_norm", F32, dev, head_norm ? dim : G * dim).data_ptr() : nullptr;
    p.eps = (float)as_double(a.eps, 0.0);
    p.freqs = n_rot ? (const double*)vector(s, a.freqs, "freqs", F64, dev, n_rot / 2).data_ptr() : nullptr;
    p.n_rot = n_rot;
    p.t = c.t;
    p.c = c.c;
    p.head_norm = head_norm;
    p.v_off = v_off;
    p.mscale = (float)as_double(a.mscale, 1.0);
    p.maps = maps;
    p.no_append = !append;
}

struct Portions {                // what a Portions8 says
    const int4* segs;
    int n, rows, per, longest;
};
Portions portions(const Signature& s, PyObject* o, long rows, c10::Device dev) {
    Ref segs(o, s_segs), r(o, s_rows), per(o, s_per), longest(o, s_longest);
    const at::Tensor& t = wide(s, piece(s, segs.o, "portions", I32, dev), "portions");
    if (t.dim() != 2 || t.size(1) != 4) refuse(s, "portions " + told(t));
    const Portions p{(const int4*)t.data_ptr(), (int)t.size(0), (int)as_long(r.o, 0), (int)as_long(per.o, 1), (int)as_long(longest.o, 0)};
    if (p.rows > rows) refuse(s, "portions of " + std::to_string(p.rows) + " rows for " + std::to_string(rows));
    return p;
}
// A tuple of n things.
PyObject* tuple_of(const Signature& s, PyObject* o, Py_ssize_t n, const char* what) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != n) refuse(s, std::string("portions whose ") + what + " are not what portions8 makes");
    return o;
}

void append8(PyObject** a) {
    const Signature& s = append_sig;
    for (int i : {A_QKV, A_K, A_V, A_TABLE, A_QOUT, A_HEADS, A_DIM, A_VDIM, A_EPS, A_NROT}) required(s, a, i);
    const at::Tensor& qkv = tensor(s, a[A_QKV], "qkv");
    const c10::Device dev = on_gpu(s, qkv);
    const Cache c = cache(s, a[A_K], a[A_V], a[A_TABLE], dev);
    Append8Args p = {};
    fill_append(s, p, qkv, c, Prep{a[A_HEADS], a[A_DIM], a[A_VDIM], a[A_QN], a[A_KN], a[A_EPS], a[A_FREQS], a[A_NROT], a[A_HEADNORM], a[A_VOFF], a[A_MSCALE], a[A_MAPS], a[A_APPEND]});
    const long n = p.rows;
    p.q_out = (float*)wide(s, shaped(s, a[A_QOUT], "q_out", F32, dev, n, p.n_heads, c.c.hd), "q_out").data_ptr();
    if (given(a[A_PORTIONS]) == (given(a[A_POS]) || given(a[A_SLOTS]))) refuse(s, "either positions and slots or portions");
    if (given(a[A_PORTIONS])) {
        const Portions q = portions(s, a[A_PORTIONS], n, dev);
        p.segs = q.segs;
        p.n_segs = q.n;
        p.per = q.per;
    } else {
        p.positions = (const int*)shaped(s, a[A_POS], "positions", I32, dev, n).data_ptr();
        p.slots = (const int*)shaped(s, a[A_SLOTS], "slots", I32, dev, n).data_ptr();
        p.per = 1;
    }
    const bool pdl = as_bool(a[A_PDL], false);
    if (!n) return;
    launched(s, unlocked(dev, [&](cudaStream_t st) { return f_append(&p, pdl, st); }));
}

// ---- read8 ----------------------------------------------------------------------------------------------------------------------
enum { R_K, R_V, R_PAGES, R_TABLE, R_KOUT, R_VOUT, R_PDL, R_CLEAN, R_N };
Signature read_sig = {"read8", 7, R_N, {"k", "v", "pages", "table", "k_out", "v_out", "pdl", "clean"}};

void read8(PyObject** a) {
    const Signature& s = read_sig;
    for (int i = 0; i < R_PDL; i++) required(s, a, i);
    const at::Tensor& pages = tensor(s, a[R_PAGES], "pages");
    const c10::Device dev = on_gpu(s, pages);
    const Cache c = cache(s, a[R_K], a[R_V], a[R_TABLE], dev);
    const long n = pages.dim() ? pages.size(0) : 0;
    wide(s, shaped(s, a[R_PAGES], "pages", I32, dev, n, 4), "pages");
    const at::Tensor &ko = wide(s, shaped(s, a[R_KOUT], "k_out", F16, dev, n, c.c.kv_heads, PAGE, c.c.hd), "k_out"),
                     &vo = wide(s, shaped(s, a[R_VOUT], "v_out", F16, dev, n, c.c.kv_heads, PAGE, c.c.hd), "v_out");
    const bool clean = as_bool(a[R_CLEAN], false), pdl = as_bool(a[R_PDL], false);
    if (!n) return;
    launched(s, unlocked(dev, [&](cudaStream_t st) { return f_read(&c.c, &c.t, pages.data_ptr(), n, ko.data_ptr(), vo.data_ptr(), clean, pdl, st); }));
}

// ---- attention ------------------------------------------------------------------------------------------------------------------
struct Mask {
    PyObject *vdim, *scale, *softcap, *chunk, *window, *keep, *gate, *diff;
};
void fill_attn(const Signature& s, Attn8Args& p, long n, long heads, PyObject* o, const Cache& c, c10::Device dev, const Mask& m) {
    const at::Tensor& out = tensor(s, o, "out");
    if ((out.scalar_type() != B16 && out.scalar_type() != F32) || out.device() != dev || out.dim() != 2 || out.size(0) != n || (out.size(1) != 1 && out.stride(1) != 1)) refuse(s, "out " + told(out));
    const long G = c.c.kv_heads, vdim = as_long(m.vdim, 0), chunk = as_long(m.chunk, 0), window = as_long(m.window, 0), keep = as_long(m.keep, 0);
    if (m.gate) p.gate = as_struct<HeadGate>(m.gate);
    if (m.diff) p.diff = as_struct<DiffHeads>(m.diff);
    p.softcap = (float)as_double(m.softcap, 0.0);
    if (heads < 1 || heads % G || vdim < 1 || vdim > c.c.hd || (p.diff.on && heads / G % 2) || out.size(1) < (p.diff.on ? heads / 2 : heads) * vdim)
        refuse(s, std::to_string(heads) + " heads on " + std::to_string(G) + " of " + std::to_string(vdim) + " columns into rows of " + std::to_string(out.size(1)));
    if (chunk < 0 || window < 0 || keep < 0 || (chunk && window) || !(p.softcap >= 0.f && p.softcap <= std::numeric_limits<float>::max()))
        refuse(s, "chunk " + std::to_string(chunk) + ", window " + std::to_string(window) + ", keep " + std::to_string(keep) + ", softcap " + std::to_string(p.softcap));
    p.rows = n;
    p.n_heads = heads;
    p.vdim = vdim;
    p.c = c.c;
    p.t = c.t;
    p.chunk = chunk;
    p.window = window;
    p.keep = keep;
    p.scale = (float)as_double(m.scale, 0.0);
    p.out = out.data_ptr();
    p.ldo = (int)row_step(s, out, "out");
    p.out16 = out.scalar_type() == B16;
}

long tiles_of(long rows, int row_tile) { return (rows + row_tile - 1) / row_tile; }
// How many query rows (of a sequence, for the heads of a KV head) and keys are taken together.  most_rows: of a sequence; tiles: row tiles of all sequences of a launch.  Returns the
// rows of partial results: an item's for each row tile and KV head, and those of as many CTAs as fit the GPU.
long tile(const Signature& s, Attn8Args& p, int row_tile, long most_rows, long tiles, c10::Device dev) {
    const long items = tiles * p.c.kv_heads;
    if (items >= 1l << 23) refuse(s, std::to_string(items) + " row tiles of all sequences and KV heads");
    p.row_tile = row_tile;
    p.turn = row_tile == 128 ? 128 : 32;
    p.tiles = (int)tiles_of(most_rows, row_tile);
    p.items = (int)items;
    p.ctas = sms_of(dev) * (row_tile == 8 ? 2 : 1);
    return (items + p.ctas) * row_tile;
}

enum { D_QKV, D_K, D_V, D_POS, D_SLOTS, D_TABLE, D_OUT, D_HEADS, D_DIM, D_VDIM, D_QN, D_KN, D_EPS, D_FREQS, D_NROT, D_SCALE, D_NCTX, D_SOFTCAP, D_CHUNK, D_WINDOW, D_KEEP, D_HEADNORM, D_VOFF, D_MSCALE,
       D_GATE, D_MAPS, D_APPEND, D_DIFF, D_PDL, D_N };
Signature decode_sig = {"attn_decode8", 7, D_N, {"qkv", "k", "v", "positions", "slots", "table", "out", "heads", "dim", "vdim", "q_norm", "k_norm", "eps", "freqs", "n_rot", "scale", "n_ctx", "softcap",
                                                 "chunk", "window", "keep", "head_norm", "v_off", "mscale", "gate", "maps", "append", "diff", "pdl"}};

void attn_decode8(PyObject** a) {
    const Signature& s = decode_sig;
    for (int i = 0; i < D_NCTX; i++)
        if (i != D_QN && i != D_KN && i != D_FREQS) required(s, a, i);
    const at::Tensor& qkv = tensor(s, a[D_QKV], "qkv");
    const c10::Device dev = on_gpu(s, qkv);
    const Cache c = cache(s, a[D_K], a[D_V], a[D_TABLE], dev);
    Append8Args p = {};
    fill_append(s, p, qkv, c, Prep{a[D_HEADS], a[D_DIM], a[D_VDIM], a[D_QN], a[D_KN], a[D_EPS], a[D_FREQS], a[D_NROT], a[D_HEADNORM], a[D_VOFF], a[D_MSCALE], a[D_MAPS], a[D_APPEND]});
    const long n = p.rows, heads = p.n_heads, hd = c.c.hd;
    p.positions = (const int*)shaped(s, a[D_POS], "positions", I32, dev, n).data_ptr();
    p.slots = (const int*)shaped(s, a[D_SLOTS], "slots", I32, dev, n).data_ptr();
    p.per = 1;
    Attn8Args t = {};
    fill_attn(s, t, n, heads, a[D_OUT], c, dev, Mask{a[D_VDIM], a[D_SCALE], a[D_SOFTCAP], a[D_CHUNK], a[D_WINDOW], a[D_KEEP], a[D_GATE], a[D_DIFF]});
    if (!n) return;
    few_rows(s, n);
    const long group = heads / c.c.kv_heads, row_tile = group <= 8 ? 8 : 16, pieces = tile(s, t, row_tile, group, std::min<long>(n, MAX_UNITS) * tiles_of(group, row_tile), dev), nq = n * heads * hd;
    t.positions = p.positions;
    t.slots = p.slots;
    const bool pdl = as_bool(a[D_PDL], false);
    launched(s, unlocked(dev, [&](cudaStream_t st) {
        const at::Tensor ws = floats(dev, nq + pieces * (hd + 2));      // rotated queries, partial results, their statistics
        float* w = (float*)ws.data_ptr();
        p.q_out = w;
        t.q = w;
        t.part_acc = w + nq;
        t.part_ml = (float2*)(w + nq + pieces * hd);
        return f_decode(&p, &t, pdl, st);
    }));
}

enum { P_Q, P_K, P_V, P_PORTIONS, P_TABLE, P_OUT, P_VDIM, P_SCALE, P_SOFTCAP, P_CHUNK, P_WINDOW, P_KEEP, P_GATE, P_DIFF, P_PDL, P_READ, P_N };
Signature prompt_sig = {"attn_prompt8", 6, P_N, {"q", "k", "v", "portions", "table", "out", "vdim", "scale", "softcap", "chunk", "window", "keep", "gate", "diff", "pdl", "read_out"}};

// The launches; 0: the pages are to be read out to f16 first, nothing is launched.  Not with read_out=False.
long attn_prompt8(PyObject** a) {
    const Signature& s = prompt_sig;
    for (int i = 0; i <= P_SCALE; i++) required(s, a, i);
    const at::Tensor& q = tensor(s, a[P_Q], "q");
    const c10::Device dev = on_gpu(s, q);
    const Cache c = cache(s, a[P_K], a[P_V], a[P_TABLE], dev);
    if (q.dim() != 3) refuse(s, "q " + told(q));
    const long n = q.size(0), heads = q.size(1), hd = c.c.hd;
    wide(s, shaped(s, a[P_Q], "q", F32, dev, n, heads, hd), "q");
    Attn8Args t = {};
    fill_attn(s, t, n, heads, a[P_OUT], c, dev, Mask{a[P_VDIM], a[P_SCALE], a[P_SOFTCAP], a[P_CHUNK], a[P_WINDOW], a[P_KEEP], a[P_GATE], a[P_DIFF]});
    const Portions po = portions(s, a[P_PORTIONS], n, dev);
    Ref masks(a[P_PORTIONS], s_masks), table(a[P_PORTIONS], s_table), sizes(a[P_PORTIONS], s_sizes);
    const int mine[3] = {t.window, t.keep, t.chunk};
    tuple_of(s, masks.o, 3, "masks");
    tuple_of(s, sizes.o, po.n, "sizes");
    for (int i = 0; i < 3; i++)
        if (as_long(PyTuple_GET_ITEM(masks.o, i), 0) != mine[i]) refuse(s, "portions that were made with another mask");
    if (const at::Tensor& own = tensor(s, table.o, "portions"); own.dim() != 2 || own.size(1) != c.t.max_pages) refuse(s, "portions that were made with another table");
    // Estimates of three forms, us (measured with 32 heads on 8 of 128, 16 on 4, and 4 on 2 of 64, 1 and 3 sequences, 5 to 512 rows behind 0 to 30000 keys; the choice costs a
    // hundredth on the mean): 16 query rows a tile 9.6 + 0.08 for each tile of a KV head + one for each 19000 of its keys, 128 rows a tile on tcgen05 12 + 0.37 + one for each 11700,
    // pages read out first 10 + 0.0107 a key for each time that the tiles of 128 rows and heads fill the GPU, for each group of portions that are read out together.  (32 heads on 8, in that order: 5 rows at 901 keys 12.3, 16.0, 21.4;
    // 64 at 6144 59.8, 30.6, 77.4; 64 at 30000 230, 59.8, 333; 512 at 6144 -, 130, 84.)
    const long group = heads / c.c.kv_heads, m = po.longest * group;
    double items16 = 0, items128 = 0, keys16 = 0, keys128 = 0, most = 0, ctas = 0, t_read = 0;
    long of = 0;
    auto group_done = [&] {
        t_read += 10 + 0.0107 * most * std::max(1.0, ctas / sms_of(dev));
        most = ctas = 0;
    };
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(sizes.o); i++) {
        PyObject* e = tuple_of(s, PyTuple_GET_ITEM(sizes.o, i), 3, "sizes");
        const double rows = as_long(PyTuple_GET_ITEM(e, 0), 0), keys = as_long(PyTuple_GET_ITEM(e, 1), 0);
        const double of16 = (double)tiles_of((long)rows * group, 16) * c.c.kv_heads, of128 = (double)tiles_of((long)rows * group, 128) * c.c.kv_heads;
        items16 += of16;
        items128 += of128;
        keys16 += of16 * keys;
        keys128 += of128 * keys;
        if (const long g = as_long(PyTuple_GET_ITEM(e, 2), 0); g != of) {
            group_done();
            of = g;
        }
        most = std::max(most, keys);
        ctas += (double)(((long)rows + 127) / 128 * heads);
    }
    group_done();
    const double t16 = 9.6 + 0.08 * items16 + keys16 / 19000, t128 = 12 + 0.37 * items128 + keys128 / 11700;
    if (as_bool(a[P_READ], true) && m > 64 && t_read < std::min(t16, t128) && t.out16 && !((uintptr_t)t.out & 15) && !(t.diff.on && t.gate.kind)) return 0;
    few_rows(s, n);
    const int row_tile = m <= 8 ? 8 : m <= 16 || t16 <= t128 ? 16 : 128;
    long tiles = 0, batch = 0;      // of the launch with most
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(sizes.o); i++) {
        if (i % MAX_UNITS == 0) batch = 0;
        batch += tiles_of(as_long(PyTuple_GET_ITEM(PyTuple_GET_ITEM(sizes.o, i), 0), 0) * group, row_tile);
        tiles = std::max(tiles, batch);
    }
    const long pieces = tile(s, t, row_tile, m, tiles, dev);
    t.q = (const float*)q.data_ptr();
    t.segs = po.segs;
    t.n_segs = po.n;
    const bool pdl = as_bool(a[P_PDL], false);
    launched(s, unlocked(dev, [&](cudaStream_t st) {
        const at::Tensor ws = floats(dev, pieces * (hd + 2));
        t.part_acc = (float*)ws.data_ptr();
        t.part_ml = (float2*)(t.part_acc + pieces * hd);
        return f_attn(&t, pdl, st);
    }));
    return 2 * tiles_of(po.n, MAX_UNITS);
}

// ---- module ---------------------------------------------------------------------------------------------------------------------
template <const Signature& S, typename F>
PyObject* called(F f, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    try {
        PyObject* a[MOST];
        parse(S, args, nargs, kwnames, a);
        if (!f_append) {
            PyErr_SetString(PyExc_RuntimeError, "the kernel library has not been bound");
            throw Raised();
        }
        return f(a);
    } catch (const Raised&) {
    } catch (const Refused& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const c10::OutOfMemoryError& e) {
        PyObject* torch = PyImport_ImportModule("torch");
        PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
        PyErr_SetString(type ? type : PyExc_MemoryError, e.what_without_backtrace());
        Py_XDECREF(type);
        Py_XDECREF(torch);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}
PyObject* none() { Py_RETURN_NONE; }

PyObject* py_append8(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
    return called<append_sig>([](PyObject** a) { append8(a); return none(); }, args, n, kw);
}
PyObject* py_read8(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
    return called<read_sig>([](PyObject** a) { read8(a); return none(); }, args, n, kw);
}
PyObject* py_attn_decode8(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
    return called<decode_sig>([](PyObject** a) { attn_decode8(a); return none(); }, args, n, kw);
}
PyObject* py_attn_prompt8(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
    return called<prompt_sig>([](PyObject** a) { return PyLong_FromLong(attn_prompt8(a)); }, args, n, kw);
}
// bind(append, attn, decode, read, exception, layout): addresses of the kernel library's entry points, what a failing launch raises, and which argument blocks the library takes
PyObject* py_bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 6) {
        PyErr_SetString(PyExc_TypeError, "bind() takes 6 arguments");
        return nullptr;
    }
    const unsigned long long layout = PyLong_AsUnsignedLongLong(args[5]);
    if (layout == (unsigned long long)-1 && PyErr_Occurred()) return nullptr;
    if (layout != PAGES8_LAYOUT) {
        PyErr_SetString(PyExc_RuntimeError, "the kernel library was built from another pages8_args.h than the calls: run python -m ollama_b200.kernels.build");
        return nullptr;
    }
    void* f[4];
    for (int i = 0; i < 4; i++)
        if (!(f[i] = PyLong_AsVoidPtr(args[i]))) return nullptr;
    Py_XSETREF(kernel_error, Py_NewRef(args[4]));
    f_attn = (decltype(f_attn))f[1];
    f_decode = (decltype(f_decode))f[2];
    f_read = (decltype(f_read))f[3];
    f_append = (decltype(f_append))f[0];
    Py_RETURN_NONE;
}

const char append8_doc[] =
    "append8(qkv, k, v, table, q_out, *, heads, dim, vdim, q_norm, k_norm, eps, freqs, n_rot, positions=None, slots=None, portions=None, head_norm=False, v_off=None, mscale=1.0, "
    "maps=1, append=True, pdl=False)\n--\n\n"
    "Norm of q and k, rotation, q to padded fp32 rows [rows, H, 64 or 128], k and v into the cache; arguments as of rows.paged_append.  Rows are one token a sequence at\n"
    "`positions` of `slots` (of rows of one slot the later ones are appended after the earlier ones), or those of `portions`.  Keys of portions turn by products of two angles' cosines\n"
    "and sines, off by 2^-23 of those of a single row: a code next to a border can depend on how the tokens were cut.";
const char read8_doc[] =
    "read8(k, v, pages, table, k_out, v_out, pdl=False, clean=False)\n--\n\n"
    "Pages as f16 values, [n, KV heads, 64, columns] each.  `pages` [n, 4] int32: slot, page of the slot, rows that are wanted (what lies behind them is written as zeros, as are\n"
    "pages that are not there), 0.  `clean`: rows of values that hold what is no number become zeros and their keys none.";
const char attn_decode8_doc[] =
    "attn_decode8(qkv, k, v, positions, slots, table, out, *, heads, dim, vdim, q_norm, k_norm, eps, freqs, n_rot, scale, n_ctx=0, softcap=0.0, chunk=0, window=0, keep=0, "
    "head_norm=False, v_off=None, mscale=1.0, gate=NO_GATE, maps=1, append=True, diff=NO_DIFF, pdl=False)\n--\n\n"
    "Decode attention on raw projections, one token a sequence: what append8 does, then attention of the rows' positions over the cache, difference of maps and gate into rows of\n"
    "`out`.  `n_ctx`, most keys that a sequence holds, is taken as the 16-bit form takes it and not needed: the work follows the positions.\n"
    "Queries and weights are rounded to f16 (2^-11 each) whatever type `out` has, so queries beyond 65504 have no result; the scores' and weights' sums are 32-bit ones.  Soft caps and\n"
    "gates use the fast exponential and quotient, some 2^-21.";

PyMethodDef methods[] = {
    {"append8", (PyCFunction)(void (*)())py_append8, METH_FASTCALL | METH_KEYWORDS, append8_doc},
    {"read8", (PyCFunction)(void (*)())py_read8, METH_FASTCALL | METH_KEYWORDS, read8_doc},
    {"attn_decode8", (PyCFunction)(void (*)())py_attn_decode8, METH_FASTCALL | METH_KEYWORDS, attn_decode8_doc},
    {"attn_prompt8", (PyCFunction)(void (*)())py_attn_prompt8, METH_FASTCALL | METH_KEYWORDS, nullptr},      // see ops/pages8.py
    {"bind", (PyCFunction)(void (*)())py_bind, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pages8", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__pages8() {
    for (Signature* s : {&append_sig, &read_sig, &decode_sig, &prompt_sig}) s->intern();
    s_codes = PyUnicode_InternFromString("codes");
    s_unit = PyUnicode_InternFromString("unit");
    s_segs = PyUnicode_InternFromString("segs");
    s_rows = PyUnicode_InternFromString("rows");
    s_per = PyUnicode_InternFromString("per");
    s_longest = PyUnicode_InternFromString("longest");
    s_masks = PyUnicode_InternFromString("masks");
    s_table = PyUnicode_InternFromString("table");
    s_sizes = PyUnicode_InternFromString("sizes");
    return PyModule_Create(&module);
}
