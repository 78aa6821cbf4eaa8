// Calls of the 4-bit cache and of packed prompts from Python: the checks of their arguments, the argument blocks, workspaces, and the entry points of the kernel library.
#include "call_args.h"

#include <queue>
#include <vector>

#include "../kernels/kv4_args.h"

namespace {

// entry points of the kernel library, set by bind()
int (*f_append)(const Append4Args*, int, cudaStream_t);
int (*f_read)(const Read4Args*, int, cudaStream_t);
int (*f_attn)(const Attn4Args*, int, cudaStream_t);
int (*f_room)(int, int, int, int);
int (*f_packed)(const PackedArgs*, int, cudaStream_t);
PyObject *s_codes, *s_scale, *s_tiles, *s_starts, *s_merges, *s_rows, *s_parts, *s_window, *s_group, *s_cache, *s_merge_rows;

// A cache as ops/kv4.py makes it; its tensors may have changed in place since.
Cache4 cache(const Signature& s, PyObject* k, PyObject* v, c10::Device dev) {
    Ref kc(k, s_codes), ks(k, s_scale), vc(v, s_codes), vs(v, s_scale);
    const at::Tensor &a = wide(s, piece(s, kc.o, "k", at::kByte, dev), "k"), &b = wide(s, piece(s, vc.o, "v", at::kByte, dev), "v");
    if (a.dim() != 4 || !a.numel() || (a.size(3) != 32 && a.size(3) != 64) || !a.sizes().equals(b.sizes()) || a.size(0) > (1l << 30) || a.size(1) > 65535 || a.size(2) > (1l << 30))
        refuse(s, "keys " + told(a) + ", values " + told(b));
    const at::Tensor &ua = wide(s, shaped(s, ks.o, "k's scales", F16, dev, a.size(0), a.size(1), a.size(2), a.size(3) / 16), "k's scales"),
                     &ub = wide(s, shaped(s, vs.o, "v's scales", F16, dev, a.size(0), a.size(1), a.size(2), a.size(3) / 16), "v's scales");
    return Cache4{(uint8_t*)a.data_ptr(), (uint8_t*)b.data_ptr(), ua.data_ptr(), ub.data_ptr(), (int)a.size(0), (int)a.size(1), (int)a.size(2), (int)a.size(3) * 2};
}

struct Prep {
    PyObject *heads, *freqs, *n_rot, *neox, *mscale, *qn, *kn, *eps;
};
void fill_rows(const Signature& s, Rows4& r, const at::Tensor& qkv, const Cache4& c, PyObject* pos, PyObject* slots, const Prep& a) {
    const c10::Device dev = qkv.device();
    if (qkv.scalar_type() != F32 || qkv.dim() != 2 || (qkv.size(1) != 1 && qkv.stride(1) != 1)) refuse(s, "qkv " + told(qkv));
    const long heads = as_long(a.heads, 0), n = qkv.size(0), n_rot = as_long(a.n_rot, 0);
    if (heads < 1 || heads % c.kv_heads || (heads + 2l * c.kv_heads) * c.hd > qkv.size(1))
        refuse(s, std::to_string(heads) + " heads on " + std::to_string(c.kv_heads) + " of " + std::to_string(c.hd) + " columns in rows of " + std::to_string(qkv.size(1)));
    if (n_rot < 0 || n_rot > c.hd || n_rot % 2) refuse(s, std::to_string(n_rot) + " rotated dimensions of " + std::to_string(c.hd));
    if (n > (1l << 30)) refuse(s, std::to_string(n) + " rows");
    r.qkv = (const float*)qkv.data_ptr();
    r.ldq = (int)row_step(s, qkv, "qkv");
    r.rows = (int)n;
    r.n_heads = (int)heads;
    r.positions = (const int*)shaped(s, pos, "positions", I32, dev, n).data_ptr();
    r.slots = (const int*)shaped(s, slots, "slots", I32, dev, n).data_ptr();
    r.inv_freq = n_rot ? (const float*)vector(s, a.freqs, "inv_freq", F32, dev, n_rot / 2).data_ptr() : nullptr;
    r.n_rot = (int)n_rot;
    r.neox = as_bool(a.neox, true);
    r.mscale = (float)as_double(a.mscale, 1.0);
    r.q_norm = given(a.qn) ? (const float*)shaped(s, a.qn, "q_norm", F32, dev, c.hd).data_ptr() : nullptr;
    r.k_norm = given(a.kn) ? (const float*)shaped(s, a.kn, "k_norm", F32, dev, c.hd).data_ptr() : nullptr;
    r.eps = (float)as_double(a.eps, 1e-6);
}

// ---- append4 --------------------------------------------------------------------------------------------------------------------
enum { A_QKV, A_K, A_V, A_POS, A_SLOTS, A_QOUT, A_HEADS, A_FREQS, A_NROT, A_NEOX, A_MSCALE, A_QN, A_KN, A_EPS, A_PDL, A_N };
Signature append_sig = {"append4", 6, A_N, {"qkv", "k", "v", "positions", "slots", "q_out", "heads", "inv_freq", "n_rot", "neox", "mscale", "q_norm", "k_norm", "eps", "pdl"}};

void append4(PyObject** a) {
    const Signature& s = append_sig;
    for (int i : {A_QKV, A_K, A_V, A_POS, A_SLOTS, A_HEADS, A_NROT}) required(s, a, i);
    const at::Tensor& qkv = tensor(s, a[A_QKV], "qkv");
    const c10::Device dev = on_gpu(s, qkv);
    Append4Args p = {};
    p.c = cache(s, a[A_K], a[A_V], dev);
    fill_rows(s, p.r, qkv, p.c, a[A_POS], a[A_SLOTS], Prep{a[A_HEADS], a[A_FREQS], a[A_NROT], a[A_NEOX], a[A_MSCALE], a[A_QN], a[A_KN], a[A_EPS]});
    if (given(a[A_QOUT])) {
        const at::Tensor& q = tensor(s, a[A_QOUT], "q_out");
        p.q16 = q.scalar_type() == F16;
        p.q_out = wide(s, shaped(s, a[A_QOUT], "q_out", p.q16 ? F16 : F32, dev, p.r.rows, p.r.n_heads, p.c.hd), "q_out").data_ptr();
    }
    const bool pdl = as_bool(a[A_PDL], false);
    if (!p.r.rows) return;
    launched(s, unlocked(dev, [&](cudaStream_t st) { return f_append(&p, pdl, st); }));
}

// ---- read4 ----------------------------------------------------------------------------------------------------------------------
enum { R_K, R_V, R_POS, R_SLOTS, R_KOUT, R_VOUT, R_PDL, R_N };
Signature read_sig = {"read4", 7, R_N, {"k", "v", "positions", "slots", "k_out", "v_out", "pdl"}};

void read4(PyObject** a) {
    const Signature& s = read_sig;
    for (int i = 0; i < R_PDL; i++) required(s, a, i);
    const at::Tensor& pos = tensor(s, a[R_POS], "positions");
    const c10::Device dev = on_gpu(s, pos);
    Read4Args p = {};
    p.c = cache(s, a[R_K], a[R_V], dev);
    const long n = pos.dim() ? pos.size(0) : 0;
    if (n > (1l << 30)) refuse(s, std::to_string(n) + " rows");
    p.positions = (const int*)shaped(s, a[R_POS], "positions", I32, dev, n).data_ptr();
    p.slots = (const int*)shaped(s, a[R_SLOTS], "slots", I32, dev, n).data_ptr();
    p.rows = (int)n;
    p.k_out = wide(s, shaped(s, a[R_KOUT], "k_out", F16, dev, n, p.c.kv_heads, p.c.hd), "k_out").data_ptr();
    p.v_out = wide(s, shaped(s, a[R_VOUT], "v_out", F16, dev, n, p.c.kv_heads, p.c.hd), "v_out").data_ptr();
    const bool pdl = as_bool(a[R_PDL], false);
    if (!n) return;
    launched(s, unlocked(dev, [&](cudaStream_t st) { return f_read(&p, pdl, st); }));
}

// ---- attention ------------------------------------------------------------------------------------------------------------------
struct Mask {
    PyObject *scale, *softcap, *window, *sinks;
};
struct Masked {
    float scale, softcap;
    int window;
    const float* sinks;
};
Masked masks(const Signature& s, const Mask& m, long heads, c10::Device dev) {
    Masked r{(float)as_double(m.scale, 0.0), (float)as_double(m.softcap, 0.0), (int)as_long(m.window, 0), nullptr};
    if (r.window < 0 || !(r.softcap >= 0.f && r.softcap <= std::numeric_limits<float>::max()) || !(r.scale >= -std::numeric_limits<float>::max() && r.scale <= std::numeric_limits<float>::max()))
        refuse(s, "scale " + std::to_string(r.scale) + ", softcap " + std::to_string(r.softcap) + ", window " + std::to_string(r.window));
    if (given(m.sinks)) r.sinks = (const float*)shaped(s, m.sinks, "sinks", F32, dev, heads).data_ptr();
    return r;
}
// Rows of results; `least`: columns.
const at::Tensor& results(const Signature& s, PyObject* o, c10::Device dev, long n, long least) {
    const at::Tensor& out = wide(s, tensor(s, o, "out"), "out");
    const auto t = out.scalar_type();
    if ((t != B16 && t != F32 && t != F16) || out.device() != dev || out.dim() != 2 || out.size(0) != n || out.size(1) < least || (out.size(1) != 1 && out.stride(1) != 1)) refuse(s, "out " + told(out));
    return out;
}
long aligned_step(const Signature& s, const at::Tensor& t, const char* name) {
    const long step = row_step(s, t, name);
    if (step * t.element_size() % 16) refuse(s, std::string(name) + " " + told(t) + " with rows " + std::to_string(step) + " apart");
    return step;
}

void run_attn(const Signature& s, Attn4Args& p, PyObject* o, const Mask& m, c10::Device dev, bool pdl) {
    const long n = p.r.rows, heads = p.r.n_heads;
    const Masked k = masks(s, m, heads, dev);
    p.scale = k.scale;
    p.softcap = k.softcap;
    p.window = k.window;
    p.sinks = k.sinks;
    const at::Tensor& out = results(s, o, dev, n, heads * p.c.hd);
    if (out.scalar_type() == F16) refuse(s, "out " + told(out));
    p.out = out.data_ptr();
    p.ldo = (int)row_step(s, out, "out");
    p.out16 = out.scalar_type() == B16;
    if (!n) return;
    few_rows(s, n);
    p.room = f_room(n, heads, p.c.kv_heads, sms_of(dev));
    launched(s, unlocked(dev, [&](cudaStream_t st) {
        const long parts = (long)p.room * heads;
        const at::Tensor ws = floats(dev, parts * (p.c.hd + 2) + 2 * n);      // partial results, their statistics, the sequences' shares
        p.part_acc = (float*)ws.data_ptr();
        p.part_ml = (float2*)(p.part_acc + parts * p.c.hd);
        p.shares = (int2*)(p.part_ml + parts);
        return f_attn(&p, pdl, st);
    }));
}

enum { D_Q, D_K, D_V, D_POS, D_SLOTS, D_OUT, D_SCALE, D_SOFTCAP, D_WINDOW, D_SINKS, D_PDL, D_N };
Signature decode_sig = {"attn_decode4", 6, D_N, {"q", "k", "v", "positions", "slots", "out", "scale", "softcap", "window", "sinks", "pdl"}};

const at::Tensor& queries(const Signature& s, PyObject* o, c10::Device dev, long hd) {
    const at::Tensor& q = wide(s, tensor(s, o, "q"), "q");
    const auto t = q.scalar_type();
    if ((t != F32 && t != F16 && t != B16) || q.device() != dev || q.dim() != 3 || q.size(1) < 1 || q.size(2) != hd) refuse(s, "q " + told(q));
    return q;
}
void heads_fit(const Signature& s, long heads, long kv_heads) {
    if (heads % kv_heads) refuse(s, std::to_string(heads) + " heads on " + std::to_string(kv_heads));
}

void attn_decode4(PyObject** a) {
    const Signature& s = decode_sig;
    for (int i = 0; i <= D_SCALE; i++) required(s, a, i);
    const c10::Device dev = on_gpu(s, tensor(s, a[D_Q], "q"));
    Attn4Args p = {};
    p.c = cache(s, a[D_K], a[D_V], dev);
    const at::Tensor& q = queries(s, a[D_Q], dev, p.c.hd);
    if (!q.is_contiguous() || q.scalar_type() == B16) refuse(s, "q " + told(q));
    heads_fit(s, q.size(1), p.c.kv_heads);
    p.q = q.data_ptr();
    p.q16 = q.scalar_type() == F16;
    p.r.rows = (int)std::min<int64_t>(q.size(0), 1 << 30);
    p.r.n_heads = (int)q.size(1);
    p.r.positions = (const int*)shaped(s, a[D_POS], "positions", I32, dev, q.size(0)).data_ptr();
    p.r.slots = (const int*)shaped(s, a[D_SLOTS], "slots", I32, dev, q.size(0)).data_ptr();
    run_attn(s, p, a[D_OUT], Mask{a[D_SCALE], a[D_SOFTCAP], a[D_WINDOW], a[D_SINKS]}, dev, as_bool(a[D_PDL], false));
}

enum { S_QKV, S_K, S_V, S_POS, S_SLOTS, S_OUT, S_HEADS, S_FREQS, S_NROT, S_SCALE, S_NEOX, S_MSCALE, S_QN, S_KN, S_EPS, S_SOFTCAP, S_WINDOW, S_SINKS, S_PDL, S_N };
Signature step_sig = {"attn_step4", 6, S_N, {"qkv", "k", "v", "positions", "slots", "out", "heads", "inv_freq", "n_rot", "scale", "neox", "mscale", "q_norm", "k_norm", "eps", "softcap", "window", "sinks", "pdl"}};

void attn_step4(PyObject** a) {
    const Signature& s = step_sig;
    for (int i = 0; i <= S_SCALE; i++)
        if (i != S_FREQS) required(s, a, i);
    const at::Tensor& qkv = tensor(s, a[S_QKV], "qkv");
    const c10::Device dev = on_gpu(s, qkv);
    Attn4Args p = {};
    p.c = cache(s, a[S_K], a[S_V], dev);
    fill_rows(s, p.r, qkv, p.c, a[S_POS], a[S_SLOTS], Prep{a[S_HEADS], a[S_FREQS], a[S_NROT], a[S_NEOX], a[S_MSCALE], a[S_QN], a[S_KN], a[S_EPS]});
    run_attn(s, p, a[S_OUT], Mask{a[S_SCALE], a[S_SOFTCAP], a[S_WINDOW], a[S_SINKS]}, dev, as_bool(a[S_PDL], false));
}

// ---- packed prompts -------------------------------------------------------------------------------------------------------------
enum { P_Q, P_K, P_V, P_PORTIONS, P_OUT, P_SCALE, P_SOFTCAP, P_WINDOW, P_SINKS, P_PDL, P_N };
Signature prompt_sig = {"attn_prompt4", 5, P_N, {"q", "k", "v", "portions", "out", "scale", "softcap", "window", "sinks", "pdl"}};
Signature packed_sig = {"attn_packed", 5, P_N, {"q", "k", "v", "portions", "out", "scale", "softcap", "window", "sinks", "pdl"}};

// Distance in elements from one of a dimension to the next, as a tensor map takes it.
long long map_step(const Signature& s, const at::Tensor& t, int dim, const char* name) {
    if (t.size(dim) == 1) return 8;
    const long long step = t.stride(dim);
    if (step < 8 || step % 8 || step >= 1ll << 39) refuse(s, std::string(name) + " " + told(t) + " with strides that are no positive multiples of 8");
    return step;
}

long prompt(const Signature& s, PyObject** a, bool codes) {
    for (int i = 0; i <= P_SCALE; i++) required(s, a, i);
    const c10::Device dev = on_gpu(s, tensor(s, a[P_Q], "q"));
    PackedArgs p = {};
    long n_ctx, slots;
    if (codes) {
        p.c = cache(s, a[P_K], a[P_V], dev);
        p.hd = p.c.hd;
        p.kv_heads = p.c.kv_heads;
        slots = p.c.slots;
        n_ctx = p.c.n_ctx;
    } else {
        const at::Tensor &k = wide(s, tensor(s, a[P_K], "k"), "k"), &v = wide(s, tensor(s, a[P_V], "v"), "v");
        const auto t = k.scalar_type();
        if ((t != F16 && t != B16) || t != v.scalar_type() || k.device() != dev || v.device() != dev || k.dim() != 4 || !k.sizes().equals(v.sizes()) || !k.numel() ||
            (k.size(3) != 64 && k.size(3) != 128) || k.stride(3) != 1 || v.stride(3) != 1 || k.size(0) > (1l << 30) || k.size(1) > 65535 || k.size(2) > (1l << 30))
            refuse(s, "keys " + told(k) + ", values " + told(v));
        p.k = k.data_ptr();
        p.v = v.data_ptr();
        p.kv_bf16 = t == B16;
        p.k_slot = map_step(s, k, 0, "k"); p.k_head = map_step(s, k, 1, "k"); p.k_row = map_step(s, k, 2, "k");
        p.v_slot = map_step(s, v, 0, "v"); p.v_head = map_step(s, v, 1, "v"); p.v_row = map_step(s, v, 2, "v");
        p.hd = (int)k.size(3);
        p.kv_heads = (int)k.size(1);
        slots = k.size(0);
        n_ctx = k.size(2);
    }
    p.slots = (int)slots;
    p.n = (int)n_ctx;
    const at::Tensor& q = queries(s, a[P_Q], dev, p.hd);
    const long n = q.size(0), heads = q.size(1);
    heads_fit(s, heads, p.kv_heads);
    if ((heads > 1 && q.stride(1) != p.hd) || q.stride(2) != 1 || n > (1l << 30) || heads > 65535) refuse(s, "q " + told(q));
    p.q = q.data_ptr();
    p.q_type = q.scalar_type() == F32 ? 0 : q.scalar_type() == F16 ? 1 : 2;
    p.q_rows = (int)n;
    p.ldq = n > 1 ? q.stride(0) : heads * p.hd;
    if (p.ldq < heads * p.hd || p.ldq >= 1ll << 39 || p.ldq * q.element_size() % 16) refuse(s, "q " + told(q) + " with rows " + std::to_string(p.ldq) + " apart");
    p.n_heads = (int)heads;
    const Masked k = masks(s, Mask{a[P_SCALE], a[P_SOFTCAP], a[P_WINDOW], a[P_SINKS]}, heads, dev);
    p.scale = k.scale;
    p.softcap = k.softcap;
    p.window = k.window;
    p.sinks = k.sinks;
    // tiles of other heads, masks or caches would point elsewhere
    PyObject* o = a[P_PORTIONS];
    Ref tiles(o, s_tiles), starts(o, s_starts), merges(o, s_merges), rows(o, s_rows), parts(o, s_parts), merge_rows(o, s_merge_rows), window(o, s_window), group(o, s_group), cached(o, s_cache);
    const long of[4] = {slots, p.kv_heads, n_ctx, p.hd};
    if (!PyTuple_Check(cached.o) || PyTuple_GET_SIZE(cached.o) != 4) refuse(s, "portions that are not what portions4 makes");
    for (int i = 0; i < 4; i++)
        if (as_long(PyTuple_GET_ITEM(cached.o, i), 0) != of[i]) refuse(s, "portions that were made with another cache");
    if (as_long(window.o, 0) != p.window) refuse(s, "portions that were made with another window");
    if (as_long(group.o, 0) * p.kv_heads != heads) refuse(s, "portions that were made for " + std::to_string(as_long(group.o, 0)) + " heads a KV head");
    if (as_long(rows.o, 0) > n) refuse(s, "portions of " + std::to_string(as_long(rows.o, 0)) + " rows for " + std::to_string(n));
    const at::Tensor &t = wide(s, piece(s, tiles.o, "portions", I32, dev), "portions"), &u = wide(s, piece(s, merges.o, "portions", I32, dev), "portions"), &w = piece(s, starts.o, "portions", I32, dev);
    if (t.dim() != 2 || t.size(1) * 4 != (long)sizeof(PackedTile) || u.dim() != 2 || u.size(1) * 4 != (long)sizeof(PackedMerge) || w.dim() != 1 || w.numel() < 2 || w.numel() - 1 > t.size(0) || t.size(0) > (1l << 30) || u.size(0) > (1l << 30)) refuse(s, "portions " + told(t));
    p.tiles = (const PackedTile*)t.data_ptr();
    p.starts = (const int*)w.data_ptr();
    p.ctas = (int)w.numel() - 1;
    p.n_tiles = (int)t.size(0);
    p.merges = (const PackedMerge*)u.data_ptr();
    p.n_merges = (int)u.size(0);
    p.parts = (int)std::max(as_long(parts.o, 0), 0l);
    p.merge_rows = (int)std::min(std::max(as_long(merge_rows.o, 0), 1l), 256l);
    const at::Tensor& out = results(s, a[P_OUT], dev, n, heads * p.hd);
    p.out = out.data_ptr();
    p.ldo = (int)aligned_step(s, out, "out");
    p.out_type = out.scalar_type() == F32 ? 0 : out.scalar_type() == F16 ? 1 : 2;
    if (n * p.ldo * out.element_size() >= 1l << 36 || 1024l * p.parts * p.hd >= 1l << 36) refuse(s, "out " + told(out) + " with rows " + std::to_string(p.ldo) + " apart");      // in 16 bytes a 32-bit number
    const bool pdl = as_bool(a[P_PDL], false);
    launched(s, unlocked(dev, [&](cudaStream_t st) {
        const long rows256 = (long)p.parts * 256;
        at::Tensor ws;
        if (rows256) {
            ws = floats(dev, rows256 * (p.hd + 2));
            p.part_acc = (float*)ws.data_ptr();
            p.part_ml = (float2*)(p.part_acc + rows256 * p.hd);
        }
        return f_packed(&p, pdl, st);
    }));
    return p.n_merges ? 2 : 1;
}

// ---- portions -------------------------------------------------------------------------------------------------------------------
// What a share's start and end, and adding up partial results, cost in the time of a tile of 128 keys.  (Over 60 drawn shapes: shares at one tile a hundredth slower on the mean, adding up at three 2 % slower, 50 at
// most, at none 2 % slower where few keys are cut, 16 % at 200 rows of 32 heads.  Shares have one tile at least; of two 7 rows behind 901 keys 12.4 for 11.0 us, of three 17.3.)
constexpr int SHARE_TILES = 2, MERGE_TILES = 1;

Signature plan_sig = {"plan", 5, 5, {"parts", "group", "kv_heads", "window", "sms"}};
// plan(parts, group, kv_heads, window, sms): shares and merges for portions [n, 5] int32 (first row, rows, slot, position, cache row of position 0), as int32 tensors [., 12] and [., 8], where
// each CTA's shares begin, the number of partial results and how many of their rows the largest sum has.  All tiles as they are, the longest first to the CTA that has least to do, where that ends about when equal shares would; else
// tiles are cut where a CTA has its share.
PyObject* plan(PyObject** a) {
    const Signature& s = plan_sig;
    for (int i = 0; i < 5; i++) required(s, a, i);
    const at::Tensor& parts = piece(s, a[0], "parts", I32, c10::Device(c10::kCPU));
    const long group = as_long(a[1], 1), heads = as_long(a[2], 1), window = as_long(a[3], 0), sms = as_long(a[4], 1);
    if (parts.dim() != 2 || parts.size(1) != 5 || group < 1 || group > 128 || heads < 1 || sms < 1 || window < 0) refuse(s, "parts " + told(parts));
    const int* from = (const int*)parts.data_ptr();
    const long step = 2 * (128 / group);
    std::vector<PackedTile> whole, out;
    std::vector<PackedMerge> merges;
    long work = 0;
    for (long i = 0; i < parts.size(0); i++, from += 5)
        for (long r = 0; r < from[1]; r += step) {
            PackedTile t = {};
            t.row = (int)(from[0] + r);
            t.rows = (int)std::min<long>(step, from[1] - r);
            t.slot = from[2];
            t.pos = (int)(from[3] + r);
            t.base = from[4];
            t.k_lo = window ? std::max(0l, t.pos - window + 1) / 128 : 0;
            t.k_hi = (t.pos + t.rows - 1) / 128 + 1;
            t.part = -1;
            for (t.kvh = 0; t.kvh < heads; t.kvh++) whole.push_back(t);
            work += heads * (t.k_hi - t.k_lo);
        }
    std::stable_sort(whole.begin(), whole.end(), [](const PackedTile& x, const PackedTile& y) { return x.k_hi - x.k_lo > y.k_hi - y.k_lo; });
    const long n = (long)whole.size(), share = std::max<long>((work + SHARE_TILES * (n + sms) + sms - 1) / sms, SHARE_TILES + 1);      // about one cut an SM
    int n_parts = 0, merge_rows = 0;
    using Load = std::pair<long, int>;       // what a CTA has to do
    using Least = std::priority_queue<Load, std::vector<Load>, std::greater<Load>>;
    std::vector<std::vector<PackedTile>> of(std::min(n, sms));
    auto all = [&] {
        Least q;
        for (int i = 0; i < (int)of.size(); i++) q.push({0, i});
        return q;
    };
    Least q = all();
    long last = 0;
    for (const PackedTile& t : whole) {
        Load x = q.top();
        q.pop();
        x.first += t.k_hi - t.k_lo + SHARE_TILES;
        last = std::max(last, x.first);
        of[x.second].push_back(t);
        q.push(x);
    }
    if (last > share + MERGE_TILES) {
        of.assign(sms, {});
        q = all();
        for (const PackedTile& t : whole) {
            int lo = t.k_lo;
            const int first = n_parts;
            while (lo < t.k_hi) {
                Load x = q.top();
                q.pop();
                const long left = t.k_hi - lo;
                const long take = std::min(left, std::max<long>(share - x.first - SHARE_TILES, 1));
                PackedTile y = t;
                y.k_lo = lo;
                y.k_hi = lo += (int)take;
                if (take < t.k_hi - t.k_lo) y.part = n_parts++;
                of[x.second].push_back(y);
                x.first += take + SHARE_TILES;
                q.push(x);
            }
            if (n_parts > first) {
                merges.push_back(PackedMerge{t.row, t.rows, first, n_parts - first, t.kvh, {}});
                merge_rows = std::max(merge_rows, (int)(t.rows <= step / 2 ? t.rows * group : 128 + (t.rows - step / 2) * group));
            }
        }
        of.erase(std::remove_if(of.begin(), of.end(), [](const auto& x) { return x.empty(); }), of.end());
    }
    for (const auto& x : of) out.push_back(x[0]);
    std::vector<int> starts(1, (int)out.size());
    for (const auto& x : of) {
        out.insert(out.end(), x.begin() + 1, x.end());
        starts.push_back((int)out.size());
    }
    auto tensor_of = [](const void* p, size_t n, int columns) {
        at::Tensor t = at::empty({(long)n, (long)columns}, at::TensorOptions().dtype(I32));
        if (n) std::memcpy(t.data_ptr(), p, n * columns * 4);
        return THPVariable_Wrap(t);
    };
    return Py_BuildValue("(NNNii)", tensor_of(out.data(), out.size(), 12), tensor_of(merges.data(), merges.size(), 8), tensor_of(starts.data(), starts.size(), 1), n_parts, merge_rows);
}

bool bound() { return f_append != nullptr; }
bool always() { return true; }

// ---- module ---------------------------------------------------------------------------------------------------------------------
PyObject* py_append4(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
    return called<append_sig, bound>([](PyObject** a) { append4(a); return none(); }, args, n, kw);
}
PyObject* py_read4(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
    return called<read_sig, bound>([](PyObject** a) { read4(a); return none(); }, args, n, kw);
}
PyObject* py_attn_decode4(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
    return called<decode_sig, bound>([](PyObject** a) { attn_decode4(a); return none(); }, args, n, kw);
}
PyObject* py_attn_step4(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
    return called<step_sig, bound>([](PyObject** a) { attn_step4(a); return none(); }, args, n, kw);
}
PyObject* py_attn_prompt4(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
    return called<prompt_sig, bound>([](PyObject** a) { return PyLong_FromLong(prompt(prompt_sig, a, true)); }, args, n, kw);
}
PyObject* py_attn_packed(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
    return called<packed_sig, bound>([](PyObject** a) { return PyLong_FromLong(prompt(packed_sig, a, false)); }, args, n, kw);
}
PyObject* py_plan(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) { return called<plan_sig, always>([](PyObject** a) { return plan(a); }, args, n, kw); }
// bind(append, read, attn, room, packed, exception, layout): addresses of the kernel library's entry points, what a failing launch raises, and which argument blocks the library takes
PyObject* py_bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 7) {
        PyErr_SetString(PyExc_TypeError, "bind() takes 7 arguments");
        return nullptr;
    }
    const unsigned long long layout = PyLong_AsUnsignedLongLong(args[6]);
    if (layout == (unsigned long long)-1 && PyErr_Occurred()) return nullptr;
    if (layout != KV4_LAYOUT) {
        PyErr_SetString(PyExc_RuntimeError, "the kernel library was built from another kv4_args.h than the calls: run python -m ollama_b200.kernels.build");
        return nullptr;
    }
    void* f[5];
    for (int i = 0; i < 5; i++)
        if (!(f[i] = PyLong_AsVoidPtr(args[i]))) return nullptr;
    Py_XSETREF(kernel_error, Py_NewRef(args[5]));
    f_read = (decltype(f_read))f[1];
    f_attn = (decltype(f_attn))f[2];
    f_room = (decltype(f_room))f[3];
    f_packed = (decltype(f_packed))f[4];
    f_append = (decltype(f_append))f[0];
    Py_RETURN_NONE;
}

const char append4_doc[] =
    "append4(qkv, k, v, positions, slots, q_out=None, *, heads, inv_freq, n_rot, neox=True, mscale=1.0, q_norm=None, k_norm=None, eps=1e-6, pdl=False)\n--\n\n"
    "Norm (`q_norm`, `k_norm` [columns], of each head) and rotation of q and k, q to rows [rows, heads, columns] of fp32 or f16, k and v into the cache.  `qkv` fp32 [rows, q heads | k heads |\n"
    "v heads].  Pairs are columns p and p + n_rot / 2 (`neox`), or 2 p and 2 p + 1; `mscale` is a factor of the rotated columns.  Rows whose position or slot the cache does not have hold no token:\n"
    "nothing is appended for them and their queries are left as they are.  What two rows of the same slot and position leave is one of them, or a mixture.";
const char read4_doc[] =
    "read4(k, v, positions, slots, k_out, v_out, pdl=False)\n--\n\n"
    "Rows as f16 values [rows, KV heads, columns]: a code's integer times its scale, rounded once.  Rows that the cache does not have are left as they are.";
const char attn_decode4_doc[] =
    "attn_decode4(q, k, v, positions, slots, out, *, scale, softcap=0.0, window=0, sinks=None, pdl=False)\n--\n\n"
    "Attention of one token a sequence, whose queries `q` [rows, heads, columns] (fp32, rounded to f16, or f16) are rotated and whose key and value are in the cache: over the positions up to its own, the last\n"
    "`window` of them where that is not 0.  `sinks` [heads] are logits in the denominator.  `out` fp32 or bf16 [rows, heads * columns].  Rows that hold no token are left as they are.\n"
    "Queries and weights are f16 numbers (2^-11 each) whatever type `out` has, so queries beyond 65504 have no result; sums are 32-bit ones.  Soft caps use the fast exponential and quotient, some 2^-21.\n"
    "Where a sequence's keys are cut follows from all sequences of the call: beside others a result is that of the sequence alone but for roundings.";
const char attn_step4_doc[] =
    "attn_step4(qkv, k, v, positions, slots, out, *, heads, inv_freq, n_rot, scale, neox=True, mscale=1.0, q_norm=None, k_norm=None, eps=1e-6, softcap=0.0, window=0, sinks=None, pdl=False)\n--\n\n"
    "A step on raw projections, one token a sequence: what append4 does, then attn_decode4 of its queries.  The rows that hold tokens are of different slots.";
const char attn_prompt4_doc[] =
    "attn_prompt4(q, k, v, portions, out, *, scale, softcap=0.0, window=0, sinks=None, pdl=False)\n--\n\n"
    "Causal attention of the rows of `portions`, made by portions4 for this cache, these heads and this window, whose keys and values are in the cache.  `q` [rows, heads, columns] fp32, f16 or bf16; `out` fp32,\n"
    "f16 or bf16 [rows, heads * columns].  Queries, weights and what the codes stand for are f16 numbers, sums 32-bit ones.  Rows behind the last portion are left as they are.  Returns the launches.";
const char attn_packed_doc[] =
    "attn_packed(q, k, v, portions, out, *, scale, softcap=0.0, window=0, sinks=None, pdl=False)\n--\n\n"
    "The same over 16-bit keys and values [slots, KV heads, positions, 64 or 128], f16 or bf16, of any strides that are multiples of 8; queries and weights are rounded to their type.  Rows packed one sequence\n"
    "after the other, [rows, KV heads, columns], are `x.transpose(0, 1)[None]`.  Keys that a row does not see do not touch its result, whatever they hold; one that it sees leaves it without one if its value is not finite.";

PyMethodDef methods[] = {
    {"append4", (PyCFunction)(void (*)())py_append4, METH_FASTCALL | METH_KEYWORDS, append4_doc},
    {"read4", (PyCFunction)(void (*)())py_read4, METH_FASTCALL | METH_KEYWORDS, read4_doc},
    {"attn_decode4", (PyCFunction)(void (*)())py_attn_decode4, METH_FASTCALL | METH_KEYWORDS, attn_decode4_doc},
    {"attn_step4", (PyCFunction)(void (*)())py_attn_step4, METH_FASTCALL | METH_KEYWORDS, attn_step4_doc},
    {"attn_prompt4", (PyCFunction)(void (*)())py_attn_prompt4, METH_FASTCALL | METH_KEYWORDS, attn_prompt4_doc},
    {"attn_packed", (PyCFunction)(void (*)())py_attn_packed, METH_FASTCALL | METH_KEYWORDS, attn_packed_doc},
    {"plan", (PyCFunction)(void (*)())py_plan, METH_FASTCALL | METH_KEYWORDS, nullptr},      // see portions4
    {"bind", (PyCFunction)(void (*)())py_bind, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kv4", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__kv4() {
    for (Signature* s : {&append_sig, &read_sig, &decode_sig, &step_sig, &prompt_sig, &packed_sig, &plan_sig}) s->intern();
    PyObject** names[] = {&s_codes, &s_scale, &s_tiles, &s_starts, &s_merges, &s_rows, &s_parts, &s_window, &s_group, &s_cache, &s_merge_rows};
    const char* texts[] = {"codes", "scale", "tiles", "starts", "merges", "rows", "parts", "window", "group", "cache", "merge_rows"};
    for (int i = 0; i < 11; i++) *names[i] = PyUnicode_InternFromString(texts[i]);
    return PyModule_Create(&module);
}
