// Attention over an 8-bit paged cache (layout: pages8.cuh).
//
//   out[row][h] = gate * softmax_k( cap(scale * q[row][h] . K[k]) ) V      k: the keys that first_key (rows.cuh) lets the row's position see
//
// Every CTA takes a row and a head and leaves (largest score, sum, unnormalised result), which a second kernel turns into rows.
#include "pages8.cuh"

namespace {

struct Attn8Args {
    const float* q;          // [rows][H][hd], rotated
    int rows, n_heads, vdim;
    Pages8 c;
    PageTable t;
    const int* positions;    // [rows], or null:
    const int* slots;
    const int4* segs;        // [n_segs] portions (first row, rows, slot, position of the first row)
    int n_segs;
    int chunk, window, keep;
    float scale, softcap;
    int n_splits;
    float* part_acc;         // [rows][H][splits][hd]
    float2* part_ml;         // [rows][H][splits] (largest score, sum); a sum below zero: the row holds no token
    void* out;               // [rows][ldo], head h at column h * vdim
    int ldo, out16;
    HeadGate gate;
    DiffHeads diff;
};

// Slot and position of a row; position -1: no token there.
__device__ __forceinline__ int2 place(const Attn8Args& a, int row) {
    int2 p = make_int2(-1, -1);
    if (a.positions) {
        p = make_int2(a.slots[row], a.positions[row]);
    } else {
        for (int i = 0; i < a.n_segs; i++) {
            const int4 s = a.segs[i];
            if (row >= s.x && row < s.x + s.y) p = make_int2(s.z, s.w + row - s.x);
        }
    }
    if ((unsigned)p.x >= (unsigned)a.t.n_slots || (unsigned)p.y >= (unsigned)a.t.max_pages * PAGE) p.y = -1;
    return p;
}

__device__ __forceinline__ float code_value(uint8_t c) { return e4m3x2_to_f2(c).x; }

// Keys in tiles of 128: a thread scores one key, the softmax statistics are merged across the CTA, then the threads own value columns.
__global__ void __launch_bounds__(128) attn8_row_kernel(const __grid_constant__ Attn8Args a) {
    __shared__ float sq[128], sp[128], red[2][4];
    const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hd = a.c.hd, g = h / (a.n_heads / a.c.kv_heads);
    pdl_launch();
    pdl_wait();
    const int2 at = place(a, row);
    const size_t pi = (size_t)row * a.n_heads + h;
    if (at.y < 0) {
        if (tid == 0) a.part_ml[pi] = make_float2(0.f, -1.f);
        return;
    }
    const int pos = at.y;
    if (tid < hd) sq[tid] = a.q[pi * hd + tid];
    __syncthreads();
    const int lo = first_key(pos, a.chunk, a.window), kept = min(a.window > 0 ? a.keep : 0, lo);
    float acc = 0.f, m = -INFINITY, l = 0.f;
    for (int k0 = kept > 0 ? 0 : lo; k0 <= pos; k0 = k0 < kept && k0 + 128 >= kept ? lo : k0 + 128) {
        const int kp = k0 + tid, last = k0 < kept ? kept - 1 : pos, n = min(128, last - k0 + 1);
        float s = -INFINITY;
        if (kp <= last) {
            const int page = max(page_at(a.t, a.c.n_pages, at.x, kp >> PAGE_SHIFT), 0);
            const size_t head = (size_t)page * a.c.kv_heads + g;
            const uint8_t* kr = a.c.k + (head * PAGE + (kp & (PAGE - 1))) * hd;
            float d = 0.f;
            for (int i = 0; i < hd; i++) d = fmaf(sq[i], code_value(kr[i]), d);
            s = d * a.c.ku[head] * a.scale;
            if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
        }
        float mx = warp_max(s);
        if (lane == 0) red[0][warp] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
        const float mn = fmaxf(m, mx), corr = expf(m - mn), p = expf(s - mn), ps = warp_sum(p);
        sp[tid] = p;
        if (lane == 0) red[1][warp] = ps;
        __syncthreads();
        l = l * corr + red[1][0] + red[1][1] + red[1][2] + red[1][3];
        m = mn;
        acc *= corr;
        for (int i = 0; i < n; i++) {
            const int page = max(page_at(a.t, a.c.n_pages, at.x, (k0 + i) >> PAGE_SHIFT), 0);
            const size_t head = (size_t)page * a.c.kv_heads + g;
            if (tid < hd) acc = fmaf(sp[i] * a.c.vu[head], code_value(a.c.v[(head * PAGE + ((k0 + i) & (PAGE - 1))) * hd + tid]), acc);
        }
        __syncthreads();
    }
    if (tid < hd) a.part_acc[pi * hd + tid] = acc;
    if (tid == 0) a.part_ml[pi] = make_float2(m, l);
}

// Splits of head h merged at column d; false: the row holds no token.
__device__ __forceinline__ bool merged(const Attn8Args& a, int row, int h, int d, float& v) {
    const size_t p0 = ((size_t)row * a.n_heads + h) * a.n_splits;
    if (a.part_ml[p0].y < 0.f) return false;
    float top = -INFINITY, o = 0.f, l = 0.f;
    for (int s = 0; s < a.n_splits; s++) top = fmaxf(top, a.part_ml[p0 + s].x);
    for (int s = 0; s < a.n_splits; s++) {
        const float2 ml = a.part_ml[p0 + s];
        if (ml.y == 0.f) continue;      // saw no key, its sums were not written
        const float w = __expf(ml.x - top);
        l = fmaf(ml.y, w, l);
        if (d < a.c.hd) o = fmaf(a.part_acc[(p0 + s) * a.c.hd + d], w, o);
    }
    v = o / l;
    return true;
}

// 128 threads, with two maps of a head 256: a half each.
__global__ void __launch_bounds__(256) attn8_merge_kernel(const __grid_constant__ Attn8Args a) {
    const int h = blockIdx.x, row = blockIdx.y, d = threadIdx.x & 127;
    pdl_launch();
    pdl_wait();
    float v = 0.f;
    if (a.diff.on) {
        __shared__ float red[4], second[128];
        const int map = threadIdx.x >> 7;
        if (!merged(a, row, 2 * h + map, d, v)) return;
        if (d >= a.vdim) v = 0.f;
        if (map) second[d] = v;
        __syncthreads();
        v -= a.diff.lambda * second[d];
        if (map) v = 0.f;
        const float s = warp_sum(v * v);
        if (!map && (d & 31) == 0) red[d >> 5] = s;
        __syncthreads();
        if (map) return;
        v *= a.diff.scale / sqrtf((red[0] + red[1] + red[2] + red[3]) / (float)a.vdim + a.diff.eps);
    } else if (!merged(a, row, h, d, v)) {
        return;
    }
    if (d >= a.vdim) return;
    if (a.gate.kind) v *= sigmoid_f(a.gate.g[(size_t)row * a.gate.ld + (a.gate.kind == 1 ? h * a.vdim + d : h)]);
    const size_t oi = (size_t)row * a.ldo + (size_t)h * a.vdim + d;
    if (a.out16) ((__nv_bfloat16*)a.out)[oi] = __float2bfloat16_rn(v);
    else ((float*)a.out)[oi] = v;
}

bool bad_args(const Attn8Args& a) {
    return !a.q || !a.c.k || !a.c.v || !a.c.ku || !a.c.vu || a.c.n_pages < 1 || (a.c.hd != 64 && a.c.hd != 128) || a.c.kv_heads < 1 || a.n_heads < 1 || a.n_heads % a.c.kv_heads ||
           a.n_heads > 65535 || a.rows < 1 || a.rows > 65535 || a.vdim < 1 || a.vdim > a.c.hd || !a.t.table || a.t.n_slots < 1 || a.t.max_pages < 1 || a.t.max_pages > (1 << 25) ||
           (!a.positions == !a.segs) || (a.positions && !a.slots) || (a.segs && a.n_segs < 1) || a.chunk < 0 || a.window < 0 || a.keep < 0 || (a.chunk && a.window) || a.softcap < 0.f ||
           a.n_splits < 1 || !a.part_acc || !a.part_ml || !a.out || a.gate.kind < 0 || a.gate.kind > 2 || (a.gate.kind && !a.gate.g) ||
           (a.diff.on && (a.n_heads / a.c.kv_heads & 1)) || a.ldo < (a.diff.on ? a.n_heads / 2 : a.n_heads) * a.vdim ||
           (((uintptr_t)a.c.k | (uintptr_t)a.c.v | (uintptr_t)a.q | (uintptr_t)a.part_acc) & 15);
}

}  // namespace

// Attention of rows of queries.  Returns a cudaError_t value.
B2_API int b2_attn8(const Attn8Args* in, int pdl, cudaStream_t st) {
    if (!in || bad_args(*in) || in->n_splits != 1) return (int)cudaErrorInvalidValue;
    Attn8Args a = *in;
    void* args[] = {&a};
    const int rc = launch_rows((const void*)attn8_row_kernel, dim3(a.rows, a.n_heads), dim3(128), 0, args, st, pdl);
    if (rc) return rc;
    return launch_rows((const void*)attn8_merge_kernel, dim3(a.diff.on ? a.n_heads / 2 : a.n_heads, a.rows), dim3(a.diff.on ? 256 : 128), 0, args, st, pdl);
}
