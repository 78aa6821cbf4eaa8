// Rows into an 8-bit paged cache and pages out of it (layout: pages8.cuh).
#include "pages8.cuh"

namespace {

constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int PAGE_WARPS = 16;               // of a CTA that appends many rows of a page
constexpr int COLS = 4;                      // columns of a head row that a lane holds

// Column i of a lane: with VEC four neighbours, so that a head row is one 16-byte load a lane, else every 32nd.
template <bool VEC>
__device__ __forceinline__ int col(int lane, int i) { return VEC ? 4 * lane + i : lane + 32 * i; }

template <bool VEC>
__device__ __forceinline__ void load_head(const float* p, int n, int lane, float (&x)[COLS]) {
    if (VEC) {
        const float4 v = 4 * lane < n ? __ldcg((const float4*)p + lane) : make_float4(0.f, 0.f, 0.f, 0.f);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
#pragma unroll
        for (int i = 0; i < COLS; i++) x[i] = lane + 32 * i < n ? p[lane + 32 * i] : 0.f;
    }
}

// x *= inv * w
template <bool VEC>
__device__ __forceinline__ void weigh(float (&x)[COLS], float inv, const float* w, int n, int lane) {
    if (VEC) {
        if (4 * lane < n) {
            const float4 v = __ldg((const float4*)w + lane);
            x[0] *= inv * v.x; x[1] *= inv * v.y; x[2] *= inv * v.z; x[3] *= inv * v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < COLS; i++)
            if (lane + 32 * i < n) x[i] *= inv * __ldg(w + lane + 32 * i);
    }
}

__device__ __forceinline__ float square_sum(const float (&x)[COLS]) { return x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3]; }

// Rotation of head rows in the half-split order (of both maps' halves of a row that has two): x = c x + s y, y the other one of a column's pair.
template <bool VEC>
struct Turn {
    float c[COLS], s[COLS];
    int other[VEC ? 1 : COLS];               // where y is: a lane (whose columns turn with this lane's), or columns

    // cs / sn: cosines and sines of the row's pairs; n: columns of the head row, of maps of dim columns
    __device__ __forceinline__ Turn(int lane, int n, int dim, int n_rot, const float* cs, const float* sn) {
        const int half = n_rot >> 1;
        if (VEC) {          // half and dim are multiples of four
            const int d = 4 * lane, in = d >= dim ? d - dim : d;
            const bool first = in < half;
            float4 co = make_float4(1.f, 1.f, 1.f, 1.f), si = make_float4(0.f, 0.f, 0.f, 0.f);
            other[0] = lane;
            if (in < n_rot && d < n) {
                co = *(const float4*)(cs + (first ? in : in - half));
                si = *(const float4*)(sn + (first ? in : in - half));
                other[0] = first ? lane + (half >> 2) : lane - (half >> 2);
            }
            const float sign = first ? -1.f : 1.f;
            c[0] = co.x; c[1] = co.y; c[2] = co.z; c[3] = co.w;
            s[0] = sign * si.x; s[1] = sign * si.y; s[2] = sign * si.z; s[3] = sign * si.w;
        } else {
#pragma unroll
            for (int i = 0; i < COLS; i++) {
                const int d = lane + 32 * i, in = d >= dim ? d - dim : d;
                const bool first = in < half, turns = in < n_rot && d < n;
                c[i] = turns ? cs[first ? in : in - half] : 1.f;
                s[i] = turns ? (first ? -sn[in] : sn[in - half]) : 0.f;
                other[VEC ? 0 : i] = turns ? (first ? d + half : d - half) : d;
            }
        }
    }
    __device__ __forceinline__ void operator()(float (&x)[COLS]) const {
        float y[COLS];
#pragma unroll
        for (int i = 0; i < COLS; i++) {
            if (VEC) {
                y[i] = __shfl_sync(0xffffffffu, x[i], other[0]);
            } else {
                const int o = other[VEC ? 0 : i];
#pragma unroll
                for (int j = 0; j < COLS; j++) {
                    const float v = __shfl_sync(0xffffffffu, x[j], o & 31);
                    if (o >> 5 == j) y[i] = v;
                }
            }
        }
        // a column that does not turn is not multiplied with another one, which may be infinite
#pragma unroll
        for (int i = 0; i < COLS; i++) x[i] = s[i] == 0.f ? x[i] * c[i] : fmaf(x[i], c[i], y[i] * s[i]);
    }
};

// A lane's codes of a head row.
template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t* row, int lane, int hd, const float (&x)[COLS], float inv) {
    const uint32_t lo = to_e4m3x2(x[0] * inv, x[1] * inv), hi = to_e4m3x2(x[2] * inv, x[3] * inv);
    if (VEC) {
        if (4 * lane < hd) ((uint32_t*)row)[lane] = lo | hi << 16;
    } else {
        const uint32_t w = lo | hi << 16;
#pragma unroll
        for (int i = 0; i < COLS; i++)
            if (lane + 32 * i < hd) row[lane + 32 * i] = (uint8_t)(w >> 8 * i);
    }
}

__device__ __forceinline__ uint32_t rescaled(uint32_t two, float f) {
    const float2 v = e4m3x2_to_f2(two);
    return to_e4m3x2(v.x * f, v.y * f);
}

// The codes of a page's head but those of rows [lo, hi), in a unit that is 1 / f of theirs.
template <int W>
__device__ void rescale_page(uint8_t* page, int hd, int lo, int hi, float f) {
    for (int c = threadIdx.x; c < PAGE * hd / 16; c += 32 * W) {
        const int r = c / (hd / 16);
        if (r >= lo && r < hi) continue;
        uint4 w = ((const uint4*)page)[c];
        uint32_t* x = &w.x;
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = rescaled(x[i], f) | rescaled(x[i] >> 16, f) << 16;
        ((uint4*)page)[c] = w;
    }
}

template <int W>
__device__ __forceinline__ float block_max(float v, float* red) {
    v = warp_max(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float m = red[0];
#pragma unroll
    for (int i = 1; i < W; i++) m = fmaxf(m, red[i]);
    return m;
}

__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ float peer_value(const float* p, int rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at));
    return v;
}

// Rows [row, row + n) at positions [pos, pos + n), all in one page, of KV head g.  PEERS: the CTAs of the cluster have a page's KV heads, and a norm over the whole row takes each
// head's sum from its CTA.
template <bool VEC, bool PEERS, int W>
__device__ void append_to_page(const Append8Args& a, int row, int n, int slot, int pos, int g, float* cs, float* red) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int half = a.n_rot >> 1, pitch = (half + 3) & ~3, kdim = a.maps * a.dim, G = a.c.kv_heads, hd = a.c.hd;
    const int nq = a.n_heads * a.dim, nk = G * kdim, off = pos & (PAGE - 1);
    float* sn = cs + (a.positions ? 1 : PAGE) * pitch;      // as many rows as the launch has shared memory for
    float k[PAGE / W][COLS], v[PAGE / W][COLS];
#pragma unroll
    for (int i = 0; i < PAGE / W; i++) {
        const int r = warp + W * i;
        if (r < n) {
            const float* p = a.qkv + (size_t)(row + r) * a.ldq;
            load_head<VEC>(p + nq + g * kdim, kdim, lane, k[i]);
            load_head<VEC>(p + a.v_off + g * a.vdim, a.vdim, lane, v[i]);
        } else if (PEERS) {
#pragma unroll
            for (int j = 0; j < COLS; j++) k[i][j] = 0.f;
        }
    }
    const int page = page_at(a.t, a.c.n_pages, slot, pos >> PAGE_SHIFT);
    if (page < 0) return;
    const size_t head = (size_t)page * G + g;
    const float old_k = a.c.ku[head], old_v = a.c.vu[head];
    __syncthreads();      // the tables may still be read for the rows before
    if (n == 1) {
        for (int p = tid; p < half; p += 32 * W) {
            float si, co;
            sincosf(rot_angle(pos, a.freqs[p]), &si, &co);
            cs[p] = co * a.mscale;
            sn[p] = si * a.mscale;
        }
    } else if (half > 0) {
        // Row 8 i + j turns by the angle of row j and that of 8 i positions more: 16 angles a pair instead of 64 (half <= 64).  The products of their cosines
        // and sines are off by some 2^-23, the codes by up to 2^-4.
        constexpr int PARTS = W / 2, EACH = 16 / PARTS;
        const int p = tid & 63, part = tid >> 6;
        float* step = sn + PAGE * pitch;      // [16][2][pitch]: rows 0 .. 7, then 0, 8 .. 56 positions
        if (p < half) {
            const double f = a.freqs[p];
#pragma unroll
            for (int i = 0; i < EACH; i++) {
                const int e = EACH * part + i;
                float si, co;
                sincosf(rot_angle(e < 8 ? pos + e : 8 * (e - 8), f), &si, &co);
                step[2 * e * pitch + p] = e < 8 ? co * a.mscale : co;
                step[(2 * e + 1) * pitch + p] = e < 8 ? si * a.mscale : si;
            }
        }
        __syncthreads();
        if (p < half)
            for (int r = part; r < n; r += PARTS) {
                const float c0 = step[2 * (r & 7) * pitch + p], s0 = step[(2 * (r & 7) + 1) * pitch + p], c1 = step[2 * (8 + (r >> 3)) * pitch + p], s1 = step[(2 * (8 + (r >> 3)) + 1) * pitch + p];
                cs[r * pitch + p] = c0 * c1 - s0 * s1;
                sn[r * pitch + p] = s0 * c1 + c0 * s1;
            }
    }
    __syncthreads();
    __shared__ float own[PAGE];              // PEERS: sums of the head's rows
    const bool whole = PEERS && a.k_norm && !a.head_norm;
    if (whole) {
#pragma unroll
        for (int i = 0; i < PAGE / W; i++) {
            const float sum = warp_sum(square_sum(k[i]));      // rows behind the last one hold nothing that is used
            if (lane == 0) own[warp + W * i] = sum;
        }
        cluster_sync();
    }
    const float per_column = 1.f / (float)(a.head_norm ? a.dim : nk);
    float top_k = 0.f, top_v = 0.f;
#pragma unroll
    for (int i = 0; i < PAGE / W; i++) {
        const int r = warp + W * i;
        if (r < n) {
            if (a.k_norm) {
                float s;
                if (a.head_norm) {
                    s = square_sum(k[i]);
                } else if (PEERS) {
                    s = lane < G ? peer_value(own + r, lane) : 0.f;
                } else {
                    const float* p = a.qkv + (size_t)(row + r) * a.ldq + nq;
                    s = 0.f;
                    for (int c = 0; c < nk; c += 128) {
                        float x[COLS];
                        load_head<VEC>(p + c, nk - c, lane, x);
                        s += square_sum(x);
                    }
                }
                weigh<VEC>(k[i], rsqrtf(warp_sum(s) * per_column + a.eps), a.k_norm + (a.head_norm ? 0 : g * kdim), kdim, lane);
            }
            if (half > 0) Turn<VEC>(lane, kdim, a.dim, a.n_rot, cs + r * pitch, sn + r * pitch)(k[i]);
#pragma unroll
            for (int j = 0; j < COLS; j++) {
                top_k = fmaxf(top_k, fabsf(k[i][j]));
                top_v = fmaxf(top_v, fabsf(v[i][j]));
            }
        }
    }
    float unit_k = unit_for(block_max<W>(top_k, red)), unit_v = unit_for(block_max<W>(top_v, red));
    uint8_t *kp = a.c.k + head * PAGE * hd, *vp = a.c.v + head * PAGE * hd;
    if (off > 0) {        // positions before these stay: the page's unit does not shrink
        unit_k = fmaxf(unit_k, old_k);
        unit_v = fmaxf(unit_v, old_v);
    }
    if (unit_k > old_k && n < PAGE) rescale_page<W>(kp, hd, off, off + n, old_k / unit_k);
    if (unit_v > old_v && n < PAGE) rescale_page<W>(vp, hd, off, off + n, old_v / unit_v);
    if (tid == 0) {
        a.c.ku[head] = unit_k;
        a.c.vu[head] = unit_v;
    }
    const float ik = 1.f / unit_k, iv = 1.f / unit_v;
#pragma unroll
    for (int i = 0; i < PAGE / W; i++) {
        const int r = warp + W * i;
        if (r < n) {
            store_codes<VEC>(kp + (off + r) * hd, lane, hd, k[i], ik);
            store_codes<VEC>(vp + (off + r) * hd, lane, hd, v[i], iv);
        }
    }
    if (whole) cluster_sync();               // a peer may still read this CTA's sums
}

// Queries of one row, a warp a head; of the first HELD heads of a warp the values stay in registers between a norm over the row and the rotation.
constexpr int HELD = 4;
template <bool VEC>
__device__ __forceinline__ void query_head(const Append8Args& a, int row, int h, float (&x)[COLS], float inv, float per_column, const Turn<VEC>& turn) {
    const int lane = threadIdx.x & 31, hd = a.c.hd;
    if (a.q_norm) {
        if (a.head_norm) inv = rsqrtf(warp_sum(square_sum(x)) * per_column + a.eps);
        weigh<VEC>(x, inv, a.q_norm + (a.head_norm ? 0 : h * a.dim), a.dim, lane);
    }
    if (a.n_rot > 0) turn(x);
    // a map's query stands in the map's columns of an otherwise empty row
    float* q = a.q_out + ((size_t)row * a.n_heads + h) * hd;
    if (VEC && a.maps == 1) {
        if (4 * lane < hd) ((float4*)q)[lane] = make_float4(x[0], x[1], x[2], x[3]);
    } else {
        const int at = a.maps > 1 && h & 1 ? a.dim : 0;
#pragma unroll
        for (int j = 0; j < COLS; j++) {
            const int d = col<VEC>(lane, j);
            if (d < a.dim) q[at + d] = x[j];
        }
        for (int d = lane; d < hd; d += 32)
            if (d < at || d >= at + a.dim) q[d] = 0.f;
    }
}
template <bool VEC>
__device__ __forceinline__ void load_heads(const Append8Args& a, int row, float (&x)[HELD][COLS]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float* p = a.qkv + (size_t)row * a.ldq;
#pragma unroll
    for (int i = 0; i < HELD; i++)
        if (warp + WARPS * i < a.n_heads) load_head<VEC>(p + (warp + WARPS * i) * a.dim, a.dim, lane, x[i]);
}
// x: load_heads of the row
template <bool VEC>
__device__ __forceinline__ void query_row(const Append8Args& a, int row, int pos, float (&x)[HELD][COLS], float* cs, float* red) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, half = a.n_rot >> 1, pitch = (half + 3) & ~3, nq = a.n_heads * a.dim;
    float* sn = cs + pitch;
    const float* p = a.qkv + (size_t)row * a.ldq;
    for (int i = tid; i < half; i += THREADS) {
        float s, c;
        sincosf(rot_angle(pos, a.freqs[i]), &s, &c);
        cs[i] = c * a.mscale;
        sn[i] = s * a.mscale;
    }
    float inv = 1.f;
    if (a.q_norm && !a.head_norm) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < HELD; i++)
            if (warp + WARPS * i < a.n_heads) s += square_sum(x[i]);
        for (int h = warp + WARPS * HELD; h < a.n_heads; h += WARPS) {
            float y[COLS];
            load_head<VEC>(p + h * a.dim, a.dim, lane, y);
            s += square_sum(y);
        }
        s = warp_sum(s);
        if (lane == 0) red[warp] = s;
        __syncthreads();
        s = 0.f;
#pragma unroll
        for (int i = 0; i < WARPS; i++) s += red[i];
        inv = rsqrtf(s / (float)nq + a.eps);
    } else {
        __syncthreads();
    }
    const float per_column = 1.f / (float)a.dim;
    const Turn<VEC> turn(lane, a.dim, a.dim, a.n_rot, cs, sn);
#pragma unroll
    for (int i = 0; i < HELD; i++)
        if (warp + WARPS * i < a.n_heads) query_head<VEC>(a, row, warp + WARPS * i, x[i], inv, per_column, turn);
    for (int h = warp + WARPS * HELD; h < a.n_heads; h += WARPS) {
        load_head<VEC>(p + h * a.dim, a.dim, lane, x[0]);
        query_head<VEC>(a, row, h, x[0], inv, per_column, turn);
    }
}

// Norm of q and k, rotation, q to padded fp32 rows; k and v become codes of the pages they go to, whose units grow so that the largest magnitude fits.  A page whose first
// position is among the rows begins anew.  Of single rows a CTA has a KV head of a row, and then one the queries of a row.
template <bool VEC>
__global__ void __launch_bounds__(THREADS, 4) append8_kernel(const __grid_constant__ Append8Args a) {
    extern __shared__ __align__(16) float cs[];
    __shared__ float red[WARPS];
    pdl_wait();
    pdl_launch();         // behind the wait: a kernel that starts now may read whatever was written before this one
    const int G = a.c.kv_heads, kv_ctas = a.no_append ? 0 : a.rows * G, b = blockIdx.x;
    if (b >= kv_ctas) {
        float x[HELD][COLS];
        load_heads<VEC>(a, b - kv_ctas, x);
        const int pos = a.positions[b - kv_ctas];
        if (!has(a.t, a.slots[b - kv_ctas], pos)) return;
        query_row<VEC>(a, b - kv_ctas, pos, x, cs, red);
        return;
    }
    // rows of one slot take their turns in one CTA: the first of them appends them all, in order
    const int g = b % G, u = b / G, slot = a.slots[u];
    uint32_t before = 0, behind = 0;      // every warp for itself
    for (int i = threadIdx.x & 31; i < ((a.rows + 31) & ~31); i += 32) {
        const bool same = i < a.rows && a.slots[i] == slot;
        before |= __ballot_sync(0xffffffffu, same && i < u);
        behind |= __ballot_sync(0xffffffffu, same && i > u);
    }
    if (before) return;
    for (int i = u; i < (behind ? a.rows : u + 1); i++) {
        if (a.slots[i] != slot || a.positions[i] < 0) continue;
        append_to_page<VEC, false, WARPS>(a, i, 1, slot, a.positions[i], g, cs, red);
        __syncthreads();      // what it wrote is read by the next one's rescaling
    }
}

// The same for portions of prompts, in two launches, since a page's rows stay in registers between the largest magnitude and the codes, and would leave the queries
// two CTAs an SM (2048 rows of 32 heads on 8: 49 us in one).  Keys and values: a KV head and a page of a portion each, 16 warps (eight: 2 us more).  Together 27.5 us, 88 MB at
// 3.2 TB/s: two waves of CTAs whose loads, norms, rotation and stores follow one another.
template <bool VEC, bool PEERS>
__global__ void __launch_bounds__(32 * PAGE_WARPS, 2) append8_pages_kernel(const __grid_constant__ Append8Args a) {
    extern __shared__ __align__(16) float cs[];
    __shared__ float red[PAGE_WARPS];
    pdl_wait();
    pdl_launch();
    const int G = a.c.kv_heads, g = blockIdx.x % G, j = blockIdx.x / G % a.per;
    const int4 s = a.segs[blockIdx.x / G / a.per];
    const int first = (s.w >> PAGE_SHIFT) + j, lo = max(s.w, first * PAGE), hi = min(s.w + s.y, (first + 1) * PAGE);
    if (s.w < 0 || s.x < 0 || s.x + s.y > a.rows || lo >= hi) return;
    append_to_page<VEC, PEERS, PAGE_WARPS>(a, s.x + lo - s.w, hi - lo, s.z, lo, g, cs, red);
}

// Queries: a row each.  `behind`: launched behind the keys and values, which it does not read, while they are under way.  Six CTAs an SM: 27.5 us instead of
// 28.7 with four.  (CTAs that take several rows and have the next one's values on their way were slower, 32.8 us where these took 31.1.)
template <bool VEC>
__global__ void __launch_bounds__(THREADS, VEC ? 6 : 4) append8_queries_kernel(const __grid_constant__ Append8Args a, int behind) {
    extern __shared__ __align__(16) float cs[];
    __shared__ float red[WARPS];
    pdl_launch();
    if (!behind) pdl_wait();
    float x[HELD][COLS];
    load_heads<VEC>(a, blockIdx.x, x);
    int pos = -1;
    for (int i = 0; i < a.n_segs; i++) {
        const int4 s = a.segs[i];
        if ((int)blockIdx.x >= s.x && (int)blockIdx.x < s.x + s.y && has(a.t, s.z, s.w + blockIdx.x - s.x)) pos = s.w + blockIdx.x - s.x;
    }
    if (pos >= 0) query_row<VEC>(a, blockIdx.x, pos, x, cs, red);
    if (behind) pdl_wait();      // the launch does not end before the one it follows
}

// Pages as f16 values.  list: (slot, page of the slot, rows that are wanted); the rows behind them, and pages that are not there, become zeros.  clean: for attention whose products
// take weights of zero times every value: a row of values that holds what is no number becomes zeros and its key none, so that only queries that see it have no result.
// A CTA a page and KV head: 8 + 8 KB in, 16 + 16 KB out for heads of 128.  A thread turns 8 codes into 16 bytes, so that a warp's stores are whole lines; all its loads are under way
// together (eight sequences of 3001 keys of 8 heads, 113 MB: 20.7 us, 5.5 TB/s; with sixteen codes a thread, a store for each half, 25.2).
template <int HD>
__global__ void __launch_bounds__(256) read8_kernel(const Pages8 c, const PageTable t, const int4* list, __half* k_out, __half* v_out, int clean) {
    constexpr int CHUNKS = HD / 8, EACH = PAGE * CHUNKS / 256;
    pdl_launch();
    pdl_wait();
    const int4 e = list[blockIdx.x];
    const int g = blockIdx.y, page = page_at(t, c.n_pages, e.x, e.y);
    const size_t head = (size_t)max(page, 0) * c.kv_heads + g, out = ((size_t)blockIdx.x * c.kv_heads + g) * PAGE * HD;
    const int rows = page < 0 ? 0 : e.z;
    uint2 w[2][EACH];
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const int at = threadIdx.x + 256 * i;
#pragma unroll
        for (int m = 0; m < 2; m++) w[m][i] = at / CHUNKS < rows ? __ldg((const uint2*)((m ? c.v : c.k) + head * PAGE * HD) + at) : make_uint2(0, 0);
    }
    const __half2 unit[2] = {__float2half2_rn(rows ? c.ku[head] : 0.f), __float2half2_rn(rows ? c.vu[head] : 0.f)};
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const int at = threadIdx.x + 256 * i;
        if (clean) {
            bool none = holds_nan(make_uint4(w[1][i].x, w[1][i].y, 0, 0));
#pragma unroll
            for (int o = 1; o < CHUNKS; o <<= 1) none |= __shfl_xor_sync(0xffffffffu, (int)none, o);
            if (none) {
                w[0][i] = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
                w[1][i] = make_uint2(0, 0);
            }
        }
#pragma unroll
        for (int m = 0; m < 2; m++) {
            const uint32_t x[2] = {w[m][i].x, w[m][i].y};
            uint32_t y[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t h = e4m3x2_to_h2(x[j >> 1] >> (j & 1) * 16);
                const __half2 f = __hmul2(*reinterpret_cast<const __half2*>(&h), unit[m]);
                y[j] = *reinterpret_cast<const uint32_t*>(&f);
            }
            ((uint4*)((m ? v_out : k_out) + out))[at] = at / CHUNKS < rows ? make_uint4(y[0], y[1], y[2], y[3]) : make_uint4(0, 0, 0, 0);
        }
    }
}

bool bad_cache(const Pages8& c, const PageTable& t) {
    return !c.k || !c.v || !c.ku || !c.vu || c.n_pages < 1 || c.kv_heads < 1 || c.kv_heads > 65535 || (c.hd != 64 && c.hd != 128) || !t.table || t.n_slots < 1 || t.max_pages < 1 ||
           (((uintptr_t)c.k | (uintptr_t)c.v) & 15);
}

}  // namespace

int append8_launch(const Append8Args& in, int pdl, cudaStream_t st) {
    const Append8Args* a = &in;
    if (bad_cache(a->c, a->t) || !a->qkv || !a->q_out || a->rows < 1 || a->n_heads < 1 || a->dim < 1 || a->vdim < 1 || a->maps < 1 || a->maps > 2 || a->n_heads % a->maps ||
        a->maps * a->dim > a->c.hd || a->vdim > a->c.hd || a->n_rot < 0 || a->n_rot > a->dim || (a->n_rot & 1) || (a->n_rot && !a->freqs) || (!a->q_norm != !a->k_norm) ||
        ((a->maps > 1 || a->no_append) && a->q_norm) || (!a->positions == !a->segs) || (a->positions && !a->slots) || (a->segs && a->n_segs < 1) || a->per < 1 || a->v_off < 0 ||
        a->ldq < a->n_heads * a->dim || ((uintptr_t)a->q_out & 15))
        return (int)cudaErrorInvalidValue;
    const int kdim = a->maps * a->dim, nq = a->n_heads * a->dim;
    if (!a->no_append && (a->ldq < nq + a->c.kv_heads * kdim || a->v_off + a->c.kv_heads * a->vdim > a->ldq)) return (int)cudaErrorInvalidValue;
    const long long ctas = a->no_append ? 0 : a->positions ? (long long)a->rows * a->c.kv_heads : (long long)a->n_segs * a->per * a->c.kv_heads;
    if (ctas + a->rows > 0x7fffffffll) return (int)cudaErrorInvalidValue;
    const bool vec = !((a->dim | a->vdim | a->ldq | a->v_off | (a->n_rot >> 1)) & 3) && !(((uintptr_t)a->qkv | (uintptr_t)a->q_norm | (uintptr_t)a->k_norm) & 15);
    const int pitch = ((a->n_rot >> 1) + 3) & ~3;
    const size_t one = 2 * sizeof(float) * (pitch ? pitch : 4);      // cosines and sines of a row
    Append8Args copy = *a;
    if (a->positions) {
        static thread_local PerDeviceOnce once;      // an SM that is set for less shared memory takes the CTAs of the attention behind this launch only when it is empty
        if (once.first()) {
            cudaFuncSetAttribute(append8_kernel<true>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
            cudaFuncSetAttribute(append8_kernel<false>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        }
        void* args[] = {&copy};
        return launch_rows(vec ? (const void*)append8_kernel<true> : (const void*)append8_kernel<false>, dim3((unsigned)(ctas + a->rows)), dim3(THREADS), one, args, st, pdl);
    }
    int behind = 0;
    if (ctas) {
        const bool peers = a->k_norm && !a->head_norm && a->c.kv_heads <= 8;      // clusters of as many CTAs
        const void* fn = peers ? (vec ? (const void*)append8_pages_kernel<true, true> : (const void*)append8_pages_kernel<false, true>)
                               : (vec ? (const void*)append8_pages_kernel<true, false> : (const void*)append8_pages_kernel<false, false>);
        void* args[] = {&copy};
        cudaLaunchAttribute at[2];
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)ctas);
        cfg.blockDim = dim3(32 * PAGE_WARPS);
        cfg.dynamicSmemBytes = (PAGE + 16) * one;
        cfg.stream = st;
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
        at[1].id = cudaLaunchAttributeClusterDimension;
        at[1].val.clusterDim.x = peers ? a->c.kv_heads : 1;
        at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 2;
        const int rc = (int)cudaLaunchKernelExC(&cfg, fn, args);
        if (rc) return rc;
        behind = 1;
    }
    void* args[] = {&copy, &behind};
    return launch_rows(vec ? (const void*)append8_queries_kernel<true> : (const void*)append8_queries_kernel<false>, dim3(a->rows), dim3(THREADS), one, args, st, pdl || behind);
}

// Which argument blocks this library takes.
B2_API unsigned long long b2_pages8_layout() { return PAGES8_LAYOUT; }

// Returns a cudaError_t value, as does the entry point below.
B2_API int b2_append8(const Append8Args* a, int pdl, cudaStream_t st) { return a ? append8_launch(*a, pdl, st) : (int)cudaErrorInvalidValue; }

B2_API int b2_read8(const Pages8* c, const PageTable* t, const int4* list, int n, __half* k_out, __half* v_out, int clean, int pdl, cudaStream_t st) {
    if (!c || !t || bad_cache(*c, *t) || !list || !k_out || !v_out || n < 1 || ((uintptr_t)list & 15) || (((uintptr_t)k_out | (uintptr_t)v_out) & 15)) return (int)cudaErrorInvalidValue;
    Pages8 cc = *c;
    PageTable tt = *t;
    void* args[] = {&cc, &tt, &list, &k_out, &v_out, &clean};
    return launch_rows(c->hd == 128 ? (const void*)read8_kernel<128> : (const void*)read8_kernel<64>, dim3(n, c->kv_heads), dim3(256), 0, args, st, pdl);
}
