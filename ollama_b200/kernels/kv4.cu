// Rows into the 4-bit cache (kv4.cuh) and back.
//
// b2_append4: norm of the query and key heads, rotation, queries out, keys and values as codes.  A warp takes a head of a token: 128 or 64 columns in its lanes' registers, so the norm's sum and a
// block's extremes are shuffles, and pairs of columns that another lane has are read from a row of shared memory.  Bound by the projections' bytes (fp32 in).
// b2_read4: rows as f16 values, a lane a word of eight codes.
#include "kv4.cuh"

namespace {

constexpr int WARPS = 8;

template <int HD>
__device__ __forceinline__ void load_head(float (&x)[HD / 32], const float* at, int lane, bool wide) {
    constexpr int N = HD / 32;
    if (wide) {
        if constexpr (N == 4) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(at) + lane);
            x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
        } else {
            const float2 v = __ldcg(reinterpret_cast<const float2*>(at) + lane);
            x[0] = v.x; x[1] = v.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; j++) x[j] = __ldcg(at + N * lane + j);
    }
}

// grid (rows, parts of the heads), 8 warps; a warp takes heads first + warp, + 8, ... of its part
template <int HD>
__global__ void __launch_bounds__(WARPS * 32) append4_kernel(const __grid_constant__ Append4Args a, int per, int wide) {
    constexpr int N = HD / 32;
    __shared__ float s_cs[HD / 2], s_sn[HD / 2];
    __shared__ __align__(16) float s_row[WARPS][HD];
    const int t = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Rows4& r = a.r;
    const int H = r.n_heads, G = a.c.kv_heads, all = H + 2 * G, end = min(all, (int)(blockIdx.y + 1) * per);
    pdl_launch();
    pdl_wait();
    const int pos = r.positions[t], slot = r.slots[t];
    if (!kv4::has_row(a.c, pos, slot)) return;
    const float* src = r.qkv + (size_t)t * r.ldq;
    int h = blockIdx.y * per + warp;
    float next[N];
    if (h < end) load_head<HD>(next, src + (size_t)h * HD, lane, wide);
    kv4::fill_angles(r, pos, s_cs, s_sn, tid, WARPS * 32);
    __syncthreads();
    const kv4::Turn<HD> turn = kv4::make_turn<HD>(r, s_cs, s_sn, lane);
    for (; h < end; h += WARPS) {
        float x[N];
#pragma unroll
        for (int j = 0; j < N; j++) x[j] = next[j];
        if (h + WARPS < end) load_head<HD>(next, src + (size_t)(h + WARPS) * HD, lane, wide);
        const bool is_q = h < H, is_k = !is_q && h < H + G;
        if (is_q && !a.q_out) continue;
        kv4::prepare_head<HD>(x, is_q ? r.q_norm : is_k ? r.k_norm : nullptr, r.eps, is_q || is_k, turn, s_row[warp], lane);
        if (is_q) {
            const size_t at = ((size_t)t * H + h) * HD + N * lane;
            if (a.q16) {
                uint32_t p[N / 2];
#pragma unroll
                for (int j = 0; j < N; j += 2) {
                    const __half2 y = __floats2half2_rn(x[j], x[j + 1]);
                    p[j / 2] = *reinterpret_cast<const uint32_t*>(&y);
                }
                if constexpr (N == 4) *reinterpret_cast<uint2*>((__half*)a.q_out + at) = make_uint2(p[0], p[1]);
                else *reinterpret_cast<uint32_t*>((__half*)a.q_out + at) = p[0];
            } else {
                if constexpr (N == 4) *reinterpret_cast<float4*>((float*)a.q_out + at) = make_float4(x[0], x[1], x[2], x[3]);
                else *reinterpret_cast<float2*>((float*)a.q_out + at) = make_float2(x[0], x[1]);
            }
        } else {
            const size_t row = kv4::row_of(a.c, pos, slot, is_k ? h - H : h - H - G);
            const kv4::Coded<HD> y = kv4::encode<HD>(x, lane);
            if (y.lead) reinterpret_cast<uint32_t*>(is_k ? a.c.k : a.c.v)[row * (HD / 8) + y.at] = y.word;
            if (y.first) reinterpret_cast<__half*>(is_k ? a.c.ks : a.c.vs)[row * (HD / 32) + y.block] = y.d;
        }
    }
}

// A thread takes a word of keys or values: HD / 8 words of each for a row and KV head.
template <int HD>
__global__ void __launch_bounds__(256) read4_kernel(const __grid_constant__ Read4Args a) {
    constexpr int W = HD / 8, NB = HD / 32;
    pdl_launch();
    pdl_wait();
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const int w = (int)(i % W), is_v = (int)(i / W) & 1;
    const long long unit = i / (2 * W);
    const int kvh = (int)(unit % a.c.kv_heads);
    const long long t = unit / a.c.kv_heads;
    if (t >= a.rows) return;
    const int pos = a.positions[t], slot = a.slots[t];
    if (!kv4::has_row(a.c, pos, slot)) return;
    const size_t row = kv4::row_of(a.c, pos, slot, kvh);
    const int b = w % NB, j = w / NB;
    uint32_t e[4];
    kv4::expand(reinterpret_cast<const uint32_t*>(is_v ? a.c.v : a.c.k)[row * W + w], e);
    const __half2 d = __half2half2(reinterpret_cast<const __half*>(is_v ? a.c.vs : a.c.ks)[row * NB + b]);
    const uint32_t dd = *reinterpret_cast<const uint32_t*>(&d);
#pragma unroll
    for (int p = 0; p < 4; p++) e[p] = kv4::hmul2_bits(e[p], dd);
    *reinterpret_cast<uint4*>((__half*)(is_v ? a.v_out : a.k_out) + ((size_t)t * a.c.kv_heads + kvh) * HD + 32 * b + 8 * j) = make_uint4(e[0], e[1], e[2], e[3]);
}

bool bad_cache(const Cache4& c) {
    return !c.k || !c.v || !c.ks || !c.vs || c.slots < 1 || c.kv_heads < 1 || c.n_ctx < 1 || (c.hd != 64 && c.hd != 128) || (((uintptr_t)c.k | (uintptr_t)c.v) & 15) || (((uintptr_t)c.ks | (uintptr_t)c.vs) & 7);
}
bool bad_rows(const Rows4& r, const Cache4& c) {
    return !r.qkv || r.rows < 0 || r.n_heads < 1 || r.n_heads % c.kv_heads || r.ldq < (r.n_heads + 2 * c.kv_heads) * c.hd || !r.positions || !r.slots || r.n_rot < 0 || r.n_rot > c.hd || (r.n_rot & 1) ||
           (r.n_rot && !r.inv_freq);
}

}  // namespace

B2_API unsigned long long b2_kv4_layout() { return KV4_LAYOUT; }

bool kv4_bad_cache(const Cache4& c) { return bad_cache(c); }
bool kv4_bad_rows(const Rows4& r, const Cache4& c) { return bad_rows(r, c); }
// Whether a head's columns can be loaded as whole vectors.
bool kv4_wide_rows(const Rows4& r) { return ((uintptr_t)r.qkv & 15) == 0 && (r.ldq & 3) == 0; }

B2_API int b2_append4(const Append4Args* in, int pdl, cudaStream_t st) {
    Append4Args a = *in;
    if (bad_cache(a.c) || bad_rows(a.r, a.c)) return (int)cudaErrorInvalidValue;
    if (!a.r.rows) return 0;
    const int all = a.r.n_heads + 2 * a.c.kv_heads;
    int per = a.r.rows > 64 ? all : WARPS;
    int wide = kv4_wide_rows(a.r);
    void* args[] = {&a, &per, &wide};
    return launch_rows(a.c.hd == 128 ? (const void*)append4_kernel<128> : (const void*)append4_kernel<64>, dim3(a.r.rows, (all + per - 1) / per), dim3(WARPS * 32), 0, args, st, pdl);
}

B2_API int b2_read4(const Read4Args* in, int pdl, cudaStream_t st) {
    Read4Args a = *in;
    if (bad_cache(a.c) || a.rows < 0 || (a.rows && (!a.positions || !a.slots || !a.k_out || !a.v_out || (((uintptr_t)a.k_out | (uintptr_t)a.v_out) & 15)))) return (int)cudaErrorInvalidValue;
    if (!a.rows) return 0;
    const long long threads = (long long)a.rows * a.c.kv_heads * (a.c.hd / 4), blocks = (threads + 255) / 256;
    if (blocks > 0x7fffffffll) return (int)cudaErrorInvalidValue;
    void* args[] = {&a};
    return launch_rows(a.c.hd == 128 ? (const void*)read4_kernel<128> : (const void*)read4_kernel<64>, dim3((unsigned)blocks), dim3(256), 0, args, st, pdl);
}
