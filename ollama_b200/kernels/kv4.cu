// Rows into the 4-bit cache (kv4.cuh) and back.
//
// b2_append4: norm of the query and key heads, rotation, queries out, keys and values as codes.  A warp takes a head of a token at a time, 128 or 64 columns in its lanes' registers, so the norm's
// sum and the other columns of pairs are shuffles.  Keys and values then stand in shared memory, where a thread takes eight columns and makes a word: with a head a warp (four columns a lane) the
// extremes of a block took three rounds of shuffles and the words two, and 2048 rows of 48 heads 29 us for what takes 20 here; their 76 MB take 12.  What is left: three waves of CTAs, each a chain
// of position, angles and heads, that issue in 65% of their cycles (five CTAs of eight warps an SM with two heads asked for ahead; four with four 21.1, three 22.6; ten CTAs of four warps 22.1).
// b2_read4: rows as f16 values, a lane a word of eight codes.
#include "kv4.cuh"

namespace {

constexpr int WARPS = 8, AHEAD = 2;      // query heads that a warp asks for at once

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

// grid (rows, parts of the heads), 8 warps; a part is `per` heads, of which the warps take one after the other
template <int HD>
__global__ void __launch_bounds__(WARPS * 32, 5) append4_kernel(const __grid_constant__ Append4Args a, int per, int wide) {
    constexpr int N = HD / 32, W = HD / 8, MANY = 2 * WARPS;      // keys and values that are coded together
    __shared__ float s_cs[HD / 2], s_sn[HD / 2];
    __shared__ __align__(16) float s_row[MANY][HD];
    const int t = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Rows4& r = a.r;
    const int H = r.n_heads, G = a.c.kv_heads, h0 = blockIdx.y * per, end = min(H + 2 * G, h0 + per), q_end = min(H, end), kv0 = max(H, h0);
    pdl_launch();
    pdl_wait();
    const int pos = r.positions[t], slot = r.slots[t];
    const float* src = r.qkv + (size_t)t * r.ldq;
    float q[AHEAD][N], kv[2][N];
    auto load_q = [&](int first) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (first + warp + i * WARPS < q_end) load_head<HD>(q[i], src + (size_t)(first + warp + i * WARPS) * HD, lane, wide);
    };
    load_q(h0);
    auto load_kv = [&](int first) {
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (first + warp + i * WARPS < end) load_head<HD>(kv[i], src + (size_t)(first + warp + i * WARPS) * HD, lane, wide);
    };
    load_kv(kv0);
    if (!kv4::has_row(a.c, pos, slot)) return;
    kv4::fill_angles(r, pos, s_cs, s_sn, tid, WARPS * 32);
    __syncthreads();
    const kv4::Turn<HD> turn = kv4::make_turn<HD>(r, s_cs, s_sn, lane);
    if (a.q_out)
        for (int first = h0; first < q_end; first += AHEAD * WARPS) {
            if (first > h0) load_q(first);
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const int h = first + warp + i * WARPS;
                if (h >= q_end) break;
                float (&x)[N] = q[i];
                kv4::prepare_head<HD>(x, r.q_norm, r.eps, true, turn, s_row[warp], lane);
                const size_t at = ((size_t)t * H + h) * HD + N * lane;
                if (a.q16) {
                    uint32_t p[N / 2];
#pragma unroll
                    for (int j = 0; j < N; j += 2) {
                        const __half2 z = __floats2half2_rn(x[j], x[j + 1]);
                        p[j / 2] = *reinterpret_cast<const uint32_t*>(&z);
                    }
                    if constexpr (N == 4) *reinterpret_cast<uint2*>((__half*)a.q_out + at) = make_uint2(p[0], p[1]);
                    else *reinterpret_cast<uint32_t*>((__half*)a.q_out + at) = p[0];
                } else {
                    if constexpr (N == 4) *reinterpret_cast<float4*>((float*)a.q_out + at) = make_float4(x[0], x[1], x[2], x[3]);
                    else *reinterpret_cast<float2*>((float*)a.q_out + at) = make_float2(x[0], x[1]);
                }
            }
        }
    for (int first = kv0; first < end; first += MANY) {
        if (first > kv0) {
            __syncthreads();
            load_kv(first);
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int h = first + warp + i * WARPS;
            if (h >= end) break;
            const bool is_k = h < H + G;
            if (is_k) kv4::prepare_head<HD>(kv[i], r.k_norm, r.eps, true, turn, s_row[warp + i * WARPS], lane);
            __syncwarp();
            if constexpr (N == 4) *reinterpret_cast<float4*>(s_row[warp + i * WARPS] + 4 * lane) = make_float4(kv[i][0], kv[i][1], kv[i][2], kv[i][3]);
            else *reinterpret_cast<float2*>(s_row[warp + i * WARPS] + 2 * lane) = make_float2(kv[i][0], kv[i][1]);
        }
        __syncthreads();
        const int rows = min(end - first, MANY);
        for (int i = tid; i - lane < rows * W; i += WARPS * 32) {      // whole warps
            const int row = min(i / W, rows - 1), c = i % W;
            float x[8];
            *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(s_row[row] + 8 * c);
            *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(s_row[row] + 8 * c + 4);
            __half d;
            const uint32_t w = kv4::encode_word(x, d);
            if (i >= rows * W) continue;
            const int h = first + row;
            const bool is_k = h < H + G;
            const size_t at = kv4::row_of(a.c, pos, slot, is_k ? h - H : h - H - G);
            reinterpret_cast<uint32_t*>(is_k ? a.c.k : a.c.v)[at * W + kv4::word_of<HD>(c)] = w;
            if ((c & 3) == 0) reinterpret_cast<__half*>(is_k ? a.c.ks : a.c.vs)[at * N + (c >> 2)] = d;
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
    // few rows: a head a warp, so that a step's many heads are worked on at once; many: a row a CTA, whose angles are made once
    const bool many = a.r.rows > 64;
    int per = many ? all : WARPS;
    int wide = kv4_wide_rows(a.r);
    void* args[] = {&a, &per, &wide};
    const void* fn = a.c.hd == 128 ? (const void*)append4_kernel<128> : (const void*)append4_kernel<64>;
    return launch_rows(fn, dim3(a.r.rows, (all + per - 1) / per), dim3(WARPS * 32), 0, args, st, pdl);
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
