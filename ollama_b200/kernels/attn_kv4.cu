// Attention of one token a sequence over the 4-bit cache (kv4.cuh), sm_100a.
//
//   out[t][h] = sum_k p_k v_k / (sum_k p_k + exp(sink)),  p_k = exp(cap(scale q . k)),  k the positions up to the token's own that its window has
//
// A key's columns cost half a byte each and two bytes more for 32, a seventh of what they weigh as fp32, so what the kernel spends is instructions: those that turn codes into operands (seven for
// eight codes of a key, half of which stay 72 too large, ten for eight of two values), the scales' products, exponentials.  Hence keys and values are the row operand of m16n8k16 products and the up to eight
// query heads of a KV head their columns (half the products of the other way round; tcgen05 would have the expanded codes written to shared memory first), codes become f16 numbers without their scale, and the
// scales, one for 32 columns, are applied to what is smaller: a key's to the fp32 sums over its blocks, a value's to the weights, which are rounded to f16 with the scale in them.  Models with more than
// eight heads a KV head take them eight at a time.
// Weights are exponents relative to a reference that follows the largest (score + log2 of the value's largest scale): with the scale in it, small values behind a large score keep their f16 digits.
// The reference moves only when something exceeds it by 2^8, and weights count from 2^7 on, so a key of 2^-21 of the heaviest is an f16 number of full precision and one of 2^-31 still counts.
// The keys of all sequences and KV heads are dealt out in runs of equal length to the CTAs that fit the GPU; four warps take 32 keys of a run in turn, through rings of their own, so that nothing
// in the loop waits for another warp.  A second launch adds up the parts.  From raw projections the CTA turns its queries itself, and the one with the token's own position also makes its codes.
// Measured, 32 heads on 8 of 128: 4 sequences, 222 MB of keys and values: 55.9 us with the sums, 4.0 TB/s, 0.60 of a copy's rate; schedulers issue in 60% of their cycles, the tensor pipe is busy in 23%: chains
// of three warps a scheduler (166 registers), and with four heads a KV head half of the products' columns and of the weights are of heads that do not exist.  Without the
// expansion of keys it took 3.0 us less, of values 6.7, without both 8.7, without the values' products 0.8: the rest is loads, scales and exponentials.  Four CTAs an SM in place of three (fewer stages) 3.6 more.
// A sequence of 6144 keys 14.0 us, two launches and the chain position, share, rows, part; 201 keys 9.3.
#include "kv4.cuh"

bool kv4_bad_cache(const Cache4& c);
bool kv4_bad_rows(const Rows4& r, const Cache4& c);
bool kv4_wide_rows(const Rows4& r);

namespace {

constexpr int WARPS = 4, TURN = 32, GRAIN = WARPS * TURN, HEADS = 8;
constexpr float LIFT = 7.f, LAG = 8.f, LOG2E = 1.4426950408889634f;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same onto other accumulators than it leaves.
__device__ __forceinline__ void mma_from(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {      // of an 8 x 8 matrix of f16
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
template <int BYTES>
__device__ __forceinline__ void copy_few(uint32_t to, const void* from) { asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(BYTES) : "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <int D>
struct Lay {
    static constexpr int NB = D / 32, ROW = D / 2, SC = D / 16;               // blocks, bytes of a row's codes and scales
    static constexpr int HALF = TURN * (ROW + SC), STAGE = 2 * HALF;          // keys (codes, scales), then values
    static constexpr int NS = 3, RING = NS * STAGE;
    static constexpr int LDQ = D + 8;
    static constexpr int Q_BYTES = HEADS * LDQ * 2, RINGS = WARPS * RING, MERGE = WARPS * HEADS * (D + 4) * 4;
    static constexpr int TOTAL = Q_BYTES + (RINGS > MERGE ? RINGS : MERGE);
};

// 16-byte piece of a row where it stands in a stage: rows that a quarter of a warp reads together (of values, every second one) are in different banks
template <int D>
__device__ __forceinline__ int piece_at(int row, int piece) { return row * (D / 2) + 16 * (D == 128 ? piece ^ ((row >> 1) & 3) : piece ^ ((row >> 2) & 1)); }

// Which keys a CTA takes: each sequence's are cut into equal shares of at most `chunk` grains, as few as leave at most `room` shares.
struct Share {
    int seq, index, count, first, end;      // count: shares of the sequence; keys first .. end - 1
};
__device__ __forceinline__ bool find_share(const Rows4& r, const Cache4& c, int window, int room, int which, int lane, Share& out) {
    const int n = r.rows;
    auto keys_at = [&](int b) {
        if (b >= n) return 0;
        const int p = r.positions[b];
        return kv4::has_row(c, p, r.slots[b]) ? p + 1 - first_key(p, 0, window) : 0;
    };
    const int mine = keys_at(lane);          // of up to 32 sequences each lane knows its own
    auto keys_of = [&](int b) { return b == lane ? mine : keys_at(b); };
    auto grains = [](int keys) { return (keys + GRAIN - 1) / GRAIN; };
    int chunk;                               // of GRAIN keys
    if (n <= 32) {
        chunk = (int)((__reduce_add_sync(0xffffffffu, (unsigned)grains(mine)) + room - 1) / room);
    } else {
        long long sum = 0;
        for (int b = lane; b < n; b += 32) sum += grains(keys_of(b));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        chunk = (int)((sum + room - 1) / room);
    }
    chunk = max(chunk, 1);
    // rounding up each sequence's last share needs at most one more for each: room is at least twice the rows, so this ends at twice the least chunk at the latest
    for (;; chunk += max(1, chunk / 32)) {
        int shares = 0;
        for (int b = lane; b < n; b += 32) shares += (grains(keys_of(b)) + chunk - 1) / chunk;
        if ((int)__reduce_add_sync(0xffffffffu, shares) <= room) break;
    }
    int before = 0;
    for (int b0 = 0; b0 < n; b0 += 32) {
        const int keys = keys_of(b0 + lane), shares = (grains(keys) + chunk - 1) / chunk;
        int upto = shares;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, which < before + upto);
        if (hit) {
            const int l = __ffs(hit) - 1;
            out.seq = b0 + l;
            out.count = __shfl_sync(0xffffffffu, shares, l);
            out.index = which - before - __shfl_sync(0xffffffffu, upto - shares, l);
            const int all = __shfl_sync(0xffffffffu, keys, l), last = r.positions[out.seq] + 1;
            out.first = last - all + (int)((long long)grains(all) * out.index / out.count) * GRAIN;      // a sequence's shares differ by a grain
            out.end = out.index + 1 == out.count ? last : last - all + (int)((long long)grains(all) * (out.index + 1) / out.count) * GRAIN;
            return true;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

template <int D>
__global__ void __launch_bounds__(WARPS * 32, 3) attn4_kernel(const __grid_constant__ Attn4Args a, int wide) {
    using L = Lay<D>;
    constexpr int NB = L::NB;
    extern __shared__ __align__(16) unsigned char smem[];
    __half* sQ = reinterpret_cast<__half*>(smem);                 // [HEADS][LDQ]
    unsigned char* rings = smem + L::Q_BYTES;
    __shared__ float s_cs[D / 2], s_sn[D / 2];
    __shared__ __align__(16) float s_row[WARPS][D];
    __shared__ __align__(16) uint32_t s_new[2][D / 8];            // the token's own key and value
    __shared__ __half s_newd[2][NB];
    __shared__ float s_m[WARPS][HEADS], s_l[WARPS][HEADS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tq = lane & 3;
    const Rows4& r = a.r;
    const int H = r.n_heads, G = a.c.kv_heads, group = H / G, tiles = (group + HEADS - 1) / HEADS;
    const int kvh = blockIdx.y / tiles, tile = blockIdx.y % tiles, head0 = kvh * group + tile * HEADS, heads = min(HEADS, group - tile * HEADS);

    pdl_launch();
    pdl_wait();
    const float freq = r.qkv && tid < (r.n_rot >> 1) ? r.inv_freq[tid] : 0.f;
    Share sh;
    if (!find_share(r, a.c, a.window, a.room, blockIdx.x, lane, sh)) return;
    const int qpos = r.positions[sh.seq], slot = r.slots[sh.seq];
    if (blockIdx.y == 0 && sh.index == 0 && tid == 0) a.shares[sh.seq] = make_int2(blockIdx.x, sh.count);
    const size_t row0 = kv4::row_of(a.c, 0, slot, kvh);
    const int turns = (sh.end - sh.first - TURN * warp + GRAIN - 1) / GRAIN;      // this warp has keys first + TURN (warp + 4 i) ..
    unsigned char* ring = rings + warp * L::RING;
    const uint32_t ring_at = smem_u32(ring);

    // a lane's pieces of a turn: rows of the same place in the swizzle, so that all but the first are constant distances away
    constexpr int PER_ROW = L::ROW / 16, STEP = 32 / PER_ROW;
    const int my_row = lane / PER_ROW, my_piece = lane % PER_ROW;
    const uint32_t to0 = ring_at + piece_at<D>(my_row, my_piece), sc0 = ring_at + TURN * L::ROW + lane * L::SC;
    size_t from0 = (row0 + sh.first + TURN * warp + my_row) * L::ROW + 16 * my_piece, scale0 = (row0 + sh.first + TURN * warp + lane) * L::SC;      // of the next turn that is asked for
    auto request = [&](int i) {      // keys behind the share repeat its last (masked below)
        if (i < turns) {
            const int n0 = sh.first + TURN * (warp + WARPS * i);
            const uint32_t at = i % L::NS * L::STAGE;
            if (n0 + TURN <= sh.end) {
#pragma unroll
                for (int v = 0; v < 2; v++) {
                    const uint8_t* from = (v ? a.c.v : a.c.k) + from0;
#pragma unroll
                    for (int p = 0; p < TURN / STEP; p++) copy16(to0 + at + v * L::HALF + p * STEP * L::ROW, from + p * STEP * L::ROW);
                    copy_few<L::SC>(sc0 + at + v * L::HALF, (const uint8_t*)(v ? a.c.vs : a.c.ks) + scale0);
                }
            } else {
#pragma unroll 1
                for (int v = 0; v < 2; v++) {
                    const uint8_t* from = v ? a.c.v : a.c.k;
#pragma unroll
                    for (int p = 0; p < TURN / STEP; p++)
                        copy16(to0 + at + v * L::HALF + p * STEP * L::ROW, from + (row0 + min(n0 + my_row + p * STEP, sh.end - 1)) * L::ROW + 16 * my_piece);
                    copy_few<L::SC>(sc0 + at + v * L::HALF, (const uint8_t*)(v ? a.c.vs : a.c.ks) + (row0 + min(n0 + lane, sh.end - 1)) * L::SC);
                }
            }
            from0 += (size_t)GRAIN * L::ROW;
            scale0 += (size_t)GRAIN * L::SC;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < L::NS - 1; i++) request(i);

    const bool fresh = r.qkv != nullptr, owner = fresh && qpos >= sh.first && qpos < sh.end;
    if (fresh) {
        // a warp takes two of the heads, warps 0 and 1 of the owner the key and the value: all asked for before the angles are made
        constexpr int N = D / 32, MINE = HEADS / WARPS;
        const float* src = r.qkv + (size_t)sh.seq * r.ldq;
        float x[MINE + 1][N];
#pragma unroll
        for (int i = 0; i <= MINE; i++) {
            const int h = warp + WARPS * i;
            const bool there = i < MINE ? h < heads : owner && warp < 2;
            const float* at = src + (size_t)(i < MINE ? head0 + h : H + warp * G + kvh) * D;
#pragma unroll
            for (int j = 0; j < N; j++) x[i][j] = 0.f;
            if (!there) continue;
            if (wide) {
                if constexpr (N == 4) {
                    const float4 y = __ldcg(reinterpret_cast<const float4*>(at) + lane);
                    x[i][0] = y.x; x[i][1] = y.y; x[i][2] = y.z; x[i][3] = y.w;
                } else {
                    const float2 y = __ldcg(reinterpret_cast<const float2*>(at) + lane);
                    x[i][0] = y.x; x[i][1] = y.y;
                }
            } else {
#pragma unroll
                for (int j = 0; j < N; j++) x[i][j] = __ldcg(at + N * lane + j);
            }
        }
        if (tid < (r.n_rot >> 1)) kv4::make_angle(r, qpos, tid, freq, s_cs, s_sn);
        __syncthreads();
        const kv4::Turn<D> turn = kv4::make_turn<D>(r, s_cs, s_sn, lane);
#pragma unroll
        for (int i = 0; i < MINE; i++) {
            const int h = warp + WARPS * i;
            if (h < heads) kv4::prepare_head<D>(x[i], r.q_norm, r.eps, true, turn, s_row[warp], lane);
#pragma unroll
            for (int j = 0; j < N; j += 2) *reinterpret_cast<uint32_t*>(sQ + h * L::LDQ + N * lane + j) = pack(x[i][j], x[i][j + 1]);
        }
        if (owner && warp < 2) {
            if (warp == 0) kv4::prepare_head<D>(x[MINE], r.k_norm, r.eps, true, turn, s_row[warp], lane);
            const size_t row = row0 + qpos;
            __syncwarp();
#pragma unroll
            for (int j = 0; j < N; j++) s_row[warp][N * lane + j] = x[MINE][j];
            __syncwarp();
            const int c = lane % (D / 8), at = kv4::word_of<D>(c);      // (D / 8 lanes do what the others repeat)
            float y[8];
            *reinterpret_cast<float4*>(y) = *reinterpret_cast<const float4*>(s_row[warp] + 8 * c);
            *reinterpret_cast<float4*>(y + 4) = *reinterpret_cast<const float4*>(s_row[warp] + 8 * c + 4);
            __half d;
            const uint32_t w = kv4::encode_word(y, d);
            if (lane < D / 8) {
                s_new[warp][at] = w;
                if (tile == 0) reinterpret_cast<uint32_t*>(warp ? a.c.v : a.c.k)[row * (D / 8) + at] = w;
                if ((c & 3) == 0) {
                    s_newd[warp][c >> 2] = d;
                    if (tile == 0) reinterpret_cast<__half*>(warp ? a.c.vs : a.c.ks)[row * NB + (c >> 2)] = d;
                }
            }
        }
    } else {
        for (int i = tid; i < HEADS * D / 8; i += WARPS * 32) {
            const int h = i / (D / 8), col = i % (D / 8) * 8;
            const size_t at = ((size_t)sh.seq * H + head0 + h) * D + col;
            uint4 y = make_uint4(0, 0, 0, 0);
            if (h < heads) {
                if (a.q16) {
                    y = __ldcg(reinterpret_cast<const uint4*>(reinterpret_cast<const __half*>(a.q) + at));
                } else {
                    const float4 lo = __ldcg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.q) + at)), hi = __ldcg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.q) + at + 4));
                    y = make_uint4(pack(lo.x, lo.y), pack(lo.z, lo.w), pack(hi.x, hi.y), pack(hi.z, hi.w));
                }
            }
            *reinterpret_cast<uint4*>(sQ + h * L::LDQ + col) = y;
        }
    }
    __syncthreads();
    // columns 32 b + 8 tq .. of head g: what lane (g, tq) of the key operand has of a row, its word of block b
    uint32_t qf[NB][4];
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const uint4 y = *reinterpret_cast<const uint4*>(sQ + g * L::LDQ + 32 * b + 8 * tq);
        qf[b][0] = y.x; qf[b][1] = y.y; qf[b][2] = y.z; qf[b][3] = y.w;
    }
    // Half of a key's columns come 72 too large: the products begin with what that makes for heads 2 tq and 2 tq + 1.  (Sums of 32 columns then lose some 2^-20 of their operands' size; all
    // columns 1032 too large would cost two instructions less and 2^-16.)
    float less[NB][2];
#pragma unroll
    for (int b = 0; b < NB; b++) {
        float sum = 0.f;
#pragma unroll
        for (int i = 1; i < 4; i += 2) {
            const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&qf[b][i]));
            sum += y.x + y.y;
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);      // of head g
#pragma unroll
        for (int e = 0; e < 2; e++) less[b][e] = -kv4::RAISED * __shfl_sync(0xffffffffu, sum, 4 * (2 * tq + e));
    }

    float o[NB][2][4];
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int i = 0; i < 8; i++) o[b][i >> 2][i & 3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;      // of heads 2 tq, 2 tq + 1
    // scores times mult are exponents of two; a key that does not count has the score that makes that -inf
    const float mult = a.softcap > 0.f ? 1.f : a.scale * LOG2E == 0.f ? 1e-37f : a.scale * LOG2E, beyond = mult > 0.f ? -INFINITY : INFINITY;
    const float inv_cap = a.softcap > 0.f ? a.scale / a.softcap : 0.f, cap2 = a.softcap * LOG2E;
    const int half = g & 1, sel = half ? 0x7632 : 0x5410;          // which half of a value word's codes: of two keys, side by side

    for (int i = 0; i < turns; i++) {
        request(i + L::NS - 1);                                                            // into the stage of the turn before
        asm volatile("cp.async.wait_group %0;" ::"n"(L::NS - 1) : "memory");
        __syncwarp();
        unsigned char* st = ring + i % L::NS * L::STAGE;
        const int n0 = sh.first + TURN * (warp + WARPS * i);
        if (owner && n0 <= qpos && qpos < n0 + TURN) {      // the token's own row did not come from the cache
            const int row = qpos - n0;
            for (int w = lane; w < D / 4; w += 32) {
                const int v = w / (D / 8), at = w % (D / 8);
                *reinterpret_cast<uint32_t*>(st + v * L::HALF + piece_at<D>(row, at >> 2) + 4 * (at & 3)) = s_new[v][at];
            }
            if (lane < 2 * NB) reinterpret_cast<__half*>(st + lane / NB * L::HALF + TURN * L::ROW)[row * NB + lane % NB] = s_newd[lane / NB][lane % NB];
            __syncwarp();
        }
        const unsigned char* vt = st + L::HALF;
        float s[2][4];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
            const int ra = 16 * u + g, rb = ra + 8;
            uint32_t ka[NB], kb[NB];
            float da[NB], db[NB];
            if constexpr (D == 128) {
                *reinterpret_cast<uint4*>(ka) = *reinterpret_cast<const uint4*>(st + piece_at<D>(ra, tq));
                *reinterpret_cast<uint4*>(kb) = *reinterpret_cast<const uint4*>(st + piece_at<D>(rb, tq));
            } else {
                *reinterpret_cast<uint2*>(ka) = *reinterpret_cast<const uint2*>(st + piece_at<D>(ra, tq >> 1) + 8 * (tq & 1));
                *reinterpret_cast<uint2*>(kb) = *reinterpret_cast<const uint2*>(st + piece_at<D>(rb, tq >> 1) + 8 * (tq & 1));
            }
            const __half2* sa = reinterpret_cast<const __half2*>(st + TURN * L::ROW + ra * L::SC);
            const __half2* sb = reinterpret_cast<const __half2*>(st + TURN * L::ROW + rb * L::SC);
#pragma unroll
            for (int b = 0; b < NB; b += 2) {
                const float2 x = __half22float2(sa[b / 2]), y = __half22float2(sb[b / 2]);
                da[b] = x.x; da[b + 1] = x.y; db[b] = y.x; db[b + 1] = y.y;
            }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                uint32_t e[4], f[4];
                kv4::expand_raised(ka[b], e);
                kv4::expand_raised(kb[b], f);
                float c[4];
                mma_from(c, e[0], f[0], e[1], f[1], qf[b][0], qf[b][1], less[b][0], less[b][1]);
                mma(c, e[2], f[2], e[3], f[3], qf[b][2], qf[b][3]);
                s[u][0] += c[0] * da[b]; s[u][1] += c[1] * da[b];
                s[u][2] += c[2] * db[b]; s[u][3] += c[3] * db[b];
            }
        }
        // s[u][0, 1]: key 16 u + g, heads 2 tq, 2 tq + 1; s[u][2, 3]: key 16 u + 8 + g.  To powers of two; the values' scales
        float dv[4][NB], big[4];
        float y0 = -INFINITY, y1 = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; k++) {      // key 8 k + g
            const __half2* sc = reinterpret_cast<const __half2*>(vt + TURN * L::ROW + (8 * k + g) * L::SC);
            float top = 5.9604644775390625e-8f;      // 2^-24: rows of zeros
#pragma unroll
            for (int b = 0; b < NB; b += 2) {
                const float2 x = __half22float2(sc[b / 2]);
                dv[k][b] = x.x;
                dv[k][b + 1] = x.y;
                top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
            }
            big[k] = lg2(top);
        }
        if (a.softcap > 0.f) {      // in powers of two from here on, mult is one
#pragma unroll
            for (int k = 0; k < 8; k++) s[k >> 2][k & 3] = cap2 * tanh_exp(s[k >> 2][k & 3] * inv_cap);
        }
        if (n0 + TURN > sh.end) {
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (n0 + 8 * k + g >= sh.end) {      // (nor do its values' scales: they may be those of a row that is being written)
                    s[k >> 1][2 * (k & 1)] = s[k >> 1][2 * (k & 1) + 1] = beyond;
                    big[k] = 0.f;
#pragma unroll
                    for (int b = 0; b < NB; b++) dv[k][b] = 0.f;
                }
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            y0 = fmaxf(y0, s[k >> 1][2 * (k & 1)] * mult + big[k]);
            y1 = fmaxf(y1, s[k >> 1][2 * (k & 1) + 1] * mult + big[k]);
        }
        if (__any_sync(0xffffffffu, y0 > m0 + LAG || y1 > m1 + LAG)) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
                y0 = fmaxf(y0, __shfl_xor_sync(0xffffffffu, y0, x));
                y1 = fmaxf(y1, __shfl_xor_sync(0xffffffffu, y1, x));
            }
            // (a head's own scores alone decide)
            const float n0m = y0 > m0 + LAG ? y0 : m0, n1m = y1 > m1 + LAG ? y1 : m1;
            const float f0 = n0m == m0 ? 1.f : ex2(m0 - n0m), f1 = n1m == m1 ? 1.f : ex2(m1 - n1m);
            m0 = n0m;
            m1 = n1m;
            l0 *= f0;
            l1 *= f1;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    o[b][t][0] *= f0; o[b][t][1] *= f1;
                    o[b][t][2] *= f0; o[b][t][3] *= f1;
                }
        }
        const float r0 = m0 == -INFINITY ? 0.f : m0 - LIFT, r1 = m1 == -INFINITY ? 0.f : m1 - LIFT;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            float& v0 = s[k >> 1][2 * (k & 1)];
            float& v1 = s[k >> 1][2 * (k & 1) + 1];
            v0 = ex2(v0 * mult - r0);
            v1 = ex2(v1 * mult - r1);
            l0 += v0;
            l1 += v1;
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            // words of block b of keys 16 u + 2 tq, + 1, + 8, + 9, of which this lane's dims are 32 b + 8 (g / 2) + 2 i + half
            const int rr = 16 * u + 2 * tq, j = g >> 1;
            uint32_t w[4][NB];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int row = rr + (k & 1) + 8 * (k >> 1);
                if constexpr (D == 128) *reinterpret_cast<uint4*>(w[k]) = *reinterpret_cast<const uint4*>(vt + piece_at<D>(row, j));
                else *reinterpret_cast<uint2*>(w[k]) = *reinterpret_cast<const uint2*>(vt + piece_at<D>(row, j >> 1) + 8 * (j & 1));
            }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const uint32_t p0 = transposed(pack(s[u][0] * dv[2 * u][b], s[u][1] * dv[2 * u][b]));
                const uint32_t p1 = transposed(pack(s[u][2] * dv[2 * u + 1][b], s[u][3] * dv[2 * u + 1][b]));
                uint32_t e[4], f[4];
                kv4::expand(__byte_perm(w[0][b], w[1][b], sel), e);
                kv4::expand(__byte_perm(w[2][b], w[3][b], sel), f);
                mma(o[b][0], e[0], e[1], f[0], f[1], p0, p1);
                mma(o[b][1], e[2], e[3], f[2], f[3], p0, p1);
            }
        }
        __syncwarp();        // every lane is done with this stage before the next turn's request overwrites it
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // the warps' parts
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, x);
        l1 += __shfl_xor_sync(0xffffffffu, l1, x);
    }
    __syncthreads();         // behind it the rings are free
    constexpr int LDO = D + 4;
    float* s_acc = reinterpret_cast<float*>(rings);      // [WARPS][HEADS][LDO]
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                s_acc[(warp * HEADS + 2 * tq + (e & 1)) * LDO + 32 * b + 8 * (g >> 1) + 2 * (2 * t + (e >> 1)) + half] = o[b][t][e];
    if (g == 0) {
        s_m[warp][2 * tq] = m0; s_m[warp][2 * tq + 1] = m1;
        s_l[warp][2 * tq] = l0; s_l[warp][2 * tq + 1] = l1;
    }
    __syncthreads();
    for (int i = tid; i < heads * (D / 4); i += WARPS * 32) {
        const int h = i / (D / 4), col = i % (D / 4) * 4;
        const float m = fmaxf(fmaxf(s_m[0][h], s_m[1][h]), fmaxf(s_m[2][h], s_m[3][h]));
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float f = s_m[w][h] == -INFINITY ? 0.f : ex2(s_m[w][h] - m);
            const float4 y = *reinterpret_cast<const float4*>(s_acc + (w * HEADS + h) * LDO + col);
            acc.x += y.x * f; acc.y += y.y * f; acc.z += y.z * f; acc.w += y.w * f;
            l += s_l[w][h] * f;
        }
        const size_t at = (size_t)blockIdx.x * H + head0 + h;
        *reinterpret_cast<float4*>(a.part_acc + at * D + col) = acc;
        if (col == 0) a.part_ml[at] = make_float2(m - LIFT, l);
    }
}

// Adds up the parts of a head: WIDE warps each, which take every WIDE-th, a lane D / 32 columns; eight warps a CTA, grid (heads * WIDE / 8, sequences).  Eight warps a head where a sequence has
// more than eight parts on the mean, else one, since CTAs then cost more than parts do.  Both launches with eight and with one: 55 parts 14.0 and 18.6 us, 4 x 14 parts of 32 heads 55.8 and
// 57.7 us, 32 x 2 parts of 64 heads 18.7 and 14.2 us.
constexpr int MERGERS = 8;
template <int D, int WIDE>
__global__ void __launch_bounds__(MERGERS * 32) merge4_kernel(const __grid_constant__ Attn4Args a) {
    constexpr int N = D / 32;
    __shared__ float s_acc[MERGERS][D];
    __shared__ float s_l[MERGERS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, H = a.r.n_heads, h = (blockIdx.x * MERGERS + warp) / WIDE, b = blockIdx.y;
    pdl_launch();
    pdl_wait();
    if (!kv4::has_row(a.c, a.r.positions[b], a.r.slots[b])) return;      // no token: the row stays as it is
    const bool there = h < H;
    const int2 sh = a.shares[b];
    float acc[N], l = 0.f, ref = 0.f, sink = -INFINITY;
#pragma unroll
    for (int j = 0; j < N; j++) acc[j] = 0.f;
    if (there) {
        float m = -INFINITY;
        for (int p = lane; p < sh.y; p += 32) m = fmaxf(m, a.part_ml[(size_t)(sh.x + p) * H + h].x);
        if (a.sinks) sink = a.sinks[h] * LOG2E;
        m = fmaxf(warp_max(m), sink);
        ref = m == -INFINITY ? 0.f : fminf(m, 3.4e38f);      // finite: relative to it an infinite sink is infinite, and the others' weights zero
#pragma unroll 8
        for (int p = warp % WIDE; p < sh.y; p += WIDE) {
            const size_t at = (size_t)(sh.x + p) * H + h;
            const float2 ml = a.part_ml[at];
            const float f = ex2(ml.x - ref);
            if constexpr (N == 4) {
                const float4 y = __ldcg(reinterpret_cast<const float4*>(a.part_acc + at * D) + lane);
                acc[0] += y.x * f; acc[1] += y.y * f; acc[2] += y.z * f; acc[3] += y.w * f;
            } else {
                const float2 y = __ldcg(reinterpret_cast<const float2*>(a.part_acc + at * D) + lane);
                acc[0] += y.x * f; acc[1] += y.y * f;
            }
            l += ml.y * f;
        }
    }
    if (WIDE > 1) {
#pragma unroll
        for (int j = 0; j < N; j++) s_acc[warp][N * lane + j] = acc[j];
        if (lane == 0) s_l[warp] = l;
        __syncthreads();
        if (warp % WIDE) return;
        l = 0.f;
#pragma unroll
        for (int j = 0; j < N; j++) acc[j] = 0.f;
#pragma unroll
        for (int w = 0; w < WIDE; w++) {
#pragma unroll
            for (int j = 0; j < N; j++) acc[j] += s_acc[warp + w][N * lane + j];
            l += s_l[warp + w];
        }
    }
    if (!there) return;
    if (a.sinks) l += ex2(sink - ref);
    const size_t at = (size_t)b * a.ldo + (size_t)h * D + N * lane;      // (rows of results stand at any distance)
#pragma unroll
    for (int j = 0; j < N; j++) {
        const float y = acc[j] / l;
        if (a.out16) reinterpret_cast<__nv_bfloat16*>(a.out)[at + j] = __float2bfloat16_rn(y);
        else reinterpret_cast<float*>(a.out)[at + j] = y;
    }
}

}  // namespace

// CTAs of a launch for one KV head and eight of its query heads, and the parts that they leave: as many as fit the GPU, at least two a sequence.
B2_API int b2_attn4_room(int rows, int n_heads, int kv_heads, int sms) {
    const long group = n_heads / kv_heads, units = (long)kv_heads * ((group + HEADS - 1) / HEADS), fit = 3l * sms / units;
    return (int)(fit > 2l * rows ? fit : 2l * rows);
}

// Two launches.  part_acc, part_ml and shares are scratch of a.room parts (b2_attn4_room) and a.r.rows sequences.
B2_API int b2_attn4(const Attn4Args* in, int pdl, cudaStream_t st) {
    Attn4Args a = *in;
    if (kv4_bad_cache(a.c) || (a.r.qkv && kv4_bad_rows(a.r, a.c)) || (!a.r.qkv && !a.q) || a.r.rows < 0 || a.r.n_heads < 1 || a.r.n_heads % a.c.kv_heads) return (int)cudaErrorInvalidValue;
    if (!a.r.rows) return 0;
    const int group = a.r.n_heads / a.c.kv_heads, tiles = (group + HEADS - 1) / HEADS;
    if (!a.r.positions || !a.r.slots || !a.out || !a.part_acc || !a.part_ml || !a.shares || a.window < 0 || a.room < 2 * a.r.rows || a.r.rows > 65535 || (long)a.c.kv_heads * tiles > 65535 ||
        a.ldo < a.r.n_heads * a.c.hd)
        return (int)cudaErrorInvalidValue;
    int wide = kv4_wide_rows(a.r);
    void* args[] = {&a, &wide};
    const bool big = a.c.hd == 128;
    const void* fn = big ? (const void*)attn4_kernel<128> : (const void*)attn4_kernel<64>;
    const int smem = big ? Lay<128>::TOTAL : Lay<64>::TOTAL;
    static thread_local PerDeviceOnce once;
    if (once.first()) {
        cudaError_t e = cudaFuncSetAttribute((const void*)attn4_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<128>::TOTAL);
        if (e == cudaSuccess) e = cudaFuncSetAttribute((const void*)attn4_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<64>::TOTAL);
        if (e != cudaSuccess) return (int)e;
    }
    const int rc = launch_rows(fn, dim3(a.room, a.c.kv_heads * tiles), dim3(WARPS * 32), smem, args, st, pdl);
    if (rc) return rc;
    void* margs[] = {&a};      // (its CTAs may wait beside the first launch's last)
    const bool many = a.room / a.r.rows > MERGERS;      // shares that a sequence has on the mean
    const void* merge = big ? (many ? (const void*)merge4_kernel<128, MERGERS> : (const void*)merge4_kernel<128, 1>) : (many ? (const void*)merge4_kernel<64, MERGERS> : (const void*)merge4_kernel<64, 1>);
    return launch_rows(merge, dim3(many ? a.r.n_heads : (a.r.n_heads + MERGERS - 1) / MERGERS, a.r.rows), dim3(MERGERS * 32), 0, margs, st, 1);
}
