// Causal attention of prompts of several sequences in one launch, on tcgen05 (sm_100a): over 16-bit keys and values of any layout, or over the 4-bit cache (kv4.cuh).
//
//   out[t][h] = sum_k p_k v_k / (sum_k p_k + exp(sink)),  p_k = exp(cap(scale q[t][h] . k)),  k the sequence's positions up to the token's own that its window has
//
// A CTA takes two tiles of 128 query rows of one KV head; a row is a token's query head (token / group, head of the group), so all heads of a group share the keys that the CTA brings, and few
// tokens of many heads still fill a tile.  Keys come in tiles of 128.  Roles: warps 0-3 and 4-7 the softmax of a tile each, a row a thread (no exchange between threads); warp 8 loads; warp 9
// issues the products; warps 12-15 make operands: of a 4-bit cache they turn codes into f16 rows in the swizzled layout, of 16-bit rows they look at tiles whose mask is not whole (below).
// Scores of one tile are computed while the other's softmax runs: S_A, then for each key tile P V of A, the next S of A, P V of B, the next S of B.  Tensor memory: S of both (128 columns each, over
// which the weights are written as 16-bit operands), O of both, accumulated there.  The weights are relative to a reference that follows a row's largest score only when that exceeds it by 2^8
// (then the thread rescales its row of O: the product before is complete by the time a tile's scores are), and count from 2^6 on, so that f16 weights keep 20 powers of two below the largest.
// Tiles that not every row sees as a whole (the diagonal, a window's edge, the end) hold keys that must not count whatever they are, and a weight of zero times a value that is no number is
// none either: in such tiles of 16-bit rows, values rows with such elements become zeros and their keys none, so that exactly the rows that see them have no result.  Cached codes are finite.
// Where tiles are few, or their keys many, the keys of a tile are shared out over several CTAs, and a second launch adds up what they leave (ops/kv4.py says which).
#include "attn_tc.cuh"
#include "kv4.cuh"

bool kv4_bad_cache(const Cache4& c);

__device__ int g_packed_status = 0;

namespace {

using namespace tc;

constexpr int BQ = 128, BKV = 128, ATOM_BYTES = 128 * 128;
constexpr int THREADS = 512;
// registers: 512 threads start with 128 each; two softmax warpgroups, the one that makes operands, the one that loads and multiplies
constexpr int SOFTMAX_REGS = 176, MAKER_REGS = 104, REST_REGS = 56;
static_assert(2 * SOFTMAX_REGS + MAKER_REGS + REST_REGS == 512, "what the block was launched with");
constexpr float LIFT = 6.f, LAG = 8.f, LOG2E = 1.4426950408889634f;
enum Form : int { F16 = 0, B16 = 1, CODES = 2 };

template <int D>
struct Lay {
    static constexpr int ATOMS = D / 64, TILE = ATOMS * ATOM_BYTES;
    static constexpr int OFF_K = 2 * TILE, OFF_V = OFF_K + 2 * TILE, OFF_BAR = OFF_V + 2 * TILE;
    static constexpr int TOTAL = OFF_BAR + 256 + 1024;
};

__device__ __forceinline__ uint32_t idesc(bool bf16, int n, int b_mn_major) { return idesc_f16(BQ, n, b_mn_major) | (bf16 ? (1u << 7) | (1u << 10) : 0u); }

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// 64 consecutive 32-bit columns of this thread's lane, waited for
__device__ __forceinline__ void tmem_ld64(uint32_t at, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
          "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]),
          "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31]), "=r"(v[32]), "=r"(v[33]), "=r"(v[34]), "=r"(v[35]), "=r"(v[36]), "=r"(v[37]), "=r"(v[38]), "=r"(v[39]),
          "=r"(v[40]), "=r"(v[41]), "=r"(v[42]), "=r"(v[43]), "=r"(v[44]), "=r"(v[45]), "=r"(v[46]), "=r"(v[47]), "=r"(v[48]), "=r"(v[49]), "=r"(v[50]), "=r"(v[51]), "=r"(v[52]),
          "=r"(v[53]), "=r"(v[54]), "=r"(v[55]), "=r"(v[56]), "=r"(v[57]), "=r"(v[58]), "=r"(v[59]), "=r"(v[60]), "=r"(v[61]), "=r"(v[62]), "=r"(v[63])
        : "r"(at)
        : "memory");
}
template <int N>
__device__ __forceinline__ void set_registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void set_registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    if (BF16) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&b);
    }
    return pack_h2(x, y);
}

// One thread's columns of a result row: n (a multiple of 8) values.
__device__ __forceinline__ void store8(void* out, int type, size_t at, const float* y) {
    if (type == 0) {
        float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at);
        p[0] = make_float4(y[0], y[1], y[2], y[3]);
        p[1] = make_float4(y[4], y[5], y[6], y[7]);
    } else if (type == 1) {
        *reinterpret_cast<uint4*>(reinterpret_cast<__half*>(out) + at) = make_uint4(pack2<false>(y[0], y[1]), pack2<false>(y[2], y[3]), pack2<false>(y[4], y[5]), pack2<false>(y[6], y[7]));
    } else {
        *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(out) + at) = make_uint4(pack2<true>(y[0], y[1]), pack2<true>(y[2], y[3]), pack2<true>(y[4], y[5]), pack2<true>(y[6], y[7]));
    }
}

template <int D, int FORM>
__global__ void __launch_bounds__(THREADS, 1) packed_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PackedArgs a) {
    using L = Lay<D>;
    constexpr bool BF16 = FORM == B16;
    constexpr int ATOMS = L::ATOMS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::OFF_BAR);
    uint64_t* k_full = bars;             // [2] each
    uint64_t* k_empty = bars + 2;
    uint64_t* v_full = bars + 4;
    uint64_t* v_empty = bars + 6;
    uint64_t* s_full = bars + 8;         // of tiles A and B
    uint64_t* p_ready = bars + 10;
    uint64_t* o_full = bars + 12;
    uint64_t* looked = bars + 14;        // of the stages
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 16);
    int* failed = reinterpret_cast<int*>(bars + 17);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wg = warp >> 2;
    pdl_wait();
    const int group = a.n_heads / a.kv_heads, tokens = BQ / group;          // tokens of a tile
    const PackedTile tile = a.tiles[blockIdx.x];
    const int kvh = blockIdx.y;
    const bool two = tile.rows > tokens;
    const int q_lo = tile.pos, q_hi = tile.pos + tile.rows - 1, n_tiles = tile.k_hi - tile.k_lo;
    const int last_lo = first_key(q_hi, 0, a.window);
    // whether some row does not see all of key tile t
    auto masked = [&](int t) { const int n0 = (tile.k_lo + t) * BKV; return n0 + BKV - 1 > q_lo || n0 < last_lo; };

    if (threadIdx.x == 0) {
        *failed = 0;
        for (int b = 0; b < 2; b++) {
            mbar_init(&k_full[b], FORM == CODES ? 4 : 1);
            mbar_init(&k_empty[b], 1);
            mbar_init(&v_full[b], FORM == CODES ? 4 : 1);
            mbar_init(&v_empty[b], FORM == CODES ? 1 : 5);      // the products, and the warps that look at values
            mbar_init(&s_full[b], 1);
            mbar_init(&p_ready[b], 4);
            mbar_init(&o_full[b], 1);
            mbar_init(&looked[b], 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (wg < 2 && (wg == 0 || two)) {        // a thread's query row, as 16-bit operands
        const int r = threadIdx.x & 127, token = wg * tokens + r / group;
        const bool live = r / group < tokens && token < tile.rows;
        const size_t at = (size_t)(tile.row + token) * a.ldq + (size_t)(kvh * group + r % group) * D;
        const float sign = a.scale < 0.f ? -1.f : 1.f;
        uint8_t* q = sm + wg * L::TILE + r * 128;
#pragma unroll 4
        for (int c = 0; c < D / 8; c++) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (live) {
                float x[8];
                if (a.q_type == 0) {
                    const float4 y0 = reinterpret_cast<const float4*>((const float*)a.q + at)[2 * c], y1 = reinterpret_cast<const float4*>((const float*)a.q + at)[2 * c + 1];
                    x[0] = y0.x; x[1] = y0.y; x[2] = y0.z; x[3] = y0.w; x[4] = y1.x; x[5] = y1.y; x[6] = y1.z; x[7] = y1.w;
                } else {
                    w = reinterpret_cast<const uint4*>((const __half*)a.q + at)[c];
                    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float2 y = a.q_type == 1 ? __half22float2(*reinterpret_cast<const __half2*>(&u[i])) : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[i]));
                        x[2 * i] = y.x;
                        x[2 * i + 1] = y.y;
                    }
                }
                w = make_uint4(pack2<BF16>(sign * x[0], sign * x[1]), pack2<BF16>(sign * x[2], sign * x[3]), pack2<BF16>(sign * x[4], sign * x[5]), pack2<BF16>(sign * x[6], sign * x[7]));
            }
            *reinterpret_cast<uint4*>(q + (c >> 3) * ATOM_BYTES + (((c & 7) ^ (r & 7)) << 4)) = w;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch();

    if (wg == 2) {
        set_registers_down<REST_REGS>();
        if (FORM != CODES && warp == 8 && lane == 0) {
            for (int t = 0; t < n_tiles; t++) {
                const int b = t & 1, y = tile.base + (tile.k_lo + t) * BKV;
                if (t >= 2 && !mbar_wait(&k_empty[b], ((t >> 1) - 1) & 1)) { atomicExch(failed, 1); break; }
                mbar_expect_tx(&k_full[b], L::TILE);
#pragma unroll
                for (int i = 0; i < ATOMS; i++) tma_load_4d(sm + L::OFF_K + b * L::TILE + i * ATOM_BYTES, &map_k, 64 * i, y, kvh, tile.slot, &k_full[b]);
                if (t >= 2 && !mbar_wait(&v_empty[b], ((t >> 1) - 1) & 1)) { atomicExch(failed, 1); break; }
                mbar_expect_tx(&v_full[b], L::TILE);
#pragma unroll
                for (int i = 0; i < ATOMS; i++) tma_load_4d(sm + L::OFF_V + b * L::TILE + i * ATOM_BYTES, &map_v, 64 * i, y, kvh, tile.slot, &v_full[b]);
            }
        } else if (warp == 9 && lane == 0) {
            const uint32_t id_s = idesc(BF16, BKV, 0), id_o = idesc(BF16, D, 1);
            bool ok = true;
            uint32_t looks = 0;      // bit b: parity of the tiles of stage b that were looked at
            auto wait_k = [&](int t) {
                const int b = t & 1;
                if (!mbar_wait(&k_full[b], (t >> 1) & 1)) ok = false;
                else if (FORM != CODES && masked(t)) {
                    if (!mbar_wait(&looked[b], looks >> b & 1)) ok = false;
                    looks ^= 1u << b;
                }
                tc_fence_after();
            };
            auto scores = [&](int x, int t) {
#pragma unroll
                for (int i = 0; i < ATOMS; i++) {
                    const uint64_t qd = umma_desc(sm + x * L::TILE + i * ATOM_BYTES), kd = umma_desc(sm + L::OFF_K + (t & 1) * L::TILE + i * ATOM_BYTES);
#pragma unroll
                    for (int k = 0; k < 4; k++) umma_f16(tmem + 128 * x, qd + 2 * k, kd + 2 * k, id_s, (i | k) != 0);
                }
                umma_commit(&s_full[x]);
            };
            auto values = [&](int x, int t) {
                const uint8_t* vt = sm + L::OFF_V + (t & 1) * L::TILE;
#pragma unroll
                for (int k = 0; k < BKV / 16; k++) umma_f16_ts(tmem + 256 + 128 * x, tmem + 128 * x + 8 * k, umma_desc_mn(vt + k * 16 * 128, ATOM_BYTES), id_o, t > 0 || k != 0);
                if (t + 1 == n_tiles) umma_commit(&o_full[x]);
            };
            wait_k(0);
            if (ok) {
                scores(0, 0);
                if (two) scores(1, 0);
                umma_commit(&k_empty[0]);
            }
            for (int t = 0; t < n_tiles && ok; t++) {
                if (!mbar_wait(&p_ready[0], t & 1) || !mbar_wait(&v_full[t & 1], (t >> 1) & 1)) { ok = false; break; }
                tc_fence_after();
                values(0, t);
                if (t + 1 < n_tiles) {
                    wait_k(t + 1);
                    if (!ok) break;
                    scores(0, t + 1);
                }
                if (two) {
                    if (!mbar_wait(&p_ready[1], t & 1)) { ok = false; break; }
                    tc_fence_after();
                    values(1, t);
                    if (t + 1 < n_tiles) scores(1, t + 1);
                }
                umma_commit(&v_empty[t & 1]);
                if (t + 1 < n_tiles) umma_commit(&k_empty[(t + 1) & 1]);
            }
            if (!ok) atomicExch(failed, 1);
        }
    } else if (wg == 3) {
        set_registers_down<MAKER_REGS>();
        const int id = threadIdx.x & 127;
        if (FORM == CODES) {
            // a thread takes 16 bytes of codes of every 32nd row (D = 128; of every 64th: D = 64); the rows of eight lanes are such that their stores go to different banks
            constexpr int NB = D / 32, PIECES = D / 32, PASSES = PIECES, STEP = BKV / PASSES;      // 16-byte pieces of a row; rows of a pass
            const int piece = id % PIECES, i = id / PIECES;
            const int row = D == 128 ? (i & ~7) | (i & 1) << 2 | (i >> 1 & 3) : (i & ~7) | (i & 1) | (i >> 1 & 1) << 2 | (i >> 2 & 1) << 1;
            const size_t row0 = kv4::row_of(a.c, tile.base, tile.slot, kvh);
            const int last = q_hi;                       // rows behind the portion repeat its last: their keys are masked
            uint4 kw[PASSES], vw[PASSES];
            uint2 kd[PASSES], vd[PASSES];
            auto fetch = [&](int t, const uint8_t* codes, const void* scales, uint4 (&w)[PASSES], uint2 (&d)[PASSES]) {
#pragma unroll
                for (int p = 0; p < PASSES; p++) {
                    const size_t at = row0 + min((tile.k_lo + t) * BKV + p * STEP + row, last);
                    w[p] = ldg16(codes + at * (D / 2) + 16 * piece);
                    if (D == 128) d[p] = ldg8((const uint8_t*)scales + at * 8);
                    else d[p].x = __ldg((const uint32_t*)scales + at);
                }
            };
            auto write = [&](uint8_t* to, const uint4 (&w)[PASSES], const uint2 (&d)[PASSES]) {
#pragma unroll
                for (int p = 0; p < PASSES; p++) {
                    const uint32_t u[4] = {w[p].x, w[p].y, w[p].z, w[p].w};
                    const int rr = p * STEP + row;
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const int b = q % NB, j = D == 128 ? piece : 2 * piece + q / NB, chunk = 4 * b + j;      // columns 32 b + 8 j ..
                        const uint32_t pair = b >> 1 ? d[p].y : d[p].x, dd = __byte_perm(pair, 0, b & 1 ? 0x3232 : 0x1010);
                        uint32_t e[4];
                        kv4::expand(u[q], e);
#pragma unroll
                        for (int x = 0; x < 4; x++) e[x] = kv4::hmul2_bits(e[x], dd);
                        *reinterpret_cast<uint4*>(to + (chunk >> 3) * ATOM_BYTES + rr * 128 + (((chunk & 7) ^ (rr & 7)) << 4)) = make_uint4(e[0], e[1], e[2], e[3]);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            };
            if (n_tiles > 0) {
                fetch(0, a.c.k, a.c.ks, kw, kd);
                fetch(0, a.c.v, a.c.vs, vw, vd);
            }
            for (int t = 0; t < n_tiles; t++) {
                const int b = t & 1;
                if (t >= 2 && !mbar_wait(&k_empty[b], ((t >> 1) - 1) & 1)) { atomicExch(failed, 1); break; }
                write(sm + L::OFF_K + b * L::TILE, kw, kd);
                if (lane == 0) mbar_arrive(&k_full[b]);
                if (t + 1 < n_tiles) fetch(t + 1, a.c.k, a.c.ks, kw, kd);
                if (t >= 2 && !mbar_wait(&v_empty[b], ((t >> 1) - 1) & 1)) { atomicExch(failed, 1); break; }
                write(sm + L::OFF_V + b * L::TILE, vw, vd);
                if (lane == 0) mbar_arrive(&v_full[b]);
                if (t + 1 < n_tiles) fetch(t + 1, a.c.v, a.c.vs, vw, vd);
            }
        } else {
            constexpr uint32_t CARRY = BF16 ? 0x00800080u : 0x04000400u;      // carries out of an exponent of ones
            // every tile is waited for and given back, so that no stage gets two phases ahead of these warps
            for (int t = 0; t < n_tiles; t++) {
                const int b = t & 1, ph = (t >> 1) & 1;
                if (!mbar_wait(&v_full[b], ph)) { atomicExch(failed, 1); break; }
                if (!masked(t)) {
                    if (lane == 0) mbar_arrive(&v_empty[b]);
                    continue;
                }
                if (!mbar_wait(&k_full[b], ph)) { atomicExch(failed, 1); break; }
                uint8_t* v = sm + L::OFF_V + b * L::TILE + id * 128;
                uint32_t odd = 0;
#pragma unroll
                for (int c = 0; c < D / 8; c++) {
                    const uint4 w = *reinterpret_cast<const uint4*>(v + (c >> 3) * ATOM_BYTES + (((c & 7) ^ (id & 7)) << 4));
                    odd |= ((w.x & 0x7fff7fffu) + CARRY) | ((w.y & 0x7fff7fffu) + CARRY) | ((w.z & 0x7fff7fffu) + CARRY) | ((w.w & 0x7fff7fffu) + CARRY);
                }
                if (odd & 0x80008000u) {
#pragma unroll 1
                    for (int c = 0; c < D / 8; c++) *reinterpret_cast<uint4*>(v + (c >> 3) * ATOM_BYTES + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint32_t*>(sm + L::OFF_K + b * L::TILE + id * 128) = 0x7fff7fffu;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&looked[b]);
                    mbar_arrive(&v_empty[b]);
                }
            }
        }
    } else {
        set_registers_up<SOFTMAX_REGS>();
        if (wg == 0 || two) {
            const int r = threadIdx.x & 127, token = wg * tokens + r / group, head = kvh * group + r % group;
            const bool live = r / group < tokens && token < tile.rows;
            const int qp = min(tile.pos + token, q_hi), lo = first_key(qp, 0, a.window);
            const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16, s_at = tmem + lane_base + 128 * wg, o_at = tmem + lane_base + 256 + 128 * wg;
            const float mult = a.softcap > 0.f ? 1.f : fmaxf(fabsf(a.scale) * LOG2E, 1e-37f),      // not zero: masked scores are -inf times this
                         cap2 = a.softcap * LOG2E, inv_cap = a.softcap > 0.f ? fabsf(a.scale) / a.softcap : 0.f;
            float m = -INFINITY, l = 0.f;                // reference of the exponents, of two; sum
            bool ok = true;
            for (int t = 0; t < n_tiles; t++) {
                const int n0 = (tile.k_lo + t) * BKV;
                if (!mbar_wait(&s_full[wg], t & 1)) { ok = false; break; }
                tc_fence_after();
                uint32_t v[BKV];
                tmem_ld64(s_at, v);
                tmem_ld64(s_at + 64, v + 64);
                if (a.softcap > 0.f) {
#pragma unroll
                    for (int j = 0; j < BKV; j++) v[j] = __float_as_uint(cap2 * tanh_exp(__uint_as_float(v[j]) * inv_cap));
                }
                if (masked(t)) {
                    const int hi = qp - n0, low = lo - n0;
#pragma unroll
                    for (int j = 0; j < BKV; j++)
                        if (j > hi || j < low) v[j] = 0xff800000u;
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < BKV; j += 4)
#pragma unroll
                    for (int i = 0; i < 4; i++) mx[i] = fmaxf(mx[i], __uint_as_float(v[j + i]));
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * mult;
                if (__any_sync(0xffffffffu, top > m + LAG)) {
                    const float next = fmaxf(m, top), f = next == -INFINITY ? 1.f : ex2(m - next);
                    m = next;
                    l *= f;
                    if (t > 0) {
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            uint32_t y[32];
                            tmem_ld32(o_at + c, y);
#pragma unroll
                            for (int j = 0; j < 32; j++) y[j] = __float_as_uint(__uint_as_float(y[j]) * f);
                            tmem_st32(o_at + c, y);
                        }
                    }
                }
                const float less = LIFT - (m == -INFINITY ? 0.f : m);
                const float2 mult2 = make_float2(mult, mult), less2 = make_float2(less, less);
                float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    uint32_t p[32];
#pragma unroll
                    for (int j = 0; j < 64; j += 2) {
                        const float2 e = fma2(make_float2(__uint_as_float(v[64 * half + j]), __uint_as_float(v[64 * half + j + 1])), mult2, less2);
                        const float2 w = make_float2(ex2(e.x), ex2(e.y));
                        sum = add2(sum, w);
                        p[j / 2] = pack2<BF16>(w.x, w.y);
                    }
                    tmem_st32(s_at + 32 * half, p);
                }
                l += sum.x + sum.y;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_ready[wg]);
            }
            if (ok && n_tiles > 0 && !mbar_wait(&o_full[wg], 0)) ok = false;
            if (!ok) atomicExch(failed, 1);
            tc_fence_after();
            if (ok) {
                const bool whole = tile.part < 0;
                float inv = 1.f;
                if (whole) {
                    if (a.sinks) l += ex2(a.sinks[head] * LOG2E - (m - LIFT));
                    inv = 1.f / l;
                }
                const size_t part = ((size_t)(whole ? 0 : tile.part) * a.kv_heads + kvh) * (2 * BQ) + wg * BQ + r;
                const size_t at = (size_t)(tile.row + token) * a.ldo + (size_t)head * D;
                if (!whole && live) a.part_ml[part] = make_float2(m - LIFT, l);
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t y[32];
                    tmem_ld32(o_at + c, y);
                    if (!live) continue;
                    float z[32];
#pragma unroll
                    for (int j = 0; j < 32; j++) z[j] = __uint_as_float(y[j]) * inv;
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {
                        if (whole) store8(a.out, a.out_type, at + c + j, z + j);
                        else store8(a.part_acc, 0, part * D + c + j, z + j);
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
    if (threadIdx.x == 0 && *failed) atomicExch(&g_packed_status, KS_TIMEOUT);
}

// Adds up the parts of query tiles: grid (tiles, KV heads, runs of 8 rows), a warp a row.
template <int D>
__global__ void __launch_bounds__(256) packed_merge_kernel(const __grid_constant__ PackedArgs a) {
    constexpr int N = D / 32;
    pdl_launch();
    pdl_wait();
    const PackedMerge u = a.merges[blockIdx.x];
    const int group = a.n_heads / a.kv_heads, tokens = BQ / group, lane = threadIdx.x & 31, kvh = blockIdx.y;
    const int row = blockIdx.z * 8 + (threadIdx.x >> 5), tile = row >> 7, r = row & 127, token = tile * tokens + r / group;
    if (r / group >= tokens || token >= u.rows) return;
    const int head = kvh * group + r % group;
    const size_t step = (size_t)a.kv_heads * (2 * BQ), first = ((size_t)u.first * a.kv_heads + kvh) * (2 * BQ) + row;
    const float sink = a.sinks ? a.sinks[head] * LOG2E : -INFINITY;
    float m = -INFINITY;
    for (int p = lane; p < u.parts; p += 32) m = fmaxf(m, a.part_ml[first + p * step].x);
    m = fmaxf(warp_max(m), sink);
    const float ref = m == -INFINITY ? 0.f : m;
    float acc[N], l = sink > -INFINITY ? ex2(sink - ref) : 0.f;
#pragma unroll
    for (int j = 0; j < N; j++) acc[j] = 0.f;
#pragma unroll 4
    for (int p = 0; p < u.parts; p++) {
        const float2 ml = a.part_ml[first + p * step];
        const float f = ex2(ml.x - ref);
        l += ml.y * f;
        const float* from = a.part_acc + (first + p * step) * D + N * lane;
        if constexpr (N == 4) {
            const float4 y = __ldcg(reinterpret_cast<const float4*>(from));
            acc[0] += y.x * f; acc[1] += y.y * f; acc[2] += y.z * f; acc[3] += y.w * f;
        } else {
            const float2 y = __ldcg(reinterpret_cast<const float2*>(from));
            acc[0] += y.x * f; acc[1] += y.y * f;
        }
    }
    const float inv = 1.f / l;
    const size_t at = (size_t)(u.row + token) * a.ldo + (size_t)head * D + N * lane;
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        const float x = acc[j] * inv, y = acc[j + 1] * inv;
        if (a.out_type == 0) *reinterpret_cast<float2*>((float*)a.out + at + j) = make_float2(x, y);
        else *reinterpret_cast<uint32_t*>((uint16_t*)a.out + at + j) = a.out_type == 1 ? pack2<false>(x, y) : pack2<true>(x, y);
    }
}

// Rows [slots][kv_heads][n][D] of 16-bit elements, D together; boxes of 64 columns x 128 rows, 128-byte swizzle, rows behind the last read as zero.
bool rows_map(CUtensorMap* map, const void* base, const PackedArgs& a, long long slot, long long head, long long row) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[4] = {(cuuint64_t)a.hd, (cuuint64_t)a.n, (cuuint64_t)a.kv_heads, (cuuint64_t)a.slots};
    cuuint64_t strides[3] = {(cuuint64_t)row * 2, (cuuint64_t)head * 2, (cuuint64_t)slot * 2};
    cuuint32_t box[4] = {64u, (cuuint32_t)BKV, 1u, 1u};
    cuuint32_t ones[4] = {1, 1, 1, 1};
    return fn(map, a.kv_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D>
const void* kernel_of(int form) {
    return form == F16 ? (const void*)packed_kernel<D, F16> : form == B16 ? (const void*)packed_kernel<D, B16> : (const void*)packed_kernel<D, CODES>;
}

}  // namespace

// One launch, two where some tile's keys are shared out.
B2_API int b2_attn_packed(const PackedArgs* in, int pdl, cudaStream_t st) {
    PackedArgs a = *in;
    const bool codes = a.k == nullptr;
    if (a.n_tiles == 0) return 0;
    if ((a.hd != 64 && a.hd != 128) || a.kv_heads < 1 || a.kv_heads > 65535 || a.n_heads < 1 || a.n_heads % a.kv_heads || a.n_heads / a.kv_heads > BQ || !a.q || !a.out || !a.tiles || a.n_tiles < 0 || a.window < 0 ||
        a.ldo < a.n_heads * a.hd || (((uintptr_t)a.q | (uintptr_t)a.out) & 15) || a.ldq % (a.q_type ? 8 : 4) || a.ldo % (a.out_type ? 8 : 4))
        return (int)cudaErrorInvalidValue;
    if (a.n_merges && (!a.merges || !a.part_acc || !a.part_ml || a.n_merges < 0)) return (int)cudaErrorInvalidValue;
    if (codes ? kv4_bad_cache(a.c) || a.c.hd != a.hd || a.c.kv_heads != a.kv_heads : !a.v || a.slots < 1 || a.n < 1) return (int)cudaErrorInvalidValue;
    CUtensorMap mk = {}, mv = {};
    if (!codes && (!rows_map(&mk, a.k, a, a.k_slot, a.k_head, a.k_row) || !rows_map(&mv, a.v, a, a.v_slot, a.v_head, a.v_row))) return (int)cudaErrorInvalidValue;
    static thread_local PerDeviceOnce once;
    if (once.first())
        for (int form = 0; form < 3; form++) {
            cudaError_t e = cudaFuncSetAttribute(kernel_of<64>(form), cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<64>::TOTAL);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel_of<128>(form), cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<128>::TOTAL);
            for (const void* fn : {kernel_of<64>(form), kernel_of<128>(form)}) {      // a block launched with fewer registers would wait for more of them
                cudaFuncAttributes at;
                if (e == cudaSuccess) e = cudaFuncGetAttributes(&at, fn);
                if (e == cudaSuccess && at.numRegs * 4 < 2 * SOFTMAX_REGS + MAKER_REGS + REST_REGS) e = cudaErrorLaunchOutOfResources;
            }
            if (e != cudaSuccess) return (int)e;
        }
    const int form = codes ? CODES : a.kv_bf16 ? B16 : F16;
    void* args[] = {&mk, &mv, &a};
    const int rc = a.hd == 128 ? launch_rows(kernel_of<128>(form), dim3(a.n_tiles, a.kv_heads), dim3(THREADS), Lay<128>::TOTAL, args, st, pdl)
                               : launch_rows(kernel_of<64>(form), dim3(a.n_tiles, a.kv_heads), dim3(THREADS), Lay<64>::TOTAL, args, st, pdl);
    if (rc || !a.n_merges) return rc;
    void* margs[] = {&a};
    return launch_rows(a.hd == 128 ? (const void*)packed_merge_kernel<128> : (const void*)packed_merge_kernel<64>, dim3(a.n_merges, a.kv_heads, 2 * BQ / 8), dim3(256), 0, margs, st, pdl);
}

// 0, or 1 once a wait has run out since the last call; synchronises.
B2_API int b2_attn_packed_status() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_packed_status, sizeof v) != cudaSuccess) return 1;
    if (v) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_packed_status, &zero, sizeof zero);
    }
    return v;
}
