// Causal attention of prompts of several sequences in one launch, on tcgen05 (sm_100a): over 16-bit keys and values of any layout, or over the 4-bit cache (kv4.cuh).
//
//   out[t][h] = sum_k p_k v_k / (sum_k p_k + exp(sink)),  p_k = exp(cap(scale q[t][h] . k)),  k the sequence's positions up to the token's own that its window has
//
// A CTA takes shares one after the other: two tiles of 128 query rows of one KV head and a run of keys; a row is a token's query head (token / group, head of the group), so all heads of a group share the keys that the CTA brings, and few
// tokens of many heads still fill a tile.  Keys come in tiles of 128.  Roles: warps 0-3 and 4-7 the softmax of a tile each, a row a thread (no exchange between threads); warp 8 loads; warp 9
// issues the products; warps 12-15 make operands: queries, of a 4-bit cache also keys and values, whose codes they turn into f16 rows in the swizzled layout; of 16-bit rows they look at tiles whose
// mask is not whole (below).  Nothing waits for a share's results to be written but the next share's first P V.
// Tensor memory: S of both tiles (128 columns each, over whose first 64 the weights are written as 16-bit operands), O of both, accumulated there.  One tile's products run under the other's softmax, and P V
// of keys 0 .. 63 while the weights of the others are still being made.  The weights are relative to a reference that follows a row's largest score only when that exceeds it by 2^8
// (then the thread rescales its row of O: the product before is complete by the time a tile's scores are), and count from 2^6 on, so that f16 weights keep 20 powers of two below the largest.
// Tiles that not every row sees as a whole (the diagonal, a window's edge, the end) hold keys that must not count whatever they are, and a weight of zero times a value that is no number is
// none either: in such tiles of 16-bit rows, values rows with such elements become zeros and their keys none, so that exactly the rows that see them have no result.  Cached codes are finite.
// The host deals the shares out to as many CTAs as SMs (plan in ops/kv4_call.cpp); where whole tiles would leave SMs without work, keys of some are cut, and a second launch adds up the parts.
#include "attn_tc.cuh"
#include "kv4.cuh"

bool kv4_bad_cache(const Cache4& c);

__device__ int g_packed_status = 0;

namespace {

using namespace tc;

constexpr int BQ = 128, BKV = 128, ATOM_BYTES = 128 * 128;
constexpr int THREADS = 512;
// registers: 512 threads start with 128 each; two softmax warpgroups, the one that makes operands, the one that loads and multiplies
constexpr int SOFTMAX_REGS = 184, MAKER_REGS = 104, REST_REGS = 40;
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
// Products and commits of a whole warp, one lane of which issues (`one`).  The warp stays together, so descriptors are in uniform registers: issued from a branch of one lane, the products of a
// tile took 4500 cycles for what the tensor cores do in 2000.
__device__ __forceinline__ uint32_t elect() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one;
}
__device__ __forceinline__ void mma_ss(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(one) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t one, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(one) : "memory");
}
__device__ __forceinline__ void commit(uint32_t one, uint64_t* bar) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)), "r"(one) : "memory");
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

// 32 bytes at once: rows of one thread each fill whole sectors
__device__ __forceinline__ void store32(void* to, const uint32_t (&w)[8], bool aligned) {
    if (aligned) {
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
    } else {
        reinterpret_cast<uint4*>(to)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4*>(to)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}
// 16 values of a result row
__device__ __forceinline__ void store16(void* out, int type, size_t at, const float* y, bool aligned) {
    uint32_t w[8];
    if (type == 0) {
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = __float_as_uint(y[i]);
        store32((float*)out + at, w, aligned);
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = __float_as_uint(y[8 + i]);
        store32((float*)out + at + 8, w, aligned);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = type == 1 ? pack2<false>(y[2 * i], y[2 * i + 1]) : pack2<true>(y[2 * i], y[2 * i + 1]);
        store32((uint16_t*)out + at, w, aligned);
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
    uint64_t* k_full = bars;             // of the stages
    uint64_t* k_empty = bars + 2;
    uint64_t* v_full = bars + 4;
    uint64_t* v_empty = bars + 6;
    uint64_t* looked = bars + 8;
    uint64_t* s_full = bars + 10;        // of tiles A and B
    uint64_t* p_half = bars + 12;        // weights of keys 0 .. 63 are there; all are:
    uint64_t* p_ready = bars + 14;
    uint64_t* o_full = bars + 16;
    uint64_t* o_empty = bars + 18;
    uint64_t* q_full = bars + 20;
    uint64_t* q_empty = bars + 21;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 22);
    int* failed = reinterpret_cast<int*>(bars + 23);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wg = warp >> 2;
    pdl_wait();
    const int group = a.n_heads / a.kv_heads, tokens = BQ / group;          // tokens of a tile
    const int behind = a.starts[blockIdx.x], shares = a.starts[blockIdx.x + 1] - behind + 1;
    // whether some row does not see all of the keys from n0 on
    auto masked = [&](const PackedTile& x, int n0) { return n0 + BKV - 1 > x.pos || n0 < first_key(x.pos + x.rows - 1, 0, a.window); };
    // keys or values of 16-bit rows, the nth tile of this CTA
    auto load = [&](const PackedTile& x, uint64_t* full, const CUtensorMap* map, int off, int t, int nth) {
        const int b = nth & 1, y = x.base + t * BKV;
        mbar_expect_tx(&full[b], L::TILE);
#pragma unroll
        for (int i = 0; i < ATOMS; i++) tma_load_4d(sm + off + b * L::TILE + i * ATOM_BYTES, map, 64 * i, y, x.kvh, x.slot, &full[b]);
    };

    // Query rows of a share as 16-bit operands, 16 bytes a thread at a time: copied where they are of the operands' type and taken as they are.
    const uint32_t per = (65536u + group - 1) / group;      // r / group = r * per >> 16 for r < 128
    auto queries = [&](const PackedTile& u, int id, int threads) {
        constexpr int PIECES = D / 8, BATCH = 8;
        const int steps = (u.rows > tokens ? 2 : 1) * BQ * PIECES / threads;      // a multiple of BATCH / 2
        const bool as_is = a.q_type == (BF16 ? 2 : 1) && a.scale >= 0.f;
        auto place = [&](int s, const void*& from, bool& live) {      // where the sth piece goes to and comes from
            const int idx = id + s * threads, c = idx % PIECES, r = idx / PIECES & 127, x = idx / (PIECES * BQ), of = r * per >> 16, token = x * tokens + of;
            live = of < tokens && token < u.rows;
            from = (const char*)a.q + ((size_t)(u.row + (live ? token : 0)) * a.ldq + (size_t)(u.kvh * group + (live ? r - of * group : 0)) * D + 8 * c) * (a.q_type ? 2 : 4);
            return sm + x * L::TILE + (c >> 3) * ATOM_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4);
        };
        if (as_is) {
#pragma unroll 4
            for (int s = 0; s < steps; s++) {
                const void* from;
                bool live;
                uint8_t* to = place(s, from, live);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(live ? 16 : 0) : "memory");
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else {
#pragma unroll 1
            for (int s0 = 0; s0 < steps; s0 += BATCH / 2) {
                uint4 w[BATCH];
#pragma unroll
                for (int s = 0; s < BATCH / 2; s++) {
                    const void* from;
                    bool live;
                    place(s0 + s, from, live);
                    w[2 * s] = w[2 * s + 1] = make_uint4(0, 0, 0, 0);
                    if (live) {
                        w[2 * s] = ((const uint4*)from)[0];
                        if (a.q_type == 0) w[2 * s + 1] = ((const uint4*)from)[1];
                    }
                }
#pragma unroll
                for (int s = 0; s < BATCH / 2; s++) {
                    const void* from;
                    bool live;
                    uint8_t* to = place(s0 + s, from, live);
                    const uint32_t z[8] = {w[2 * s].x, w[2 * s].y, w[2 * s].z, w[2 * s].w, w[2 * s + 1].x, w[2 * s + 1].y, w[2 * s + 1].z, w[2 * s + 1].w};
                    uint32_t y[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float2 f = a.q_type == 0   ? make_float2(__uint_as_float(z[2 * j]), __uint_as_float(z[2 * j + 1]))
                                         : a.q_type == 1 ? __half22float2(*reinterpret_cast<const __half2*>(&z[j]))
                                                         : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&z[j]));
                        y[j] = pack2<BF16>(f.x, f.y) ^ (a.scale < 0.f ? 0x80008000u : 0u);
                    }
                    *reinterpret_cast<uint4*>(to) = make_uint4(y[0], y[1], y[2], y[3]);
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    };
    const PackedTile u0 = a.tiles[blockIdx.x];
    auto share = [&](int i) { return i == 0 ? u0 : a.tiles[behind + i - 1]; };

    if (warp == 8 && lane == 0) {        // the loading thread makes the barriers and asks for the first tiles before anything else
        *failed = 0;
        for (int b = 0; b < 2; b++) {
            mbar_init(&k_full[b], FORM == CODES ? 4 : 1);
            mbar_init(&k_empty[b], 1);
            mbar_init(&v_full[b], FORM == CODES ? 4 : 1);
            mbar_init(&v_empty[b], FORM == CODES ? 1 : 5);      // the products, and the warps that look at values
            mbar_init(&looked[b], 4);
            mbar_init(&s_full[b], 1);
            mbar_init(&p_half[b], 4);
            mbar_init(&p_ready[b], 4);
            mbar_init(&o_full[b], 1);
            mbar_init(&o_empty[b], 4);
        }
        mbar_init(q_full, 4);
        mbar_init(q_empty, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (FORM != CODES) {
            load(u0, k_full, &map_k, L::OFF_K, u0.k_lo, 0);
            load(u0, v_full, &map_v, L::OFF_V, u0.k_lo, 0);
        }
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    queries(u0, threadIdx.x, THREADS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch();

    if (wg == 2) {
        set_registers_down<REST_REGS>();
        if (FORM != CODES && warp == 8 && lane == 0) {
            int nth = 0;
            bool ok = true;
            for (int i = 0; i < shares && ok; i++) {
                const PackedTile x = share(i);
                for (int t = x.k_lo; t < x.k_hi; t++, nth++) {
                    const int b = nth & 1, ph = ((nth >> 1) - 1) & 1;
                    if (nth == 0) continue;
                    if (nth >= 2 && !mbar_wait(&k_empty[b], ph)) { ok = false; break; }
                    load(x, k_full, &map_k, L::OFF_K, t, nth);
                    if (nth >= 2 && !mbar_wait(&v_empty[b], ph)) { ok = false; break; }
                    load(x, v_full, &map_v, L::OFF_V, t, nth);
                }
            }
            if (!ok) atomicExch(failed, 1);
        } else if (warp == 9) {
            const uint32_t one = elect();
            const uint32_t id_s = idesc(BF16, BKV, 0), id_o = idesc(BF16, D, 1);
            bool ok = true;
            uint32_t looks = 0;          // bit b: parity of the tiles of stage b that were looked at
            uint32_t sp = 0, op = 0;     // bit x: parity of the scores, of the results of tile x
            int nth = 0;
            auto expect = [&](uint64_t* bar, int parity) {
                if (!mbar_wait(bar, parity)) ok = false;
                tc_fence_after();
            };
            auto wait_k = [&](int at, bool look) {
                const int b = at & 1;
                expect(&k_full[b], (at >> 1) & 1);
                if (look) {
                    expect(&looked[b], looks >> b & 1);
                    looks ^= 1u << b;
                }
            };
            auto scores = [&](int x, int at) {
#pragma unroll
                for (int i = 0; i < ATOMS; i++) {
                    const uint64_t qd = umma_desc(sm + x * L::TILE + i * ATOM_BYTES), kd = umma_desc(sm + L::OFF_K + (at & 1) * L::TILE + i * ATOM_BYTES);
#pragma unroll
                    for (int k = 0; k < 4; k++) mma_ss(one, tmem + 128 * x, qd + 2 * k, kd + 2 * k, id_s, (i | k) != 0);
                }
                commit(one, &s_full[x]);
            };
            auto values = [&](int x, int at, int half, bool more) {
                const uint8_t* vt = sm + L::OFF_V + (at & 1) * L::TILE;
#pragma unroll
                for (int k = 4 * half; k < 4 * half + 4; k++)
                    mma_ts(one, tmem + 256 + 128 * x, tmem + 128 * x + 8 * k, umma_desc_mn(vt + k * 16 * 128, ATOM_BYTES), id_o, more || k != 0);
            };
            PackedTile next = u0;
            for (int i = 0; i < shares && ok; i++) {
                const PackedTile u = next;
                if (i + 1 < shares) next = share(i + 1);
                const int n_tiles = u.k_hi - u.k_lo, n_x = u.rows > tokens ? 2 : 1;
                auto looks_at = [&](int t) { return FORM != CODES && masked(u, (u.k_lo + t) * BKV); };
                if (i) expect(q_full, (i - 1) & 1);      // (the first share's queries were there before)
                if (ok) wait_k(nth, looks_at(0));
                if (!ok) break;
                for (int x = 0; x < n_x; x++) scores(x, nth);
                commit(one, &k_empty[nth & 1]);
                if (n_tiles == 1) commit(one, q_empty);
                for (int t = 0; t < n_tiles && ok; t++, nth++) {
                    const bool more = t + 1 < n_tiles, look = more && looks_at(t + 1);
                    if (more && !look) wait_k(nth + 1, false);      // (tiles that are looked at come later: their scores are not waited for ahead of this tile's values)
                    for (int x = 0; x < n_x && ok; x++) {
                        if (x == 0) expect(&v_full[nth & 1], (nth >> 1) & 1);
                        if (t == 0) {      // the result before has been read: the first one finds the place empty
                            expect(&o_empty[x], op >> x & 1 ^ 1);
                            op ^= 1u << x;
                        }
                        expect(&p_half[x], sp >> x & 1);
                        if (!ok) break;
                        values(x, nth, 0, t > 0);
                        expect(&p_ready[x], sp >> x & 1);
                        sp ^= 1u << x;
                        if (!ok) break;
                        values(x, nth, 1, true);
                        if (more) {
                            if (look && x == 0) wait_k(nth + 1, true);
                            if (!ok) break;
                            scores(x, nth + 1);
                        } else {
                            commit(one, &o_full[x]);
                        }
                    }
                    commit(one, &v_empty[nth & 1]);
                    if (more) commit(one, &k_empty[(nth + 1) & 1]);
                    if (t + 2 == n_tiles) commit(one, q_empty);
                }
            }
            if (!ok && lane == 0) atomicExch(failed, 1);
        }
    } else if (wg == 3) {
        set_registers_down<MAKER_REGS>();
        const int id = threadIdx.x & 127;
        bool ok = true;
        auto next_queries = [&](const PackedTile& u, int i) {
            if (i == 0) return true;
            if (!mbar_wait(q_empty, (i - 1) & 1)) return false;
            queries(u, id, 128);
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
            return true;
        };
        int nth = 0;
        if (FORM == CODES) {
            // a thread takes 16 bytes of codes of every 32nd row (D = 128; of every 64th: D = 64); the rows of eight lanes are such that their stores go to different banks
            constexpr int NB = D / 32, PIECES = D / 32, PASSES = PIECES, STEP = BKV / PASSES;      // 16-byte pieces of a row; rows of a pass
            const int piece = id % PIECES, i8 = id / PIECES;
            const int row = D == 128 ? (i8 & ~7) | (i8 & 1) << 2 | (i8 >> 1 & 3) : (i8 & ~7) | (i8 & 1) | (i8 >> 1 & 1) << 2 | (i8 >> 2 & 1) << 1;
            uint4 kw[PASSES], vw[PASSES];
            uint2 kd[PASSES], vd[PASSES];
            // rows behind the portion repeat its last: their keys are masked
            auto fetch = [&](const PackedTile& u, int t, const uint8_t* codes, const void* scales, uint4 (&w)[PASSES], uint2 (&d)[PASSES]) {
                const size_t row0 = kv4::row_of(a.c, u.base, u.slot, u.kvh);
#pragma unroll
                for (int p = 0; p < PASSES; p++) {
                    const size_t at = row0 + min(t * BKV + p * STEP + row, u.pos + u.rows - 1);
                    w[p] = ldg16(codes + at * (D / 2) + 16 * piece);
                    if (D == 128) d[p] = ldg8((const uint8_t*)scales + at * 8);
                    else d[p].x = __ldg((const uint32_t*)scales + at);
                }
            };
            auto write = [&](uint8_t* to, const uint4 (&w)[PASSES], const uint2 (&d)[PASSES]) {
#pragma unroll
                for (int p = 0; p < PASSES; p++) {
                    const uint32_t z[4] = {w[p].x, w[p].y, w[p].z, w[p].w};
                    const int rr = p * STEP + row;
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const int b = q % NB, j = D == 128 ? piece : 2 * piece + q / NB, chunk = 4 * b + j;      // columns 32 b + 8 j ..
                        const uint32_t pair = b >> 1 ? d[p].y : d[p].x, dd = __byte_perm(pair, 0, b & 1 ? 0x3232 : 0x1010);
                        uint32_t e[4];
                        kv4::expand(z[q], e);
#pragma unroll
                        for (int x = 0; x < 4; x++) e[x] = kv4::hmul2_bits(e[x], dd);
                        *reinterpret_cast<uint4*>(to + (chunk >> 3) * ATOM_BYTES + rr * 128 + (((chunk & 7) ^ (rr & 7)) << 4)) = make_uint4(e[0], e[1], e[2], e[3]);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            };
            PackedTile u = u0;
            fetch(u, u.k_lo, a.c.k, a.c.ks, kw, kd);
            fetch(u, u.k_lo, a.c.v, a.c.vs, vw, vd);
            for (int i = 0; i < shares && ok; i++) {
                PackedTile next = u;
                if (i + 1 < shares) next = share(i + 1);
                for (int t = u.k_lo; t < u.k_hi && ok; t++, nth++) {
                    const int b = nth & 1, ph = ((nth >> 1) - 1) & 1;
                    const bool more = t + 1 < u.k_hi, any = more || i + 1 < shares;
                    if (nth >= 2 && !mbar_wait(&k_empty[b], ph)) { ok = false; break; }
                    write(sm + L::OFF_K + b * L::TILE, kw, kd);
                    if (lane == 0) mbar_arrive(&k_full[b]);
                    if (t == u.k_lo && !next_queries(u, i)) { ok = false; break; }
                    if (any) fetch(more ? u : next, more ? t + 1 : next.k_lo, a.c.k, a.c.ks, kw, kd);
                    if (nth >= 2 && !mbar_wait(&v_empty[b], ph)) { ok = false; break; }
                    write(sm + L::OFF_V + b * L::TILE, vw, vd);
                    if (lane == 0) mbar_arrive(&v_full[b]);
                    if (any) fetch(more ? u : next, more ? t + 1 : next.k_lo, a.c.v, a.c.vs, vw, vd);
                }
                u = next;
            }
        } else {
            constexpr uint32_t CARRY = BF16 ? 0x00800080u : 0x04000400u;      // carries out of an exponent of ones
            for (int i = 0; i < shares && ok; i++) {
                const PackedTile u = share(i);
                if (!next_queries(u, i)) { ok = false; break; }
                // every tile is waited for and given back, so that no stage gets two phases ahead of these warps
                for (int t = u.k_lo; t < u.k_hi && ok; t++, nth++) {
                    const int b = nth & 1, ph = (nth >> 1) & 1;
                    if (!mbar_wait(&v_full[b], ph)) { ok = false; break; }
                    if (!masked(u, t * BKV)) {
                        if (lane == 0) mbar_arrive(&v_empty[b]);
                        continue;
                    }
                    if (!mbar_wait(&k_full[b], ph)) { ok = false; break; }
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
        }
        if (!ok) atomicExch(failed, 1);
    } else {
        set_registers_up<SOFTMAX_REGS>();
        const int r = threadIdx.x & 127, of = r / group, token = wg * tokens + of;
        const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16, s_at = tmem + lane_base + 128 * wg, o_at = tmem + lane_base + 256 + 128 * wg;
        const float mult = a.softcap > 0.f ? 1.f : fmaxf(fabsf(a.scale) * LOG2E, 1e-37f),      // not zero: masked scores are -inf times this
                    cap2 = a.softcap * LOG2E, inv_cap = a.softcap > 0.f ? fabsf(a.scale) / a.softcap : 0.f;
        const bool aligned = ((uintptr_t)a.out & 31) == 0 && a.ldo % (a.out_type ? 16 : 8) == 0;
        bool ok = true;
        uint32_t sp = 0, op = 0;
        for (int i = 0; i < shares && ok; i++) {
            const PackedTile u = share(i);
            if (wg == 1 && u.rows <= tokens) continue;
            const bool live = of < tokens && token < u.rows;
            const int qp = min(u.pos + token, u.pos + u.rows - 1), lo = first_key(qp, 0, a.window), head = u.kvh * group + r - of * group;
            float m = -INFINITY, l = 0.f;                // reference of the exponents, of two; sum
            for (int t = u.k_lo; t < u.k_hi; t++) {
                if (!mbar_wait(&s_full[wg], sp)) { ok = false; break; }
                sp ^= 1;
                tc_fence_after();
                uint32_t v[BKV];
                tmem_ld64(s_at, v);
                tmem_ld64(s_at + 64, v + 64);
                if (a.softcap > 0.f) {
#pragma unroll
                    for (int j = 0; j < BKV; j++) v[j] = __float_as_uint(cap2 * tanh_exp(__uint_as_float(v[j]) * inv_cap));
                }
                if (masked(u, t * BKV)) {
                    const int hi = qp - t * BKV, low = lo - t * BKV;
#pragma unroll
                    for (int j = 0; j < BKV; j++)
                        if (j > hi || j < low) v[j] = 0xff800000u;
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < BKV; j += 8)
#pragma unroll
                    for (int e = 0; e < 4; e++) mx[e] = fmaxf(fmaxf(mx[e], __uint_as_float(v[j + e])), __uint_as_float(v[j + 4 + e]));
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * mult;
                if (__any_sync(0xffffffffu, top > m + LAG)) {
                    const float to = fmaxf(m, top), f = to == -INFINITY ? 1.f : ex2(m - to);
                    m = to;
                    l *= f;
                    if (t > u.k_lo) {
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
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(half ? &p_ready[wg] : &p_half[wg]);
                }
                l += sum.x + sum.y;
            }
            if (ok && !mbar_wait(&o_full[wg], op)) ok = false;
            op ^= 1;
            if (!ok) break;
            tc_fence_after();
            const bool whole = u.part < 0;
            float inv = 1.f;
            if (whole) {
                if (a.sinks) l += ex2(a.sinks[head] * LOG2E - (m - LIFT));
                inv = 1.f / l;
            }
            const size_t part = (size_t)(whole ? 0 : u.part) * (2 * BQ) + wg * BQ + r;
            const size_t at = (size_t)(u.row + token) * a.ldo + (size_t)head * D;
            if (!whole && live) a.part_ml[part] = make_float2(m - LIFT, l);
#pragma unroll
            for (int c = 0; c < D; c += 64) {
                uint32_t y[64];
                tmem_ld64(o_at + c, y);
                if (c + 64 == D) {       // all of it has been read
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&o_empty[wg]);
                }
                if (live) {
#pragma unroll
                    for (int j = 0; j < 64; j += 16) {
                        float z[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) z[e] = __uint_as_float(y[j + e]) * inv;
                        if (whole) store16(a.out, a.out_type, at + c + j, z, aligned);
                        else store16(a.part_acc, 0, part * D + c + j, z, true);
                    }
                }
                __syncwarp();
            }
        }
        if (!ok) atomicExch(failed, 1);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
    if (threadIdx.x == 0 && *failed) atomicExch(&g_packed_status, KS_TIMEOUT);
}

// Adds up the parts of query tiles: grid (tiles, runs of 8 rows), a warp a row.
template <int D>
__global__ void __launch_bounds__(256) packed_merge_kernel(const __grid_constant__ PackedArgs a) {
    constexpr int N = D / 32;
    pdl_launch();
    pdl_wait();
    const PackedMerge u = a.merges[blockIdx.x];
    const int group = a.n_heads / a.kv_heads, tokens = BQ / group, lane = threadIdx.x & 31, kvh = u.kvh;
    const int row = blockIdx.y * 8 + (threadIdx.x >> 5), tile = row >> 7, r = row & 127, token = tile * tokens + r / group;
    if (r / group >= tokens || token >= u.rows) return;
    const int head = kvh * group + r % group;
    const size_t step = 2 * BQ, first = (size_t)u.first * step + row;
    const float sink = a.sinks ? a.sinks[head] * LOG2E : -INFINITY;
    float m = -INFINITY;
    for (int p = lane; p < u.parts; p += 32) m = fmaxf(m, a.part_ml[first + p * step].x);
    m = fmaxf(warp_max(m), sink);
    const float ref = m == -INFINITY ? 0.f : m;
    float acc[N], l = sink > -INFINITY ? ex2(sink - ref) : 0.f;
#pragma unroll
    for (int j = 0; j < N; j++) acc[j] = 0.f;
#pragma unroll 8
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
    if (a.ctas == 0) return 0;
    if ((a.hd != 64 && a.hd != 128) || a.kv_heads < 1 || a.kv_heads > 65535 || a.n_heads < 1 || a.n_heads % a.kv_heads || a.n_heads / a.kv_heads > BQ || !a.q || !a.out || !a.tiles || !a.starts || a.ctas < 0 || a.window < 0 ||
        a.ldo < a.n_heads * a.hd || (((uintptr_t)a.q | (uintptr_t)a.out) & 15) || a.ldq % (a.q_type ? 8 : 4) || a.ldo % (a.out_type ? 8 : 4))
        return (int)cudaErrorInvalidValue;
    if (a.n_merges && (!a.merges || !a.part_acc || !a.part_ml || a.n_merges < 0 || ((uintptr_t)a.part_acc & 31))) return (int)cudaErrorInvalidValue;
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
    const int rc = a.hd == 128 ? launch_rows(kernel_of<128>(form), dim3(a.ctas), dim3(THREADS), Lay<128>::TOTAL, args, st, pdl)
                               : launch_rows(kernel_of<64>(form), dim3(a.ctas), dim3(THREADS), Lay<64>::TOTAL, args, st, pdl);
    if (rc || !a.n_merges) return rc;
    void* margs[] = {&a};      // (its CTAs may wait beside the first launch's last)
    return launch_rows(a.hd == 128 ? (const void*)packed_merge_kernel<128> : (const void*)packed_merge_kernel<64>, dim3(a.n_merges, 2 * BQ / 8), dim3(256), 0, margs, st, 1);
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
