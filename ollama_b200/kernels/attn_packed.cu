// Causal attention of prompts of several sequences in one launch, on tcgen05 (sm_100a): over 16-bit keys and values of any layout, or over the 4-bit cache (kv4.cuh).
//
//   out[t][h] = sum_k p_k v_k / (sum_k p_k + exp(sink)),  p_k = exp(cap(scale q[t][h] . k)),  k the sequence's positions up to the token's own that its window has
//
// A CTA takes shares one after the other: two tiles of 128 query rows of one KV head and a run of keys; a row is a token's query head (token / group, head of the group), so all heads of a group
// share the keys that the CTA brings, and few tokens of many heads still fill a tile.  Keys come in tiles of 128.  Roles: warps 0-3 and 4-7 the softmax of a tile each, a row a thread (no exchange
// between threads); warp 8 loads keys and values, warp 10 queries; warp 9 issues the products; warps 12-15 make operands: queries that are not of the operands' type, of a 4-bit cache also keys and
// values, whose codes they turn into f16 rows in the swizzled layout; of 16-bit rows they look at tiles whose mask is not whole (below).  The next share's first scores are computed behind the last
// products of this one; nothing waits for a share's results to be written but the next one's first P V.
// Tensor memory: S of both tiles (128 columns each, over whose first 64 the weights are written as 16-bit operands), O of both, accumulated there.  One tile's products run under the other's softmax, and P V
// of keys 0 .. 63 while the weights of the others are still being made.  The weights are relative to a reference that follows a row's largest score only when that exceeds it by 2^8
// (then the thread rescales its row of O: the product before is complete by the time a tile's scores are), and count from 2^6 on, so that f16 weights keep 20 powers of two below the largest (of bf16 rows
// weights are bf16: both operands of a product have one type).
// Tiles that not every row sees as a whole (the diagonal, a window's edge, the end) hold keys that must not count whatever they are, and a weight of zero times a value that is no number is
// none either: in such tiles of 16-bit rows, values rows with such elements become zeros and their keys none, so that exactly the rows that see them have no result.  Cached codes are finite.
// The host deals the shares out to as many CTAs as SMs (plan in ops/kv4_call.cpp); where whole tiles would leave SMs without work, keys of some are cut, and a second launch adds up the parts.
// What bounds it: the products of a tile of keys (2 x 128 rows, 128 columns) keep the tensor cores busy for 2048 cycles and its exponentials the units that make them for as many; a tile takes some
// 3500 in the middle of a share (1.9 us, 1.3 PFLOP/s on 148 SMs, where power allows 1.4 in a long product), since a row's scores, weights and products wait for one another and there is room for two rows
// of tiles only.  Both pipes are busy in 50 to 54% of all cycles; a share's ends cost 4.5 us more.  Measured, 32 heads on 8 of 128: 2048 rows behind 6144 cached keys 234 us, 1.03 PFLOP/s of what the mask
// leaves; five prompts of 4096 f16 rows 342, 1.05 (400 one after the other, under the power cap); 64 rows behind 30000 46.7; nine short ones 18.5. Of a tile's chain scores to weights are 2200 cycles and products 1100.
// Tried: exponentials as polynomials (12 % of them 350 us for 349, 37 % 364), scores in halves of 64 keys (3.6 us a tile), weights handed over as 96 and 32 keys (no difference).
#include "attn_tc.cuh"
#include "kv4.cuh"

bool kv4_bad_cache(const Cache4& c);

__device__ int g_packed_status = 0;

namespace {

using namespace tc;

constexpr int BQ = 128, BKV = 128, ATOM_BYTES = 128 * 128;
constexpr int THREADS = 512;
constexpr float LIFT = 6.f, LAG = 8.f, LOG2E = 1.4426950408889634f;
enum Form : int { F16 = 0, B16 = 1, CODES = 2 };

template <int D>
struct Lay {
    static constexpr int ATOMS = D / 64, TILE = ATOMS * ATOM_BYTES;
    static constexpr int OFF_K = 2 * TILE, OFF_V = OFF_K + 2 * TILE, OFF_OUT = OFF_V + 2 * TILE;
    static constexpr int OFF_BAR = OFF_OUT + 8 * 32 * 128, TOTAL = OFF_BAR + 256 + 1024;      // 32 rows of 128 bytes for each softmax warp's results
};

__device__ __forceinline__ uint32_t idesc(bool bf16, int n, int b_mn_major) { return idesc_f16(BQ, n, b_mn_major) | (bf16 ? (1u << 7) | (1u << 10) : 0u); }

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}
// 32 consecutive 32-bit columns of this thread's lane, without waiting for them, and the wait, which hands them on: what uses them comes behind it
__device__ __forceinline__ void tmem_ask32(uint32_t at, uint32_t (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(at));
}
__device__ __forceinline__ void tmem_have32(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])::"memory");
}
// 16 columns, not waited for
__device__ __forceinline__ void tmem_put16(uint32_t at, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void tmem_put_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Bounded like mbar_wait, in fewer instructions; the hint lets a thread sleep in the hardware.
__device__ __forceinline__ bool arrived(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
    for (int i = 0; i < 1 << 16; i++) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 20000;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
        if (ok) return true;
    }
    return false;
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
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    if (BF16) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&b);
    }
    return pack_h2(x, y);
}

template <int D, int FORM>
__global__ void __launch_bounds__(THREADS, 1) packed_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_q,
                                                                const __grid_constant__ PackedArgs a) {
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
    const int behind = a.starts[blockIdx.x], shares = min(max(a.starts[blockIdx.x + 1] - behind, 0), a.n_tiles) + 1;
    // whether some row does not see all of the keys from n0 on
    auto masked = [&](const PackedTile& x, int n0) { return n0 + BKV - 1 > x.pos || n0 < first_key(x.pos + x.rows - 1, 0, a.window); };
    // keys or values of 16-bit rows, the nth tile of this CTA
    auto load = [&](const PackedTile& x, uint64_t* full, const CUtensorMap* map, int off, int t, int nth) {
        const int b = nth & 1, y = x.base + t * BKV;
        mbar_expect_tx(&full[b], L::TILE);
#pragma unroll
        for (int i = 0; i < ATOMS; i++) tma_load_4d(sm + off + b * L::TILE + i * ATOM_BYTES, map, 64 * i, y, x.kvh, x.slot, &full[b]);
    };

    // Query rows of a share as 16-bit operands: those of the operands' type are copied, row token * group + head of a tile one after the other as a box of (64 columns, group heads, tokens) lays
    // them (rows behind the portion's are others', whose results nothing reads); others are rounded, 16 bytes a thread at a time.
    const uint32_t per = (65536u + group - 1) / group;      // r / group = r * per >> 16 for r < 128
    const bool as_is = a.q_type == (BF16 ? 2 : 1) && a.scale >= 0.f;
    auto copy_queries = [&](const PackedTile& u) {
        const int n_x = u.rows > tokens ? 2 : 1;
        mbar_expect_tx(q_full, n_x * tokens * group * D * 2);
        for (int x = 0; x < n_x; x++)
#pragma unroll
            for (int i = 0; i < ATOMS; i++)
                tma_load_3d(sm + x * L::TILE + i * ATOM_BYTES, &map_q, 64 * i, u.kvh * group, u.row + x * tokens, q_full);
    };
    auto round_queries = [&](const PackedTile& u, int id, int threads) {
        constexpr int PIECES = D / 8, BATCH = 4;
        const int steps = (u.rows > tokens ? 2 : 1) * BQ * PIECES / threads;
#pragma unroll 1
        for (int s0 = 0; s0 < steps; s0 += BATCH) {
            uint4 w[2 * BATCH];
            auto place = [&](int s, size_t& from) {      // where the sth piece goes to and comes from: whether there is one
                const int idx = id + (s0 + s) * threads, c = idx % PIECES, r = idx / PIECES & 127, x = idx / (PIECES * BQ), of = r * per >> 16, token = x * tokens + of;
                from = (size_t)(u.row + token) * a.ldq + (size_t)(u.kvh * group + r - of * group) * D + 8 * c;
                return of < tokens && token < u.rows ? x * L::TILE + (c >> 3) * ATOM_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4) : -1;
            };
#pragma unroll
            for (int s = 0; s < BATCH; s++) {
                size_t from;
                if (place(s, from) < 0) continue;
                const uint4* at = (const uint4*)((const char*)a.q + from * (a.q_type ? 2 : 4));
                w[2 * s] = at[0];
                if (a.q_type == 0) w[2 * s + 1] = at[1];
            }
#pragma unroll
            for (int s = 0; s < BATCH; s++) {
                size_t from;
                const int to = place(s, from);
                if (to < 0) continue;
                const uint32_t z[8] = {w[2 * s].x, w[2 * s].y, w[2 * s].z, w[2 * s].w, w[2 * s + 1].x, w[2 * s + 1].y, w[2 * s + 1].z, w[2 * s + 1].w};
                uint32_t y[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 f = a.q_type == 0   ? make_float2(__uint_as_float(z[2 * j]), __uint_as_float(z[2 * j + 1]))
                                     : a.q_type == 1 ? __half22float2(*reinterpret_cast<const __half2*>(&z[j]))
                                                     : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&z[j]));
                    y[j] = pack2<BF16>(f.x, f.y) ^ (a.scale < 0.f ? 0x80008000u : 0u);
                }
                *reinterpret_cast<uint4*>(sm + to) = make_uint4(y[0], y[1], y[2], y[3]);
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    };
    // Lists are on the device, so what they say is checked here: a tile that reaches beyond the queries, the cache or the partial results becomes one without rows, which writes nothing.
    auto tile_of = [&](int at) {
        PackedTile x = a.tiles[min(max(at, 0), a.n_tiles - 1)];
        const bool fits = x.row >= 0 && x.rows > 0 && x.rows <= 2 * tokens && x.row <= a.q_rows - x.rows && (unsigned)x.slot < (unsigned)a.slots && (unsigned)x.kvh < (unsigned)a.kv_heads && x.base >= 0 &&
                          x.pos >= 0 && x.base <= a.n - x.rows && x.pos <= a.n - x.rows - x.base && x.k_lo >= 0 && x.k_lo < x.k_hi && x.k_hi <= (x.pos + x.rows - 1) / BKV + 1 && x.part < a.parts;
        return fits ? x : PackedTile{0, 0, 0, 1, 0, 0, 1, -1, 0, {}};
    };
    const PackedTile u0 = tile_of(blockIdx.x);
    auto share = [&](int i) { return i == 0 ? u0 : tile_of(behind + i - 1); };

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
        mbar_init(q_full, as_is ? 1 : 4);
        mbar_init(q_empty, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (as_is) copy_queries(u0);
        if (FORM != CODES) {
            load(u0, k_full, &map_k, L::OFF_K, u0.k_lo, 0);
            load(u0, v_full, &map_v, L::OFF_V, u0.k_lo, 0);
        }
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (!as_is) round_queries(u0, threadIdx.x, THREADS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch();

    if (wg == 2) {
        if (FORM != CODES && warp == 8 && lane == 0) {
            int nth = 0;
            bool ok = true;
            for (int i = 0; i < shares && ok; i++) {
                const PackedTile x = share(i);
                for (int t = x.k_lo; t < x.k_hi; t++, nth++) {
                    const int b = nth & 1, ph = ((nth >> 1) - 1) & 1;
                    if (nth == 0) continue;
                    if (nth >= 2 && !arrived(&k_empty[b], ph)) { ok = false; break; }
                    load(x, k_full, &map_k, L::OFF_K, t, nth);
                    if (nth >= 2 && !arrived(&v_empty[b], ph)) { ok = false; break; }
                    load(x, v_full, &map_v, L::OFF_V, t, nth);
                }
            }
            if (!ok) atomicExch(failed, 1);
        } else if (warp == 10 && lane == 0 && as_is) {
            bool ok = true;
            for (int i = 1; i < shares && ok; i++) {
                const PackedTile u = share(i);
                if (arrived(q_empty, (i - 1) & 1)) copy_queries(u);
                else ok = false;
            }
            if (!ok) atomicExch(failed, 1);
        } else if (warp == 9) {
            // (with a warp for each tile the products of both interleave, and each chain waits for all of them: 2.3 us a tile of keys instead of 1.9)
            const uint32_t one = elect(), id_s = idesc(BF16, BKV, 0), id_o = idesc(BF16, D, 1);
            bool ok = true;
            uint32_t looks = 0;          // bit b: parity of the tiles of stage b that were looked at
            uint32_t sp = 0, op = 0;     // bit x: parity of the scores, of the results of tile x
            int nth = 0;
            auto expect = [&](uint64_t* bar, int parity) {
                if (!arrived(bar, parity)) ok = false;
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
                const uint64_t qd = umma_desc(sm + x * L::TILE), kd = umma_desc(sm + L::OFF_K + (at & 1) * L::TILE);
#pragma unroll
                for (int k = 0; k < D / 16; k++) mma_ss(one, tmem + 128 * x, qd + (k >> 2) * (ATOM_BYTES / 16) + 2 * (k & 3), kd + (k >> 2) * (ATOM_BYTES / 16) + 2 * (k & 3), id_s, k != 0);
                commit(one, &s_full[x]);
            };
            auto values = [&](int x, int at, int half, bool more) {
                const uint64_t vd = umma_desc_mn(sm + L::OFF_V + (at & 1) * L::TILE + half * 64 * 128, ATOM_BYTES);
#pragma unroll
                for (int k = 0; k < 4; k++) mma_ts(one, tmem + 256 + 128 * x, tmem + 128 * x + 32 * half + 8 * k, vd + k * (16 * 128 / 16), id_o, more || k != 0);
            };
            auto looks_at = [&](const PackedTile& y, int t) { return FORM != CODES && masked(y, (y.k_lo + t) * BKV); };
            PackedTile next = u0;
            for (int i = 0; i < shares && ok; i++) {
                const PackedTile u = next;
                if (i + 1 < shares) next = share(i + 1);
                const int n_tiles = u.k_hi - u.k_lo, n_x = u.rows > tokens ? 2 : 1;
                if (i == 0) {
                    if (as_is) expect(q_full, 0);      // (others were there before)
                    if (ok) wait_k(0, looks_at(u, 0));
                    if (!ok) break;
                    for (int x = 0; x < n_x; x++) scores(x, 0);
                    commit(one, &k_empty[0]);
                    if (n_tiles == 1) commit(one, q_empty);
                }
                for (int t = 0; t < n_tiles && ok; t++, nth++) {
                    // the tile behind this one, which may be the next share's first
                    const bool more = t + 1 < n_tiles, any = more || i + 1 < shares, look = any && (more ? looks_at(u, t + 1) : looks_at(next, 0));
                    const int n_then = more ? n_x : any ? (next.rows > tokens ? 2 : 1) : 0;
                    const bool late = look || !more;      // (tiles that are looked at, and queries, come late: their scores are not waited for ahead of this tile's values)
                    if (any && !late) wait_k(nth + 1, false);
                    for (int x = 0; x < max(n_x, n_then) && ok; x++) {
                        if (x < n_x) {
                            if (x == 0) expect(&v_full[nth & 1], (nth >> 1) & 1);
                            if (t == 0) {      // the result before has been read: the first one finds the place empty
                                expect(&o_empty[x], op >> x & 1 ^ 1);
                                op ^= 1u << x;
                            }
                            expect(&p_half[x], sp >> x & 1);
                            if (!ok) break;
                            tc_fence_after();
                            values(x, nth, 0, t > 0);
                            expect(&p_ready[x], sp >> x & 1);
                            sp ^= 1u << x;
                            if (!ok) break;
                            tc_fence_after();
                            values(x, nth, 1, true);
                            if (!more) commit(one, &o_full[x]);
                        }
                        if (x < n_then) {
                            if (late && x == 0) {
                                if (!more) expect(q_full, as_is ? (i + 1) & 1 : i & 1);
                                if (ok) wait_k(nth + 1, look);
                            }
                            if (!ok) break;
                            scores(x, nth + 1);
                        }
                    }
                    commit(one, &v_empty[nth & 1]);
                    if (any) commit(one, &k_empty[(nth + 1) & 1]);
                    if (any && (more ? t + 2 == n_tiles : next.k_hi - next.k_lo == 1)) commit(one, q_empty);
                }
            }
            if (!ok && lane == 0) atomicExch(failed, 1);
        }
    } else if (wg == 3) {
        const int id = threadIdx.x & 127;
        bool ok = true;
        auto next_queries = [&](int i) {
            if (i == 0 || as_is) return true;
            if (!arrived(q_empty, (i - 1) & 1)) return false;
            round_queries(share(i), id, 128);
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
            size_t row0 = kv4::row_of(a.c, u0.base, u0.slot, u0.kvh);
            int last = u0.pos + u0.rows - 1, lo = u0.k_lo, hi = u0.k_hi;
            auto fetch = [&](int t, const uint8_t* codes, const void* scales, uint4 (&w)[PASSES], uint2 (&d)[PASSES]) {
#pragma unroll
                for (int p = 0; p < PASSES; p++) {
                    const size_t at = row0 + min(t * BKV + p * STEP + row, last);
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
            fetch(lo, a.c.k, a.c.ks, kw, kd);
            fetch(lo, a.c.v, a.c.vs, vw, vd);
            int i = 0, t = lo;           // share and tile
            for (; ok; nth++) {
                const int b = nth & 1, ph = ((nth >> 1) - 1) & 1;
                if (nth >= 2 && !arrived(&k_empty[b], ph)) { ok = false; break; }
                write(sm + L::OFF_K + b * L::TILE, kw, kd);
                if (lane == 0) mbar_arrive(&k_full[b]);
                if (t == lo && !next_queries(i)) { ok = false; break; }
                const bool more = t + 1 < hi, any = more || i + 1 < shares;
                t++;
                if (!more && any) {      // on to the next share
                    const PackedTile u = share(++i);
                    row0 = kv4::row_of(a.c, u.base, u.slot, u.kvh);
                    last = u.pos + u.rows - 1;
                    t = lo = u.k_lo;
                    hi = u.k_hi;
                }
                if (any) fetch(t, a.c.k, a.c.ks, kw, kd);
                if (nth >= 2 && !arrived(&v_empty[b], ph)) { ok = false; break; }
                write(sm + L::OFF_V + b * L::TILE, vw, vd);
                if (lane == 0) mbar_arrive(&v_full[b]);
                if (!any) break;
                fetch(t, a.c.v, a.c.vs, vw, vd);
            }
        } else {
            constexpr uint32_t CARRY = BF16 ? 0x00800080u : 0x04000400u;      // carries out of an exponent of ones
            for (int i = 0; i < shares && ok; i++) {
                const PackedTile u = share(i);
                if (!next_queries(i)) { ok = false; break; }
                // every tile is waited for and given back, so that no stage gets two phases ahead of these warps
                for (int t = u.k_lo; t < u.k_hi && ok; t++, nth++) {
                    const int b = nth & 1, ph = (nth >> 1) & 1;
                    if (!arrived(&v_full[b], ph)) { ok = false; break; }
                    if (!masked(u, t * BKV)) {
                        if (lane == 0) mbar_arrive(&v_empty[b]);
                        continue;
                    }
                    if (!arrived(&k_full[b], ph)) { ok = false; break; }
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
        const int r = threadIdx.x & 127, of = r / group, token = wg * tokens + of;
        const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16, s_at = tmem + lane_base + 128 * wg, o_at = tmem + lane_base + 256 + 128 * wg;
        const float mult = a.softcap > 0.f ? 1.f : fmaxf(fabsf(a.scale) * LOG2E, 1e-37f),      // not zero: masked scores are -inf times this
                    cap2 = a.softcap * LOG2E, inv_cap = a.softcap > 0.f ? fabsf(a.scale) / a.softcap : 0.f;
        bool ok = true;
        uint32_t sp = 0, op = 0;
        for (int i = 0; i < shares && ok; i++) {
            const PackedTile u = share(i);
            if (wg == 1 && u.rows <= tokens) continue;
            const bool live = of < tokens && token < u.rows;
            const int qp = min(u.pos + token, u.pos + u.rows - 1), lo = first_key(qp, 0, a.window), head = u.kvh * group + r - of * group;
            const int q_first = __shfl_sync(0xffffffffu, qp, 0), lo_last = __shfl_sync(0xffffffffu, lo, 31);      // of the warp's rows
            float m = -INFINITY, l = 0.f;                // reference of the exponents, of two; sum
            for (int t = u.k_lo; t < u.k_hi; t++) {
                if (!arrived(&s_full[wg], sp)) { ok = false; break; }
                sp ^= 1;
                tc_fence_after();
                const bool edge = masked(u, t * BKV);
                if (edge || a.softcap > 0.f) {      // scores that change before they count are written back
                    const int hi = qp - t * BKV, low = lo - t * BKV;
#pragma unroll 1
                    for (int c = 0; c < BKV; c += 32) {
                        const bool all = c + 31 <= q_first - t * BKV && c >= lo_last - t * BKV;      // the warp's rows see all of these keys
                        if (all && !(a.softcap > 0.f)) continue;
                        uint32_t v[32];
                        tmem_ld32(s_at + c, v);
                        if (a.softcap > 0.f) {
#pragma unroll
                            for (int j = 0; j < 32; j++) v[j] = __float_as_uint(cap2 * tanh_exp(__uint_as_float(v[j]) * inv_cap));
                        }
                        if (!all) {
                            const int upto = hi - c, from = low - c;
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                if (j > upto) v[j] = 0xff800000u;
                            if (from > 0) {
#pragma unroll
                                for (int j = 0; j < 32; j++)
                                    if (j < from) v[j] = 0xff800000u;
                            }
                            __syncwarp();
                        }
                        tmem_st32(s_at + c, v);
                    }
                }
                // Scores are read twice, 32 at a time, the next while these are worked on: with all 128 in registers, which cannot be indexed, the loop's code was longer than the
                // instruction caches keep for warps that are out of step.  (16 at a time: 2.0 us a tile of keys instead of 1.9.)
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                uint32_t v[2][32];
                tmem_ask32(s_at, v[0]);
#pragma unroll 1
                for (int c = 0; c < BKV; c += 64)
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        tmem_have32(v[k]);
                        tmem_ask32(s_at + ((c + 32 * k + 32) & (BKV - 1)), v[k ^ 1]);      // behind the last, the first again
#pragma unroll
                        for (int j = 0; j < 32; j += 8)
#pragma unroll
                            for (int e = 0; e < 4; e++) mx[e] = fmaxf(fmaxf(mx[e], __uint_as_float(v[k][j + e])), __uint_as_float(v[k][j + 4 + e]));
                    }
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * mult;
                if (__any_sync(0xffffffffu, live && top > m + LAG)) {
                    // (a row's own scores alone decide: rows of a tile do not touch one another; where keys are cut, and with it a sum's order, follows from all portions of a step)
                    const float to = top > m + LAG ? top : m, f = to == m ? 1.f : ex2(m - to);
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
                // (weights take half the columns of their scores, so none is overwritten that has not been read)
#pragma unroll 1
                for (int c = 0; c < BKV; c += 64) {
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        tmem_have32(v[k]);
                        if (k == 0 || c == 0) tmem_ask32(s_at + c + 32 * k + 32, v[k ^ 1]);
                        uint32_t p[16];
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            const float2 e = fma2(make_float2(__uint_as_float(v[k][j]), __uint_as_float(v[k][j + 1])), mult2, less2);
                            const float2 w = make_float2(ex2(e.x), ex2(e.y));
                            sum = add2(sum, w);
                            p[j / 2] = pack2<BF16>(w.x, w.y);
                        }
                        tmem_put16(s_at + (c + 32 * k) / 2, p);
                    }
                    tmem_put_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(c ? &p_ready[wg] : &p_half[wg]);
                }
                l += sum.x + sum.y;
            }
            if (ok && !arrived(&o_full[wg], op)) ok = false;
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
            if (!whole && live) a.part_ml[part] = make_float2(m - LIFT, l);
            // through the warp's rows of shared memory, 128 bytes of each at a time, to whole lines
            uint8_t* mine = sm + L::OFF_OUT + warp * 32 * 128;
            const bool wide = !whole || a.out_type == 0;
            const uint32_t row_at = live ? (uint32_t)((whole ? ((size_t)(u.row + token) * a.ldo + (size_t)head * D) * (wide ? 4 : 2) : part * D * 4) >> 4) : 0xffffffffu;      // in 16 bytes
            uint4* const to = reinterpret_cast<uint4*>(whole ? a.out : (void*)a.part_acc) + (lane & 7);
            uint32_t rows_at[8];                     // of rows 4 k + lane / 8
#pragma unroll
            for (int k = 0; k < 8; k++) rows_at[k] = __shfl_sync(0xffffffffu, row_at, 4 * k + (lane >> 3));
            auto flush = [&](int col) {      // byte col of the rows on
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const int row = 4 * k + (lane >> 3);
                    const uint4 y = *reinterpret_cast<const uint4*>(mine + row * 128 + (((lane ^ row) & 7) << 4));
                    if (rows_at[k] != 0xffffffffu) to[rows_at[k] + (col >> 4)] = y;
                }
                __syncwarp();
            };
            auto put = [&](int c, uint32_t x, uint32_t y, uint32_t z, uint32_t w) { *reinterpret_cast<uint4*>(mine + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_uint4(x, y, z, w); };
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t y[32];
                tmem_ld32(o_at + c, y);
                if (c + 32 == D) {       // all of it has been read
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&o_empty[wg]);
                }
#pragma unroll
                for (int j = 0; j < 32; j++) y[j] = __float_as_uint(__uint_as_float(y[j]) * inv);
                if (wide) {
#pragma unroll
                    for (int k = 0; k < 8; k++) put(k, y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]);
                    flush(4 * c);
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const float e0 = __uint_as_float(y[j]), e1 = __uint_as_float(y[j + 1]);
                        y[j / 2] = a.out_type == 1 ? pack2<false>(e0, e1) : pack2<true>(e0, e1);
                    }
                    const int to4 = c >> 3 & 4;      // the first or the second 64 bytes
#pragma unroll
                    for (int k = 0; k < 4; k++) put(to4 + k, y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]);
                    if (to4) flush(2 * c - 64);
                }
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

// Adds up the parts of query tiles: grid (tiles, rows * WIDE / 8), WIDE warps a row, which take every WIDE-th part.
constexpr int MERGERS = 8;
template <int D, int WIDE>
__global__ void __launch_bounds__(MERGERS * 32) packed_merge_kernel(const __grid_constant__ PackedArgs a) {
    constexpr int N = D / 32;
    __shared__ __align__(16) float s_acc[WIDE > 1 ? MERGERS : 1][D];
    __shared__ float s_l[MERGERS];
    pdl_launch();
    pdl_wait();
    const PackedMerge u = a.merges[blockIdx.x];
    if (u.row < 0 || u.row > a.q_rows - u.rows || (unsigned)u.kvh >= (unsigned)a.kv_heads || u.first < 0 || u.parts < 1 || u.first > a.parts - u.parts) return;      // as above
    const int group = a.n_heads / a.kv_heads, tokens = BQ / group, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kvh = u.kvh;
    const int row = (blockIdx.y * MERGERS + warp) / WIDE, tile = row >> 7, r = row & 127, token = tile * tokens + r / group;
    if (r / group >= tokens || token >= u.rows) return;      // (all of a row's warps)
    const int head = kvh * group + r % group;
    const size_t step = 2 * BQ, first = (size_t)u.first * step + row;
    const float sink = a.sinks ? a.sinks[head] * LOG2E : -INFINITY;
    float m = -INFINITY;
    for (int p = lane; p < u.parts; p += 32) m = fmaxf(m, a.part_ml[first + p * step].x);
    m = fmaxf(warp_max(m), sink);
    const float ref = m == -INFINITY ? 0.f : fminf(m, 3.4e38f);      // finite: relative to it an infinite sink is infinite, and the others' weights zero
    float acc[N], l = a.sinks && warp % WIDE == 0 ? ex2(sink - ref) : 0.f;
#pragma unroll
    for (int j = 0; j < N; j++) acc[j] = 0.f;
#pragma unroll 8
    for (int p = warp % WIDE; p < u.parts; p += WIDE) {
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
    if constexpr (WIDE > 1) {
#pragma unroll
        for (int j = 0; j < N; j++) s_acc[warp][N * lane + j] = acc[j];
        if (lane == 0) s_l[warp] = l;
        __syncthreads();
        if (warp) return;
#pragma unroll
        for (int w = 1; w < WIDE; w++) {
#pragma unroll
            for (int j = 0; j < N; j++) acc[j] += s_acc[w][N * lane + j];
            l += s_l[w];
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

// Queries [rows][heads][D] of 16-bit elements; boxes of 64 columns x the heads of a KV head x the tokens of a tile.
bool queries_map(CUtensorMap* map, const PackedArgs& a) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const int group = a.n_heads / a.kv_heads;
    cuuint64_t dims[3] = {(cuuint64_t)a.hd, (cuuint64_t)a.n_heads, (cuuint64_t)a.q_rows};
    cuuint64_t strides[2] = {(cuuint64_t)a.hd * 2, (cuuint64_t)a.ldq * 2};
    cuuint32_t box[3] = {64u, (cuuint32_t)group, (cuuint32_t)(BQ / group)};
    cuuint32_t ones[3] = {1, 1, 1};
    return fn(map, a.q_type == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(a.q), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
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
    if ((a.hd != 64 && a.hd != 128) || a.kv_heads < 1 || a.kv_heads > 65535 || a.n_heads < 1 || a.n_heads % a.kv_heads || a.n_heads / a.kv_heads > BQ || !a.q || a.q_rows < 1 || !a.out || !a.tiles || !a.starts || a.ctas < 0 || a.n_tiles < a.ctas || a.window < 0 ||
        a.ldo < a.n_heads * a.hd || (((uintptr_t)a.q | (uintptr_t)a.out) & 15) || a.ldq % (a.q_type ? 8 : 4) || a.ldo % (a.out_type ? 8 : 4))
        return (int)cudaErrorInvalidValue;
    if (a.n_merges < 0 || a.parts < 0 || (a.n_merges && (a.merge_rows < 1 || a.merge_rows > 2 * BQ)) || (a.n_merges && !a.merges) || (a.parts && (!a.part_acc || !a.part_ml || ((uintptr_t)a.part_acc & 15)))) return (int)cudaErrorInvalidValue;
    if (codes ? kv4_bad_cache(a.c) || a.c.hd != a.hd || a.c.kv_heads != a.kv_heads : !a.v || a.slots < 1 || a.n < 1) return (int)cudaErrorInvalidValue;
    CUtensorMap mk = {}, mv = {}, mq = {};
    if (a.q_type && !queries_map(&mq, a)) return (int)cudaErrorInvalidValue;
    if (!codes && (!rows_map(&mk, a.k, a, a.k_slot, a.k_head, a.k_row) || !rows_map(&mv, a.v, a, a.v_slot, a.v_head, a.v_row))) return (int)cudaErrorInvalidValue;
    static thread_local PerDeviceOnce once;
    if (once.first())
        for (int form = 0; form < 3; form++) {
            cudaError_t e = cudaFuncSetAttribute(kernel_of<64>(form), cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<64>::TOTAL);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel_of<128>(form), cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<128>::TOTAL);
            if (e != cudaSuccess) return (int)e;
        }
    const int form = codes ? CODES : a.kv_bf16 ? B16 : F16;
    void* args[] = {&mk, &mv, &mq, &a};
    const int rc = a.hd == 128 ? launch_rows(kernel_of<128>(form), dim3(a.ctas), dim3(THREADS), Lay<128>::TOTAL, args, st, pdl)
                               : launch_rows(kernel_of<64>(form), dim3(a.ctas), dim3(THREADS), Lay<64>::TOTAL, args, st, pdl);
    if (rc || !a.n_merges) return rc;
    void* margs[] = {&a};      // (its CTAs may wait beside the first launch's last)
    static_assert(MERGERS == 8, "a row's warps are one or all of a CTA's");
    // Eight warps a row where a sum has more than four parts on the mean (35, of 2 x 10 rows behind 5581 keys: 22.5 us with one, 11.9 with eight; 8, of 7 behind 901: 10.9, 10.1; 2, of 2048 behind 6144:
    // 234, 294) and there are at most eight rows, each a CTA then, for an SM, which has room for five: beyond two rounds of CTAs these cost more than parts do (19 parts of 1024 rows 35.4 us with one
    // warp, 31.6 with eight; of 2048 rows 45.7, 47.1; of 4096 46.1, 52.2).
    int dev = 0, sms = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const bool many = a.parts / a.n_merges > 4 && (long)a.n_merges * a.merge_rows <= 8l * sms;
    const void* merge = a.hd == 128 ? (many ? (const void*)packed_merge_kernel<128, MERGERS> : (const void*)packed_merge_kernel<128, 1>) : (many ? (const void*)packed_merge_kernel<64, MERGERS> : (const void*)packed_merge_kernel<64, 1>);
    return launch_rows(merge, dim3(a.n_merges, many ? a.merge_rows : (a.merge_rows + MERGERS - 1) / MERGERS), dim3(MERGERS * 32), 0, margs, st, 1);
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
