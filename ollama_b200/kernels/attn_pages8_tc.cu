// Attention of tens to hundreds of query rows over an 8-bit paged cache on tcgen05 (layout: pages8.cuh, how it is dealt out: attn_pages8.cuh).
//
// An item is 128 rows of (row of a portion, query head of a KV head), so that a few rows for all heads of a KV head fill a tile, and its keys are shared by several CTAs: 64 rows of
// four heads behind a long context are 256 rows a KV head, which rows of 16 read (and expand) the cache for 16 times, and a tile a head leaves most SMs idle.
// Tiles of 128 keys: bulk copies bring the codes into a ring of three boxes, in the order in which the products take them; eight warps turn them into swizzled f16 tiles, exactly
// (code times unit is an f16 number), two buffers of keys and of values.  S = Q K^T and P V: two score buffers in tensor memory, probabilities over the scores they came from, S of
// tile t + 2 issued behind P V of tile t.  Even and odd tiles have a softmax group and a result in tensor memory each, which P V adds to and which is scaled only where a score passes
// the group's reference by a factor of 2^LAG: no group waits for the other, and nothing is read back per tile.  The groups' results meet in shared memory at the end.
// Warps: 0-3 and 4-7 softmax (a thread a row), 8 bulk copies, 9 products and tensor memory, 12-19 codes.  Every wait is bounded; one that runs out sets KS_TIMEOUT, and all roles
// leave their loops.
// Measured: 64 rows of 32 heads on 8 of 128 columns behind 30000 keys, 59 us with the merge, 1.4 us a tile.  A group's turn is 1.5 us of softmax (exponentials, at 16 a
// cycle, and rounding 0.95, loads from tensor memory and maximum 0.6) and 1.1 until its next scores are there; two groups take 1.4 a tile, the tensor cores busy for 0.6 of them.
// Leaving the expansion's stores out changed nothing.  Slower: boxes in the order K(t), V(t), six code warps and one softmax group that reads each P V back, 88; a second look at the
// keys of masked tiles, 10 us in instruction misses; sixteen softmax warps, 60.7; a quarter of the exponentials as cubics on the FMA units, 63.7, half of them 68.
#include "attn_pages8.cuh"
#include "attn_tc.cuh"

__device__ int g_attn8_tc_status = 0;

namespace {

using namespace tc;

constexpr int BQ = 128, BKV = 128;
constexpr int ATOM_BYTES = 128 * 128;        // 128 rows x 64 f16
constexpr int SOFTMAX_WARPS = 8, CODE_WARPS = 8, TEAM = CODE_WARPS / 2, FIRST_CODE_WARP = 12, THREADS = 32 * (FIRST_CODE_WARP + CODE_WARPS);      // whole groups of four warps, whose registers are split
constexpr int BOXES = 3;
constexpr uint32_t TMEM_COLS = 512;
constexpr float LAG = 8.f;
constexpr float LIFT = 6.f;                  // weights count from 2^LIFT for the reference on (see attn_pages8.cu), so that they end at 2^14, within f16

template <int D>
struct Lay {
    static constexpr int ATOMS = D / 64, TILE = ATOMS * ATOM_BYTES, BOX = BKV * D;
    static constexpr int OFF_K = TILE, OFF_V = OFF_K + 2 * TILE, OFF_BOX = OFF_V + 2 * TILE, TOTAL = OFF_BOX + BOXES * BOX + 1024;
};

__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void tmem_ld8(uint32_t at, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(at));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// bits 0 .. n - 1
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? 0xffffffffu : n > 0 ? (1u << n) - 1 : 0u; }
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * SOFTMAX_WARPS) : "memory"); }

// 16 codes times the unit as f16 at p (the first eight of x) and q
__device__ __forceinline__ void put_codes(uint8_t* p, uint8_t* q, const uint32_t (&x)[4], __half2 unit) {
    uint32_t y[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uint32_t h = e4m3x2_to_h2(x[j >> 1] >> (j & 1) * 16);
        const __half2 f = __hmul2(*reinterpret_cast<const __half2*>(&h), unit);
        y[j] = *reinterpret_cast<const uint32_t*>(&f);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(y[0], y[1], y[2], y[3]);
    *reinterpret_cast<uint4*>(q) = make_uint4(y[4], y[5], y[6], y[7]);
}

template <int D>
__global__ void __launch_bounds__(THREADS, 1) attn8_tc_kernel(const __grid_constant__ Attn8Args a) {
    using L = Lay<D>;
    constexpr int OH = D / 2, PITCH = D + 4, CHUNKS = D / 16, CODE_THREADS = 32 * TEAM, EACH = BKV * CHUNKS / CODE_THREADS;      // 16 codes at a time of a code thread
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t bars[20];
    __shared__ DealRoom room;
    __shared__ uint32_t tmem_slot;
    __shared__ int failed;
    __shared__ float2 units8[BOXES];             // of the two pages in a box
    __shared__ uint8_t no_number[2][BKV];        // of a tile that some row does not see all of: keys whose values hold what is no number
    __shared__ float2 x_ml[2][128];              // of the two groups: reference, sum
    uint64_t *full8 = bars, *empty8 = bars + 3, *k_full = bars + 6, *k_empty = bars + 8, *v_full = bars + 10, *v_empty = bars + 12, *s_full = bars + 14, *p_ready = bars + 16,
             *o_full = bars + 18;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n_units = a.positions ? a.rows : a.n_segs, G = a.c.kv_heads, group = a.n_heads / G;
    pdl_wait();
    pdl_launch();        // behind the wait, so that what the merging kernel reads before its own has been written
    Unit s;
    uint32_t first;
    if (!find_unit<true>(a, n_units, blockIdx.x, room, s, first)) return;
    const int part = (blockIdx.x - first) % s.parts, item = (blockIdx.x - first) / s.parts, kvh = item % G, m0 = BQ * (item / G), rows_m = min(BQ, s.rows * group - m0);
    Unit own = s;                    // the tile's rows, whose keys may be fewer than the unit's: some CTA may have none
    own.pos += m0 / group;
    own.rows = (m0 + rows_m - 1) / group - m0 / group + 1;
    const Keys ks = keys_of(a, own);
    const int x0 = (int)((long long)ks.turns * part / s.parts), n_tiles = (int)((long long)ks.turns * (part + 1) / s.parts) - x0;
    // positions of the tile's first and last row, the last one's first key
    const int first_pos = own.pos, last_pos = own.pos + own.rows - 1, last_lo = first_key(last_pos, a.chunk, a.window), keep = a.window > 0 ? a.keep : 0;
    auto n0_of = [&](int t) { return first_of(ks, BKV, x0 + t); };
    auto masked = [&](int n0) { return n0 + BKV - 1 > first_pos || (n0 < last_lo && n0 + BKV > keep); };      // some row does not see some key

    // The boxes in the order in which the products take them: K(0), K(1), V(0), K(2), V(1), ... V(n - 1).  x: tile, y: 1 with values
    auto box_of = [&](int j) { return j == 2 * n_tiles - 1 ? make_int2(n_tiles - 1, 1) : j > 0 && (j & 1) == 0 ? make_int2(j / 2 - 1, 1) : make_int2((j + 1) / 2, 0); };

    if (warp == 8 && lane == 0) {
        failed = 0;
        for (int i = 0; i < BOXES; i++) {
            mbar_init(&full8[i], 1);
            mbar_init(&empty8[i], TEAM);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&k_full[b], TEAM);
            mbar_init(&k_empty[b], 1);
            mbar_init(&v_full[b], TEAM);
            mbar_init(&v_empty[b], 1);
            mbar_init(&s_full[b], 1);
            mbar_init(&p_ready[b], SOFTMAX_WARPS / 2);
            mbar_init(&o_full[b], 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // Warp 8, the copies: its lanes look up the pages of 32 boxes at a time.
    const int last_page = last_pos >> PAGE_SHIFT;
    int head[2] = {}, asked = 0;                     // boxes
    float2 un = make_float2(0.f, 0.f);
    auto look_up = [&](int j0) {
        if (j0 + lane < 2 * n_tiles) {
            const int2 of = box_of(j0 + lane);
            const int p0 = n0_of(of.x) >> PAGE_SHIFT;
            const float* units = of.y ? a.c.vu : a.c.ku;
            for (int i = 0; i < 2; i++) head[i] = max(page_at(a.t, a.c.n_pages, s.slot, min(p0 + i, last_page)), 0) * G + kvh;
            un = make_float2(units[head[0]], units[head[1]]);
        }
    };
    auto ask = [&](int j) {
        const size_t h0 = __shfl_sync(0xffffffffu, head[0], j & 31), h1 = __shfl_sync(0xffffffffu, head[1], j & 31);
        const float2 u = make_float2(__shfl_sync(0xffffffffu, un.x, j & 31), __shfl_sync(0xffffffffu, un.y, j & 31));
        if (lane == 0) {
            const int slot = j % BOXES;
            uint8_t* box = sm + L::OFF_BOX + slot * L::BOX;
            const uint8_t* from = box_of(j).y ? a.c.v : a.c.k;
            units8[slot] = u;
            mbar_expect_tx(&full8[slot], L::BOX);
            bulk_copy(box, from + h0 * PAGE * D, PAGE * D, &full8[slot]);
            bulk_copy(box + PAGE * D, from + h1 * PAGE * D, PAGE * D, &full8[slot]);
        }
        asked++;
        __syncwarp();
    };
    if (warp == 8) {                 // the first of them before anything else
        look_up(0);
        for (int j = 0; j < min(2 * n_tiles, BOXES); j++) ask(j);
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp < SOFTMAX_WARPS || warp >= FIRST_CODE_WARP) {      // queries: whole rows by neighbouring threads
        constexpr int N = 32 * (SOFTMAX_WARPS + CODE_WARPS), QUADS = D / 4, LOADS = BQ * QUADS / N;
        const int t0 = tid - (warp < SOFTMAX_WARPS ? 0 : 32 * (FIRST_CODE_WARP - SOFTMAX_WARPS));
        const float sign = a.scale > 0.f ? 1.f : a.scale < 0.f ? -1.f : 0.f;      // the running maximum is one of plain scores, which takes a scale above zero
        float4 x[LOADS];
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int r = (t0 + N * i) / QUADS, col = (t0 + N * i) % QUADS * 4, m = m0 + r;
            x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < rows_m) x[i] = *(const float4*)(a.q + ((size_t)(s.row + m / group) * a.n_heads + kvh * group + m % group) * D + col);
        }
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int r = (t0 + N * i) / QUADS, col = (t0 + N * i) % QUADS * 4;
            *(uint2*)(sm + (col >> 6) * ATOM_BYTES + r * 128 + ((((col & 63) >> 3) ^ (r & 7)) << 4) + (col & 4) * 2) = make_uint2(pack_h2(sign * x[i].x, sign * x[i].y), pack_h2(sign * x[i].z, sign * x[i].w));
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    // 60 K registers: 168 a softmax thread, 48 a thread of the other three groups
    if (warp >= SOFTMAX_WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (warp == 8) {
            bool ok = true;
            for (int j = BOXES; j < 2 * n_tiles; j++) {
                if ((j & 31) == 0) look_up(j);
                if (!mbar_wait(&empty8[j % BOXES], (j / BOXES - 1) & 1)) {
                    ok = false;
                    break;
                }
                ask(j);
            }
            if (!ok && lane == 0) atomicExch(&failed, 1);
            for (int i = max(0, asked - BOXES); i < asked; i++) mbar_wait(&full8[i % BOXES], (i / BOXES) & 1);      // no copy is under way when the CTA leaves
        } else if (warp >= FIRST_CODE_WARP) {
            // Two teams of four warps take every second box each: what one waits for behind its stores is covered by the other
            const int t0 = tid - 32 * FIRST_CODE_WARP & CODE_THREADS - 1, team = warp - FIRST_CODE_WARP >= TEAM;      // its chunks of a box are t0 + CODE_THREADS i
            // Row, columns 16 col .. 16 col + 15 of its first chunk; the others' rows lie multiples of eight on, so that the swizzle is the same.  Columns below 64 and above, whose atoms have
            // the same banks, begin with different halves.
            const int r0 = t0 / CHUNKS, col = t0 % CHUNKS, swap = col >> 2 & 1;
            const int at0 = (col >> 2) * ATOM_BYTES + r0 * 128 + ((2 * (col & 3) + swap ^ (r0 & 7)) << 4), at1 = at0 ^ 16;
            static_assert(CODE_THREADS / CHUNKS % 8 == 0, "rows of a thread's chunks");
            bool ok = true;
            for (int j = team; j < 2 * n_tiles; j += 2) {
                const int slot = j % BOXES, tile = box_of(j).x, is_v = box_of(j).y, b = tile & 1;
                if (!mbar_wait(&full8[slot], (j / BOXES) & 1)) { ok = false; break; }
                if (tile >= 2 && !mbar_wait(is_v ? &v_empty[b] : &k_empty[b], ((tile >> 1) - 1) & 1)) { ok = false; break; }
                const bool look = is_v && masked(n0_of(tile));
                const uint4* box = reinterpret_cast<const uint4*>(sm + L::OFF_BOX + slot * L::BOX);
                const float2 un = units8[slot];
                uint8_t* to = sm + (is_v ? L::OFF_V : L::OFF_K) + b * L::TILE;
#pragma unroll
                for (int h = 0; h < 2; h++) {          // a page
                    const __half2 unit = __float2half2_rn(h ? un.y : un.x);
                    uint4 w[EACH / 2];             // all of them before anything is stored: the compiler keeps loads behind stores
#pragma unroll
                    for (int i = 0; i < EACH / 2; i++) w[i] = box[t0 + CODE_THREADS * (h * EACH / 2 + i)];
                    if (look) {       // a weight of zero times what is no number: such values become zeros, and their keys' scores none
#pragma unroll
                        for (int i = 0; i < EACH / 2; i++) {
                            const int at = t0 + CODE_THREADS * (h * EACH / 2 + i);
                            uint32_t none = holds_nan(w[i]);
#pragma unroll
                            for (int o = 1; o < CHUNKS; o <<= 1) none |= __shfl_xor_sync(0xffffffffu, none, o);
                            if (none) w[i] = make_uint4(0, 0, 0, 0);
                            if (at % CHUNKS == 0) no_number[b][at / CHUNKS] = none != 0;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < EACH / 2; i++) {
                        const int rows = CODE_THREADS / CHUNKS * (h * EACH / 2 + i) * 128;
                        const uint32_t x[4] = {swap ? w[i].z : w[i].x, swap ? w[i].w : w[i].y, swap ? w[i].x : w[i].z, swap ? w[i].y : w[i].w};
                        put_codes(to + at0 + rows, to + at1 + rows, x, unit);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(is_v ? &v_full[b] : &k_full[b]);
                    mbar_arrive(&empty8[slot]);
                }
            }
            if (!ok) atomicExch(&failed, 1);
        } else if (warp == 9 && lane == 0) {
            {
                constexpr uint32_t id_s = idesc_f16(BQ, BKV, 0), id_o = idesc_f16(BQ, D, 1);
                bool ok = true;
                auto issue_s = [&](int t) {          // S(t) = Q K(t)^T into score buffer t & 1
                    const int b = t & 1;
                    if (!mbar_wait(&k_full[b], (t >> 1) & 1)) { ok = false; return; }
                    tc_fence_after();
                    const uint8_t* kt = sm + L::OFF_K + b * L::TILE;
#pragma unroll
                    for (int at = 0; at < L::ATOMS; at++) {
                        const uint64_t qd = umma_desc(sm + at * ATOM_BYTES), kd = umma_desc(kt + at * ATOM_BYTES);
#pragma unroll
                        for (int k = 0; k < 4; k++) umma_f16(tmem + 128 * b, qd + 2 * k, kd + 2 * k, id_s, (at | k) != 0);
                    }
                    umma_commit(&s_full[b]);
                    umma_commit(&k_empty[b]);
                };
                if (n_tiles > 0) issue_s(0);
                if (ok && n_tiles > 1) issue_s(1);
                for (int t = 0; t < n_tiles && ok; t++) {
                    const int b = t & 1, ph = (t >> 1) & 1;
                    if (!mbar_wait(&p_ready[b], ph) || !mbar_wait(&v_full[b], ph)) { ok = false; break; }
                    tc_fence_after();
                    const uint8_t* vt = sm + L::OFF_V + b * L::TILE;
#pragma unroll
                    for (int kk = 0; kk < BKV / 16; kk++)      // P(t) V(t) onto its group's result; P sits in the first 64 columns of its score buffer
                        umma_f16_ts(tmem + 256 + 128 * b, tmem + 128 * b + 8 * kk, umma_desc_mn(vt + kk * 16 * 128, ATOM_BYTES), id_o, t >= 2 || kk != 0);
                    if (t + 2 >= n_tiles) umma_commit(&o_full[b]);
                    umma_commit(&v_empty[b]);
                    if (t + 2 < n_tiles) issue_s(t + 2);       // runs behind P V(t), which still reads the buffer it overwrites
                }
                if (!ok) atomicExch(&failed, 1);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
        // Warps 0-3 have the even tiles, 4-7 the odd ones: a thread a row, with a reference, a sum and a result (in tensor memory) of its own, so that one group's exponentials run
        // beside the other's products.  The reference is a score that none passes by more than a factor of 2^LAG; the result is scaled when one does.
        const int q = warp & 3, c = warp >> 2, r = 32 * q + lane;
        const int qp = s.pos + min((m0 + r) / group, s.rows - 1), row_lo = first_key(qp, a.chunk, a.window);
        const float size = a.scale == 0.f ? 1.f : fabsf(a.scale), mult = a.softcap > 0.f ? 1.f : size * LOG2E, inv_cap = a.softcap > 0.f ? size / a.softcap : 0.f, cap2 = a.softcap * LOG2E;
        const uint32_t lane_base = (uint32_t)(32 * q) << 16, scores = tmem + lane_base + 128 * c, result = scores + 256;
        float m_ref = NONE, l_run = 0.f;
        bool ok = true;
        for (int t = c; t < n_tiles; t += 2) {
            const int n0 = n0_of(t);
            if (!mbar_wait(&s_full[c], (t >> 1) & 1)) { ok = false; break; }
            tc_fence_after();
            uint32_t v[4][32];
#pragma unroll
            for (int i = 0; i < 4; i++) tmem_ld32(scores + 32 * i, v[i]);
            if (a.softcap > 0.f) {
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 32; j++) v[i][j] = __float_as_uint(cap2 * tanh_exp(__uint_as_float(v[i][j]) * inv_cap));
            }
            if (masked(n0)) {
                if (!mbar_wait(&v_full[c], (t >> 1) & 1)) { ok = false; break; }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int k0 = n0 + 32 * i;
                    const uint32_t none = __ballot_sync(0xffffffffu, no_number[c][32 * i + lane]), seen = below(qp + 1 - k0) & (~below(row_lo - k0) | below(keep - k0));
                    if (none) {
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (none >> j & 1) v[i][j] = 0x7fffffffu;
                    }
#pragma unroll
                    for (int j = 0; j < 32; j++)
                        if (!(seen >> j & 1)) v[i][j] = 0xff800000u;
                }
            }
            float top[4] = {NONE, NONE, NONE, NONE};
#pragma unroll
            for (int j = 0; j < 32; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) top[i] = fmaxf(top[i], __uint_as_float(v[i][j]));
            const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            if (__any_sync(0xffffffffu, (mx - m_ref) * mult > LAG)) {
                const float m_new = fmaxf(m_ref, mx), corr = ex2((m_ref - m_new) * mult);
                m_ref = m_new;
                l_run *= corr;
                if (t >= 2) {        // S(t) is behind P V(t - 2)
#pragma unroll 1
                    for (int j = 0; j < D; j += 8) {
                        uint32_t o[8];
                        tmem_ld8(result + j, o);
#pragma unroll
                        for (int i = 0; i < 8; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                        tmem_st8(result + j, o);
                    }
                }
            }
            const float2 mult2 = make_float2(mult, mult), less = make_float2(fmaf(-m_ref, mult, LIFT), fmaf(-m_ref, mult, LIFT));
            float2 ls2[2] = {};
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t pw[32];
#pragma unroll
                for (int j = 0; j < 32; j++) {
                    const int i = 2 * h + (j >> 4), k = 2 * j & 31;
                    const float2 e = fma2(make_float2(__uint_as_float(v[i][k]), __uint_as_float(v[i][k + 1])), mult2, less);
                    const float2 pr = make_float2(ex2(e.x), ex2(e.y));
                    ls2[j & 1] = add2(ls2[j & 1], pr);
                    pw[j] = pack_h2(pr.x, pr.y);
                }
                tmem_st32(scores + 32 * h, pw);      // over scores that have been read
            }
            l_run += ls2[0].x + ls2[0].y + (ls2[1].x + ls2[1].y);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[c]);
        }
        // The groups' sums become one, in shared memory that the products no longer read, and go out in whole rows
        if (ok && c < n_tiles && !mbar_wait(&o_full[c], 0)) ok = false;
        if (!ok) atomicExch(&failed, 1);
        tc_fence_after();
        x_ml[c][r] = make_float2(m_ref * mult, l_run);
        softmax_sync();
        const float2 x0 = x_ml[0][r], x1 = x_ml[1][r];
        const float top = fmaxf(x0.x, x1.x), w = ex2((c ? x1.x : x0.x) - top);
        float* row = reinterpret_cast<float*>(sm + L::OFF_K) + r * PITCH;
        for (int add = 0; add < 2; add++) {          // a half of the columns: first the other group's, then its own
            const int j0 = OH * (c ^ 1 ^ add);
            if (c < n_tiles || add) {
#pragma unroll 1
                for (int j = j0; j < j0 + OH; j += 32) {
                    uint32_t o[32];
                    if (c < n_tiles) tmem_ld32(result + j, o);
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        float4 y = add && (c ^ 1) < n_tiles ? *reinterpret_cast<float4*>(row + j + i) : make_float4(0.f, 0.f, 0.f, 0.f);
                        if (c < n_tiles) {
                            y.x = fmaf(__uint_as_float(o[i]), w, y.x);
                            y.y = fmaf(__uint_as_float(o[i + 1]), w, y.y);
                            y.z = fmaf(__uint_as_float(o[i + 2]), w, y.z);
                            y.w = fmaf(__uint_as_float(o[i + 3]), w, y.w);
                        }
                        *reinterpret_cast<float4*>(row + j + i) = y;
                    }
                }
            }
            softmax_sync();
        }
        const size_t at = (size_t)blockIdx.x * BQ;
        float4* to = reinterpret_cast<float4*>(a.part_acc + at * D);
        for (int i = tid; i < rows_m * (D / 4); i += 32 * SOFTMAX_WARPS) to[i] = *reinterpret_cast<const float4*>(sm + L::OFF_K + ((i / (D / 4)) * PITCH + 4 * (i % (D / 4))) * 4);
        if (c == 0 && r < rows_m) a.part_ml[at + r] = make_float2(top, x0.y * w + x1.y * ex2(x1.x - top));
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
    if (tid == 0 && failed) atomicExch(&g_attn8_tc_status, KS_TIMEOUT);
}

template <int D>
int launch(Attn8Args& a, int grid, int pdl, cudaStream_t st) {
    static thread_local PerDeviceOnce once;
    if (once.first()) cudaFuncSetAttribute(attn8_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<D>::TOTAL);
    void* args[] = {&a};
    return launch_rows((const void*)attn8_tc_kernel<D>, dim3(grid), dim3(THREADS), Lay<D>::TOTAL, args, st, pdl);
}

}  // namespace

int attn8_tc_launch(const Attn8Args& in, int grid, int pdl, cudaStream_t st) {
    Attn8Args a = in;
    return a.c.hd == 128 ? launch<128>(a, grid, pdl, st) : launch<64>(a, grid, pdl, st);
}

int attn8_tc_status() {
    int v = 0, none = 0;
    if (cudaMemcpyFromSymbol(&v, g_attn8_tc_status, sizeof(int)) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(g_attn8_tc_status, &none, sizeof(int));
    return v;
}
