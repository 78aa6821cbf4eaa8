// Attention over an 8-bit paged cache (layout: pages8.cuh).
//
//   out[row][h] = gate * softmax_k( cap(scale * q[row][h] . K[k]) ) V      k: the keys that first_key (rows.cuh) lets the row's position see
//
// Few rows: the cache is read once and everything else has to keep up with that.  Keys (then columns of values) are the rows of m16n8k16 products, the rows of a sequence for
// the query heads of a KV head their columns, eight or sixteen of them (an item: sequence, so many rows, KV head): with the four heads of grouped-query models as the rows, three
// quarters of every product, of its sums and of the exponentials were padding.  Codes become f16 operands in registers, exactly; the units multiply scores and sums.  An item's
// keys, in turns of 32, are shared by as many CTAs as its part of all turns is of the CTAs that fit the GPU, so that a CTA has one item (CTAs with an equal share of all turns each
// took 80 to 86 us where one item ended inside it and 60 to 72 elsewhere; twice and three times as many CTAs an item, 88 and 96 us instead of 87); its warps take the turns in rotation, each through a ring of its own that TMA fills, so that nothing in
// the loop waits for another warp.  A CTA leaves (largest score, sum, unnormalised result), which the merge kernel adds up.
// In a decode step the launch runs behind the append's start: what does not depend on the appended rows (shares, places, boxes of closed pages) is under way when the append ends.
// Measured, whole steps with append and merge in a graph, 128 columns: four sequences of 60000 keys, 32 heads on 8, 77 us, 5.1 TB/s of the 6.5 that a copy reaches (the SMs fetch
// unevenly: CTAs end between 51 and 74 us); one of 6144 keys 13 us and 32 sequences with windows of 1024, 16 heads on 4, 20 us, of which the three launches' latencies are most.
#include "attn_pages8.cuh"
#include "attn_tc.cuh"

__device__ int g_attn8_status = 0;

namespace {

using namespace tc;

constexpr int TURN = 32;                     // keys
constexpr int BATCH = 128;                   // turns whose places are looked up at a time
constexpr int MERGE_COLUMNS = 256;
// Weights count from 2^LIFT for the largest score on, so that f16 keeps those down to 2^-(24 + LIFT) of it (and 2^-25 as zero without: a book of faint keys lost its part of the sum
// beside one that stands out).  Taken off the maximum, the one place where it is rounded; a power beyond 7 could become 2^16 there, with scores whose last digit counts 16.
constexpr float LIFT = 7.f;

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The transpose of an 8 x 8 matrix of 16-bit values, a row's two neighbours a register.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// NB: blocks of eight query rows.  Of CTAs with one, two fit an SM.
template <int D, int NB>
struct Lay {
    static constexpr int WARPS = 8, THREADS = 32 * WARPS, ROWS = 8 * NB, PER_SM = NB == 1 ? 2 : 1;
    static constexpr int BOX = TURN * D;                     // bytes of a turn's keys, or of its values
    static constexpr int RING = 192 * 1024 / PER_SM, SLOTS = RING / (WARPS * BOX);
    static constexpr int PITCH = D + 4;                      // floats of a row of results in shared memory: banks of their own for the four rows of a store
    static constexpr int TOTAL = RING + 1024;
    static_assert(ROWS * PITCH * 4 <= RING / WARPS);
    // 16-byte chunk of a row as the tensor map's swizzle (128 or 64 bytes) places it
    __device__ static int at(int row, int chunk) {
        const int off = row * D + chunk * 16;
        return off ^ (off >> 3 & (D == 128 ? 0x70 : 0x30));
    }
};

struct Place {
    int y;                   // row of the tensor maps
    int n0;                  // first key; all bits flipped where the page is one that rows of this step go to
};

__device__ __forceinline__ Place place_of(const Attn8Args& a, const Unit& s, const Keys& k, int g, int turn) {
    const int n0 = first_of(k, TURN, turn), page = max(page_at(a.t, a.c.n_pages, s.slot, n0 >> PAGE_SHIFT), 0);
    return Place{(int)(((size_t)page * a.c.kv_heads + g) * PAGE) + (n0 & (PAGE - 1)), n0 >> PAGE_SHIFT >= s.open ? ~n0 : n0};
}
// Units of the keys and values there.
__device__ __forceinline__ float2 units_of(const Attn8Args& a, const Place& p) { return make_float2(__ldcg(a.c.ku + p.y / PAGE), __ldcg(a.c.vu + p.y / PAGE)); }

template <int D, int NB>
__global__ void __launch_bounds__(Lay<D, NB>::THREADS, Lay<D, NB>::PER_SM)
    attn8_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Attn8Args a) {
    using L = Lay<D, NB>;
    constexpr int WARPS = L::WARPS, THREADS = L::THREADS, SLOTS = L::SLOTS, CHUNKS = D / 16;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t bars[WARPS * SLOTS];
    __shared__ Place places[2 * BATCH];
    __shared__ float2 code_units[2 * BATCH];
    __shared__ DealRoom room;
    __shared__ float2 s_ml[WARPS][L::ROWS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tq = lane & 3;
    const int units = a.positions ? a.rows : a.n_segs, G = a.c.kv_heads, group = a.n_heads / G;
    if (tid < WARPS * SLOTS) mbar_init(&bars[tid], 1);
    if (tid == 0) asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (!a.behind) pdl_wait();
    pdl_launch();         // what the merging kernel reads before its own wait has been written
    Unit s;
    uint32_t first;
    if (!find_unit<true>(a, units, blockIdx.x, room, s, first)) {
        if (a.behind) pdl_wait();      // the launch does not end before the one it follows
        return;
    }
    const Keys ks = keys_of(a, s);
    const int part = (blockIdx.x - first) % s.parts, item = (blockIdx.x - first) / s.parts, kvh = item % G, m0 = L::ROWS * (item / G), rows_m = min(L::ROWS, s.rows * group - m0);
    const int x0 = (int)((long long)ks.turns * part / s.parts), turns = (int)((long long)ks.turns * (part + 1) / s.parts) - x0;
    const bool looks = tid < min(turns, 2 * BATCH);
    Place here = {};
    if (looks) here = places[tid] = place_of(a, s, ks, kvh, x0 + tid);
    __syncthreads();

    // Box 2 k of the warp's ring is the keys of its turn k, box 2 k + 1 the values.
    uint8_t* ring = sm + warp * SLOTS * L::BOX;
    uint64_t* full = bars + warp * SLOTS;
    const int boxes = warp < turns ? 2 * ((turns - warp + WARPS - 1) / WARPS) : 0;
    auto issue = [&](int j, int slot) {
        if (j < boxes && lane == 0) {
            mbar_expect_tx(&full[slot], L::BOX);
            tma_load_2d(ring + slot * L::BOX, j & 1 ? &map_v : &map_k, 0, places[(warp + WARPS * (j >> 1)) % (2 * BATCH)].y, &full[slot]);
        }
    };
    int asked = 0;                          // boxes that have been requested
    if (a.behind) {
        // The rows are still being appended: pages that none of them goes to can be fetched, and their units are what they were.
        for (; asked < min(boxes, SLOTS) && places[warp + WARPS * (asked >> 1)].n0 >= 0; asked++) issue(asked, asked);
        pdl_wait();
    }
    for (; asked < SLOTS; asked++) issue(asked, asked);

    int j = 0, slot = 0, phase = 0;         // the warp's next box and where it is
    bool ok = true;
    auto consumed = [&]() {                 // the warp has read box j
        __syncwarp();
        issue(j + SLOTS, slot);
        j++;
        if (++slot == SLOTS) {
            slot = 0;
            phase ^= 1;
        }
    };
    {
        // query row 8 n + g, columns in the order in which a lane holds a key's codes
        uint32_t qf[NB][CHUNKS][2];
        int pos[NB][2], lo[NB][2];          // of query rows 8 n + 2 tq and the next one, whose scores the lane holds
#pragma unroll
        for (int n = 0; n < NB; n++) {
            const int m = m0 + 8 * n + g, row = m / group;
            const bool live = 8 * n + g < rows_m;
            const float* q = a.q + ((size_t)(s.row + row) * a.n_heads + kvh * group + m % group) * D + 4 * tq;
#pragma unroll
            for (int c = 0; c < CHUNKS; c++) {
                const float4 v = live ? __ldcg((const float4*)(q + 16 * c)) : make_float4(0.f, 0.f, 0.f, 0.f);
                qf[n][c][0] = pack_h2(v.x, v.y);
                qf[n][c][1] = pack_h2(v.z, v.w);
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                pos[n][i] = s.pos + min((m0 + 8 * n + 2 * tq + i) / group, s.rows - 1);
                lo[n][i] = first_key(pos[n][i], a.chunk, a.window);
            }
        }
        const int first_pos = s.pos + m0 / group, last_lo = first_key(s.pos + min(s.rows - 1, (m0 + L::ROWS - 1) / group), a.chunk, a.window), keep = a.window > 0 ? a.keep : 0;
        float o[NB][CHUNKS][4];             // columns 16 c + 2 g and 16 c + 2 g + 1 of query rows 8 n + 2 tq, 8 n + 2 tq + 1
        float m_run[NB][2], l_run[NB][2], v_unit = 1.f;
#pragma unroll
        for (int n = 0; n < NB; n++) {
            m_run[n][0] = m_run[n][1] = NONE;
            l_run[n][0] = l_run[n][1] = 0.f;
#pragma unroll
            for (int c = 0; c < CHUNKS; c++) o[n][c][0] = o[n][c][1] = o[n][c][2] = o[n][c][3] = 0.f;
        }

        if (looks) code_units[tid] = units_of(a, here);
        __syncthreads();
        for (int batch = 0; batch * BATCH < turns; batch++) {
            // the places of the batch after the next one, which replace this one's
            const int next = BATCH * (batch + 2) + tid, end = min(turns, BATCH * (batch + 1));
            Place ahead = {};
            float2 ahead_units = {};
            if (tid < BATCH && next < turns) {
                ahead = place_of(a, s, ks, kvh, x0 + next);
                ahead_units = units_of(a, ahead);
            }
            while (ok && warp + WARPS * (j >> 1) < end) {
                Place p = places[(warp + WARPS * (j >> 1)) % (2 * BATCH)];
                const float2 un = code_units[(warp + WARPS * (j >> 1)) % (2 * BATCH)];
                p.n0 = max(p.n0, ~p.n0);
                if (!mbar_wait(&full[slot], phase)) {
                    ok = false;
                    break;
                }
                // scores: element e of block b is key n0 + 16 b + g + 8 (e >> 1), query row 8 n + 2 tq + (e & 1)
                float sc[NB][2][4];
#pragma unroll
                for (int b = 0; b < 2; b++) {
#pragma unroll
                    for (int n = 0; n < NB; n++) sc[n][b][0] = sc[n][b][1] = sc[n][b][2] = sc[n][b][3] = 0.f;
#pragma unroll
                    for (int c = 0; c < CHUNKS; c += 2) {
                        uint32_t kb[4];     // chunk c of keys 0-7 and 8-15, chunk c + 1 of both
                        ldsm_x4(kb, smem_u32(ring + slot * L::BOX + L::at(16 * b + (lane & 15), c + (lane >> 4))));
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const uint32_t ka[4] = {e4m3x2_to_h2(kb[2 * i]), e4m3x2_to_h2(kb[2 * i + 1]), e4m3x2_to_h2(kb[2 * i] >> 16), e4m3x2_to_h2(kb[2 * i + 1] >> 16)};
#pragma unroll
                            for (int n = 0; n < NB; n++) mma_f16(sc[n][b], ka, qf[n][c + i][0], qf[n][c + i][1]);
                        }
                    }
                }
                consumed();
                const bool all = p.n0 + TURN - 1 <= first_pos && (p.n0 >= last_lo || p.n0 + TURN <= keep);      // every row sees every key
                uint32_t bad = 0;
                if (!all) {
                    // A value that is no number would reach the rows that do not see it through a weight of zero: it becomes zero, and its key's scores none, of the rows that do.
                    if (!mbar_wait(&full[slot], phase)) {
                        ok = false;
                        break;
                    }
                    uint4* row = reinterpret_cast<uint4*>(ring + slot * L::BOX + lane * D);
                    bool none = false;
#pragma unroll
                    for (int c = 0; c < CHUNKS; c++) none |= holds_nan(row[c]);
                    bad = __ballot_sync(0xffffffffu, none);
                    if (none) {
#pragma unroll
                        for (int c = 0; c < CHUNKS; c++) row[c] = make_uint4(0, 0, 0, 0);
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    __syncwarp();
                }
                const float f = a.scale * un.x * (a.softcap > 0.f ? 1.f / a.softcap : LOG2E);
                const float turn_unit = __fdividef(v_unit, un.y);      // sums count in the unit of the last turn's values
                bool still = v_unit == un.y;                           // sums stay as they are
                v_unit = un.y;
                uint32_t pf[NB][2][2];
                float corr[NB][2];
#pragma unroll
                for (int n = 0; n < NB; n++) {
                    float mx[2] = {NONE, NONE};
#pragma unroll
                    for (int b = 0; b < 2; b++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            float v = sc[n][b][e] * f;
                            if (a.softcap > 0.f) v = a.softcap * LOG2E * tanh_exp(v);
                            if (!all) {
                                const int i = 16 * b + g + 8 * (e >> 1), kp = p.n0 + i;
                                if (bad >> i & 1) v = __int_as_float(0x7fffffff);
                                if (!(kp <= pos[n][e & 1] && (kp >= lo[n][e & 1] || kp < keep))) v = -INFINITY;
                            }
                            sc[n][b][e] = v;
                            mx[e & 1] = fmaxf(mx[e & 1], v);
                        }
#pragma unroll
                    for (int i = 0; i < 2; i++) {
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], d));
                        const float m_new = fmaxf(m_run[n][i], mx[i] - LIFT);
                        still &= m_new == m_run[n][i];
                        corr[n][i] = ex2(m_run[n][i] - m_new);
                        m_run[n][i] = m_new;
                        l_run[n][i] *= corr[n][i];
                        corr[n][i] *= turn_unit;
                    }
#pragma unroll
                    for (int b = 0; b < 2; b++) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            sc[n][b][e] = ex2(sc[n][b][e] - m_run[n][e & 1]);
                            l_run[n][e & 1] += sc[n][b][e];
                        }
                        pf[n][b][0] = transposed(pack_h2(sc[n][b][0], sc[n][b][1]));
                        pf[n][b][1] = transposed(pack_h2(sc[n][b][2], sc[n][b][3]));
                    }
                }
                if (!__all_sync(0xffffffffu, still)) {
#pragma unroll
                    for (int n = 0; n < NB; n++)
#pragma unroll
                        for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[n][c][e] *= corr[n][e & 1];
                }
                if (!mbar_wait(&full[slot], phase)) {
                    ok = false;
                    break;
                }
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int c = 0; c < CHUNKS; c += 2) {
                        uint32_t vb[4];     // chunk c of keys 0-7 and 8-15, chunk c + 1 of both; columns 2 g and 2 g + 1 of two keys each
                        ldsm_x4_trans(vb, smem_u32(ring + slot * L::BOX + L::at(16 * b + (lane & 15), c + (lane >> 4))));
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const uint32_t w0 = __byte_perm(vb[2 * i], 0, 0x3120), w1 = __byte_perm(vb[2 * i + 1], 0, 0x3120);
                            const uint32_t va[4] = {e4m3x2_to_h2(w0), e4m3x2_to_h2(w0 >> 16), e4m3x2_to_h2(w1), e4m3x2_to_h2(w1 >> 16)};
#pragma unroll
                            for (int n = 0; n < NB; n++) mma_f16(o[n][c + i], va, pf[n][b][0], pf[n][b][1]);
                        }
                    }
                consumed();
            }
            if (BATCH * (batch + 2) < turns) {
                __syncthreads();
                if (tid < BATCH) {
                    places[(batch & 1) * BATCH + tid] = ahead;
                    code_units[(batch & 1) * BATCH + tid] = ahead_units;
                }
                __syncthreads();
            }
        }

        // The warps' sums become one: they leave them in their rings, which have served, or after a wait that ran out, when what is still under way has come.
        if (!ok) {
            for (int i = j; i < min(boxes, j + SLOTS); i++) {
                mbar_wait(&full[slot], phase);
                if (++slot == SLOTS) {
                    slot = 0;
                    phase ^= 1;
                }
            }
            if (lane == 0) atomicExch(&g_attn8_status, KS_TIMEOUT);
        }
        constexpr int RANK = SLOTS * L::BOX / 4;
        float* dump = reinterpret_cast<float*>(sm);
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int row = 8 * n + 2 * tq + i;
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l_run[n][i] += __shfl_xor_sync(0xffffffffu, l_run[n][i], d);
                if (row >= rows_m) continue;
                if (g == 0) s_ml[warp][row] = make_float2(m_run[n][i], l_run[n][i]);
#pragma unroll
                for (int c = 0; c < CHUNKS; c++)
                    *reinterpret_cast<float2*>(dump + warp * RANK + row * L::PITCH + 16 * c + 2 * g) = make_float2(o[n][c][i] * v_unit, o[n][c][i + 2] * v_unit);
            }
        __syncthreads();
        for (int i = tid; i < rows_m * (D / 4); i += THREADS) {
            const int row = i / (D / 4), d = 4 * (i % (D / 4));
            float top = NONE, l = 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; w++) top = fmaxf(top, s_ml[w][row].x);
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                const float f = ex2(s_ml[w][row].x - top);
                const float4 y = *reinterpret_cast<const float4*>(dump + w * RANK + row * L::PITCH + d);
                l += f * s_ml[w][row].y;
                v.x += f * y.x;
                v.y += f * y.y;
                v.z += f * y.z;
                v.w += f * y.w;
            }
            const size_t at = (size_t)blockIdx.x * L::ROWS + row;
            *reinterpret_cast<float4*>(a.part_acc + at * D + d) = v;
            if (d == 0) a.part_ml[at] = make_float2(top, l);
        }
    }
}

// Sums of an item's row m at column d, over the CTAs from .. to - 1: unnormalised result, sum, largest score.
template <int BATCH>        // CTAs whose sums are requested together
__device__ __forceinline__ float3 merged(const Attn8Args& a, int hd, uint32_t from, uint32_t to, int m, int d) {
    float top = NONE, v = 0.f, l = 0.f;
    for (uint32_t c = from; c < to; c += BATCH) {
        float2 ml[BATCH];
        float x[BATCH], mn = top;
#pragma unroll
        for (int i = 0; i < BATCH; i++) {
            const size_t at = (size_t)(c + i) * a.row_tile + m;
            ml[i] = c + i < to ? __ldcg(a.part_ml + at) : make_float2(NONE, 0.f);
            x[i] = c + i < to ? __ldcg(a.part_acc + at * hd + d) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < BATCH; i++) mn = fmaxf(mn, ml[i].x);
        const float w = ex2(top - mn);
        v *= w;
        l *= w;
        top = mn;
#pragma unroll
        for (int i = 0; i < BATCH; i++) {
            const float f = ex2(ml[i].x - mn);
            v = fmaf(x[i], f, v);
            l = fmaf(ml[i].y, f, l);
        }
    }
    return make_float3(v, l, top);
}

// A CTA a row and MERGE_COLUMNS columns of its heads (maps), a thread a column.  With HALVES two threads share a column, each with half of the CTAs' sums, and ask for
// more of them together.
template <int HALVES>
__global__ void __launch_bounds__(MERGE_COLUMNS * HALVES) attn8_merge_kernel(const __grid_constant__ Attn8Args a) {
    constexpr int HALF = MERGE_COLUMNS, BATCH = 8 * HALVES;
    __shared__ DealRoom room;
    __shared__ float3 theirs[HALVES == 2 ? HALF : 1];
    __shared__ float second[HALF], red[HALF / 32];
    const int hd = a.c.hd, tid = threadIdx.x % HALF, half = threadIdx.x / HALF, G = a.c.kv_heads, group = a.n_heads / G, units = a.positions ? a.rows : a.n_segs;
    const int h = blockIdx.x * (HALF / hd) + tid / hd, d = tid % hd, row = blockIdx.y;
    pdl_launch();
    int u = -1;
    if (a.positions) {
        u = row;
    } else {
        for (int i = 0; i < units; i++) {
            const int4 s = a.segs[i];
            if (row >= s.x && row < s.x + s.y) u = i;
        }
    }
    const int ho = a.diff.on ? h >> 1 : h;
    const bool in = h < a.n_heads, out = in && half == 0 && d < a.vdim && !(a.diff.on && h & 1);
    float gate = 1.f;
    if (out && a.gate.kind) gate = sigmoid_f(a.gate.g[(size_t)row * a.gate.ld + (a.gate.kind == 1 ? ho * a.vdim + d : ho)]);
    Unit s;
    uint32_t first;
    const bool any = u >= 0 && find_unit<false>(a, units, u, room, s, first);
    pdl_wait();
    if (!any) return;
    float3 x = make_float3(0.f, 1.f, 0.f);
    if (in) {
        const int m = (row - s.row) * group + h % group;
        const uint32_t from = first + (m / a.row_tile * G + h / group) * s.parts, to = from + s.parts, middle = HALVES == 2 ? from + (s.parts + 1) / 2 : to;
        x = merged<BATCH>(a, hd, half ? middle : from, half ? to : middle, m % a.row_tile, d);
    }
    if (HALVES == 2) {
        if (half) theirs[tid] = x;
        __syncthreads();
        const float3 y = theirs[tid];
        const float top = fmaxf(x.z, y.z), f = ex2(x.z - top), g = ex2(y.z - top);
        x.x = x.x * f + y.x * g;
        x.y = x.y * f + y.y * g;
    }
    float v = x.x / x.y;
    if (a.diff.on) {        // threads of even maps take the odd ones' results
        if (d >= a.vdim) v = 0.f;
        if (!half) second[tid] = v;
        __syncthreads();
        const int map = tid / hd & 1;
        if (!map) v -= a.diff.lambda * second[tid + hd];
        const float sq = warp_sum(v * v);
        if (!half && (tid & 31) == 0) red[tid >> 5] = sq;
        __syncthreads();
        float sum = 0.f;
        for (int w = 0; w < hd / 32; w++) sum += red[tid / hd * (hd / 32) + w];
        v *= a.diff.scale / sqrtf(sum / (float)a.vdim + a.diff.eps);
    }
    if (!out) return;
    v *= gate;
    const size_t oi = (size_t)row * a.ldo + (size_t)ho * a.vdim + d;
    if (a.out16) ((__nv_bfloat16*)a.out)[oi] = __float2bfloat16_rn(v);
    else ((float*)a.out)[oi] = v;
}

bool bad_args(const Attn8Args& a) {
    // counts of (turn, item) pairs, of 256 sequences' items and of rows times heads are 32 bits wide
    if (a.items < 1 || a.items >> 23 || (unsigned long long)a.items * ((unsigned long long)a.t.max_pages * PAGE / 32 + 2) >> 32 || (long long)a.rows * a.n_heads >> 31 ||
        (long long)a.tiles * a.row_tile >> 31)
        return true;
    return !a.q || !a.c.k || !a.c.v || !a.c.ku || !a.c.vu || a.c.n_pages < 1 || (a.c.hd != 64 && a.c.hd != 128) || a.c.kv_heads < 1 || a.n_heads < 1 || a.n_heads % a.c.kv_heads ||
           a.n_heads > 65535 || a.rows < 1 || a.rows > 65535 || a.vdim < 1 || a.vdim > a.c.hd || !a.t.table || a.t.n_slots < 1 || a.t.max_pages < 1 || a.t.max_pages > (1 << 24) ||
           (!a.positions == !a.segs) || (a.positions && !a.slots) || (a.segs && a.n_segs < 1) || a.chunk < 0 || a.window < 0 || a.keep < 0 || (a.chunk && a.window) || a.softcap < 0.f ||
           !((a.row_tile == 128 && a.turn == 128) || ((a.row_tile == 8 || a.row_tile == 16) && a.turn == TURN)) || a.tiles < 1 || a.ctas < 1 || !a.part_acc || !a.part_ml || !a.out || a.gate.kind < 0 || a.gate.kind > 2 || (a.gate.kind && !a.gate.g) ||
           (a.diff.on && (a.n_heads / a.c.kv_heads & 1)) || a.ldo < (a.diff.on ? a.n_heads / 2 : a.n_heads) * a.vdim ||
           (((uintptr_t)a.c.k | (uintptr_t)a.c.v | (uintptr_t)a.q | (uintptr_t)a.part_acc) & 15) || ((uintptr_t)a.part_ml & 7) || (size_t)a.c.n_pages * a.c.kv_heads * PAGE >= ((size_t)1 << 31);
}

// Codes [rows][D], a turn's rows of a head as the box, each row one swizzle span.
template <int D>
bool code_map(CUtensorMap* map, const void* base, size_t rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)D};
    cuuint32_t box[2] = {(cuuint32_t)D, (cuuint32_t)TURN};
    cuuint32_t estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int NB>
int launch(Attn8Args& a, int pdl, cudaStream_t st) {
    using L = Lay<D, NB>;
    CUtensorMap mk, mv;
    const size_t rows = (size_t)a.c.n_pages * a.c.kv_heads * PAGE;
    if (!code_map<D>(&mk, a.c.k, rows) || !code_map<D>(&mv, a.c.v, rows)) return (int)cudaErrorNotSupported;
    static thread_local PerDeviceOnce once;
    if (once.first()) cudaFuncSetAttribute(attn8_kernel<D, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL);
    void* args[] = {&mk, &mv, &a};
    // at most one CTA an item more than fit the GPU: parts are rounded down but to one
    return launch_rows((const void*)attn8_kernel<D, NB>, dim3(a.ctas + a.items), dim3(L::THREADS), L::TOTAL, args, st, pdl);
}
int launch(Attn8Args& a, int pdl, cudaStream_t st) {
    if (a.row_tile == 128) return attn8_tc_launch(a, a.ctas + a.items, pdl, st);
    if (a.c.hd == 128) return a.row_tile == 8 ? launch<128, 1>(a, pdl, st) : launch<128, 2>(a, pdl, st);
    return a.row_tile == 8 ? launch<64, 1>(a, pdl, st) : launch<64, 2>(a, pdl, st);
}

}  // namespace

static int attn8_launch(const Attn8Args& in, int pdl, cudaStream_t st) {
    if (bad_args(in)) return (int)cudaErrorInvalidValue;
    static thread_local PerDeviceOnce once;      // an SM that is set for less shared memory takes the attention kernel's CTAs only when it is empty
    if (once.first()) {
        cudaFuncSetAttribute(attn8_merge_kernel<1>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        cudaFuncSetAttribute(attn8_merge_kernel<2>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    }
    int dev = 0, sms = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const int units = in.positions ? in.rows : in.n_segs, heads = MERGE_COLUMNS / in.c.hd;
    for (int u = 0; u < units; u += MAX_UNITS) {
        Attn8Args a = in;
        a.keep = min(a.keep, a.t.max_pages * PAGE);      // tiles of kept keys are counted in 32 bits
        const int n = units - u < MAX_UNITS ? units - u : MAX_UNITS;
        if (a.positions) {
            a.positions += u;
            a.slots += u;
            a.rows = n;
            a.items = min(a.items, n * a.tiles * a.c.kv_heads);
            a.q += (size_t)u * a.n_heads * a.c.hd;
            a.out = (char*)a.out + (size_t)u * a.ldo * (a.out16 ? 2 : 4);
            if (a.gate.kind) a.gate.g += (size_t)u * a.gate.ld;
        } else {
            a.segs += u;
            a.n_segs = n;
        }
        a.behind = in.behind && units <= MAX_UNITS;
        int rc = launch(a, pdl || a.behind, st);
        if (rc) return rc;
        void* args[] = {&a};
        const dim3 grid((a.n_heads + heads - 1) / heads, a.rows);
        // Two threads a column while there are no more CTAs than SMs (16 heads at 6144: 16.6 -> 13.0 us a step); beyond, other CTAs' loads fill the time, and two cost
        // (64 rows of 32 heads at 30000: 88 -> 103 us).
        const bool wide = grid.x * grid.y <= (unsigned)sms;
        rc = launch_rows(wide ? (const void*)attn8_merge_kernel<2> : (const void*)attn8_merge_kernel<1>, grid, dim3(wide ? 2 * MERGE_COLUMNS : MERGE_COLUMNS), 0, args, st, 1);
        if (rc) return rc;
        pdl = 1;
    }
    return 0;
}

// Attention of rows of queries.  Returns a cudaError_t value, as does the entry point below.
B2_API int b2_attn8(const Attn8Args* a, int pdl, cudaStream_t st) {
    if (!a) return (int)cudaErrorInvalidValue;
    Attn8Args c = *a;
    c.behind = 0;
    return attn8_launch(c, pdl, st);
}

// A decode step: the rows are appended, then their attention, which begins while they are.
B2_API int b2_decode8(const Append8Args* p, const Attn8Args* a, int pdl, cudaStream_t st) {
    if (!p || !a || !p->positions || bad_args(*a) || p->rows != a->rows) return (int)cudaErrorInvalidValue;
    const int rc = append8_launch(*p, pdl, st);
    if (rc) return rc;
    Attn8Args c = *a;
    c.behind = 1;
    return attn8_launch(c, 1, st);
}

// 0, or KS_TIMEOUT once a wait of the attention kernel has run out since the last call.
B2_API int b2_attn8_status() {
    int v = 0, none = 0;
    if (cudaMemcpyFromSymbol(&v, g_attn8_status, sizeof(int)) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(g_attn8_status, &none, sizeof(int));
    return v | attn8_tc_status();
}
