// Attention over an 8-bit paged cache (layout: pages8.cuh).
//
//   out[row][h] = gate * softmax_k( cap(scale * q[row][h] . K[k]) ) V      k: the keys that first_key (rows.cuh) lets the row's position see
//
// Few rows: the cache is read once and everything else has to keep up with that.  The rows of a sequence and the query heads of a KV head are the 16 rows of m16n8k16 products
// (an item: sequence, 16 such rows, KV head); codes become f16 operands in registers, exactly, and the units multiply scores and sums.  All items' keys, in turns of 32, are
// dealt out to one CTA an SM in equal runs, whatever the sequences' lengths; eight warps take the turns of a run in rotation, each through a ring of its own that TMA fills,
// so that nothing in the loop waits for another warp.  A run that ends inside an item leaves (largest score, sum, unnormalised result), which the merge kernel adds up.
#include "pages8.cuh"
#include "tc_common.cuh"

__device__ int g_attn8_status = 0;

namespace {

using namespace tc;

constexpr int TURN = 32;                     // keys
constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int MAX_UNITS = THREADS;           // sequences of a launch
constexpr int BATCH = THREADS / 2;           // turns whose places are looked up at a time
constexpr float LOG2E = 1.4426950408889634f;
constexpr float NONE = -1e30f;               // largest score of no keys

// The rows of one sequence in the launch.
struct Unit {
    int row, rows, slot, pos;                // first row, rows (0: no token), slot, position of the first row
    int open;                                // first page of the slot that rows of the step go to
};

__device__ __forceinline__ Unit unit_at(const Attn8Args& a, int u) {
    Unit s;
    if (a.positions) {
        s = Unit{u, 1, a.slots[u], a.positions[u], 0};
    } else {
        const int4 g = a.segs[u];
        s = Unit{g.x, g.y, g.z, g.w, 0};
    }
    if ((unsigned)s.slot >= (unsigned)a.t.n_slots || s.pos < 0 || s.row < 0 || s.row + s.rows > a.rows || s.pos + s.rows > a.t.max_pages * PAGE) s.rows = 0;
    s.open = s.pos >> PAGE_SHIFT;
    return s;
}

// Turns of a unit's items: those with kept keys first, then the ones from the first row's first key on.
struct Keys {
    int base, front, turns;
};
__device__ __forceinline__ Keys keys_of(const Attn8Args& a, const Unit& s) {
    Keys k;
    k.base = first_key(s.pos, a.chunk, a.window) & ~(TURN - 1);
    k.front = a.window > 0 ? kept_tiles(a.keep, k.base, TURN) : 0;
    k.turns = s.rows > 0 ? k.front + (s.pos + s.rows - k.base + TURN - 1) / TURN : 0;
    return k;
}
__device__ __forceinline__ int first_of(const Keys& k, int turn) { return turn < k.front ? turn * TURN : k.base + (turn - k.front) * TURN; }

// Items of a unit: 16 rows of (row, head of the KV head) each, of every KV head.
__device__ __forceinline__ int row_tiles(const Attn8Args& a, const Unit& s) { return (s.rows * (a.n_heads / a.c.kv_heads) + 15) >> 4; }

// Where an item's first sums go, less the CTA they are of: an item after another has a larger number, so that no two runs' ends meet.
__device__ __forceinline__ size_t piece_of(const Attn8Args& a, int u, uint32_t item) { return (size_t)u * a.tiles * a.c.kv_heads + item; }

// All units, the turns before each (prefix[u]) and in all (prefix[units]).
__device__ __forceinline__ void count_turns(const Attn8Args& a, int units, Unit* list, uint32_t* prefix, uint32_t* sums) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t n = 0;
    if (tid < units) {
        const Unit s = unit_at(a, tid);
        list[tid] = s;
        n = (uint32_t)keys_of(a, s).turns * row_tiles(a, s) * a.c.kv_heads;
    }
    uint32_t x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    for (int w = 0; w < warp; w++) x += sums[w];
    if (tid <= units) prefix[tid] = x - n;
    if (tid == units - 1) prefix[units] = x;
    if (a.behind && tid < units) {      // other rows of the slot may go to earlier pages
        int open = list[tid].open;
        for (int i = 0; i < units; i++)
            if (list[i].slot == list[tid].slot && list[i].pos >= 0) open = min(open, list[i].pos >> PAGE_SHIFT);
        list[tid].open = open;
    }
    __syncthreads();
}

// Turns of a CTA's run: at least one a warp.
__device__ __forceinline__ uint32_t share_of(uint32_t total, int ctas) { return max((total + ctas - 1) / ctas, (uint32_t)WARPS); }

__device__ __forceinline__ int unit_of(const uint32_t* prefix, int units, uint32_t x) {
    int lo = 0, hi = units - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (prefix[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    while (lo < units - 1 && prefix[lo + 1] <= x) lo++;      // units without turns
    return lo;
}

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <int D>
struct Lay {
    static constexpr int HALF = TURN * D;                    // bytes of a turn's keys
    static constexpr int STAGE = 2 * HALF, NS = D == 128 ? 3 : 6;
    static constexpr int RING = WARPS * NS * STAGE;          // 192 KB
    static constexpr int MERGE = 16 * 1024;
    static constexpr int TOTAL = RING + MERGE + 1024;
    // 16-byte chunk of a row as the tensor map's swizzle (128 or 64 bytes) places it
    __device__ static int at(int row, int chunk) {
        const int off = row * D + chunk * 16;
        return off ^ (off >> 3 & (D == 128 ? 0x70 : 0x30));
    }
};

struct Place {
    int y;                   // row of the tensor maps
    float ku, vu;
    int n0;                  // first key; all bits flipped where the page is one that rows of this step go to
};

__device__ __forceinline__ Place place_of(const Attn8Args& a, const Unit* list, const uint32_t* prefix, int units, uint32_t x) {
    const int u = unit_of(prefix, units, x);
    const Unit s = list[u];
    const Keys k = keys_of(a, s);
    const uint32_t in = x - prefix[u], item = in / k.turns;
    Place p;
    const int n0 = first_of(k, in - item * k.turns);
    const int g = item % a.c.kv_heads, page = max(page_at(a.t, a.c.n_pages, s.slot, n0 >> PAGE_SHIFT), 0);
    const size_t head = (size_t)page * a.c.kv_heads + g;
    p.y = (int)(head * PAGE) + (n0 & (PAGE - 1));
    p.ku = __ldcg(a.c.ku + head);
    p.vu = __ldcg(a.c.vu + head);
    p.n0 = n0 >> PAGE_SHIFT >= s.open ? ~n0 : n0;
    return p;
}

template <int D>
__global__ void __launch_bounds__(THREADS, 1) attn8_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Attn8Args a) {
    using L = Lay<D>;
    constexpr int NS = L::NS, CHUNKS = D / 16;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t bars[WARPS * NS];
    __shared__ Place places[2 * BATCH];
    __shared__ Unit list[MAX_UNITS];
    __shared__ uint32_t prefix[MAX_UNITS + 1], sums[WARPS];
    __shared__ float2 s_ml[WARPS][16];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tq = lane & 3;
    const int units = a.positions ? a.rows : a.n_segs, G = a.c.kv_heads, group = a.n_heads / G;
    if (tid < WARPS * NS) mbar_init(&bars[tid], 1);
    if (tid == 0) asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    pdl_launch();
    if (!a.behind) pdl_wait();
    count_turns(a, units, list, prefix, sums);
    const uint32_t total = prefix[units], share = share_of(total, gridDim.x);
    const uint32_t x0 = blockIdx.x * share, x1 = min(total, x0 + share);
    if (x0 >= x1) {
        if (a.behind) pdl_wait();      // the launch does not end before the one it follows
        return;
    }
    if (x0 + tid < x1) places[tid] = place_of(a, list, prefix, units, x0 + tid);
    __syncthreads();

    uint8_t* ring = sm + warp * NS * L::STAGE;
    uint64_t* full = bars + warp * NS;
    const int mine = x0 + warp < x1 ? (int)((x1 - x0 - warp + WARPS - 1) / WARPS) : 0;      // turns of this warp
    auto issue = [&](int k) {
        if (k < mine && lane == 0) {
            const int y = places[(warp + WARPS * k) % (2 * BATCH)].y, s = k % NS;
            mbar_expect_tx(&full[s], L::STAGE);
            tma_load_2d(ring + s * L::STAGE, &map_k, 0, y, &full[s]);
            tma_load_2d(ring + s * L::STAGE + L::HALF, &map_v, 0, y, &full[s]);
        }
    };
    int asked = 0;                          // turns that have been requested
    if (a.behind) {
        // The rows are still being appended: pages that none of them goes to can be fetched, and their units are what they were.
        for (; asked < min(mine, NS - 1) && places[warp + WARPS * asked].n0 >= 0; asked++) issue(asked);
        pdl_wait();
        if (x0 + tid < x1 && places[tid].n0 < 0) places[tid] = place_of(a, list, prefix, units, x0 + tid);
        __syncthreads();
    }
    for (; asked < NS - 1; asked++) issue(asked);

    int k = 0, batch = 0;                   // the warp's next turn; the CTA's batch
    bool ok = true;
    auto look_ahead = [&]() {               // the places of the batch after the next one, which replace this one's
        const uint32_t x = x0 + (uint32_t)BATCH * (batch + 2) + tid;
        return tid < BATCH && x < x1 ? place_of(a, list, prefix, units, x) : Place{};
    };
    Place ahead = look_ahead();
    for (uint32_t xa = x0; xa < x1;) {      // items of the run
        const int u = unit_of(prefix, units, xa);
        const Unit s = list[u];
        const Keys ks = keys_of(a, s);
        const uint32_t item = (xa - prefix[u]) / ks.turns, xb = min(x1, prefix[u] + (item + 1) * ks.turns);
        const int kvh = item % G, m0 = 16 * (item / G), rows_m = min(16, s.rows * group - m0);
        // the lane's query rows g and g + 8, columns in the order in which a lane holds a key's codes
        uint32_t qf[CHUNKS][4];
        int pos[2], lo[2];
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int m = m0 + g + 8 * r, row = m / group;
            const bool live = g + 8 * r < rows_m;
            pos[r] = s.pos + (live ? row : s.rows - 1);
            lo[r] = first_key(pos[r], a.chunk, a.window);
            const float* q = a.q + ((size_t)(s.row + row) * a.n_heads + kvh * group + m % group) * D + 4 * tq;
#pragma unroll
            for (int c = 0; c < CHUNKS; c++) {
                const float4 v = live ? __ldcg((const float4*)(q + 16 * c)) : make_float4(0.f, 0.f, 0.f, 0.f);
                qf[c][r] = pack_h2(v.x, v.y);
                qf[c][r + 2] = pack_h2(v.z, v.w);
            }
        }
        const int first_pos = s.pos + m0 / group, last_lo = first_key(s.pos + min(s.rows - 1, (m0 + 15) / group), a.chunk, a.window), keep = a.window > 0 ? a.keep : 0;
        float o[CHUNKS][2][4];
#pragma unroll
        for (int c = 0; c < CHUNKS; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) o[c][e >> 2][e & 3] = 0.f;
        float m_run[2] = {NONE, NONE}, l_run[2] = {0.f, 0.f}, v_unit = 1.f;

        for (;;) {
        const uint32_t batch_end = x0 + (uint32_t)BATCH * (batch + 1), end = min(xb, batch_end);
        for (; ok && x0 + warp + (uint32_t)WARPS * k < end; k++) {
            issue(k + NS - 1);
            Place p = places[(warp + WARPS * k) % (2 * BATCH)];
            p.n0 = max(p.n0, ~p.n0);
            const int st = k % NS;
            if (!mbar_wait(&full[st], (k / NS) & 1)) {
                ok = false;
                break;
            }
            uint8_t* kt = ring + st * L::STAGE;
            uint8_t* vt = kt + L::HALF;
            float sc[4][4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
#pragma unroll
                for (int c4 = 0; c4 < CHUNKS; c4 += 4) {
                    uint32_t kb[4];
                    ldsm_x4(kb, smem_u32(kt + L::at(8 * j + (lane & 7), c4 + (lane >> 3))));
#pragma unroll
                    for (int c = 0; c < 4; c++) mma_f16(sc[j], qf[c4 + c], e4m3x2_to_h2(kb[c]), e4m3x2_to_h2(kb[c] >> 16));
                }
            }
            const bool all = p.n0 + TURN - 1 <= first_pos && (p.n0 >= last_lo || p.n0 + TURN <= keep);      // every row sees every key
            // element e of block j: row g + 8 (e >> 1), key n0 + 8 j + 2 tq + (e & 1)
            uint32_t bad = 0;
            if (!all) {
                // A value that is no number would reach the rows that do not see it through a weight of zero: its row becomes zeros, and its key's scores none, of the rows that do.
                bool none = false;
                uint4* row = (uint4*)(vt + lane * D);
#pragma unroll
                for (int c = 0; c < CHUNKS; c++) {
                    const uint4 w = row[c];
                    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int i = 0; i < 4; i++) none |= (((ws[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
                }
                bad = __ballot_sync(0xffffffffu, none);
                if (none) {
#pragma unroll
                    for (int c = 0; c < CHUNKS; c++) row[c] = make_uint4(0, 0, 0, 0);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                __syncwarp();
            }
            const float f = a.scale * p.ku * (a.softcap > 0.f ? 1.f / a.softcap : LOG2E);
            float mx[2] = {NONE, NONE};
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float v = sc[j][e] * f;
                    if (a.softcap > 0.f) v = a.softcap * LOG2E * tanh_exp(v);
                    if (!all) {
                        const int i = 8 * j + 2 * tq + (e & 1), kp = p.n0 + i;
                        if (bad >> i & 1) v = __int_as_float(0x7fffffff);
                        if (!(kp <= pos[e >> 1] && (kp >= lo[e >> 1] || kp < keep))) v = -INFINITY;
                    }
                    sc[j][e] = v;
                    mx[e >> 1] = fmaxf(mx[e >> 1], v);
                }
            float corr[2];
            const float turn_unit = v_unit / p.vu;      // sums count in the unit of the last turn's values
            v_unit = p.vu;
#pragma unroll
            for (int r = 0; r < 2; r++) {
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                const float m_new = fmaxf(m_run[r], mx[r]);
                corr[r] = ex2(m_run[r] - m_new);
                m_run[r] = m_new;
                l_run[r] *= corr[r];
                corr[r] *= turn_unit;
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float w = ex2(sc[j][e] - m_run[e >> 1]);
                    sc[j][e] = w;
                    l_run[e >> 1] += w;
                }
#pragma unroll
            for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                for (int e = 0; e < 8; e++) o[c][e >> 2][e & 3] *= corr[(e & 3) >> 1];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t pa[4] = {pack_h2(sc[2 * h][0], sc[2 * h][1]), pack_h2(sc[2 * h][2], sc[2 * h][3]), pack_h2(sc[2 * h + 1][0], sc[2 * h + 1][1]),
                                        pack_h2(sc[2 * h + 1][2], sc[2 * h + 1][3])};
#pragma unroll
                for (int c = 0; c < CHUNKS; c += 2) {
                    uint32_t vb[4];
                    ldsm_x4_trans(vb, smem_u32(vt + L::at(16 * h + (lane & 15), c + (lane >> 4))));
                    // a register holds columns 2 g and 2 g + 1 of two keys: those of the even column, then of the odd one
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const uint32_t w0 = __byte_perm(vb[2 * i], 0, 0x3120), w1 = __byte_perm(vb[2 * i + 1], 0, 0x3120);
                        mma_f16(o[c + i][0], pa, e4m3x2_to_h2(w0), e4m3x2_to_h2(w1));
                        mma_f16(o[c + i][1], pa, e4m3x2_to_h2(w0 >> 16), e4m3x2_to_h2(w1 >> 16));
                    }
                }
            }
            __syncwarp();
        }
        if (batch_end < x1 && end == batch_end) {
            __syncthreads();
            if (tid < BATCH) places[(batch & 1) * BATCH + tid] = ahead;
            __syncthreads();
            batch++;
            ahead = look_ahead();
        }
        if (end == xb) break;
        }

#pragma unroll
        for (int r = 0; r < 2; r++) {
            l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
            l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
            if (tq == 0) s_ml[warp][g + 8 * r] = make_float2(m_run[r], l_run[r]);
#pragma unroll
            for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    o[c][e][2 * r] *= v_unit;
                    o[c][e][2 * r + 1] *= v_unit;
                }
        }
        // The warps' sums become one: they leave them in shared memory, as many rows at a time as there is room for (all, in their rings, once those have served).
        const size_t piece = piece_of(a, u, item) + blockIdx.x;
        const bool last = xb == x1;
        const int step = last ? 16 : L::MERGE / (WARPS * D * 4), pitch = last ? NS * L::STAGE / 16 : step * (D / 4);
        float4* dump = reinterpret_cast<float4*>(sm + (last ? 0 : L::RING));
        for (int r0 = 0; r0 < rows_m; r0 += step) {
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int row = g + 8 * r - r0;
                if (row < 0 || row >= min(step, rows_m - r0)) continue;
#pragma unroll
                for (int c = 0; c < CHUNKS; c++)
                    dump[warp * pitch + row * (D / 4) + 4 * c + tq] = make_float4(o[c][0][2 * r], o[c][1][2 * r], o[c][0][2 * r + 1], o[c][1][2 * r + 1]);
            }
            __syncthreads();
            for (int i = tid; i < min(step, rows_m - r0) * (D / 4); i += THREADS) {
                const int row = r0 + i / (D / 4);
                float top = NONE, l = 0.f;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < WARPS; w++) top = fmaxf(top, s_ml[w][row].x);
#pragma unroll
                for (int w = 0; w < WARPS; w++) {
                    const float f = ex2(s_ml[w][row].x - top);
                    const float4 y = dump[w * pitch + i];
                    l += f * s_ml[w][row].y;
                    v.x += f * y.x;
                    v.y += f * y.y;
                    v.z += f * y.z;
                    v.w += f * y.w;
                }
                ((float4*)(a.part_acc + (piece * 16 + row) * D))[i % (D / 4)] = v;
                if (i % (D / 4) == 0) a.part_ml[piece * 16 + row] = make_float2(top, l);
            }
            __syncthreads();
        }
        xa = xb;
        // a wait that ran out: everyone leaves, after the copies that are still under way
        if (__syncthreads_or(!ok)) {
            for (int i = k; i < min(mine, k + NS - ok); i++) mbar_wait(&full[i % NS], (i / NS) & 1);
            if (tid == 0) atomicExch(&g_attn8_status, KS_TIMEOUT);
            return;
        }
    }
}

// Sums of an item's row at column d, over the runs that hold a part of the item.
__device__ __forceinline__ float merged(const Attn8Args& a, int hd, size_t piece, uint32_t from, uint32_t turns, uint32_t share, int m, int d) {
    const int c0 = from / share, c1 = (from + turns - 1) / share;
    float top = NONE, v = 0.f, l = 0.f;
    for (int c = c0; c <= c1; c++) {
        const size_t at = (piece + c) * 16 + m;
        const float2 ml = __ldcg(a.part_ml + at);
        const float x = __ldcg(a.part_acc + at * hd + d), mn = fmaxf(top, ml.x), w0 = ex2(top - mn), w1 = ex2(ml.x - mn);
        v = v * w0 + x * w1;
        l = l * w0 + ml.y * w1;
        top = mn;
    }
    return v / l;
}

// A CTA a row and THREADS / hd heads (maps), a thread a column.
__global__ void __launch_bounds__(THREADS) attn8_merge_kernel(const __grid_constant__ Attn8Args a) {
    __shared__ Unit list[MAX_UNITS];
    __shared__ uint32_t prefix[MAX_UNITS + 1], sums[WARPS];
    __shared__ float second[THREADS], red[WARPS];
    const int hd = a.c.hd, tid = threadIdx.x, G = a.c.kv_heads, group = a.n_heads / G, units = a.positions ? a.rows : a.n_segs;
    const int h = blockIdx.x * (THREADS / hd) + tid / hd, d = tid % hd, row = blockIdx.y;
    pdl_launch();
    if (!a.behind) pdl_wait();
    count_turns(a, units, list, prefix, sums);
    int u = -1;
    if (a.positions) {
        u = row;
    } else {
        for (int i = 0; i < units; i++) {
            const int4 s = a.segs[i];
            if (row >= s.x && row < s.x + s.y) u = i;
        }
    }
    if (a.behind) pdl_wait();
    if (u < 0) return;
    const Unit s = list[u];
    const uint32_t turns = keys_of(a, s).turns;
    if (turns == 0) return;
    const bool in = h < a.n_heads;
    float v = 0.f;
    if (in) {
        const int m = (row - s.row) * group + h % group;
        const uint32_t item = (m >> 4) * G + h / group;
        v = merged(a, hd, piece_of(a, u, item), prefix[u] + item * turns, turns, share_of(prefix[units], a.ctas), m & 15, d);
    }
    int ho = h;
    if (a.diff.on) {        // threads of even maps take the odd ones' results
        if (d >= a.vdim) v = 0.f;
        second[tid] = v;
        __syncthreads();
        const int map = tid / hd & 1;
        if (!map) v -= a.diff.lambda * second[tid + hd];
        const float sq = warp_sum(v * v);
        if ((tid & 31) == 0) red[tid >> 5] = sq;
        __syncthreads();
        if (map) return;
        float sum = 0.f;
        for (int w = 0; w < hd / 32; w++) sum += red[tid / hd * (hd / 32) + w];
        v *= a.diff.scale / sqrtf(sum / (float)a.vdim + a.diff.eps);
        ho = h >> 1;
    }
    if (!in || d >= a.vdim) return;
    if (a.gate.kind) v *= sigmoid_f(a.gate.g[(size_t)row * a.gate.ld + (a.gate.kind == 1 ? ho * a.vdim + d : ho)]);
    const size_t oi = (size_t)row * a.ldo + (size_t)ho * a.vdim + d;
    if (a.out16) ((__nv_bfloat16*)a.out)[oi] = __float2bfloat16_rn(v);
    else ((float*)a.out)[oi] = v;
}

bool bad_args(const Attn8Args& a) {
    return !a.q || !a.c.k || !a.c.v || !a.c.ku || !a.c.vu || a.c.n_pages < 1 || (a.c.hd != 64 && a.c.hd != 128) || a.c.kv_heads < 1 || a.n_heads < 1 || a.n_heads % a.c.kv_heads ||
           a.n_heads > 65535 || a.rows < 1 || a.rows > 65535 || a.vdim < 1 || a.vdim > a.c.hd || !a.t.table || a.t.n_slots < 1 || a.t.max_pages < 1 || a.t.max_pages > (1 << 24) ||
           (!a.positions == !a.segs) || (a.positions && !a.slots) || (a.segs && a.n_segs < 1) || a.chunk < 0 || a.window < 0 || a.keep < 0 || (a.chunk && a.window) || a.softcap < 0.f ||
           a.tiles < 1 || a.ctas < 1 || !a.part_acc || !a.part_ml || !a.out || a.gate.kind < 0 || a.gate.kind > 2 || (a.gate.kind && !a.gate.g) ||
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

template <int D>
int launch(Attn8Args& a, int pdl, cudaStream_t st) {
    CUtensorMap mk, mv;
    const size_t rows = (size_t)a.c.n_pages * a.c.kv_heads * PAGE;
    if (!code_map<D>(&mk, a.c.k, rows) || !code_map<D>(&mv, a.c.v, rows)) return (int)cudaErrorNotSupported;
    static PerDeviceOnce once;
    if (once.first()) cudaFuncSetAttribute(attn8_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<D>::TOTAL);
    void* args[] = {&mk, &mv, &a};
    return launch_rows((const void*)attn8_kernel<D>, dim3(a.ctas), dim3(THREADS), Lay<D>::TOTAL, args, st, pdl);
}

}  // namespace

static int attn8_launch(const Attn8Args& in, int pdl, cudaStream_t st) {
    if (bad_args(in)) return (int)cudaErrorInvalidValue;
    const int units = in.positions ? in.rows : in.n_segs, heads = THREADS / in.c.hd;
    for (int u = 0; u < units; u += MAX_UNITS) {
        Attn8Args a = in;
        const int n = units - u < MAX_UNITS ? units - u : MAX_UNITS;
        if (a.positions) {
            a.positions += u;
            a.slots += u;
            a.rows = n;
            a.q += (size_t)u * a.n_heads * a.c.hd;
            a.out = (char*)a.out + (size_t)u * a.ldo * (a.out16 ? 2 : 4);
            if (a.gate.kind) a.gate.g += (size_t)u * a.gate.ld;
        } else {
            a.segs += u;
            a.n_segs = n;
        }
        a.behind = in.behind && units <= MAX_UNITS;
        int rc = a.c.hd == 128 ? launch<128>(a, pdl || a.behind, st) : launch<64>(a, pdl || a.behind, st);
        if (rc) return rc;
        void* args[] = {&a};
        rc = launch_rows((const void*)attn8_merge_kernel, dim3((a.n_heads + heads - 1) / heads, a.rows), dim3(THREADS), 0, args, st, 1);
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
    return v;
}
