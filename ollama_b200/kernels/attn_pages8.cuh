// How attention over an 8-bit paged cache is dealt out to CTAs; shared by its kernels (attn_pages8.cu, attn_pages8_tc.cu) and their merge.
#pragma once
#include "pages8.cuh"

namespace {

constexpr int MAX_UNITS = 256;               // sequences of a launch
constexpr int LEAST = 256;                   // keys of a CTA, where there are as many
constexpr float LOG2E = 1.4426950408889634f;
constexpr float NONE = -1e30f;               // largest score of no keys

// The rows of one sequence in the launch.
struct Unit {
    int row, rows, slot, pos;                // first row, rows (0: no token), slot, position of the first row
    int open;                                // first page of the slot that rows of the step go to
    int parts;                               // CTAs of each of its items
};

__device__ __forceinline__ Unit unit_at(const Attn8Args& a, int u) {
    Unit s;
    if (a.positions) {
        s = Unit{u, 1, a.slots[u], a.positions[u], 0, 0};
    } else {
        const int4 g = a.segs[u];
        s = Unit{g.x, g.y, g.z, g.w, 0, 0};
    }
    if ((unsigned)s.slot >= (unsigned)a.t.n_slots || s.pos < 0 || s.row < 0 || s.rows < 0 || s.rows > a.rows - s.row || s.rows > a.t.max_pages * PAGE - s.pos ||
        s.rows * (a.n_heads / a.c.kv_heads) > a.tiles * a.row_tile)
        s.rows = 0;
    s.open = s.pos >> PAGE_SHIFT;
    return s;
}

// Turns of a unit's items: those with kept keys first, then the ones from the first row's first key on.
struct Keys {
    int base, front, turns;
};
__device__ __forceinline__ Keys keys_of(const Attn8Args& a, const Unit& s) {
    const int turn = a.turn;
    Keys k;
    k.base = first_key(s.pos, a.chunk, a.window) & ~(turn - 1);
    k.front = a.window > 0 ? kept_tiles(a.keep, k.base, turn) : 0;
    k.turns = s.rows > 0 ? k.front + (s.pos + s.rows - k.base + turn - 1) / turn : 0;
    return k;
}
__device__ __forceinline__ int first_of(const Keys& k, int turn, int i) { return i < k.front ? i * turn : k.base + (i - k.front) * turn; }

// Items of a unit: row_tile rows of (row, head of the KV head) each, of every KV head.
__device__ __forceinline__ int row_tiles(const Attn8Args& a, const Unit& s) { return (s.rows * (a.n_heads / a.c.kv_heads) + a.row_tile - 1) / a.row_tile; }
// Their number, as far as there is room for them; below 2^24, so that those of MAX_UNITS units fit 32 bits.
__device__ __forceinline__ uint32_t items_of(const Attn8Args& a, const Unit& s) { return min(row_tiles(a, s) * a.c.kv_heads, a.items + 1); }

// Sum of the threads' numbers up to each and over all; at least MAX_UNITS threads, `sums` has one place a warp.
__device__ __forceinline__ uint32_t scan(uint32_t x, uint32_t* sums, uint32_t& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    all = 0;
    for (int w = 0; w < MAX_UNITS / 32; w++) {
        if (w == warp) x += all;
        all += sums[w];
    }
    return x;
}

// CTAs of each item of a unit, of so many turns in all.
__device__ __forceinline__ uint32_t parts_of(const Attn8Args& a, uint32_t turns, uint32_t total) {
    return turns ? max(1u, min((uint32_t)((unsigned long long)turns * a.ctas / total), (turns * a.turn + LEAST - 1) / LEAST)) : 0;
}

// All units, and the CTAs before each one's (prefix[u]) and in all (prefix[units]); none where the units have more items than there is room for.
__device__ __forceinline__ void deal_out(const Attn8Args& a, int units, Unit* list, uint32_t* prefix, uint32_t* sums) {
    const int tid = threadIdx.x;
    Unit s;
    uint32_t turns = 0, items = 0, total, ctas;
    if (tid < units) {
        s = unit_at(a, tid);
        list[tid] = s;
        turns = keys_of(a, s).turns;
        items = items_of(a, s);
    }
    if (!a.positions) {      // portions that say less than they hold
        scan(items, sums, total);
        if (total > (uint32_t)a.items) turns = 0;
    }
    scan(turns * items, sums, total);
    const uint32_t parts = parts_of(a, turns, total);
    const uint32_t x = scan(parts * items, sums, ctas);
    if (tid < units) {
        prefix[tid] = x - parts * items;
        if (a.behind)        // other rows of the slot may go to earlier pages
            for (int i = 0; i < units; i++)
                if (list[i].slot == s.slot && list[i].pos >= 0) s.open = min(s.open, list[i].pos >> PAGE_SHIFT);
    }
    if (tid == 0) prefix[units] = ctas;
    __syncthreads();
    if (tid < units) {
        s.parts = parts;
        list[tid] = s;
    }
    __syncthreads();
}

__device__ __forceinline__ int unit_of(const uint32_t* prefix, int units, uint32_t x) {
    int lo = 0, hi = units - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (prefix[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;               // of units without turns, the one behind them
}

struct DealRoom {
    Unit list[MAX_UNITS];
    uint32_t prefix[MAX_UNITS + 1], sums[32];
};
// The unit of CTA x (BY_CTA) or unit x, and the first of its CTAs; false: there is none.  Of up to 32 units every warp finds out by itself: with the block's scans a small step took
// 2 us more.
template <bool BY_CTA>
__device__ __forceinline__ bool find_unit(const Attn8Args& a, int units, uint32_t x, DealRoom& room, Unit& s, uint32_t& first) {
    if (units > 32) {
        deal_out(a, units, room.list, room.prefix, room.sums);
        if (BY_CTA && x >= room.prefix[units]) return false;
        const int u = BY_CTA ? unit_of(room.prefix, units, x) : x;
        s = room.list[u];
        first = room.prefix[u];
        return s.parts > 0;
    }
    constexpr uint32_t ALL = 0xffffffffu;
    const int lane = threadIdx.x & 31;
    Unit m = {};
    uint32_t turns = 0, items = 0;
    if (lane < units) {
        m = unit_at(a, lane);
        turns = keys_of(a, m).turns;
        items = items_of(a, m);
    }
    if (!a.positions && __reduce_add_sync(ALL, items) > (uint32_t)a.items) return false;      // portions that say less than they hold
    const uint32_t parts = parts_of(a, turns, __reduce_add_sync(ALL, turns * items)), n = parts * items;
    uint32_t end = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(ALL, end, o);
        if (lane >= o) end += y;
    }
    const uint32_t mine = __ballot_sync(ALL, BY_CTA ? x >= end - n && x < end : lane == (int)x && n > 0);
    if (!mine) return false;
    const int u = __ffs(mine) - 1;
    s.row = __shfl_sync(ALL, m.row, u);
    s.rows = __shfl_sync(ALL, m.rows, u);
    s.slot = __shfl_sync(ALL, m.slot, u);
    s.pos = __shfl_sync(ALL, m.pos, u);
    s.parts = __shfl_sync(ALL, (int)parts, u);
    first = __shfl_sync(ALL, end - n, u);
    // other rows of the slot may go to earlier pages
    s.open = __reduce_min_sync(ALL, lane < units && m.slot == s.slot && m.pos >= 0 ? m.pos >> PAGE_SHIFT : 0x7fffffff);
    return true;
}

}  // namespace

// Attention of tiles of 128 query rows, the sums to be merged as those of attn8_kernel; a cudaError_t value (attn_pages8_tc.cu).
int attn8_tc_launch(const Attn8Args& a, int grid, int pdl, cudaStream_t st);
// 0, KS_TIMEOUT once a wait of it has run out since the last call, or -1.
int attn8_tc_status();
