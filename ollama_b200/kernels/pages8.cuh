// 8-bit paged cache: pages of 64 positions [page][kv head][64][hd] of E4M3 codes (hd = 64 or 128, pad columns zero), which count in a unit of their own for each page and
// KV head, [page][kv head].  Units are powers of two between 2^-15 and 2^7, so that every value of the cache, code times unit, is an f16 number too
// (448 * 2^7 = 57344, 2^-9 * 2^-15 the least subnormal), and a unit that grows leaves old codes as they are but for the subnormal ones.
#pragma once
#include "rows.cuh"

constexpr int UNIT_LOW = -15, UNIT_HIGH = 7;
constexpr float E4M3_MAX = 448.f;

// Keys and values of one layer run.
struct Pages8 {
    uint8_t* k;
    float* ku;
    uint8_t* v;
    float* vu;
    int n_pages, kv_heads, hd;
};
// Where the pages of a slot are: table[slot][i] holds positions 64 i .. 64 i + 63.
struct PageTable {
    const int* table;
    int n_slots, max_pages;
};

// What rows are appended, b2_append8.
struct Append8Args {
    const float* qkv;        // [rows][ldq]: q heads | k heads | ..., value heads from column v_off on
    int ldq, rows, n_heads, dim, vdim;
    const float* q_norm;     // see PagedAppendArgs
    const float* k_norm;
    float eps;
    const double* freqs;     // [n_rot / 2]
    int n_rot;
    const int* positions;    // [rows], one row a sequence; or null:
    const int* slots;
    const int4* segs;        // [n_segs] portions (first row, rows, slot, position of the first row), of slots of their own
    int n_segs, per;         // per: most pages that a portion touches
    PageTable t;
    float* q_out;            // [rows][H][hd]
    Pages8 c;
    int head_norm, v_off;
    float mscale;
    int maps, no_append;
};

// Attention of rows, b2_attn8 (attn_pages8.cu).
struct Attn8Args {
    const float* q;          // [rows][H][hd], rotated
    int rows, n_heads, vdim;
    Pages8 c;
    PageTable t;
    const int* positions;    // [rows], or null:
    const int* slots;
    const int4* segs;        // [n_segs] portions (first row, rows, slot, position of the first row)
    int n_segs;
    int chunk, window, keep;
    float scale, softcap;
    int row_tile, turn;      // query rows (of a sequence, for the heads of a KV head) and keys that are taken together: 8 or 16 and 32, 128 and 128
    int tiles;               // most row tiles of a sequence
    int ctas;                // that fit the GPU at once
    float* part_acc;         // [items + ctas][row_tile][hd]
    float2* part_ml;         // [items + ctas][row_tile] (largest score, sum)
    void* out;               // [rows][ldo], head h at column h * vdim
    int ldo, out16;
    HeadGate gate;
    DiffHeads diff;
    int behind;              // the launch follows the one that appends the rows, which writes neither positions, slots nor tables
};

// Codes of two values (the first in the low byte), rounded to nearest even; magnitudes beyond 448 become 448, what is no number stays none.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// Two codes as f16 values, exact.
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t two) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
    return r;
}
__device__ __forceinline__ float2 e4m3x2_to_f2(uint32_t two) {
    const uint32_t h = e4m3x2_to_h2(two);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Whether one of 16 codes is no number.
__device__ __forceinline__ bool holds_nan(const uint4& w) {
    return ((((w.x & 0x7f7f7f7fu) + 0x01010101u) | ((w.y & 0x7f7f7f7fu) + 0x01010101u) | ((w.z & 0x7f7f7f7fu) + 0x01010101u) | ((w.w & 0x7f7f7f7fu) + 0x01010101u)) & 0x80808080u) != 0;
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// The unit in which a magnitude is at most 448 = 1.75 * 2^8: the least such power of two, within the limits.
__device__ __forceinline__ float unit_for(float top) {
    const uint32_t b = __float_as_uint(top);
    const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u);
    return pow2(min(max(e, UNIT_LOW), UNIT_HIGH));
}

// The page of a slot's positions 64 i .. 64 i + 63; -1 for a slot, a position or a page that is not there.
__device__ __forceinline__ int page_at(const PageTable& t, int n_pages, int slot, int i) {
    if ((unsigned)slot >= (unsigned)t.n_slots || (unsigned)i >= (unsigned)t.max_pages) return -1;
    const int p = __ldg(t.table + (size_t)slot * t.max_pages + i);
    return (unsigned)p < (unsigned)n_pages ? p : -1;
}

// A cudaError_t value.
int append8_launch(const Append8Args& a, int pdl, cudaStream_t st);
