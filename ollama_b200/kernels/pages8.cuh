// 8-bit paged cache: pages of 64 positions [page][kv head][64][hd] of E4M3 codes (hd = 64 or 128, pad columns zero), which count in a unit of their own for each page and
// KV head, [page][kv head].  Units are powers of two between 2^-15 and 2^7, so that every value of the cache, code times unit, is an f16 number too
// (448 * 2^7 = 57344, 2^-9 * 2^-15 the least subnormal), and a unit that grows leaves old codes as they are but for the subnormal ones.
#pragma once
#include "pages8_args.h"
#include "rows.cuh"

constexpr int UNIT_LOW = -15, UNIT_HIGH = 7;
constexpr float E4M3_MAX = 448.f;

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

// Whether the table has the position.
__device__ __forceinline__ bool has(const PageTable& t, int slot, int pos) {
    return (unsigned)slot < (unsigned)t.n_slots && pos >= 0 && pos >> PAGE_SHIFT < t.max_pages;
}
// The page of a slot's positions 64 i .. 64 i + 63; -1 for a slot, a position or a page that is not there.
__device__ __forceinline__ int page_at(const PageTable& t, int n_pages, int slot, int i) {
    if ((unsigned)slot >= (unsigned)t.n_slots || (unsigned)i >= (unsigned)t.max_pages) return -1;
    const int p = __ldg(t.table + (size_t)slot * t.max_pages + i);
    return (unsigned)p < (unsigned)n_pages ? p : -1;
}

// A cudaError_t value.
int append8_launch(const Append8Args& a, int pdl, cudaStream_t st);
