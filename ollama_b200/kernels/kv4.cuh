// The 4-bit cache: what a row's bytes say, and the device functions that read and make them.
//
// A row of hd columns (64 or 128) is hd / 2 bytes of codes 0 .. 15 and an f16 scale d for every 32 columns; a value is d (code - 8).  Eight neighbouring columns are a 32-bit word: column 2 i of
// them in bits 4 i .., column 2 i + 1 in bits 16 + 4 i .., so that one mask takes two neighbours into the halves of a register.  Word j of a block of 32 columns stands before word j + 1 of any
// (word j * (hd / 32) + b of the row is columns 32 b + 8 j ..): the lanes of a matrix product's operand, which want the same word of every block, find theirs side by side.
// d is minus an eighth of the value of largest magnitude (of two, the negative one), rounded to f16 and at most 8188, eight times which is an f16 number; a code is the quotient rounded to the
// nearest, ties to even.  So the largest value is held to f16's precision and the others within half a step, but for one of the other sign as large as it, which is one step smaller.  Values
// that are no number are held as zero.
#pragma once
#include "kv4_args.h"
#include "rows.cuh"

namespace kv4 {

constexpr float TOP = 8188.f;

// Codes of two columns (or of a column of two rows) to f16 pairs: pair i is nibble i of the word's halves.  1024 + n and 1024 + 16 n are f16 numbers whose low bits are the nibble, and so are
// n - 8 and its products by a power of two: nothing is rounded.  Nine instructions for eight codes.
__device__ __forceinline__ uint32_t hsub2_bits(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t hfma2_bits(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t hmul2_bits(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
template <uint32_t MASK>
__device__ __forceinline__ uint32_t masked_or_1024(uint32_t w) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(w), "n"(MASK), "r"(0x64006400u));      // (w & MASK) | 0x64006400
    return d;
}
__device__ __forceinline__ void expand(uint32_t w, uint32_t (&e)[4]) {
    constexpr uint32_t LOW = 0x64086408u, SIXTEENTH = 0x2C002C00u, MINUS_72 = 0xD480D480u;      // 1032, 1 / 16, -72
    const uint32_t w8 = w >> 8;
    e[0] = hsub2_bits(masked_or_1024<0x000f000fu>(w), LOW);
    e[1] = hfma2_bits(masked_or_1024<0x00f000f0u>(w), SIXTEENTH, MINUS_72);
    e[2] = hsub2_bits(masked_or_1024<0x000f000fu>(w8), LOW);
    e[3] = hfma2_bits(masked_or_1024<0x00f000f0u>(w8), SIXTEENTH, MINUS_72);
}

__device__ __forceinline__ bool has_row(const Cache4& c, int pos, int slot) { return (unsigned)pos < (unsigned)c.n_ctx && (unsigned)slot < (unsigned)c.slots; }
__device__ __forceinline__ size_t row_of(const Cache4& c, int pos, int slot, int kvh) { return ((size_t)slot * c.kv_heads + kvh) * c.n_ctx + pos; }

// What turns a lane's columns N lane .. N lane + N - 1 of any head of a token: x cos + y sin, y the pair's other column.
template <int HD>
struct Turn {
    static constexpr int N = HD / 32;
    float c[N], s[N];
    int at[N];               // the other column, -1 of a column that is not turned
};

// cs, sn: cosines and sines of the token's pairs.
template <int HD>
__device__ __forceinline__ Turn<HD> make_turn(const Rows4& r, const float* cs, const float* sn, int lane) {
    Turn<HD> t;
#pragma unroll
    for (int j = 0; j < Turn<HD>::N; j++) {
        const int i = Turn<HD>::N * lane + j, half = r.n_rot >> 1;
        t.at[j] = -1;
        t.c[j] = 1.f;
        t.s[j] = 0.f;
        if (i < r.n_rot) {
            const bool first = r.neox ? i < half : !(i & 1);
            const int p = r.neox ? (first ? i : i - half) : i >> 1;
            t.at[j] = r.neox ? (first ? i + half : i - half) : i ^ 1;
            t.c[j] = cs[p];
            t.s[j] = first ? -sn[p] : sn[p];
        }
    }
    return t;
}

// The angles are formed in double: in 32 bits a position of 100000 would leave 0.004 of a radian.
__device__ __forceinline__ void fill_angles(const Rows4& r, int pos, float* cs, float* sn, int tid, int threads) {
    for (int p = tid; p < (r.n_rot >> 1); p += threads) {
        float s, c;
        sincosf(rot_angle(pos, (double)r.inv_freq[p]), &s, &c);
        sn[p] = s * r.mscale;
        cs[p] = c * r.mscale;
    }
}

// Norm and rotation of a head by a warp: x[N] are its columns N lane ..; `row`: HD floats of the warp's own.
template <int HD>
__device__ __forceinline__ void prepare_head(float (&x)[HD / 32], const float* norm, float eps, bool turned, const Turn<HD>& t, float* row, int lane) {
    constexpr int N = HD / 32;
    if (norm) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < N; j++) s += x[j] * x[j];
        const float inv = 1.f / sqrtf(warp_sum(s) / (float)HD + eps);
#pragma unroll
        for (int j = 0; j < N; j++) x[j] = x[j] * inv * norm[N * lane + j];
    }
    if (!turned) return;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < N; j++) row[N * lane + j] = x[j];
    __syncwarp();
#pragma unroll
    for (int j = 0; j < N; j++)
        if (t.at[j] >= 0) x[j] = x[j] * t.c[j] + row[t.at[j]] * t.s[j];
}

// A warp makes the codes of a row.  Lane l has columns N l ..; the lane of a word's first columns gets the word (where `lead`), that of a block's first the scale (`first`).
template <int HD>
struct Coded {
    uint32_t word;
    int at;                  // which word of the row
    bool lead, first;
    __half d;
    int block;
};
template <int HD>
__device__ __forceinline__ Coded<HD> encode(const float (&in)[HD / 32], int lane) {
    constexpr int N = HD / 32, PER_BLOCK = 32 / N, PER_WORD = 8 / N;
    float x[N], hi = -INFINITY, lo = INFINITY;
#pragma unroll
    for (int j = 0; j < N; j++) {
        x[j] = in[j] == in[j] ? in[j] : 0.f;
        hi = fmaxf(hi, x[j]);
        lo = fminf(lo, x[j]);
    }
#pragma unroll
    for (int o = 1; o < PER_BLOCK; o <<= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    const float far = hi > -lo ? hi : lo;
    Coded<HD> r;
    r.d = __float2half_rn(fminf(fmaxf(far * -0.125f, -TOP), TOP));
    const float d = __half2float(r.d);
    const int i0 = (lane % PER_WORD) * N;      // first of the lane's columns in its word
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < N; j++) {
        const float q = d != 0.f ? fminf(fmaxf(rintf(x[j] / d) + 8.f, 0.f), 15.f) : 8.f;
        const int i = i0 + j;
        w |= (uint32_t)q << (4 * (i >> 1) + 16 * (i & 1));
    }
#pragma unroll
    for (int o = 1; o < PER_WORD; o <<= 1) w |= __shfl_xor_sync(0xffffffffu, w, o);
    r.word = w;
    r.block = lane / PER_BLOCK;
    r.at = lane % PER_BLOCK / PER_WORD * (HD / 32) + r.block;
    r.lead = lane % PER_WORD == 0;
    r.first = lane % PER_BLOCK == 0;
    return r;
}

}  // namespace kv4
