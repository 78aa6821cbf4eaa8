// The 4-bit cache: what a row's bytes say, and the device functions that read and make them.
//
// A row of hd columns (64 or 128) is hd / 2 bytes of codes 0 .. 15 and an f16 scale d for every 32 columns; a value is d (code - 8).  Eight neighbouring columns are a 32-bit word: column 2 i of
// them in bits 4 i .., column 2 i + 1 in bits 16 + 4 i .., so that one mask takes two neighbours into the halves of a register.  Word j of a block of 32 columns stands before word j + 1 of any
// (word j * (hd / 32) + b of the row is columns 32 b + 8 j ..): the lanes of a matrix product's operand, which want the same word of every block, find theirs side by side.
// d is minus an eighth of the value of largest magnitude (of two, the negative one), rounded to f16 and at most 8188, eight times which is an f16 number; a code is the quotient rounded to the
// nearest.  So the largest value is held to f16's precision and the others within half a step, but for one of the other sign as large as it, which is one step smaller.  Values
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

// The same but for what a product can take off at once: pairs 0 and 2 as n - 8, pairs 1 and 3 as 64 + n, seven instructions.
constexpr float RAISED = 72.f;       // what pairs 1 and 3 are too large by
__device__ __forceinline__ void expand_raised(uint32_t w, uint32_t (&e)[4]) {
    constexpr uint32_t LOW = 0x64086408u;
    const uint32_t w8 = w >> 8;
    uint32_t e1, e3;
    asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xEA;" : "=r"(e1) : "r"(w), "r"(0x54005400u));
    asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xEA;" : "=r"(e3) : "r"(w8), "r"(0x54005400u));
    e[0] = hsub2_bits(masked_or_1024<0x000f000fu>(w), LOW);
    e[1] = e1;
    e[2] = hsub2_bits(masked_or_1024<0x000f000fu>(w8), LOW);
    e[3] = e3;
}

__device__ __forceinline__ bool has_row(const Cache4& c, int pos, int slot) { return (unsigned)pos < (unsigned)c.n_ctx && (unsigned)slot < (unsigned)c.slots; }
__device__ __forceinline__ size_t row_of(const Cache4& c, int pos, int slot, int kvh) { return ((size_t)slot * c.kv_heads + kvh) * c.n_ctx + pos; }

// What turns a lane's columns N lane .. N lane + N - 1 of any head of a token: x cos + y sin, y the pair's other column.
enum Other : int { HERE, LANE, ROW };        // where that is: the lane's own neighbour, the same place of another lane, anywhere in the row
template <int HD>
struct Turn {
    static constexpr int N = HD / 32;
    float c[N], s[N];
    bool all;                // every column is turned
    int other, from;         // from: LANE: which; ROW: how far behind the lane's columns of the first half
};

// cs, sn: cosines and sines of the token's pairs.
template <int HD>
__device__ __forceinline__ Turn<HD> make_turn(const Rows4& r, const float* cs, const float* sn, int lane) {
    constexpr int N = HD / 32;
    Turn<HD> t;
    const int half = r.n_rot >> 1, i0 = N * lane;
    t.all = r.n_rot == HD;
    t.other = !r.neox ? HERE : half % N == 0 ? LANE : ROW;
    t.from = t.other == LANE ? (i0 < half ? lane + half / N : i0 < r.n_rot ? lane - half / N : lane) : half;
#pragma unroll
    for (int j = 0; j < N; j++) {
        const int i = i0 + j;
        t.c[j] = 1.f;
        t.s[j] = 0.f;
        if (i < r.n_rot) {
            const bool first = r.neox ? i < half : !(i & 1);
            const int p = r.neox ? (first ? i : i - half) : i >> 1;
            t.c[j] = cs[p];
            t.s[j] = first ? -sn[p] : sn[p];
        }
    }
    return t;
}

// The angles are formed in double: in 32 bits a position of 100000 would leave 0.004 of a radian.
__device__ __forceinline__ void make_angle(const Rows4& r, int pos, int p, float freq, float* cs, float* sn) {
    float s, c;
    sincosf(rot_angle(pos, (double)freq), &s, &c);
    sn[p] = s * r.mscale;
    cs[p] = c * r.mscale;
}
__device__ __forceinline__ void fill_angles(const Rows4& r, int pos, float* cs, float* sn, int tid, int threads) {
    for (int p = tid; p < (r.n_rot >> 1); p += threads) make_angle(r, pos, p, r.inv_freq[p], cs, sn);
}

// (Roundings are spelled out, so that a row is the same whichever kernel makes it.)
// Norm and rotation of a head by a warp: x[N] are its columns N lane ..; `row`: HD floats of the warp's own.
template <int HD>
__device__ __forceinline__ void prepare_head(float (&x)[HD / 32], const float* norm, float eps, bool turned, const Turn<HD>& t, float* row, int lane) {
    constexpr int N = HD / 32;
    if (norm) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < N; j++) s = __fmaf_rn(x[j], x[j], s);
        const float inv = 1.f / sqrtf(warp_sum(s) / (float)HD + eps);
#pragma unroll
        for (int j = 0; j < N; j++) x[j] = __fmul_rn(__fmul_rn(x[j], inv), norm[N * lane + j]);
    }
    if (!turned) return;
    float y[N];
    if (t.other == HERE) {
#pragma unroll
        for (int j = 0; j < N; j++) y[j] = x[j ^ 1];
    } else if (t.other == LANE) {
#pragma unroll
        for (int j = 0; j < N; j++) y[j] = __shfl_sync(0xffffffffu, x[j], t.from);
    } else {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < N; j++) row[N * lane + j] = x[j];
        __syncwarp();
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int i = N * lane + j;
            y[j] = i < t.from ? row[i + t.from] : i < 2 * t.from ? row[i - t.from] : 0.f;
        }
    }
    if (t.all) {
#pragma unroll
        for (int j = 0; j < N; j++) x[j] = __fmaf_rn(x[j], t.c[j], __fmul_rn(y[j], t.s[j]));
    } else {
#pragma unroll
        for (int j = 0; j < N; j++)
            if (t.s[j] != 0.f || t.c[j] != 1.f) x[j] = __fmaf_rn(x[j], t.c[j], __fmul_rn(y[j], t.s[j]));      // columns that are not turned stay, whatever stands beside them
    }
}

// A lane makes a word of a row's codes from its eight columns; the four lanes of a block stand side by side, all 32 of the warp take part.  d: the block's scale.
__device__ __forceinline__ uint32_t encode_word(const float (&in)[8], __half& scale) {
    float x[8], hi = -INFINITY, lo = INFINITY;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        x[j] = in[j] == in[j] ? in[j] : 0.f;
        hi = fmaxf(hi, x[j]);
        lo = fminf(lo, x[j]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    scale = __float2half_rn(fminf(fmaxf((hi > -lo ? hi : lo) * -0.125f, -TOP), TOP));
    const float d = __half2float(scale), inv = d != 0.f ? __frcp_rn(d) : 0.f;
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        // 1.5 * 2^23 + 8: the sum's low bits are the code.  (By the reciprocal: a quotient within 2^-23 of a border may go either way.)
        const uint32_t q = __float_as_uint(fminf(fmaxf(x[j] * inv, -8.f), 7.f) + 12582920.f) & 15u;
        w |= q << (4 * (j >> 1) + 16 * (j & 1));
    }
    return w;
}
// Lane or thread i of a row's HD / 8: which word of the row it makes, from columns 32 b + 8 j on.
template <int HD>
__device__ __forceinline__ int word_of(int i) { return (i & 3) * (HD / 32) + (i >> 2); }

}  // namespace kv4
