// Argument blocks of the 8-bit paged cache's entry points, for device code and for host code that fills them in (ops/pages8_call.cpp).  Plain C++.
#pragma once
#include <stdint.h>
#include <vector_types.h>

// Follows from this file (kernels/build.py): the library and the calls compare theirs before the first call.
#ifndef PAGES8_LAYOUT
#define PAGES8_LAYOUT 0ull
#endif

// Sigmoid gate of attention results: kind 1 one number per element, 2 one per head; before the sigmoid.
struct HeadGate {
    const float* g;          // [rows][ld]
    int ld, kind;
};
// Differential attention: a head's result is a1 - lambda a2 of its two maps, divided by its root mean square, times `scale`.
struct DiffHeads {
    float lambda, scale, eps;
    int on;
};

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
    int items;               // most row tiles of a launch's sequences together, times KV heads: partial results and CTAs are counted by them, since a step has long portions beside single tokens
    int ctas;                // that fit the GPU at once
    float* part_acc;         // [items + ctas][row_tile][hd]
    float2* part_ml;         // [items + ctas][row_tile] (largest score, sum)
    void* out;               // [rows][ldo], head h at column h * vdim
    int ldo, out16;
    HeadGate gate;
    DiffHeads diff;
    int behind;              // the launch follows the one that appends the rows, which writes neither positions, slots nor tables
};
