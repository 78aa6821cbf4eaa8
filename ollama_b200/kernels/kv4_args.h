// Argument blocks of the 4-bit cache's and the packed prompts' entry points, for device code and for host code that fills them in (ops/kv4_call.cpp).  Plain C++.
#pragma once
#include <stdint.h>
#include <vector_types.h>

// Follows from this file (kernels/build.py): the library and the calls compare theirs before the first call.
#ifndef KV4_LAYOUT
#define KV4_LAYOUT 0ull
#endif

// Keys and values of one layer: codes [slots][kv_heads][n_ctx][hd / 2], f16 scales [slots][kv_heads][n_ctx][hd / 32] (kv4.cuh).
struct Cache4 {
    uint8_t* k;
    uint8_t* v;
    void* ks;
    void* vs;
    int slots, kv_heads, n_ctx, hd;
};

// Rows of raw projections and what is done to them before they are used: norm of the query and key heads, rotation.
struct Rows4 {
    const float* qkv;        // [rows][ldq]: q heads | k heads | v heads of hd columns
    int ldq, rows, n_heads;
    const int* positions;    // [rows]
    const int* slots;        // [rows]
    const float* inv_freq;   // [n_rot / 2]
    int n_rot, neox;         // pairs (p, p + n_rot / 2), or (2 p, 2 p + 1)
    float mscale;            // factor of the rotated columns
    const float* q_norm;     // [hd] or null
    const float* k_norm;
    float eps;
};

struct Append4Args {
    Rows4 r;
    Cache4 c;
    void* q_out;             // [rows][n_heads][hd], or null
    int q16;                 // f16, else fp32
};

struct Read4Args {
    Cache4 c;
    const int* positions;    // [rows]
    const int* slots;
    int rows;
    void* k_out;             // f16 [rows][kv_heads][hd]
    void* v_out;
};

// Attention of one token a sequence (attn_kv4.cu).
struct Attn4Args {
    Rows4 r;                 // qkv null: queries come rotated from q and the rows are in the cache
    Cache4 c;
    const void* q;           // [rows][n_heads][hd]
    int q16;
    float scale, softcap;
    int window;              // 0: none; key k is visible to the token at position p when p - k < window
    const float* sinks;      // [n_heads] or null
    void* out;               // [rows][ldo], head h at column h * hd
    int ldo, out16;          // out16: bf16, else fp32
    int room;                // shares of keys, of all sequences together, that there are CTAs and room for
    float* part_acc;         // [room][n_heads][hd]
    float2* part_ml;         // [room][n_heads] (reference of the exponents, sum)
    int2* shares;            // [rows] (first share, shares) of each sequence
};

// A run of key tiles for a tile of query rows of one portion and KV head (attn_packed.cu): up to 2 x floor(128 / group) tokens.
struct alignas(16) PackedTile {
    int row, rows;           // query rows
    int slot, pos;           // of the cache; position of the first row
    int base;                // cache row of the sequence's position 0
    int k_lo, k_hi;          // tiles of 128 keys
    int part;                // -1: all that the rows see; else which partial result it leaves
    int kvh;
    int pad[3];
};
// What a merge adds up: `parts` partial results from `first` on of `rows` query rows.
struct alignas(16) PackedMerge {
    int row, rows, first, parts, kvh;
    int pad[3];
};

struct PackedArgs {
    const void* q;           // [rows][n_heads][hd], ldq elements a row
    int q_type;              // 0 fp32, 1 f16, 2 bf16
    int q_rows;
    long long ldq;
    int n_heads, kv_heads, hd;
    const void* k;           // 16-bit rows [slots][kv_heads][n][hd], elements from one to the next in ld_*; null: codes of c
    const void* v;
    int kv_bf16;
    long long k_slot, k_head, k_row, v_slot, v_head, v_row;
    int slots, n;
    Cache4 c;
    const PackedTile* tiles;
    const int* starts;       // [ctas + 1]: CTA i takes tile i, then starts[i] .. starts[i + 1] - 1
    int ctas, n_tiles;
    const PackedMerge* merges;
    int n_merges, parts;
    int merge_rows;          // rows of partial results, of the 256, that the merges' largest has
    float scale, softcap;
    int window;
    const float* sinks;
    void* out;               // [rows][ldo], head h at column h * hd
    int ldo, out_type;       // 0 fp32, 1 f16, 2 bf16
    float* part_acc;         // [parts][256][hd]
    float2* part_ml;         // [parts][256]
};
