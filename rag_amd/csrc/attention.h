// attention.h — internal interface of attention.hip (packed attention with grouped heads and a relative position bias).
#pragma once
#include "common.h"

#define MI_ATTN_MAX_BUCKETS 64
#define MI_ATTN_MAX_DISTANCE 1024

// One operand or result: rows of head_dim 16-bit elements, row (token t, head h) at ptr + t * ts + h * hs (elements).
struct mi_attn_rows {
    uint16_t* p = nullptr;
    int64_t ts = 0, hs = 0;
};

// Everything a kernel of attention.hip reads besides the tensors' elements (passed by value).
struct mi_attn_args {
    mi_attn_rows q, k, v, out, dout, dq, dk, dv;
    float* lse = nullptr;                 // [heads][tokens] natural log-sum-exp of a row's scores; may be NULL in the forward pass
    const int32_t* offsets = nullptr;     // [nseq + 1], or NULL: nseq sequences of `uniform_len` rows each
    const int32_t* key_mask = nullptr;    // [tokens], 0 = the row is no key; or NULL
    const float* table = nullptr;         // [buckets][heads], or NULL
    float* delta = nullptr;               // backward workspace [heads][tokens]: sum of p dp over a row
    float* lse2 = nullptr;                // backward workspace [heads][tokens]: lse in log2 units, +inf where it is -inf
    float* partial = nullptr;             // backward workspace [heads][dq tiles][64]: the table gradient's block sums
    float* parts_kv = nullptr;            // backward workspace [splits][dk | dv][tokens][key heads][hd], where splits > 1
    int splits = 1, share_heads = 1;      // shares of a group's query heads in the dK / dV kernel
    float* dtable = nullptr;              // [buckets][heads]
    int dq_tiles = 0, dtable_row = 0;     // `partial`'s tiles; the row of the dK / dV grid whose blocks sum them
    int64_t tokens = 0;
    int nseq = 0, uniform_len = 0;
    int heads = 0, group = 1, hd = 0;     // group = query heads per key head
    int causal = 0, zero_tail = 0;
    float scale_log2 = 0.0f, scale = 0.0f, scale_inv = 0.0f;   // score = scale * q.k; the kernels exponentiate in base 2
    // bucket(r), r = key - query: two_sided: n = buckets / 2, + n for r > 0, d = |r|; else n = buckets, d = max(-r, 0).
    // d < exact: d; else exact + #{t : d >= border[t]}.  From d = reach on the bucket no longer changes.
    int buckets = 0, two_sided = 0, side = 0, exact = 0, nborder = 0, reach = 0;
    int32_t border[MI_ATTN_MAX_BUCKETS + 8];   // from nborder on: beyond any distance
    // block -> (head, tile): see at_work in attention.hip
    int tiles = 0, parts_log2 = 0, units_per_xcd = 0;
    uint32_t group_inv = 0, splits_inv = 0;   // ceil(2^32 / x), 0 for x = 1
};

// Fills two_sided .. border for a bucket scheme; MI_ERR_* (with a message) when it is not one.
int mi_attn_buckets(const char* who, mi_attn_args* a, int buckets, int max_distance, int bidirectional);
// The forward pass on device pointers (arguments already checked).
int mi_launch_attention(hipStream_t st, mi_attn_args a, int dtype);

// Bytes of workspace of the backward pass (fields offsets, tokens, nseq, uniform_len, heads, group, hd, table, buckets), and the pass itself.
size_t mi_attn_backward_bytes(const mi_attn_args& a);
int mi_launch_attention_backward(hipStream_t st, mi_attn_args a, int dtype, void* workspace);
