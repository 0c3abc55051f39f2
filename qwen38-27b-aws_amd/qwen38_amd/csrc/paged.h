// Arguments and launchers of the paged 8-bit cache's kernels (paged.hip).
#pragma once

#include "../../../include/q38.h"
#include "common.h"

typedef q38_paged_cache PagedCache;
typedef q38_paged_rows PagedRows;

struct PagedAppendArgs {
    PagedCache c;
    PagedRows r;
    const bf16_t *k, *v, *q;
    bf16_t* q_out;           // [tokens][q_heads][head_dim]
    long long k_token, k_head, v_token, v_head, q_token, q_head;  // strides in elements
    int q_heads, rot;
    const bf16_t *cos, *sin;  // [tokens][rot]
    const bf16_t *q_norm, *k_norm;
    float eps;
    int visits, kv_blocks;   // set by the launcher: pages that a row may touch; workgroups of keys and values
};

struct PagedAttnArgs {
    PagedCache c;
    PagedRows r;
    const bf16_t* q;         // [tokens][q_heads][head_dim]
    bf16_t* out;
    int q_heads;
    float scale, cap;
    int window;
    const float* slopes;     // [q_heads] or null
    const int* prefix;       // [rows] or null
};

hipError_t q38_paged_append(const PagedAppendArgs& a, hipStream_t stream);
hipError_t q38_paged_attention(const PagedAttnArgs& a, hipStream_t stream);
