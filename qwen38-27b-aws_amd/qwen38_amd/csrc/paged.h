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

// How a call of the attention is cut: from the host's sizes and the device's CUs, the same for the scratch's size and the launch.
struct PagedPlan {
    int few;                 // rows with at most this many (token, query head) pairs per KV head stream their positions, 16 pairs a tile
    int target;              // workgroups that their positions are cut into, about
    int items, slots, joins;  // workgroups of those at most; of them those that leave partial sums; pairs of a row at most
    int tiles, parts, cus;   // workgroups of tiles of query rows; parts that few tiles' work is cut into (0: they are many); the device's CUs
    size_t table, part, cuts, cut_part, bytes;  // places in the scratch: the (row, KV head)s' first slot and count and their partial
                                                // sums; the number of parts, the PagedCuts of them 256 bytes on, their sums; its size
};
PagedPlan paged_attention_plan(const PagedCache& c, const PagedRows& r, int q_heads);

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
    PagedPlan plan;
    uint8_t* scratch;
};

constexpr float QNAN = __builtin_nanf("");

// A row's new tokens: [t0, t0 + n) of the call's, at positions p0 .. p0 + n - 1 (p0 at most the table's end, past which no
// page is found). A row to be skipped has n = 0.
struct PagedRow {
    int t0, n, p0;
    bool skip;
};

__device__ __forceinline__ PagedRow paged_row(const PagedRows& a, int row, int page_size) {
    PagedRow r;
    int t1;
    if (a.q_start) {
        r.t0 = a.q_start[row];
        t1 = a.q_start[row + 1];
    } else {
        r.t0 = row * a.max_tokens;
        t1 = r.t0 + a.max_tokens;
    }
    r.t0 = min(max(r.t0, 0), a.tokens);
    t1 = min(max(t1, r.t0), a.tokens);
    const int p = a.position[row];
    r.skip = p < 0;
    r.n = min(t1 - r.t0, a.max_tokens);
    r.p0 = min(p, a.max_pages * page_size);
    return r;
}

// The page that holds position p of the row whose table entries are at `table`, or -1.
__device__ __forceinline__ int paged_find(const PagedRows& a, const int* table, int page, int pages) {
    const int id = table[min(max(page, 0), a.max_pages - 1)];  // read in any case: a choice, not a branch
    return ((page >= 0) & (page < a.max_pages) & (id >= 0) & (id < pages)) ? id : -1;
}

hipError_t q38_paged_append(const PagedAppendArgs& a, hipStream_t stream);
// The engine's glue: a step's positions with -1 for rows that are not active; a prefill call's one row (its page numbers, its
// position, where its n_valid (null: all) tokens start and end; the position -1 if the chunk does not fit or there is no such
// row); and the attention's outputs, gated, as the o projection's e5m2 input tiles (tokens past q_start[1]: zeros).
hipError_t q38_paged_positions(const int* position, const float* active, int rows, int* out, hipStream_t stream);
hipError_t q38_paged_slot(const int* slot, const int* start, const int* n_valid, int tokens, int rows, int seq, const int* table, int max_pages,
                          int* position, int* q_start, int* pages, hipStream_t stream);
hipError_t q38_paged_gate(const bf16_t* o, const bf16_t* qkv, int ld, int tokens, int q_heads, const int* q_start, uint8_t* act, hipStream_t stream);
hipError_t q38_paged_attention(const PagedAttnArgs& a, hipStream_t stream);
bool paged_attention_fits(const PagedCache& c, const PagedRows& r, int q_heads);
