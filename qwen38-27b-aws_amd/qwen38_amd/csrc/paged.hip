// A key/value cache in pages of 8-bit values (include/q38.h, q38_paged_cache): appending a step's tokens, and attention over it.
//
// A page of a KV head holds page_size keys, e4m3 [page_size][head_dim], and values, e4m3 [page_size / 16][head_dim][16] (sixteen
// positions of a dim side by side: what a lane feeds the matrix cores for weights x V), each times one power of two, held as an
// E8M0 byte b (2^(b - 127)): the smallest that the largest value so far fits in +-448. Powers of two, because a page whose scale
// has to grow codes what it held again, and halving an e4m3 value is exact but for subnormals.
//
// A token whose key or value is not finite is stored as a key of NaN and a value of zero: whoever sees the position answers
// NaN, and nobody else does, whatever weight zero times its value would be.
#include "kernels.h"
#include "paged.h"

namespace {

// The scale byte that values up to amax need: 448 = 1.75 x 2^8.
__device__ __forceinline__ int paged_need(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    const int b = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);
    return min(max(b, 1), 254);
}

__device__ __forceinline__ uint32_t e4m3_four(float a, float b, float c, float d) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}

// Four e4m3 codes times 2^-shift, coded again.
__device__ __forceinline__ uint32_t e4m3_shift(uint32_t w, int shift) {
    typedef float v2f_ __attribute__((ext_vector_type(2)));
    const v2f_ a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.0f, true);
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(ldexpf(a[0], -shift), ldexpf(a[1], -shift), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(ldexpf(b[0], -shift), ldexpf(b[1], -shift), lo, true);
}

// How a wave holds head vectors: HD / 8 lanes each, eight dims per lane in two runs of four, from `lo` and from `hi`. The lanes of
// the rotated dims hold both halves of their pairs, so that nothing moves between lanes.
struct HeadLane {
    int vec, lo, hi;  // the lane's vector of the wave's 64 / (HD / 8)
    bool turns;
};

template <int HD>
__device__ __forceinline__ HeadLane head_lane(int lane, int rot) {
    const int i = lane % (HD / 8), n = rot / 8;  // the first n lanes: pairs
    return i < n ? HeadLane{lane / (HD / 8), 4 * i, rot / 2 + 4 * i, true} : HeadLane{lane / (HD / 8), 8 * i, 8 * i + 4, false};
}

typedef uint32_t words2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ void load_dims(const bf16_t* p, const HeadLane& l, words2& lo, words2& hi) {
    lo = *(const words2*)(p + l.lo);
    hi = *(const words2*)(p + l.hi);
}

__device__ __forceinline__ void widen_dims(words2 lo, words2 hi, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        x[2 * e] = lo_bf(lo[e]), x[2 * e + 1] = hi_bf(lo[e]);
        x[4 + 2 * e] = lo_bf(hi[e]), x[5 + 2 * e] = hi_bf(hi[e]);
    }
}

// RMS norm with weights 1 + w (gain: those; normed false: none), then the rotation. False if the norm is of something not
// finite, the sum of the squares included: else large finite values would come out as zeros.
template <int HD>
__device__ __forceinline__ bool norm_rotate(float (&x)[8], bool normed, const float (&gain)[8], float eps, const HeadLane& l, const bf16_t* cos,
                                            const bf16_t* sin) {
    bool fine = true;
    if (normed) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
#pragma unroll
        for (int o = 1; o < HD / 8; o <<= 1) ss += __shfl_xor(ss, o);
        fine = ss < INFINITY;
        const float f = 1.0f / sqrtf(ss * (1.0f / HD) + eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * f * gain[e];
    }
    if (l.turns) {
        words2 a, b;
        float c[8], s[8];
        load_dims(cos, l, a, b);
        widen_dims(a, b, c);
        load_dims(sin, l, a, b);
        widen_dims(a, b, s);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float lo = x[e], hi = x[4 + e];
            x[e] = lo * c[e] - hi * s[e];
            x[4 + e] = hi * c[4 + e] + lo * s[4 + e];
        }
    }
    return fine;
}

__device__ __forceinline__ void load_gain(const bf16_t* w, const HeadLane& l, float (&gain)[8]) {
    words2 lo = {}, hi = {};
    if (w) load_dims(w, l, lo, hi);
    widen_dims(lo, hi, gain);
#pragma unroll
    for (int e = 0; e < 8; ++e) gain[e] += 1.0f;
}

// Queries and codes are written past the caches (nontemporal): nothing reads them again in this kernel, and lines that wait in L2 to be
// written slow the inputs' reads down (37 ragged prompts 80 us against 101, 8 chunks of 2,048 tokens 114 against 134).
template <typename T>
__device__ __forceinline__ void store_past(void* p, T x) {
    __builtin_nontemporal_store(x, (T*)p);
}

constexpr int QUERY_STEPS = 2;  // a lane's vectors of the queries (those prompts with 1 and 4: 91 and 90 us)

// Vectors that nw waves hold at `steps` to a lane: of a page all new ones, in their registers.
constexpr int append_room(int head_dim, int nw, int steps) { return nw * (64 / (head_dim / 8)) * steps; }

}  // namespace

// Grid: per row, page it may touch and KV head one workgroup; then the queries, QUERY_STEPS vectors per lane. A workgroup has all
// of its page's new tokens, so the page's largest value is known before any of them is coded, and every input is read once.
// Bound: memory; for a few tokens a launch's and four loads' time, one after another. With 24 query and 4 KV heads of 256: one token
// 4.4 us, 64 rows of 4 tokens 5.9, 2,048 tokens of a prompt 17 (3.7 TB/s); 37 prompts, 32 and 8 heads of 128, pages of 16, 77 us (5.4 TB/s).
template <int HD, int NW, int STEPS>
__global__ __launch_bounds__(NW * 64) void paged_append_kernel(const PagedAppendArgs a) {
    constexpr int VECS = 64 / (HD / 8);  // vectors of a wave at a time
    __shared__ float amax[2][NW];
    constexpr int ROOM = append_room(HD, NW, STEPS);
    __shared__ __attribute__((aligned(16))) uint8_t codes[(ROOM < 128 ? ROOM : 128) * HD];  // the new values, [token][dim]
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int Hkv = a.c.kv_heads, ps = a.c.page_size;
    const HeadLane l = head_lane<HD>(lane, a.rot);
    float gain[8];
    if ((int)blockIdx.x >= a.kv_blocks) {
        const long long tokens = a.r.q_start ? min(a.r.q_start[a.r.rows], a.r.tokens) : a.r.tokens;
        const long long first = ((long long)((int)blockIdx.x - a.kv_blocks) * NW + wv) * (VECS * QUERY_STEPS) + l.vec;
        words2 lo[QUERY_STEPS], hi[QUERY_STEPS];
#pragma unroll
        for (int i = 0; i < QUERY_STEPS; ++i) {
            const long long u = first + i * VECS;
            const int t = (int)(u / a.q_heads), h = (int)(u % a.q_heads);
            lo[i] = hi[i] = (words2){0, 0};
            if (t < tokens) load_dims(a.q + t * a.q_token + h * a.q_head, l, lo[i], hi[i]);
        }
        load_gain(a.q_norm, l, gain);
#pragma unroll
        for (int i = 0; i < QUERY_STEPS; ++i) {
            const long long u = first + i * VECS;
            const int t = (int)(u / a.q_heads), at = min(t, a.r.tokens - 1);
            float x[8];
            widen_dims(lo[i], hi[i], x);
            if (!norm_rotate<HD>(x, a.q_norm != nullptr, gain, a.eps, l, a.cos + (size_t)at * a.rot, a.sin + (size_t)at * a.rot))
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = QNAN;
            if (t < tokens) {
                store_past(a.q_out + u * HD + l.lo, (words2){pk_bf16(x[0], x[1]), pk_bf16(x[2], x[3])});
                store_past(a.q_out + u * HD + l.hi, (words2){pk_bf16(x[4], x[5]), pk_bf16(x[6], x[7])});
            }
        }
        return;
    }
    const int kvh = blockIdx.x % Hkv, y = blockIdx.x / Hkv % a.visits, row = blockIdx.x / Hkv / a.visits;
    const PagedRow r = paged_row(a.r, row, ps);
    if (r.skip || r.n <= 0) return;
    const int page = r.p0 / ps + y, base = page * ps;
    const int lo = max(r.p0 - base, 0), hi = min(r.p0 + r.n - base, ps);  // the new tokens' slots
    if (lo >= hi) return;
    float k[STEPS][8], km = 0.0f, vm = 0.0f;
    words2 w[STEPS][4];  // the new keys and values
    const int t0 = r.t0 + base - r.p0;  // the token of slot 0
    auto slot_of = [&](int i) { return lo + (i * NW + wv) * VECS + l.vec; };
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        if (lo + (i * NW + wv) * VECS >= hi) continue;
        const size_t t = t0 + min(slot_of(i), hi - 1);
        load_dims(a.k + t * a.k_token + kvh * a.k_head, l, w[i][0], w[i][1]);
        load_dims(a.v + t * a.v_token + kvh * a.v_head, l, w[i][2], w[i][3]);
    }
    const int id = paged_find(a.r, a.r.pages + (size_t)row * a.r.max_pages, page, a.c.pages);
    if (id < 0) return;
    const size_t head = (size_t)id * Hkv + kvh, at = head * ps * HD;
    const int k_old = min((int)a.c.k_scale[head], 254), v_old = min((int)a.c.v_scale[head], 254);  // 255 is no scale: nothing was appended
    load_gain(a.k_norm, l, gain);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        if (lo + (i * NW + wv) * VECS >= hi) continue;
        const size_t t = t0 + min(slot_of(i), hi - 1);  // past the last token: that one again
        widen_dims(w[i][0], w[i][1], k[i]);
        float v[8];
        widen_dims(w[i][2], w[i][3], v);
        int fine = norm_rotate<HD>(k[i], a.k_norm != nullptr, gain, a.eps, l, a.cos + t * a.rot, a.sin + t * a.rot);
        float ka = 0.0f, va = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            fine &= (int)(fabsf(k[i][e]) < INFINITY) & (int)(fabsf(v[e]) < INFINITY);
            ka = fmaxf(ka, fabsf(k[i][e]));
            va = fmaxf(va, fabsf(v[e]));
        }
#pragma unroll
        for (int o = 1; o < HD / 8; o <<= 1) fine &= __shfl_xor(fine, o);
        if (fine) {
            km = fmaxf(km, ka);
            vm = fmaxf(vm, va);
        } else {
            w[i][2] = w[i][3] = (words2){0, 0};
#pragma unroll
            for (int e = 0; e < 8; ++e) k[i][e] = QNAN;
        }
    }
    km = warp_max(km);
    vm = warp_max(vm);
    if (lane == 0) amax[0][wv] = km, amax[1][wv] = vm;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NW; ++j) km = fmaxf(km, amax[0][j]), vm = fmaxf(vm, amax[1][j]);
    int kb = paged_need(km), vb = paged_need(vm);
    if (lo > 0) {  // the page goes on: what it holds stays, coded again if the scale grows
        kb = max(kb, k_old);
        vb = max(vb, v_old);
        if (kb > k_old)
            for (int i = threadIdx.x; i < lo * HD / 4; i += NW * 64) {
                uint32_t* w4 = (uint32_t*)(a.c.k + at) + i;
                *w4 = e4m3_shift(*w4, kb - k_old);
            }
        if (vb > v_old)
            for (int i = threadIdx.x; i < (lo + 15) / 16 * HD * 4; i += NW * 64) {
                uint32_t* w4 = (uint32_t*)(a.c.v + at) + i;
                const int left = lo - (i / (HD * 4) * 16 + i % 4 * 4);  // of the word's four slots those before lo
                if (left <= 0) continue;
                const uint32_t mask = left >= 4 ? 0xffffffffu : (1u << 8 * left) - 1, o = *w4;
                *w4 = (e4m3_shift(o, vb - v_old) & mask) | (o & ~mask);
            }
    }
    const float kf = __uint_as_float((uint32_t)(254 - kb) << 23), vf = __uint_as_float((uint32_t)(254 - vb) << 23);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int slot = slot_of(i);
        if (slot >= hi) continue;
        uint8_t *ko = a.c.k + at + (size_t)slot * HD, *vo = codes + (slot - lo) * HD;
        float v[8];
        widen_dims(w[i][2], w[i][3], v);
        store_past(ko + l.lo, e4m3_four(k[i][0] * kf, k[i][1] * kf, k[i][2] * kf, k[i][3] * kf));
        store_past(ko + l.hi, e4m3_four(k[i][4] * kf, k[i][5] * kf, k[i][6] * kf, k[i][7] * kf));
        *(uint32_t*)(vo + l.lo) = e4m3_four(v[0] * vf, v[1] * vf, v[2] * vf, v[3] * vf);
        *(uint32_t*)(vo + l.hi) = e4m3_four(v[4] * vf, v[5] * vf, v[6] * vf, v[7] * vf);
    }
    __syncthreads();  // also: the page's words coded again are written before new bytes go into them
    // Values: a thread takes a dim of a group of sixteen slots.
    for (int i = threadIdx.x; i < ((hi + 15) / 16 - lo / 16) * HD; i += NW * 64) {
        const int g = lo / 16 + i / HD, d = i % HD;
        uint8_t* vo = a.c.v + at + ((size_t)g * HD + d) * 16;
        const int s0 = max(lo, g * 16), s1 = min(hi, g * 16 + 16);
        const uint8_t* from = codes + d;
        if (s1 - s0 == 16) {
            typedef uint32_t words4 __attribute__((ext_vector_type(4)));
            words4 w4 = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int b = 0; b < 4; ++b) w4[j] |= (uint32_t)from[(s0 - lo + j * 4 + b) * HD] << 8 * b;
            store_past(vo, w4);
        } else {
            for (int s = s0; s < s1; ++s) vo[s - g * 16] = from[(s - lo) * HD];
        }
    }
    if (threadIdx.x == 0) {
        a.c.k_scale[head] = (uint8_t)kb;
        a.c.v_scale[head] = (uint8_t)vb;
    }
}

hipError_t q38_paged_append(const PagedAppendArgs& a0, hipStream_t stream) {
    PagedAppendArgs a = a0;
    const int ps = a.c.page_size;
    a.visits = (a.r.max_tokens + ps - 2) / ps + 1;
    // The fewest waves and registers that have room for a page's new tokens: a workgroup's time is a few loads', one after
    // another, and with one vector per lane eight workgroups share a CU (37 ragged prompts in pages of 16).
    const int hd = a.c.head_dim, most = a.r.max_tokens < ps ? a.r.max_tokens : ps;
    const int nw = most <= append_room(hd, 4, 4) ? 4 : 16, steps = most <= append_room(hd, 4, 1) ? 1 : most <= append_room(hd, 4, 4) ? 4 : most <= append_room(hd, 16, 2) ? 2 : 4;
    const long long kv = (long long)a.r.rows * a.visits * a.c.kv_heads, vectors = a.q ? (long long)a.r.tokens * a.q_heads : 0;
    const long long grid = kv + (vectors + append_room(hd, nw, QUERY_STEPS) - 1) / append_room(hd, nw, QUERY_STEPS);
    if (grid * nw * 64 > 0xffffffffLL) return hipErrorInvalidConfiguration;  // a grid's threads are counted in 32 bits
    a.kv_blocks = (int)kv;
#define APPEND1(HD, NW, STEPS) hipLaunchKernelGGL((paged_append_kernel<HD, NW, STEPS>), dim3(grid), dim3(NW * 64), 0, stream, a)
#define APPEND(HD)                \
    do {                          \
        if (nw == 4 && steps == 1) \
            APPEND1(HD, 4, 1);    \
        else if (nw == 4)         \
            APPEND1(HD, 4, 4);    \
        else if (steps == 2)      \
            APPEND1(HD, 16, 2);   \
        else                      \
            APPEND1(HD, 16, 4);   \
    } while (0)
    switch (a.c.head_dim) {
        case 64: APPEND(64); break;
        case 128: APPEND(128); break;
        case 256: APPEND(256); break;
        default: return hipErrorInvalidValue;
    }
#undef APPEND
#undef APPEND1
    return hipGetLastError();
}

// ---- The engine's glue.
__global__ void paged_positions_kernel(const int* position, const float* active, int rows, int* out) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b < rows) out[b] = active[b] > 0.5f ? position[b] : -1;
}

hipError_t q38_paged_positions(const int* position, const float* active, int rows, int* out, hipStream_t stream) {
    hipLaunchKernelGGL(paged_positions_kernel, dim3((rows + 255) / 256), dim3(256), 0, stream, position, active, rows, out);
    return hipGetLastError();
}

__global__ __launch_bounds__(256) void paged_slot_kernel(const int* slot, const int* start, const int* n_valid, int tokens, int rows, int seq, const int* table,
                                                         int max_pages, int* position, int* q_start, int* pages) {
    const int b = *slot, p = *start;
    const bool row = b >= 0 && b < rows;
    if (threadIdx.x == 0) {
        *position = row && p >= 0 && p <= seq - tokens ? p : -1;
        q_start[0] = 0;
        q_start[1] = n_valid ? min(max(*n_valid, 0), tokens) : tokens;
    }
    for (int i = threadIdx.x; i < max_pages; i += 256) pages[i] = row ? table[(size_t)b * max_pages + i] : -1;
}

hipError_t q38_paged_slot(const int* slot, const int* start, const int* n_valid, int tokens, int rows, int seq, const int* table, int max_pages,
                          int* position, int* q_start, int* pages, hipStream_t stream) {
    hipLaunchKernelGGL(paged_slot_kernel, dim3(1), dim3(256), 0, stream, slot, start, n_valid, tokens, rows, seq, table, max_pages, position, q_start, pages);
    return hipGetLastError();
}

// Four dims per thread: bf16(o) x bf16(sigmoid(gate)) in bf16, then e5m2 (reference model.py:637-638, as every projection input).
__global__ __launch_bounds__(256) void paged_gate_kernel(const bf16_t* o, const bf16_t* qkv, int ld, int tokens, int q_heads, const int* q_start, uint8_t* act) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    const int t = (int)(i / (q_heads * 64)), x = (int)(i % (q_heads * 64)) * 4;
    if (t >= tokens) return;
    uint32_t r = 0;
    if (!q_start || t < q_start[1]) {
        const uint2 v = *(const uint2*)(o + (size_t)t * q_heads * 256 + x), g = *(const uint2*)(qkv + (size_t)t * ld + x / 256 * 512 + 256 + x % 256);
        r = pk_e5m2(rbf(lo_bf(v.x) * rbf(sigmoidf_(lo_bf(g.x)))), rbf(hi_bf(v.x) * rbf(sigmoidf_(hi_bf(g.x)))),
                    rbf(lo_bf(v.y) * rbf(sigmoidf_(lo_bf(g.y)))), rbf(hi_bf(v.y) * rbf(sigmoidf_(hi_bf(g.y)))));
    }
    *(uint32_t*)(act + act_offset(t, x, q_heads * 256)) = r;
}

hipError_t q38_paged_gate(const bf16_t* o, const bf16_t* qkv, int ld, int tokens, int q_heads, const int* q_start, uint8_t* act, hipStream_t stream) {
    hipLaunchKernelGGL(paged_gate_kernel, dim3(((size_t)tokens * q_heads * 64 + 255) / 256), dim3(256), 0, stream, o, qkv, ld, tokens, q_heads, q_start, act);
    return hipGetLastError();
}

// ---- The C ABI (include/q38.h).
namespace {

const char* paged_bad(const q38_paged_cache* c, const q38_paged_rows* r) {
    if (!c || !r) return "null argument";
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !r->position || !r->pages) return "null argument";
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return "paged cache: head_dim must be 64, 128 or 256";
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
        return "paged cache: page_size must be 16, 32, 64 or 128";
    if (c->pages < 1 || c->kv_heads < 1) return "paged cache: pages and kv_heads must be positive";
    if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16) return "paged cache: keys and values must be 16-byte aligned";
    if (r->rows < 1 || r->max_pages < 1 || r->tokens < 1 || r->max_tokens < 1) return "paged rows: rows, max_pages, tokens and max_tokens must be positive";
    if (r->max_tokens > r->tokens) return "paged rows: max_tokens above tokens";
    if (!r->q_start && (long long)r->rows * r->max_tokens != r->tokens) return "paged rows: without q_start tokens must be rows * max_tokens";
    if ((long long)r->max_pages * c->page_size > (1 << 30)) return "paged rows: more than 2^30 positions";
    if ((long long)r->rows * c->kv_heads >= 1 << 18) return "paged rows: rows * kv_heads too large for one call";
    if ((long long)r->rows * (r->max_tokens + 2) > (1 << 24) || (long long)r->rows * r->max_tokens * c->kv_heads > (1 << 28))
        return "paged rows: rows * max_tokens too large for one call";
    return nullptr;
}

}  // namespace

extern "C" {

int q38_paged_append(const q38_paged_cache* c, const q38_paged_rows* r, const q38_paged_tokens* t, void* stream) {
    if (const char* bad = paged_bad(c, r)) return q38_report(bad);
    if (!t || !t->k || !t->v) return q38_report("null argument");
    if (t->rotary_dim < 0 || t->rotary_dim > c->head_dim || t->rotary_dim % 8) return q38_report("paged append: rotary_dim must be a multiple of 8 up to head_dim");
    if (t->rotary_dim && (!t->cos || !t->sin)) return q38_report("null argument");
    if ((t->q != nullptr) != (t->q_out != nullptr)) return q38_report("paged append: q and q_out go together");
    if (t->q && (t->q_heads < 1 || t->q_heads > 65536)) return q38_report("paged append: q_heads must be 1 to 65536");
    if (t->k_token % 4 || t->k_head % 4 || t->v_token % 4 || t->v_head % 4 || (t->q && (t->q_token % 4 || t->q_head % 4)))
        return q38_report("paged append: strides must be multiples of 4 elements");
    if ((uintptr_t)t->k % 8 || (uintptr_t)t->v % 8 || (uintptr_t)t->q % 8 || (uintptr_t)t->q_out % 8)
        return q38_report("paged append: keys, values and queries must be 8-byte aligned");
    if ((uintptr_t)t->q_norm % 8 || (uintptr_t)t->k_norm % 8 || (t->rotary_dim && ((uintptr_t)t->cos % 8 || (uintptr_t)t->sin % 8)))
        return q38_report("paged append: norms, cos and sin must be 8-byte aligned");
    if (!(t->eps >= 0.0f)) return q38_report("paged append: eps must not be negative");
    PagedAppendArgs a{};
    a.c = *c;
    a.r = *r;
    a.k = t->k;
    a.v = t->v;
    a.q = t->q;
    a.q_out = t->q_out;
    a.k_token = t->k_token;
    a.k_head = t->k_head;
    a.v_token = t->v_token;
    a.v_head = t->v_head;
    a.q_token = t->q_token;
    a.q_head = t->q_head;
    a.q_heads = t->q ? t->q_heads : 0;
    a.cos = t->cos;
    a.sin = t->sin;
    a.rot = t->rotary_dim;
    a.q_norm = t->q_norm;
    a.k_norm = t->k_norm;
    a.eps = t->eps;
    const hipError_t e = q38_paged_append(a, (hipStream_t)stream);
    return e == hipSuccess ? 0 : q38_report(hipGetErrorString(e));
}

size_t q38_paged_attention_scratch(const q38_paged_cache* c, const q38_paged_rows* r, int q_heads) {
    if (paged_bad(c, r) || q_heads < 1 || q_heads % c->kv_heads || q_heads / c->kv_heads > 64 || !paged_attention_fits(*c, *r, q_heads)) return 0;
    return paged_attention_plan(*c, *r, q_heads).bytes;
}

int q38_paged_attention(const q38_paged_cache* c, const q38_paged_rows* r, const q38_paged_query* q, void* scratch, size_t scratch_bytes,
                        void* stream) {
    if (const char* bad = paged_bad(c, r)) return q38_report(bad);
    if (!q || !q->q || !q->out) return q38_report("null argument");
    if (q->q_heads < 1 || q->q_heads % c->kv_heads || q->q_heads / c->kv_heads > 64)
        return q38_report("paged attention: q_heads must be 1 to 64 times kv_heads");
    if (!(q->scale > 0.0f && q->scale < INFINITY)) return q38_report("paged attention: scale must be positive and finite");
    if (!(q->cap >= 0.0f && q->cap < INFINITY)) return q38_report("paged attention: cap must be finite and not negative");
    if (q->window < 0) return q38_report("paged attention: window must not be negative");
    if (q->window && q->prefix) return q38_report("paged attention: a window and a prefix exclude each other");
    if ((uintptr_t)q->q % 16 || (uintptr_t)q->out % 16) return q38_report("paged attention: queries and outputs must be 16-byte aligned");
    if (!paged_attention_fits(*c, *r, q->q_heads)) return q38_report("paged attention: query rows too many for one call");
    PagedAttnArgs a{};
    a.c = *c;
    a.r = *r;
    a.q = q->q;
    a.out = q->out;
    a.q_heads = q->q_heads;
    a.scale = q->scale;
    a.cap = q->cap;
    a.window = q->window;
    a.slopes = q->slopes;
    a.prefix = q->prefix;
    a.plan = paged_attention_plan(*c, *r, q->q_heads);
    if (a.plan.bytes > scratch_bytes || (a.plan.bytes && !scratch)) return q38_report("paged attention: the scratch is smaller than q38_paged_attention_scratch says");
    if ((uintptr_t)scratch % 256) return q38_report("paged attention: the scratch must be 256-byte aligned");
    a.scratch = (uint8_t*)scratch;
    const hipError_t e = q38_paged_attention(a, (hipStream_t)stream);
    return e == hipSuccess ? 0 : q38_report(hipGetErrorString(e));
}

}  // extern "C"
