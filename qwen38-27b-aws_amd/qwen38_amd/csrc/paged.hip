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

__device__ __forceinline__ uint32_t e4m3_byte(float x) { return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false) & 0xffu; }

// Four e4m3 codes times 2^-shift, coded again.
__device__ __forceinline__ uint32_t e4m3_shift(uint32_t w, int shift) {
    typedef float v2f_ __attribute__((ext_vector_type(2)));
    const v2f_ a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.0f, true);
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(ldexpf(a[0], -shift), ldexpf(a[1], -shift), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(ldexpf(b[0], -shift), ldexpf(b[1], -shift), lo, true);
}

// One head's vector in a wave, E = hd / 64 dims per lane: RMS norm with weight 1 + w (w null: none), then the rotation of its
// first `rot` dims (dim d with d +- rot / 2, rot / 2 a multiple of E).
template <int E>
__device__ __forceinline__ void norm_rotate(float (&x)[E], const bf16_t* w, float eps, const bf16_t* cos, const bf16_t* sin, int rot, int lane,
                                            bool& fine) {
    constexpr int HD = E * 64;
    if (w) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) ss += x[e] * x[e];
        ss = warp_sum(ss);
        fine = fine && ss < INFINITY;  // else the norm of large finite values would be zero
        const float f = 1.0f / sqrtf(ss * (1.0f / HD) + eps);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = x[e] * f * (1.0f + bf2f(w[lane * E + e]));
    }
    if (rot) {
        const int half = rot / 2;
        const bool low = lane * E < half;
        const int other = low ? lane + half / E : lane - half / E;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float p = __shfl(x[e], other & 63);
            const int d = lane * E + e;
            if (d < rot) x[e] = x[e] * bf2f(cos[d]) + (low ? -p : p) * bf2f(sin[d]);
        }
    }
}

template <int E>
__device__ __forceinline__ void load_dims(const bf16_t* p, float (&x)[E]) {
    if constexpr (E == 4) {
        const uint2 w = *(const uint2*)p;
        x[0] = lo_bf(w.x), x[1] = hi_bf(w.x), x[2] = lo_bf(w.y), x[3] = hi_bf(w.y);
    } else if constexpr (E == 2) {
        const uint32_t w = *(const uint32_t*)p;
        x[0] = lo_bf(w), x[1] = hi_bf(w);
    } else {
        x[0] = bf2f(*p);
    }
}

constexpr int APPEND_TOKENS = 8;  // a wave's tokens of one page at most: their keys and values stay in its registers
constexpr int APPEND_HEADS = 8;   // a wave's query heads of one token

}  // namespace

// Grid: per row, page it may touch and KV head one workgroup; then the queries, a wave per token and APPEND_HEADS heads.
// A workgroup has all of its page's new tokens, so the page's largest value is known before any of them is coded, and every
// input is read once.
template <int E, int NW>
__global__ __launch_bounds__(NW * 64) void paged_append_kernel(const PagedAppendArgs a) {
    constexpr int HD = E * 64;
    __shared__ float amax[2][NW];
    __shared__ __attribute__((aligned(16))) uint8_t codes[NW * APPEND_TOKENS * HD];  // the new values, [token][dim]
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int Hkv = a.c.kv_heads, ps = a.c.page_size;
    if ((int)blockIdx.x >= a.kv_blocks) {
        const int groups = (a.q_heads + APPEND_HEADS - 1) / APPEND_HEADS, id = (blockIdx.x - a.kv_blocks) * NW + wv;
        const int t = id / groups, h0 = id % groups * APPEND_HEADS;
        const int tokens = a.r.q_start ? min(a.r.q_start[a.r.rows], a.r.tokens) : a.r.tokens;
        if (t >= tokens) return;
        float x[APPEND_HEADS][E];
#pragma unroll
        for (int h = 0; h < APPEND_HEADS; ++h)
            if (h0 + h < a.q_heads) load_dims<E>(a.q + t * a.q_token + (h0 + h) * a.q_head + lane * E, x[h]);
#pragma unroll
        for (int h = 0; h < APPEND_HEADS; ++h) {
            if (h0 + h >= a.q_heads) break;
            bool fine = true;
            norm_rotate<E>(x[h], a.q_norm, a.eps, a.cos + (size_t)t * a.rot, a.sin + (size_t)t * a.rot, a.rot, lane, fine);
            if (!fine)
#pragma unroll
                for (int e = 0; e < E; ++e) x[h][e] = QNAN;
            bf16_t* o = a.q_out + ((size_t)t * a.q_heads + h0 + h) * HD + lane * E;
            if constexpr (E == 4)
                *(uint2*)o = make_uint2(pk_bf16(x[h][0], x[h][1]), pk_bf16(x[h][2], x[h][3]));
            else if constexpr (E == 2)
                *(uint32_t*)o = pk_bf16(x[h][0], x[h][1]);
            else
                *o = f2bf(x[h][0]);
        }
        return;
    }
    const int kvh = blockIdx.x % Hkv, y = blockIdx.x / Hkv % a.visits, row = blockIdx.x / Hkv / a.visits;
    const PagedRow r = paged_row(a.r, row, ps);
    if (r.skip || r.n <= 0) return;
    const int page = r.p0 / ps + y, base = page * ps;
    const int lo = max(r.p0 - base, 0), hi = min(r.p0 + r.n - base, ps);  // the new tokens' slots
    if (lo >= hi) return;
    const int id = paged_find(a.r, a.r.pages + (size_t)row * a.r.max_pages, page, a.c.pages);
    if (id < 0) return;

    float k[APPEND_TOKENS][E], v[APPEND_TOKENS][E];
    float km = 0.0f, vm = 0.0f;
    const int t0 = r.t0 + base - r.p0;  // the token of slot 0
#pragma unroll
    for (int i = 0; i < APPEND_TOKENS; ++i) {
        const int slot = lo + i * NW + wv;
        if (slot >= hi) continue;
        const size_t t = t0 + slot;
        load_dims<E>(a.k + t * a.k_token + kvh * a.k_head + lane * E, k[i]);
        load_dims<E>(a.v + t * a.v_token + kvh * a.v_head + lane * E, v[i]);
    }
#pragma unroll
    for (int i = 0; i < APPEND_TOKENS; ++i) {
        const int slot = lo + i * NW + wv;
        if (slot >= hi) continue;
        const size_t t = t0 + slot;
        bool fine = true;
        norm_rotate<E>(k[i], a.k_norm, a.eps, a.cos + t * a.rot, a.sin + t * a.rot, a.rot, lane, fine);
        float ka = 0.0f, va = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            fine = fine && fabsf(k[i][e]) < INFINITY && fabsf(v[i][e]) < INFINITY;
            ka = fmaxf(ka, fabsf(k[i][e]));
            va = fmaxf(va, fabsf(v[i][e]));
        }
        if (__all(fine)) {
            km = fmaxf(km, ka);
            vm = fmaxf(vm, va);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) k[i][e] = QNAN, v[i][e] = 0.0f;
        }
    }
    km = warp_max(km);
    vm = warp_max(vm);
    if (lane == 0) amax[0][wv] = km, amax[1][wv] = vm;
    const size_t head = (size_t)id * Hkv + kvh, at = head * ps * HD;
    const int k_old = a.c.k_scale[head], v_old = a.c.v_scale[head];
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) km = fmaxf(km, amax[0][w]), vm = fmaxf(vm, amax[1][w]);
    int kb = paged_need(km), vb = paged_need(vm);
    if (lo > 0) {  // the page goes on: what it holds stays, coded again if the scale grows
        kb = max(kb, k_old);
        vb = max(vb, v_old);
        if (kb > k_old)
            for (int i = threadIdx.x; i < lo * HD / 4; i += NW * 64) {
                uint32_t* w = (uint32_t*)(a.c.k + at) + i;
                *w = e4m3_shift(*w, kb - k_old);
            }
        if (vb > v_old)
            for (int i = threadIdx.x; i < (lo + 15) / 16 * HD * 4; i += NW * 64) {
                uint32_t* w = (uint32_t*)(a.c.v + at) + i;
                const int left = lo - (i / (HD * 4) * 16 + i % 4 * 4);  // of the word's four slots those before lo
                if (left <= 0) continue;
                const uint32_t mask = left >= 4 ? 0xffffffffu : (1u << 8 * left) - 1, o = *w;
                *w = (e4m3_shift(o, vb - v_old) & mask) | (o & ~mask);
            }
    }
    const float kf = __uint_as_float((uint32_t)(254 - kb) << 23), vf = __uint_as_float((uint32_t)(254 - vb) << 23);
#pragma unroll
    for (int i = 0; i < APPEND_TOKENS; ++i) {
        const int slot = lo + i * NW + wv;
        if (slot >= hi) continue;
        uint8_t* ko = a.c.k + at + (size_t)slot * HD + lane * E;
        uint8_t* vo = codes + (i * NW + wv) * HD + lane * E;
        if constexpr (E == 4) {
            *(uint32_t*)ko = e4m3_byte(k[i][0] * kf) | e4m3_byte(k[i][1] * kf) << 8 | e4m3_byte(k[i][2] * kf) << 16 | e4m3_byte(k[i][3] * kf) << 24;
            *(uint32_t*)vo = e4m3_byte(v[i][0] * vf) | e4m3_byte(v[i][1] * vf) << 8 | e4m3_byte(v[i][2] * vf) << 16 | e4m3_byte(v[i][3] * vf) << 24;
        } else if constexpr (E == 2) {
            *(uint16_t*)ko = (uint16_t)(e4m3_byte(k[i][0] * kf) | e4m3_byte(k[i][1] * kf) << 8);
            *(uint16_t*)vo = (uint16_t)(e4m3_byte(v[i][0] * vf) | e4m3_byte(v[i][1] * vf) << 8);
        } else {
            *ko = (uint8_t)e4m3_byte(k[i][0] * kf);
            *vo = (uint8_t)e4m3_byte(v[i][0] * vf);
        }
    }
    __syncthreads();  // also: the page's words coded again are written before new bytes go into them
    // Values: a thread takes a dim of a group of sixteen slots.
    for (int i = threadIdx.x; i < ((hi + 15) / 16 - lo / 16) * HD; i += NW * 64) {
        const int g = lo / 16 + i / HD, d = i % HD;
        uint8_t* vo = a.c.v + at + ((size_t)g * HD + d) * 16;
        const int s0 = max(lo, g * 16), s1 = min(hi, g * 16 + 16);
        const uint8_t* from = codes + d;
        if (s1 - s0 == 16) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = 0;
#pragma unroll
                for (int b = 0; b < 4; ++b) w[j] |= (uint32_t)from[(s0 - lo + j * 4 + b) * HD] << 8 * b;
            }
            *(uint4*)vo = make_uint4(w[0], w[1], w[2], w[3]);
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
    // Four waves while a page's new tokens fit their registers, else sixteen.
    const bool few = (a.r.max_tokens < ps ? a.r.max_tokens : ps) <= 4 * APPEND_TOKENS;
    const int nw = few ? 4 : 16;
    a.kv_blocks = a.r.rows * a.visits * a.c.kv_heads;
    const int groups = (a.q_heads + APPEND_HEADS - 1) / APPEND_HEADS;
    const int grid = a.kv_blocks + (a.q ? (int)(((size_t)a.r.tokens * groups + nw - 1) / nw) : 0);
    if (!grid) return hipSuccess;
#define APPEND(E)                                                                                                   \
    do {                                                                                                            \
        if (few)                                                                                                    \
            hipLaunchKernelGGL((paged_append_kernel<E, 4>), dim3(grid), dim3(256), 0, stream, a);                   \
        else                                                                                                        \
            hipLaunchKernelGGL((paged_append_kernel<E, 16>), dim3(grid), dim3(1024), 0, stream, a);                 \
    } while (0)
    switch (a.c.head_dim) {
        case 64: APPEND(1); break;
        case 128: APPEND(2); break;
        case 256: APPEND(4); break;
        default: return hipErrorInvalidValue;
    }
#undef APPEND
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
    if (paged_bad(c, r) || q_heads < 1 || q_heads % c->kv_heads || q_heads / c->kv_heads > 64) return 0;
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
