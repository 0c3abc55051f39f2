// Attention over the paged 8-bit cache (paged.hip, include/q38.h): o_i = sum_j softmax_j(score_ij) v_j over the positions j that
// token i sees.
//
// Keys and values are widened to bf16 in registers, exactly (an e4m3 value times a power of two), for the bf16 matrix cores;
// scores, their maxima and the sums stay in float32, the weights are rounded to bf16 for the second product (2^-8 of each, as
// the output's own rounding) and summed unrounded. Exponentials are powers of two: scores carry log2 e.
//
// The maximum that the weights are relative to is raised, and the sums so far rescaled, only when a score passes it by
// SLACK: until then weights reach 2^SLACK, which float32 and bf16 hold as exactly as those below one.
#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "paged.h"

namespace {

constexpr float LOG2E = 1.44269504088896340736f, SLACK = 8.0f;

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Sum over the lanes up to this one: within rows of 16 lanes by shifts, then each row's last lane added to the rows after it. (By
// ds_bpermute the six steps take some 400 clocks, and a tile's lookup has three such sums one after another.)
__device__ __forceinline__ uint32_t lanes_up_to(uint32_t x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast 31 into rows 2 and 3
    return x;
}

__device__ __forceinline__ int lane_of(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }  // lane: uniform

// A workgroup's row: the same in every lane, and known to be.
__device__ __forceinline__ PagedRow paged_row_uniform(const PagedRows& a, int row, int page_size) {
    const PagedRow r = paged_row(a, row, page_size);
    return {uniform(r.t0), uniform(r.n), uniform(r.p0), uniform(r.skip) != 0};
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// What a packed query row (token r / G, query head r % G of the KV head's G) sees: positions [lo, hi); at is its own.
struct PagedSight {
    int lo, hi, at;
};

__device__ __forceinline__ PagedSight paged_sight(const PagedAttnArgs& a, const PagedRow& r, int prefix, int i) {
    const int at = r.p0 + i;
    return {a.window ? max(0, at + 1 - a.window) : 0, min(r.p0 + r.n, max(at + 1, prefix)), at};
}

// Eight e4m3 codes times a power of two as one bf16 matrix operand.
__device__ __forceinline__ v8bf16 paged_widen(uint32_t w0, uint32_t w1, float scale) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    const u4 r = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true))};
    return __builtin_bit_cast(v8bf16, r);
}

// A page's scale; of one that no token wrote it may be any byte, and stays finite, so that zeros times it are zeros.
__device__ __forceinline__ float paged_scale(int byte) { return __uint_as_float((uint32_t)min(byte, 254) << 23); }

// Of a word with four positions' bytes those from `from` on and below `to`.
__device__ __forceinline__ uint32_t paged_bytes(int from, int to) {
    auto below = [](int n) { return n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << 8 * n) - 1; };
    return below(to) & ~below(from);
}

// Scores to powers of two: capped and biased as the call asks.
template <int N>
__device__ __forceinline__ void paged_scores(const PagedAttnArgs& a, float (&s)[N], float slope2, int j0, int at) {
    if (a.cap > 0.0f) {
        const float in = a.scale * 2.0f * LOG2E / a.cap, out = a.cap * LOG2E;  // tanh x = 1 - 2 / (e^2x + 1)
#pragma unroll
        for (int e = 0; e < N; ++e) s[e] = out - 2.0f * out * __builtin_amdgcn_rcpf(exp2_(s[e] * in) + 1.0f);
        if (a.slopes)
#pragma unroll
            for (int e = 0; e < N; ++e) s[e] += slope2 * (float)(j0 + e - at);
    } else {
        const float f = a.scale * LOG2E, bias = slope2 * (float)(j0 - at);  // 0 without slopes
#pragma unroll
        for (int e = 0; e < N; ++e) s[e] = __builtin_fmaf(s[e], f, __builtin_fmaf(slope2, (float)e, bias));
    }
}

}  // namespace

// ---- Few query rows (decode, verify): the positions streamed once from memory, straight into registers.
//
// A wave takes a tile of 4 PT positions of one (row, KV head) at a time, its four lane groups g of 16 lanes PT each, with all of the
// row's query rows as columns (16 per tile of the matrix cores, NT tiles). Keys are A (a 16-position block's rows permuted, so
// that a lane's 16 scores of the four blocks are its group's 16 positions in order: they are the second product's B operand
// as they stand, without moving between lanes); values are A of the second product, sixteen positions of a dim being one 16-byte load.
// Nothing goes through LDS until a workgroup's four waves, which take tiles in turn, put their sums together.
//
// Bound: the cache's bytes from memory. With one tile of query rows two waves share a SIMD, with a tile's loads in flight each (16
// or 32 KB); with more, the sums and the queries mostly take the whole register file, and one wave is left. 64 rows of 8,192 positions, 4 KV
// heads of 256 and six query heads to each: 181 us, 5.2 TB/s; 16 rows of 4 tokens after 32,768: 186 us, 5.1 TB/s; one row of 262,144
// positions, 8 heads of 128: 97 us, 5.5 TB/s. Blocks of 16 positions per lane group (PT) where the registers hold them,
// 8 for heads of 256: with 16 those spilled (decode 197 us, verify 237).
//
// The work is cut on the device, where the lengths are: units of 256 positions (a tile or two for each wave) of every row and KV head, as
// many per workgroup as give PAGED_PER_CU workgroups per CU, but PAGED_LEAST of them while the CUs have one each, rows in order. A (row, KV head) that one workgroup has all of is written
// out by it; the others' sums go to scratch slots, which paged_join_kernel puts together.
namespace {

// Workgroups that the work is cut into, per CU. Each begins with a few loads one after another (its place in the work, queries, first
// pages) and ends with its sums; more of them even out the CUs. One tile of query rows, heads of 256: 64 rows of 8,192 positions 188,
// 181 and 176 us with 2, 3 and 4, 16 of 16,384 91, 92 and 98, one of 262,144 98, 102 and 114; heads of 128: 64 rows of 8,192 164 and 196
// with 1 and 2, one of 262,144 97 and 101. Two tiles, heads of 256, 16 rows of 4 after 32,768: 186 and 201 with 2 and 3. Three
// tiles, 16 rows after 32,768, heads of 256 356 and 312 with 2 and 4, of 128 159 and 146.
constexpr int PAGED_PER_CU(int hd, int tiles) { return tiles > 2 ? 4 : tiles == 2 ? 2 : hd > 128 ? 3 : 1; }
// 64 rows of 4 tokens after 512 positions, heads of 256: 28 us, with a unit each 51; one token each 19 and 25.
constexpr int PAGED_LEAST = 3;

struct PagedItem {
    int row, kvh, chunk, chunks, slot;  // slot: the item's place among the partial sums, -1 if it has its (row, KV head) whole
};

// Units of a row that streams; 0 for one that does not.
__device__ __forceinline__ int paged_units(const PagedAttnArgs& a, int row, int G) {
    const PagedRow r = paged_row(a.r, row, a.c.page_size);
    if (r.n <= 0 || r.n * G > a.plan.few) return 0;
    if (r.skip) return 1;
    const int lo = a.window ? max(0, r.p0 + 1 - a.window) / 64 : 0;
    return max(1, ((r.p0 + r.n + 63) / 64 - lo + 3) / 4);
}

__device__ __forceinline__ bool paged_item(const PagedAttnArgs& a, int id, int G, PagedItem& it) {
    const int lane = threadIdx.x & 63, Hkv = a.c.kv_heads;
    const int units0 = lane < a.r.rows ? paged_units(a, lane, G) : 0;  // of the first 64 rows, for both rounds
    double total = units0;
    for (int row = lane + 64; row < a.r.rows; row += 64) total += paged_units(a, row, G);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o);
    total *= Hkv;
    const int target = a.plan.target, cus = a.plan.cus;
    const int per = max(max(1, (int)((total + (target - 1)) / target)), min(PAGED_LEAST, (int)((total + (cus - 1)) / cus)));
    int before = 0, slots = 0;  // items and slots of the rows so far
    for (int base = 0; base < a.r.rows; base += 64) {
        const int row = base + lane;
        const int units = base == 0 ? units0 : row < a.r.rows ? paged_units(a, row, G) : 0, n = (units + per - 1) / per, m = n > 1 ? n : 0;
        const int ends = lanes_up_to(n), slot_ends = lanes_up_to(m);
        const unsigned long long past = __ballot(before + ends * Hkv > id);
        if (past) {
            const int l = __ffsll(past) - 1;
            const int chunks = lane_of(n, l), first = before + (lane_of(ends, l) - chunks) * Hkv,
                      slot0 = slots + (lane_of(slot_ends, l) - (chunks > 1 ? chunks : 0)) * Hkv;
            it.row = base + l;
            it.chunks = chunks;
            it.kvh = (id - first) / chunks;
            it.chunk = (id - first) % chunks;
            it.slot = chunks > 1 ? slot0 + id - first : -1;
            return true;
        }
        before += lane_of(ends, 63) * Hkv;
        slots += lane_of(slot_ends, 63) * Hkv;
    }
    return false;
}

}  // namespace

// Waves that share a SIMD: two while the sums and queries leave room for the loads (16 rows of 32,768 positions, 4 KV heads of 64, two and
// three tiles 59 and 66 us against 87 and 99 with one; four tiles 131 against 120, and two tiles of heads of 128 152 against 130).
constexpr int PAGED_WAVES(int hd, int tiles) { return tiles == 1 || hd * tiles <= 192 ? 2 : 1; }

template <int HD, int NT, int PT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(PAGED_WAVES(HD, NT), PAGED_WAVES(HD, NT)))) void paged_stream_kernel(const PagedAttnArgs a) {
    constexpr int KB = HD / 64, DB = HD / 16, LD = HD + 4, NB = PT / 4, TILE = 4 * PT;
    typedef uint32_t words __attribute__((ext_vector_type(PT / 4)));
    __shared__ __attribute__((aligned(16))) float sums[4 * 16 * LD];
    __shared__ float tops[4][16 * NT], totals[4][16 * NT];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int Hkv = a.c.kv_heads, G = a.q_heads / Hkv, ps = a.c.page_size, shift = __builtin_ctz(ps);
    PagedItem it;
    if (!paged_item(a, blockIdx.x, G, it)) return;
    it = {uniform(it.row), uniform(it.kvh), uniform(it.chunk), uniform(it.chunks), uniform(it.slot)};
    const PagedRow r = paged_row_uniform(a.r, it.row, ps);
    const int R = r.n * G, total = r.p0 + r.n;
    if (it.chunk == 0 && threadIdx.x == 0) {
        int2* t = (int2*)(a.scratch + a.plan.table);
        t[it.row * Hkv + it.kvh] = make_int2(it.slot, it.chunks);
    }
    const int prefix = a.prefix ? uniform(a.prefix[it.row]) : 0;
    const int lo_all = a.window ? max(0, r.p0 + 1 - a.window) : 0, t_first = lo_all / TILE, t_count = r.skip ? 0 : (total + TILE - 1) / TILE - t_first;
    const int t0 = t_first + (int)((long long)t_count * it.chunk / it.chunks), t1 = t_first + (int)((long long)t_count * (it.chunk + 1) / it.chunks);
    const int lo_last = a.window ? max(0, total - a.window) : 0, hi_first = min(total, max(r.p0 + 1, prefix));  // what every token sees
    const int* table = a.r.pages + (size_t)it.row * a.r.max_pages;

    // The queries as B operands: in registers, or where those are full in LDS (rows spread over the banks by 16 bytes).
    constexpr bool QL = NT * HD > 512;
    __shared__ __attribute__((aligned(16))) bf16_t qs[QL ? NT * 16 * (HD + 8) : 8];
    v8bf16 qf[QL ? 1 : NT][QL ? 1 : KB][2];
    auto query = [&](int nt, int j, int u) __attribute__((always_inline)) {
        if constexpr (QL)
            return *(const v8bf16*)(qs + (nt * 16 + col) * (HD + 8) + j * 64 + g * 16 + u * 8);
        else
            return qf[nt][j][u];
    };
    PagedSight see[NT];
    float slope2[NT], top[NT], sum[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = nt * 16 + col, i = row / G, head = it.kvh * G + row % G;
        const bool live = row < R;
        see[nt] = live ? paged_sight(a, r, prefix, i) : PagedSight{0, 0, 0};
        slope2[nt] = live && a.slopes ? a.slopes[head] * LOG2E : 0.0f;
        top[nt] = -INFINITY;
        sum[nt] = 0.0f;
        const bf16_t* qp = a.q + ((size_t)(r.t0 + (live ? i : 0)) * a.q_heads + (live ? head : 0)) * HD + g * 16;
#pragma unroll
        for (int j = 0; j < KB; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                v8bf16 x = *(const v8bf16*)(qp + j * 64 + u * 8);
                if (!live) x = (v8bf16)(__bf16)0.0f;
                if constexpr (!QL)
                    qf[nt][j][u] = x;
                else if (wv == 0)
                    *(v8bf16*)(qs + row * (HD + 8) + j * 64 + g * 16 + u * 8) = x;
            }
    }
    if constexpr (QL) __syncthreads();
    v4f o[NT][DB];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int d = 0; d < DB; ++d) o[nt][d] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};

    // Keys and values are read past the caches (nontemporal), each byte once: over caches in turn, so that none is left from the call
    // before, 64 rows of 8,192 positions 180 us against 188, one of 262,144 97 against 104.
    // The pages of a tile's key rows (lane group col / 4 of each block) and of its values (lane group g); -1: none.
    auto find = [&](int t, int group) { return paged_find(a.r, table, (t * TILE + group * PT) >> shift, a.c.pages); };
    typedef uint32_t words4 __attribute__((ext_vector_type(4)));
    words4 kr[NB][KB];
    words vr[DB];
    int ks, vs;  // scale bytes: made scales where they are used, as doing it here would wait for them
    auto load_keys = [&](int t, int id) __attribute__((always_inline)) {
        const size_t head = (size_t)max(id, 0) * Hkv + it.kvh;
        const int slot = (t * TILE + (col >> 2) * PT + (col & 3)) & (ps - 1);
        const uint8_t* p = a.c.k + (head * ps + slot) * HD + g * 16;
        ks = a.c.k_scale[head];
#pragma unroll
        for (int j = 0; j < KB; ++j)
#pragma unroll
            for (int b = 0; b < NB; ++b) kr[b][j] = __builtin_nontemporal_load((const words4*)(p + b * 4 * HD + j * 64));
    };
    auto load_values = [&](int t, int id) __attribute__((always_inline)) {
        const size_t head = (size_t)max(id, 0) * Hkv + it.kvh;
        const int slot = (t * TILE + g * PT) & (ps - 1);
        const uint8_t* p = a.c.v + head * ps * HD + ((size_t)(slot >> 4) * HD + col) * 16 + (slot & 15);
        vs = a.c.v_scale[head];
#pragma unroll
        for (int d = 0; d < DB; ++d) vr[d] = __builtin_nontemporal_load((const words*)(p + d * 256));
    };
    // Loads run a tile ahead (the pages' numbers two), always, so that what is waited for does not depend on the path here:
    // past its last tile a wave loads that one again.
    int t = t0 + wv;
    if (t < t1) {
        const int last = t + (t1 - 1 - t) / 4 * 4;
        int idk = find(t, col >> 2), idv = find(t, g), next_k = find(min(t + 4, last), col >> 2), next_v = find(min(t + 4, last), g);
        load_keys(t, idk);
        load_values(t, idv);
        for (; t < t1; t += 4) {
            float s[NT][PT];
            {
                v4f c[NT][NB];
                const float scale = paged_scale(ks);
#pragma unroll
                for (int j = 0; j < KB; ++j) {
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            const v8bf16 kf = u ? paged_widen(kr[b][j].z, kr[b][j].w, scale) : paged_widen(kr[b][j].x, kr[b][j].y, scale);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                c[nt][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, query(nt, j, u), j + u ? c[nt][b] : (v4f){0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
                        }
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < PT; ++e) s[nt][e] = c[nt][e >> 2][e & 3];
            }
            const int after_k = find(min(t + 8, last), col >> 2), after_v = find(min(t + 8, last), g);
            load_keys(min(t + 4, last), next_k);
            __builtin_amdgcn_sched_barrier(0);
            const int base = t * TILE, mine = base + g * PT;
            const bool edge = base < lo_last || base + TILE > hi_first || __any(idv < 0);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                paged_scores<PT>(a, s[nt], slope2[nt], mine, see[nt].at);
                if (edge)
#pragma unroll
                    for (int e = 0; e < PT; ++e) s[nt][e] = ((mine + e < see[nt].lo) | (mine + e >= see[nt].hi)) ? -INFINITY : idv < 0 ? QNAN : s[nt][e];
                float m = s[nt][0];
#pragma unroll
                for (int e = 1; e < PT; ++e) m = fmaxf(m, s[nt][e]);
                m = fmaxf(m, __shfl_xor(m, 16));
                m = fmaxf(m, __shfl_xor(m, 32));
                if (__any((m > top[nt] + SLACK) | ((top[nt] == -INFINITY) & (m > -INFINITY)))) {
                    const float up = fmaxf(top[nt], m), f = up == -INFINITY ? 1.0f : exp2_(top[nt] - up);
                    top[nt] = up;
                    sum[nt] *= f;
#pragma unroll
                    for (int d = 0; d < DB; ++d)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[nt][d][e] *= f;
                }
                const float from = top[nt] == -INFINITY ? 0.0f : top[nt];
#pragma unroll
                for (int e = 0; e < PT; ++e) {
                    s[nt][e] = exp2_(s[nt][e] - from);
                    sum[nt] += s[nt][e];
                }
            }
            // What no token of the row sees may be anything: bytes behind its end, a freed page's before its window. Weight zero times
            // NaN is none.
            if (base + TILE > total || base < lo_all || __any(idv < 0)) {
                const int first = lo_all - mine, live = idv < 0 ? 0 : total - mine;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int x = 0; x < PT / 4; ++x) vr[d][x] &= paged_bytes(first - 4 * x, live - 4 * x);
            }
            v8bf16 pf[NT][PT / 8];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int u = 0; u < PT / 8; ++u) {
                    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
                    const u4 w = {pk_bf16(s[nt][8 * u], s[nt][8 * u + 1]), pk_bf16(s[nt][8 * u + 2], s[nt][8 * u + 3]),
                                  pk_bf16(s[nt][8 * u + 4], s[nt][8 * u + 5]), pk_bf16(s[nt][8 * u + 6], s[nt][8 * u + 7])};
                    pf[nt][u] = __builtin_bit_cast(v8bf16, w);
                }
            const float scale = paged_scale(vs);
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                if (d % 4 == 0) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < PT / 8; ++u) {
                    const v8bf16 vf = paged_widen(vr[d][2 * u], vr[d][2 * u + 1], scale);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) o[nt][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[nt][u], o[nt][d], 0, 0, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            load_values(min(t + 4, last), next_v);
            idk = next_k;
            idv = next_v;
            next_k = after_k;
            next_v = after_v;
        }
    }

    // The waves' sums together.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        sum[nt] += __shfl_xor(sum[nt], 16);
        sum[nt] += __shfl_xor(sum[nt], 32);
        if (g == 0) tops[wv][nt * 16 + col] = top[nt], totals[wv][nt * 16 + col] = sum[nt];
    }
    __syncthreads();
    float* part = (float*)(a.scratch + a.plan.part) + (size_t)max(it.slot, 0) * a.plan.few * (HD + 2);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        if (nt * 16 >= R) break;
        const int mine = nt * 16 + col;
        const float up = fmaxf(fmaxf(tops[0][mine], tops[1][mine]), fmaxf(tops[2][mine], tops[3][mine]));
        const float f = up == -INFINITY ? 1.0f : exp2_(top[nt] - up);
        if (nt) __syncthreads();
#pragma unroll
        for (int d = 0; d < DB; ++d)
            *(v4f*)(sums + (wv * 16 + col) * LD + d * 16 + g * 4) = (v4f){o[nt][d][0] * f, o[nt][d][1] * f, o[nt][d][2] * f, o[nt][d][3] * f};
        __syncthreads();
        for (int x = threadIdx.x; x < 16 * HD / 4; x += 256) {
            const int c = x / (HD / 4), d = x % (HD / 4) * 4, row = nt * 16 + c;
            if (row >= R) continue;
            v4f v = *(const v4f*)(sums + c * LD + d);
#pragma unroll
            for (int w = 1; w < 4; ++w) v += *(const v4f*)(sums + (w * 16 + c) * LD + d);
            const float m = fmaxf(fmaxf(tops[0][row], tops[1][row]), fmaxf(tops[2][row], tops[3][row]));
            float l = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) l += totals[w][row] * (m == -INFINITY ? 1.0f : exp2_(tops[w][row] - m));
            if (it.slot < 0) {
                const float inv = r.skip ? 0.0f : 1.0f / l;
                *(uint2*)(a.out + ((size_t)(r.t0 + row / G) * a.q_heads + it.kvh * G + row % G) * HD + d) =
                    make_uint2(pk_bf16(v[0] * inv, v[1] * inv), pk_bf16(v[2] * inv, v[3] * inv));
            } else {
                *(v4f*)(part + (size_t)row * HD + d) = v;
                if (d == 0) *(float2*)(part + (size_t)a.plan.few * HD + row * 2) = make_float2(m, l);
            }
        }
    }
}

// The parts of one (row, KV head)'s query row put together, W waves every W-th of them each, four under way at a time. Grid: rows x
// KV heads x query rows. Sixteen waves where parts are many (one row of 262,144 positions has 128 per KV head: 7 us against 15 with
// four waves), four where they are few and the workgroups many (64 rows of 8,192 positions: 189 us in all against 204 with
// sixteen).
template <int E, int W>
__device__ __forceinline__ void paged_join(const PagedAttnArgs& a, int block) {
    constexpr int HD = E * 64;
    __shared__ float sums[W][HD], totals[W];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, Hkv = a.c.kv_heads, G = a.q_heads / Hkv;
    const int n = a.plan.joins, q = block % n, kvh = block / n % Hkv, row = block / n / Hkv;
    const PagedRow r = paged_row(a.r, row, a.c.page_size);
    if (q >= r.n * G || r.n * G > a.plan.few) return;
    const int2 t = ((const int2*)(a.scratch + a.plan.table))[row * Hkv + kvh];
    if (t.y <= 1) return;
    const size_t step = (size_t)a.plan.few * (HD + 2);
    const float* part = (const float*)(a.scratch + a.plan.part) + (size_t)t.x * step;
    const float* stats = part + (size_t)a.plan.few * HD + q * 2;
    float top = -INFINITY;
    for (int c = lane; c < t.y; c += 64) top = fmaxf(top, stats[c * step]);
    top = warp_max(top);
    float o[E] = {}, l = 0.0f;
    for (int c0 = wv; c0 < t.y; c0 += 4 * W) {
        float2 s[4];
        float v[4][E];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const size_t c = min(c0 + i * W, t.y - 1);
            s[i] = *(const float2*)(stats + c * step);
#pragma unroll
            for (int e = 0; e < E; ++e) v[i][e] = part[c * step + (size_t)q * HD + e * 64 + lane];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (c0 + i * W >= t.y) break;
            const float f = s[i].x == -INFINITY ? (s[i].y == 0.0f ? 0.0f : 1.0f) : exp2_(s[i].x - top);  // no weights, or only NaN ones
            l += s[i].y * f;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += v[i][e] * f;
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sums[wv][e * 64 + lane] = o[e];
    if (lane == 0) totals[wv] = l;
    __syncthreads();
    bf16_t* out = a.out + ((size_t)(r.t0 + q / G) * a.q_heads + kvh * G + q % G) * HD;
    for (int d = threadIdx.x; d < HD; d += W * 64) {
        float all = 0.0f, x = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) all += totals[w], x += sums[w][d];
        out[d] = f2bf(x / all);
    }
}

template <int E, int W>
__global__ __launch_bounds__(W * 64) void paged_join_kernel(const PagedAttnArgs a) {
    paged_join<E, W>(a, blockIdx.x);
}

// ---- Many query rows (prefill chunks): tiles of 256 query rows (tokens x the KV head's query heads) per workgroup.
//
// A wave has 32 query rows as a B operand's columns; keys are A, 32 positions at a time, their rows permuted so that a lane's
// scores are the eight consecutive positions that it feeds to each step of weights x V, where values are A (a lane then holds
// four consecutive dims of one query row). Each tile of 32 positions is read from its pages once per workgroup, widened to bf16 by
// its threads and put into one of three LDS buffers, from which its eight waves read it: widening in the waves' own registers
// would take as long as their MFMAs. Two waves share a SIMD, one half a tile behind the other, so that one's exponentials
// run beside the other's MFMAs.
//
// Bound: the matrix cores and the exponentials together. A tile of heads of 256 takes 4,100 to 4,500 clocks, of which its MFMAs
// are 2,048 and its LDS reads 2,300 (2,048 tokens after 14,336, 24 and 4 heads of 256: 0.72 to 0.83 ms, 0.9 to 1.07 PFLOP/s); of heads
// of 128 some 2,600, of which 1,024; of heads of 64, whose registers let two workgroups share a CU, 1,500 of 512. Four waves of 64 rows read LDS half
// as often, but have no second wave to fill a SIMD's pauses: 0.83 ms.
//
// While tiles are few, the sub-blocks of 32 positions of all of them, one after another, and the beginning of each, are dealt out to
// the CUs in equal parts: a workgroup ends one tile, takes some whole and begins another. What it has of a tile that others share goes to scratch
// in float32 (256 KB for heads of 256, a dozen sub-blocks' time), and paged_join_tiles_kernel puts it together.
namespace {

constexpr int PT_TILE = 256;
constexpr int PT_FEW = 3;  // tiles per CU: with as many they go whole, a workgroup each
// Sub-blocks of a part. Beginning a tile costs some 15,000 clocks (its work found, its first pages and queries read), as much as
// five sub-blocks of heads of 128: 777 tokens after none in parts of 12 took 78 us, of 8 (more of them) 59, whole 46.
// Of heads of 64 a sub-block takes half as long, but two workgroups begin beside each other: parts of 8 (4 prompts of 624 to 1,000 with
// slopes 71 us against 74, 777 tokens after none 31 against 37).
constexpr int PT_LEAST(int head_dim) { return head_dim > 64 ? 16 : 8; }
// What beginning a tile counts as, in sub-blocks (fewer than a part has); a part that would end within it leaves the tile to the next. 4
// prompts with slopes 62 us, counting nothing 66; 777 tokens after 4,000 59 and 66. For larger heads, whose sub-blocks take
// longer, nothing: what it saves there (2% of short calls) their loops lose by the registers that it takes.
constexpr int PT_START(int head_dim) { return head_dim > 64 ? 0 : 7; }
constexpr int PT_PER_CU(int head_dim) { return head_dim > 64 ? 1 : 2; }  // workgroups that a CU holds
__device__ __forceinline__ v8bf16 paged_frag(uint32_t at) {
    return *(const __attribute__((address_space(3))) v8bf16*)(uintptr_t)at;
}

// The sub-blocks [lo, hi) that a tile's query rows see.
struct PagedSpan {
    int lo, hi;
};

__device__ __forceinline__ PagedSpan paged_span(const PagedAttnArgs& a, const PagedRow& r, int prefix, int tile, int G) {
    const int first = tile * PT_TILE, lo = paged_sight(a, r, prefix, first / G).lo / 32;
    return {lo, r.skip ? lo : (paged_sight(a, r, prefix, min((first + PT_TILE - 1) / G, r.n - 1)).hi + 31) / 32};
}

__device__ __forceinline__ int paged_row_tiles(const PagedAttnArgs& a, const PagedRow& r, int G) {
    return r.n <= 0 || (a.plan.items && r.n * G <= a.plan.few) ? 0 : (r.n * G + PT_TILE - 1) / PT_TILE;
}

// a / b of 0 <= a < 2^52, b > 0: rounding the reciprocal and the product leaves the quotient one off at most.
__device__ __forceinline__ long long quotient(long long a, long long b) {
    long long q = (long long)((double)a * (1.0 / (double)b));
    const long long left = a - q * b;
    return left < 0 ? q - 1 : left >= b ? q + 1 : q;
}

// The call's work: `total` units, sub-blocks of its tiles in order (row, tile, KV head) or, `whole`, tiles; in equal `parts`, one
// per workgroup.
struct PagedWork {
    long long total;
    int jobs, parts;
    bool whole, kept;
    long long each, longer;  // units of a part; the first `longer` have one more
    __device__ __forceinline__ long long start(int w) const { return each * w + min((long long)w, longer); }
    __device__ __forceinline__ int part(long long u) const {  // that unit u is in
        const long long l = longer * (each + 1);
        return u < l ? (int)quotient(u, each + 1) : (int)(longer + quotient(u - l, each));
    }
};

// The tile that unit u of the call's work is in, and its first unit.
struct PagedJob {
    int row, tile, kvh;
    long long start;
    int units;
};

__device__ __forceinline__ long long uniform(long long x) {
    return (long long)uniform((int)(x >> 32)) << 32 | (uint32_t)uniform((int)x);
}

// Goes over the tiles, a lane for each: 64 rows' numbers of tiles at a time, then 64 of their tiles, whose rows the lanes look up among
// them. Without `find` it returns the work's total of sub-blocks per KV head, number of tiles and longest tile in job.start, tile and units; with it
// the job of unit u. `keep` receives the lanes' first tiles.
typedef int PagedKept[4][64];  // sub-blocks up to the tile's end, its own, its row, its place in the row

template <int HD>
__device__ __forceinline__ PagedJob paged_tiles_list(const PagedAttnArgs& a, int G, bool find, long long u, bool whole, PagedKept* keep) {
    const int lane = threadIdx.x & 63, Hkv = a.c.kv_heads;
    long long before = 0;
    int tiles = 0, longest = 1;
    for (int base = 0; base < a.r.rows; base += 64) {
        const int at = min(base + lane, a.r.rows - 1);
        PagedRow r = paged_row(a.r, at, a.c.page_size);
        const int prefix = a.prefix ? a.prefix[at] : 0, n = base + lane < a.r.rows ? paged_row_tiles(a, r, G) : 0;
        const int ends = lanes_up_to(n), count = lane_of(ends, 63);
        for (int k0 = 0; k0 < count; k0 += 64) {
            const int k = k0 + lane;
            int l = 0;  // the first lane whose rows' tiles end past k
#pragma unroll
            for (int o = 32; o > 0; o >>= 1)
                if (__shfl(ends, l + o - 1) <= k) l += o;
            l = min(l, 63);
            PagedRow mine;
            mine.n = __shfl(r.n, l);
            mine.p0 = __shfl(r.p0, l);
            mine.skip = __shfl((int)r.skip, l) != 0;
            mine.t0 = 0;
            const int tile = __shfl(ends, l) - 1 - k;  // the latest tokens, the longest tiles, first
            const PagedSpan s = paged_span(a, mine, __shfl(prefix, l), max(tile, 0), G);
            const int units = k >= count ? 0 : whole ? 1 : max(1, s.hi - s.lo) + PT_START(HD);
            longest = max(longest, units);
            const uint32_t sum = lanes_up_to(units);  // of 64 tiles of up to 2^25 sub-blocks and a token's
            if (keep && base == 0 && k0 == 0 && threadIdx.x < 64) {
                (*keep)[0][lane] = (int)sum;
                (*keep)[1][lane] = units;
                (*keep)[2][lane] = l;
                (*keep)[3][lane] = tile;
            }
            const unsigned long long past = find ? __ballot(before + (long long)sum * Hkv > u) : 0;
            if (past) {
                const int f = __ffsll(past) - 1;
                PagedJob job;
                job.row = base + lane_of(l, f);
                job.tile = lane_of(tile, f);
                job.units = lane_of(units, f);
                const long long first = before + (long long)(uint32_t)lane_of(sum - units, f) * Hkv;
                job.kvh = (int)quotient(u - first, job.units);
                job.start = first + (long long)job.kvh * job.units;
                return job;
            }
            before += (long long)(uint32_t)lane_of(sum, 63) * (find ? Hkv : 1);
        }
        tiles += count;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) longest = max(longest, __shfl_xor(longest, o));
    return {-1, tiles, 0, before, uniform(longest)};
}

// The job of unit u: from the kept tiles where those are all (looking it up again takes 4,000 clocks of each tile), or from the list.
// Not for heads of 256: the registers that this takes push others out of the loop (a prompt's chunk 855 us against 805).
template <int HD>
__device__ __forceinline__ PagedJob paged_tiles_find(const PagedAttnArgs& a, int G, long long u, bool whole, bool kept, const PagedKept& keep) {
    if (!kept) return paged_tiles_list<HD>(a, G, true, u, whole, nullptr);
    const int lane = threadIdx.x & 63, Hkv = a.c.kv_heads, units = keep[1][lane];
    const uint32_t sum = keep[0][lane];
    const int f = whole ? (int)u / Hkv : __ffsll((unsigned long long)__ballot((long long)sum * Hkv > u)) - 1;
    PagedJob job;
    job.row = lane_of(keep[2][lane], f);
    job.tile = lane_of(keep[3][lane], f);
    job.units = whole ? 1 : lane_of(units, f);
    const long long first = whole ? (long long)f * Hkv : (long long)(uint32_t)lane_of(sum - units, f) * Hkv;
    job.kvh = (int)quotient(u - first, job.units);
    job.start = first + (long long)job.kvh * job.units;
    return job;
}

template <int HD>
__device__ __forceinline__ PagedWork paged_work(const PagedAttnArgs& a, int G, PagedKept* keep) {
    const PagedJob all = paged_tiles_list<HD>(a, G, false, 0, false, keep);
    const int jobs = all.tile * a.c.kv_heads;
    const long long total = all.start * a.c.kv_heads;
    const bool kept = keep && a.r.rows <= 64 && all.tile <= 64;
    if (!a.plan.parts || jobs >= PT_FEW * a.plan.cus || all.units <= 2 * PT_LEAST(HD) + PT_START(HD)) return {jobs, jobs, jobs, true, kept, 1, 0};
    const int parts = (int)max(1LL, min((long long)a.plan.parts, total / PT_LEAST(HD)));
    const long long each = quotient(total, parts);
    return {total, jobs, parts, false, kept, each, total - each * parts};
}

// A cut tile in the scratch's table, at the workgroup that begins it: which workgroups' sums make it.
struct PagedCut {
    int row, tile, kvh, slot, first, last;  // slot: where the first one's are; a later workgroup w's are in slot 2 w
};

}  // namespace

template <int HD>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2 * PT_PER_CU(HD), 2 * PT_PER_CU(HD)))) void paged_tiles_kernel(const PagedAttnArgs a) {
    constexpr int KM = HD / 16, VD = HD / 32, HALF = 32 * HD * 2, BUF = 2 * HALF;  // MFMA steps; bytes of a buffer's keys, of a buffer
    constexpr int PIECES = 2 * HD;       // 16-byte pieces of a tile's keys, and of its values: one of each per thread, or of either
    constexpr bool BOTH = HD == 256;
    constexpr int STEPS = BOTH ? 4 : 2;  // half pieces to widen
    constexpr int DEEP = HD > 128 ? 2 : 4;  // operands read ahead from LDS
    __shared__ __attribute__((aligned(1024))) uint8_t ring[3 * BUF];
    __shared__ int lost[3][2];
    __shared__ float slopes[PT_TILE];
    const int lane = threadIdx.x & 63, wv = uniform((int)threadIdx.x >> 6), l32 = lane & 31, h = lane >> 5;
    const int Hkv = a.c.kv_heads, G = a.q_heads / Hkv, ps = a.c.page_size, shift = __builtin_ctz(ps);
    constexpr bool KEEP = HD <= 128;
    __shared__ PagedKept keep;
    const PagedWork work = paged_work<HD>(a, G, KEEP ? &keep : nullptr);
    const int w = blockIdx.x;
    if (w == 0 && threadIdx.x == 0 && a.plan.parts) *(int*)(a.scratch + a.plan.cuts) = work.whole || !work.jobs ? 0 : work.parts;
    if (!work.jobs || w >= work.parts) return;
    if constexpr (KEEP) __syncthreads();
    const long long begin = work.start(w), end = work.start(w + 1);
    for (long long unit = begin; unit < end;) {
    const PagedJob job = paged_tiles_find<HD>(a, G, unit, work.whole, KEEP && work.kept, keep);
    if (job.row < 0) return;
    const PagedRow r = paged_row_uniform(a.r, job.row, ps);
    const int R = r.n * G, total = r.p0 + r.n, prefix = a.prefix ? uniform(a.prefix[job.row]) : 0;
    const int lo_all = a.window ? max(0, r.p0 + 1 - a.window) : 0;
    const int* table = a.r.pages + (size_t)job.row * a.r.max_pages;
    // This part's tiles of 32 positions of those that any of the workgroup's query rows sees.
    const PagedSpan span = paged_span(a, r, prefix, job.tile, G);
    const long long stop = min(end, job.start + job.units);
    int begun = (int)(unit - job.start), ended = (int)(stop - job.start);
    bool left = false;
    if constexpr (PT_START(HD) > 0) {
        begun = max(begun - PT_START(HD), 0);
        ended -= PT_START(HD);
        left = !work.whole && ended <= 0;
    }
    const int T0 = span.lo + (work.whole ? 0 : begun), T1 = work.whole ? span.hi : min(span.hi, span.lo + ended);
    const bool first = PT_START(HD) ? work.whole || begun == 0 : unit == job.start, alone = first && stop == job.start + job.units;
    const int slot = 2 * w + (unit > begin);
    // The tile that this part begins and others end: this part's last, at most one.
    if (stop == end && !work.whole && threadIdx.x == 0)
        ((PagedCut*)(a.scratch + a.plan.cuts + 256))[w] = {job.row, job.tile, job.kvh, slot, w, first && !alone && !left ? work.part(job.start + job.units - 1) : w};
    if (left) return;
    unit = stop;

    // The wave's query rows, a lane's (and lane ^ 32's) one, as B operands.
    const int row0 = job.tile * PT_TILE + wv * 32, row = row0 + l32, token = row < R ? row / G : -1, head = job.kvh * G + row % G;
    if (h == 0) slopes[wv * 32 + l32] = token >= 0 && a.slopes ? a.slopes[head] * LOG2E : 0.0f;
    // For heads of 256 the first QS of them wait in LDS: with all in registers the loop would reload something from scratch memory,
    // each time behind every load under way.
    constexpr int QS = HD > 128 ? 4 : 0;
    __shared__ __attribute__((aligned(16))) v8bf16 q_wait[QS ? QS * 512 : 1];
    v8bf16 qf[KM];
    {
        const bf16_t* qp = a.q + ((size_t)(r.t0 + max(token, 0)) * a.q_heads + (token >= 0 ? head : 0)) * HD + h * 8;
#pragma unroll
        for (int m = 0; m < KM; ++m) {
            v8bf16 x = *(const v8bf16*)(qp + m * 16);
            if (token < 0) x = (v8bf16)(__bf16)0.0f;
            if (m < QS)
                q_wait[m * 512 + threadIdx.x] = x;
            else
                qf[m] = x;
        }
    }
    const int lo_whole = uniform(paged_sight(a, r, prefix, min(row0 + 31, R - 1) / G).lo), hi_whole = uniform(paged_sight(a, r, prefix, min(row0, R - 1) / G).hi);

    // This thread's pieces of a tile: 16 dims of one key and 16 positions of one value dim, in position group vg0 (of 16).
    const bool keys = BOTH || wv * 64 < PIECES, vals = BOTH || (wv * 64 >= PIECES && wv * 64 < 2 * PIECES);
    const int c0 = (int)threadIdx.x & (PIECES - 1), vg0 = uniform(c0 / HD);
    uint4 rk, rv;
    int id, found, ks, vs;  // this tile's page; the next one's as read; scale bytes
    // Zero, but not for the compiler: it would take the scale bytes for uniform and move them to scalar registers as soon as they
    // are asked for, which waits for them in every tile.
    uint32_t zero;
    asm("v_mov_b32 %0, 0" : "=v"(zero));
    // Tiles go from the part's last to its first: the nearest positions first, whose scores are the largest where distance takes from
    // them. A tile's page number is read a tile before its keys and values, so that no load waits for another.
    auto look = [&](int T) __attribute__((always_inline)) { found = table[min((max(T, T0) * 32 + vg0 * 16) >> shift, a.r.max_pages - 1)]; };
    auto load = [&](int T) __attribute__((always_inline)) {
        const int p = max(T, T0) * 32 + vg0 * 16;
        id = uniform(found);
        id = ((id < a.c.pages) & (p >> shift < a.r.max_pages)) ? id : -1;
        const size_t hd = (size_t)max(id, 0) * Hkv + job.kvh, at = (hd * ps + (p & (ps - 1))) * HD + c0 % HD * 16;
        if constexpr (BOTH) {
            ks = (a.c.k_scale + hd)[zero];
            vs = (a.c.v_scale + hd)[zero];
            rk = *(const uint4*)(a.c.k + at);
            rv = *(const uint4*)(a.c.v + at);
        } else {
            ks = ((keys ? a.c.k_scale : a.c.v_scale) + hd)[zero];
            rk = *(const uint4*)((keys ? a.c.k : a.c.v) + at);
        }
    };
    // Step x of widening the loaded tile T into buffer b. Keys: row (position), its 16-byte chunks spread over the banks;
    // values: per dim 32 positions, likewise.
    const uint32_t lds0 = (uint32_t)(uintptr_t)LDS_PTR(&ring[0]);
    const int kp0 = c0 / (HD / 16), kc0 = c0 % (HD / 16) * 2, vd0 = c0 % HD;
    const uint32_t put_k = kp0 * HD * 2 + ((kc0 ^ (HD > 64 ? kp0 & 15 : (kp0 >> 1) & 7)) << 4);
    const uint32_t put_v = HALF + vd0 * 64 + ((vg0 * 2 ^ ((vd0 >> 1) & 3) ^ ((vd0 >> 3) & 1)) << 4);
    auto widen = [&](int T, int b, int x) __attribute__((always_inline)) {
        const uint32_t buf = lds0 + b * BUF;
        const int u = x & 1;
        const bool key = BOTH ? x < 2 : keys;
        if (x == 0) {
            // What no token of the row sees may be anything: weight zero times NaN is none.
            if ((T * 32 + 32 > total) | (T * 32 < lo_all) | (id < 0)) {
                const int at = T * 32 + vg0 * 16, first = lo_all - at, left = id < 0 ? 0 : total - at;
                uint32_t* w4 = (uint32_t*)(BOTH ? &rv : &rk);
                if (vals)
#pragma unroll
                    for (int y = 0; y < 4; ++y) w4[y] &= paged_bytes(first - 4 * y, left - 4 * y);
            }
            if (vd0 == 0) lost[b][vg0] = id < 0;
        }
        const uint4 w4 = !BOTH || key ? rk : rv;
        const uint32_t at = key ? put_k ^ (u << 4) : put_v ^ (u << 4);
        if (keys | vals)
            *(__attribute__((address_space(3))) v8bf16*)(uintptr_t)(buf + at) =
                u ? paged_widen(w4.z, w4.w, paged_scale(!BOTH || key ? ks : vs)) : paged_widen(w4.x, w4.y, paged_scale(!BOTH || key ? ks : vs));
    };

    const int kp = (l32 & ~12) | (l32 & 4) << 1 | (l32 & 8) >> 1;  // the position of this lane's key row
    const uint32_t kl = kp * HD * 2 + ((h ^ (HD > 64 ? kp & 15 : (kp >> 1) & 7)) << 4);
    const uint32_t vl = HALF + l32 * 64 + ((h ^ ((l32 >> 1) & 3) ^ ((l32 >> 3) & 1)) << 4);
    v16f o[VD], s;
    typedef uint32_t u4_ __attribute__((ext_vector_type(4)));
    u4_ pw[2];
    // Scores in powers of two: times scale log2 e beside the exponential, or capped and biased (`bent`) before the maxima.
    const bool bent = a.cap > 0.0f || a.slopes;
    const float mul = bent ? 1.0f : a.scale * LOG2E;
    // What a query row's weights are relative to is the largest score of the first tile that it sees anything of, and stays:
    // floats hold weights of up to 2^LEAP as exactly as others. Only if some score leaps further than that are the item's sums
    // formed again, relative to the largest score, which is known by then. (Raising it on the way costs the loop copies of the
    // sums even where it never happens: the compiler keeps them out of the MFMAs' registers for it.)
    constexpr float LEAP = 40.0f, UNSEEN = -3e38f;
    float top = UNSEEN, most = -INFINITY, sum;
    bool unseen = true;  // some row's reference is not known yet
    // The largest of three, NaN ones passed over.
    auto max3 = [](float x, float y, float z) __attribute__((always_inline)) {
        float m;
        asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(x), "v"(y), "v"(z));
        return m;
    };
    // Scores of tile T in buffer b, with the loaded tile T - 1 widened beside their MFMAs and the one after it asked for; then its weights.
    auto scores = [&](int T, int b, int next) __attribute__((always_inline)) {
        const uint32_t ka = lds0 + b * BUF + kl;
        const int gone0 = lost[b][0], gone1 = lost[b][1];
        v8bf16 kf[DEEP], qx[DEEP];
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
        for (int m = 0; m < DEEP; ++m) {
            kf[m] = paged_frag(ka ^ (m << 5));
            if (m < QS) qx[m] = q_wait[m * 512 + threadIdx.x];
        }
#pragma unroll
        for (int m = 0; m < KM; ++m) {
            __builtin_amdgcn_sched_barrier(0);
            const v8bf16 q = m < QS ? qx[m % DEEP] : qf[m];
            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[m % DEEP], q, s, 0, 0, 0);
            if (m + DEEP < QS) qx[m % DEEP] = q_wait[(m + DEEP) * 512 + threadIdx.x];
            if (m + DEEP < KM) kf[m % DEEP] = paged_frag(ka ^ ((m + DEEP) << 5));
            if (m >= KM - STEPS) widen(T - 1, next, m - (KM - STEPS));
        }
        __builtin_amdgcn_sched_barrier(0);
        load(T - 2);
        look(T - 3);
        const int p0 = T * 32, lost0 = uniform(gone0), lost1 = uniform(gone1);
        if (bent)
#pragma unroll
            for (int k = 0; k < 2; ++k) {  // the lane's positions: 8 from p0 + 16 k + 8 h on
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = s[8 * k + e];
                paged_scores<8>(a, y, slopes[wv * 32 + l32], p0 + 16 * k + 8 * h, r.p0 + token);
#pragma unroll
                for (int e = 0; e < 8; ++e) s[8 * k + e] = y[e];
            }
        if (!((p0 >= lo_whole) & (p0 + 32 <= hi_whole) & !(lost0 | lost1))) {
            const PagedSight see = paged_sight(a, r, prefix, max(token, 0));
            const int lo = see.lo - p0 - 8 * h, hi = token < 0 ? -64 : see.hi - p0 - 8 * h;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int p = 16 * (e >> 3) + (e & 7);
                const float x = (e >> 3 ? lost1 : lost0) ? QNAN : s[e];
                s[e] = ((p < lo) | (p >= hi)) ? -INFINITY : x;
            }
        }
        float m = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; e += 2) m = max3(s[e], s[e + 1], m);
        most = fmaxf(most, m);
        if (unseen) {
            m = fmaxf(m, __shfl_xor(m, 32)) * mul;
            top = ((top == UNSEEN) & (m > -INFINITY)) ? m : top;
            unseen = __any(top == UNSEEN);
        }
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            const float p = exp2_(__builtin_fmaf(s[e], mul, -top)), q = exp2_(__builtin_fmaf(s[e + 1], mul, -top));
            sum += p;
            sum += q;
            pw[e >> 3][(e >> 1) & 3] = pk_bf16(p, q);
        }
    };
    // Weights x V of the tile in buffer b.
    auto values = [&](int b) __attribute__((always_inline)) {
        const uint32_t va = lds0 + b * BUF + vl;
        auto frag = [&](int x) __attribute__((always_inline)) { return paged_frag((va ^ (x / VD << 5)) + x % VD * 2048); };
        v8bf16 vf[DEEP];
#pragma unroll
        for (int x = 0; x < DEEP; ++x) vf[x] = frag(x);
#pragma unroll
        for (int x = 0; x < 2 * VD; ++x) {
            __builtin_amdgcn_sched_barrier(0);
            o[x % VD] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[x % DEEP], __builtin_bit_cast(v8bf16, pw[x / VD]), o[x % VD], 0, 0, 0);
            if (x + DEEP < 2 * VD) vf[x % DEEP] = frag(x + DEEP);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // A tile's beginning: what the waves have widened is in LDS.
    auto meet = [&]() __attribute__((always_inline)) { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

    for (int pass = 0;; ++pass) {
        sum = 0.0f;
#pragma unroll
        for (int d = 0; d < VD; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
        if (T0 >= T1) break;
        look(T1 - 1);
        load(T1 - 1);
        look(T1 - 2);
#pragma unroll
        for (int x = 0; x < STEPS; ++x) widen(T1 - 1, 0, x);
        load(T1 - 2);
        look(T1 - 3);
        // The buffers go round. A tile is in its own, widened there before its beginning, which the first four waves meet before their scores of it, the
        // other four, which share the SIMDs with them, before their weights x V of the tile before: so one of a SIMD's two waves
        // forms weights while the other feeds the matrix cores. A tile goes into the buffer of the one three before, whose
        // last weights x V lie before the meeting before.
        for (int T = T1 - 1, b = 0; T >= T0; --T) {
            const int next = b == 2 ? 0 : b + 1;
            if (wv < 4 || T == T1 - 1) meet();
            scores(T, b, next);
            if (wv >= 4 && T > T0) meet();
            values(b);
            b = next;
        }
        most = fmaxf(most, __shfl_xor(most, 32)) * mul;
        if (pass || !__syncthreads_or(most > top + LEAP)) break;
        top = fmaxf(top, most);
    }

    const float l = sum + __shfl_xor(sum, 32);
    if (alone) {
        const float inv = r.skip ? 0.0f : 1.0f / l;
        if (token >= 0) {
            bf16_t* out = a.out + ((size_t)(r.t0 + token) * a.q_heads + head) * HD + h * 4;
#pragma unroll
            for (int d = 0; d < VD; ++d)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *(uint2*)(out + d * 32 + q * 8) = make_uint2(pk_bf16(o[d][4 * q] * inv, o[d][4 * q + 1] * inv), pk_bf16(o[d][4 * q + 2] * inv, o[d][4 * q + 3] * inv));
        }
    } else {
        // [slot][wave][d][q][lane] of four dims, then per query row what its weights are relative to and their sum.
        float* part = (float*)(a.scratch + a.plan.cut_part) + (size_t)slot * (PT_TILE * (HD + 2));
        if (h == 0) *(float2*)(part + PT_TILE * HD + (wv * 32 + l32) * 2) = make_float2(top, l);
#pragma unroll
        for (int d = 0; d < VD; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *(v4f*)(part + (((wv * VD + d) * 4 + q) * 64 + lane) * 4) = (v4f){o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
    }
    __syncthreads();  // the ring and the slopes are the next tile's
    }
}

// The parts of cut tiles put together. Grid: parts (the tile that each begins, if it is cut) x the tile's eight groups of 32 query
// rows x dims in blocks of 32; behind those of the rows that streamed, if some may have been cut: one launch for both.
template <int HD>
__global__ __launch_bounds__(256) void paged_join_tiles_kernel(const PagedAttnArgs a, int streamed) {
    if ((int)blockIdx.x < streamed) return paged_join<HD / 64, 4>(a, blockIdx.x);
    constexpr int VD = HD / 32;
    const int lane = threadIdx.x & 63, q = threadIdx.x >> 6, l32 = lane & 31, h = lane >> 5;
    const int Hkv = a.c.kv_heads, G = a.q_heads / Hkv, block = blockIdx.x - streamed;
    const int d = block % VD, group = block / VD % 8, j = block / VD / 8;
    if (j >= *(const int*)(a.scratch + a.plan.cuts)) return;
    const PagedCut job = ((const PagedCut*)(a.scratch + a.plan.cuts + 256))[j];
    if (job.first == job.last) return;
    const PagedRow r = paged_row(a.r, job.row, a.c.page_size);
    const int row = job.tile * PT_TILE + group * 32 + l32;
    if (row >= r.n * G) return;
    const size_t step = PT_TILE * (HD + 2);
    const float* part = (const float*)(a.scratch + a.plan.cut_part);
    const size_t stats = PT_TILE * HD + (group * 32 + l32) * 2, dims = ((((size_t)group * VD + d) * 4 + q) * 64 + lane) * 4;
    auto slot = [&](int w) { return (w == job.first ? job.slot : 2 * w) * step; };
    float top = -INFINITY, l = 0.0f;
    for (int w = job.first; w <= job.last; ++w) top = fmaxf(top, part[slot(w) + stats]);
    v4f o = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
    for (int w = job.first; w <= job.last; ++w) {
        const float2 s = *(const float2*)(part + slot(w) + stats);
        const float f = s.x == top ? 1.0f : exp2_(s.x - top);  // the same where no part saw anything, or only NaN
        l += s.y * f;
        o += *(const v4f*)(part + slot(w) + dims) * f;
    }
    const float inv = r.skip ? 0.0f : 1.0f / l;
    *(uint2*)(a.out + ((size_t)(r.t0 + row / G) * a.q_heads + job.kvh * G + row % G) * HD + d * 32 + q * 8 + h * 4) =
        make_uint2(pk_bf16(o[0] * inv, o[1] * inv), pk_bf16(o[2] * inv, o[3] * inv));
}

PagedPlan paged_attention_plan(const PagedCache& c, const PagedRows& r, int q_heads) {
    PagedPlan p{};
    const int G = q_heads / c.kv_heads;
    const long long most = (long long)r.max_tokens * G;
    // All rows stream while their query rows fit four tiles, three for heads of 256 (the fourth's sums do not fit the registers: 16 rows of
    // 32,768 positions, 64 query rows, 1,627 us against 473 as a tile of 256). In a ragged call with longer rows those of the other
    // rows' usual number of tokens, if that many fit, or else of one token: a single token pays for the tiles that it does not
    // fill (heads of 256, two tiles for one 240 us against 191), a verify row that goes as a tile of 256 takes twice as long.
    const int limit = c.head_dim > 128 ? 48 : 64;
    const bool any = most <= limit || (r.q_start && G <= limit);
    const long long others = std::max(0, r.tokens - r.max_tokens), usual = (others + r.rows - 2) / std::max(1, r.rows - 1) * G;
    p.few = !any ? 0 : (int)((most <= limit ? most : usual <= limit ? std::max<long long>(usual, G) : G) + 15) / 16 * 16;
    p.cus = q38_device_cus();
    p.target = PAGED_PER_CU(c.head_dim, p.few / 16) * p.cus;
    const long long heads = (long long)r.rows * c.kv_heads, units = ((long long)r.max_pages * c.page_size + r.max_tokens + 63) / 64 / 4 + 2;
    p.joins = (int)std::min<long long>(most, p.few);
    p.items = any ? (int)std::min<long long>(p.target + heads, heads * units) : 0;
    p.slots = units > 1 ? std::min(2 * p.target, p.items) : 0;
    p.bytes = 0;
    if (any) {
        p.table = 0;
        p.part = (size_t)heads * 8 + 255 & ~(size_t)255;
        p.bytes = p.part + (size_t)p.slots * p.few * (c.head_dim + 2) * 4;
    }
    if (most > p.few) {
        // Of a ragged call's tokens at most so many tiles (a workgroup that finds no work still takes its turn on a CU: 24 rows, one of
        // 777 tokens, 155 us with a workgroup for as many in each row).
        const long long jobs = std::min(heads * ((most + PT_TILE - 1) / PT_TILE), c.kv_heads * ((long long)r.tokens * G / PT_TILE + r.rows));
        const long long blocks = ((long long)r.max_pages * c.page_size + r.max_tokens + 31) / 32 + 1;
        const bool many = jobs >= (long long)PT_FEW * p.cus;
        p.parts = many && !r.q_start ? 0 : (int)std::min<long long>(p.cus * PT_PER_CU(c.head_dim), std::max<long long>(1, jobs * blocks / PT_LEAST(c.head_dim)));
        p.tiles = (int)std::max<long long>(p.parts, jobs);
        if (p.parts) {
            p.cuts = p.bytes + 255 & ~(size_t)255;
            p.cut_part = p.cuts + 256 + (size_t)p.parts * sizeof(PagedCut) + 255 & ~(size_t)255;
            p.bytes = p.cut_part + (size_t)2 * p.parts * PT_TILE * (c.head_dim + 2) * 4;
        }
    }
    return p;
}

// A grid's threads are counted in 32 bits.
bool paged_attention_fits(const PagedCache& c, const PagedRows& r, int q_heads) {
    return (long long)r.rows * c.kv_heads * (((long long)r.max_tokens * (q_heads / c.kv_heads) + PT_TILE - 1) / PT_TILE) < 1 << 23;
}

hipError_t q38_paged_attention(const PagedAttnArgs& a, hipStream_t stream) {
    const int few = a.plan.few, G = a.q_heads / a.c.kv_heads;
    int joins = 0;
    if (a.plan.items) {
#define STREAM(HD, NT) hipLaunchKernelGGL((paged_stream_kernel<HD, NT, (HD > 128 ? 8 : 16)>), dim3(a.plan.items), dim3(256), 0, stream, a)
        switch (a.c.head_dim * 8 + few / 16) {
            case 64 * 8 + 1: STREAM(64, 1); break;
            case 64 * 8 + 2: STREAM(64, 2); break;
            case 64 * 8 + 3: STREAM(64, 3); break;
            case 64 * 8 + 4: STREAM(64, 4); break;
            case 128 * 8 + 1: STREAM(128, 1); break;
            case 128 * 8 + 2: STREAM(128, 2); break;
            case 128 * 8 + 3: STREAM(128, 3); break;
            case 128 * 8 + 4: STREAM(128, 4); break;
            case 256 * 8 + 1: STREAM(256, 1); break;
            case 256 * 8 + 2: STREAM(256, 2); break;
            case 256 * 8 + 3: STREAM(256, 3); break;
            default: return hipErrorInvalidValue;
        }
#undef STREAM
        const int heads = a.r.rows * a.c.kv_heads;
        joins = a.plan.slots ? heads * a.plan.joins : 0;
        if ((long long)a.r.max_tokens * G <= few) {
#define JOIN(E)                                                                                                              \
    do {                                                                                                                     \
        if (heads * 8 <= a.plan.cus)                                                                                         \
            hipLaunchKernelGGL((paged_join_kernel<E, 16>), dim3(joins), dim3(1024), 0, stream, a);                           \
        else                                                                                                                 \
            hipLaunchKernelGGL((paged_join_kernel<E, 4>), dim3(joins), dim3(256), 0, stream, a);                             \
    } while (0)
            switch (joins ? a.c.head_dim : 0) {
                case 64: JOIN(1); break;
                case 128: JOIN(2); break;
                case 256: JOIN(4); break;
            }
#undef JOIN
            return hipGetLastError();
        }
    }
#define TILES(HD)                                                                                                             \
    do {                                                                                                                     \
        hipLaunchKernelGGL((paged_tiles_kernel<HD>), dim3(a.plan.tiles), dim3(512), 0, stream, a);                           \
        if (joins || a.plan.parts)                                                                                           \
            hipLaunchKernelGGL((paged_join_tiles_kernel<HD>), dim3(joins + a.plan.parts * 8 * (HD / 32)), dim3(256), 0, stream, a, joins); \
    } while (0)
    switch (a.c.head_dim) {
        case 64: TILES(64); break;
        case 128: TILES(128); break;
        case 256: TILES(256); break;
        default: return hipErrorInvalidValue;
    }
#undef TILES
    return hipGetLastError();
}
