// Attention of one new token per sequence over a few pages of its cache.
//
// Each page keeps, per KV head and dim, its least and its largest key (mn, mx),
// rounded outwards to bf16.  No key of the page scores more with a query q than
//   bound = sum_d max(q_d mn_d, q_d mx_d) = sum_d max(q_d, 0) mx_d + min(q_d, 0) mn_d,
// and the pages with the largest bounds (of the largest among a KV head's query
// heads) are those that can matter most.  Three steps: bounds kept beside the
// pages as they are written; scores of all pages but the newest (which is always
// taken) and the choice among them; the one-token attention over a table of the
// chosen pages, one for each KV head.
//
// The choice is that of scores in 64 bits, where products of 16-bit numbers are
// exact and their sums nearly so: it does not depend on the order of evaluation, and
// equal bounds (pages that hold the same keys) go to the lower page.  Scores in 32
// bits, on the matrix cores, leave few pages undecided, those nearer to the last one
// taken than both may be off; these, 2 or 3 of 2047, are scored in 64 bits.  (All of
// them in 64 bits, by v_mfma_f64_16x16x4, took the scores of 16 sequences of up to
// 1024 pages from 14 us to 33, of one sequence of 2048 from 5 to 8.5.)
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "fkv_paged.h"

namespace fkv {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------------------
// bounds
// ---------------------------------------------------------------------------

struct BoundArgs {
    PageView pg;
    TableView table;
    PositionsView start;
    const int32_t* n_new;
    uint16_t* bounds;  // (n_pages, H, 2, D) bf16
    int32_t L, touched;  // pages that a sequence's tokens may lie in
    uint32_t units;
};

// The nearest bf16 number that is not above (UP: not below) x.
template <bool UP>
__device__ inline uint32_t outward(float x) {
    const uint32_t b = __float_as_uint(x), cut = b >> 16;
    const bool negative = b >> 31;
    return cut + ((b & 0xFFFFu) != 0 && negative != UP ? 1 : 0);
}

// A wave takes one page of one KV head: its rows by D / 8 (E4M3: D / 16) lanes
// each, 16 bytes a lane.  Bound by the keys' bytes, read once and not kept in the
// caches: a prompt of 64K tokens, 8 KV heads of 128 dims in bf16, 134 MB, takes 24 us,
// 5.6 TB/s (as other loads 28.5; a kernel that only reads them 20 to 24).
template <int D, int FMT>
__global__ void __launch_bounds__(256, FMT <= FKV_PAGES_BF16 ? 6 : 2) paged_bound_kernel(BoundArgs a) {
    constexpr bool k16 = FMT <= FKV_PAGES_BF16;
    constexpr int RB = k16 ? 2 * D : D, LPR = RB / 16, ROWS = 64 / LPR, N = k16 ? 8 : 16;
    const int lane = threadIdx.x & 63, chunk = lane % LPR;
    const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (unit >= a.units) return;
    const int h = unit % a.pg.H;
    const uint32_t rest = unit / a.pg.H;
    const int b = rest / a.touched, i = rest - b * a.touched;
    // tokens [first, last) of the sequence are new; pages from first's on
    int64_t first = position_of(a.start, b, 0);
    const int64_t cap = (int64_t)a.table.n * a.pg.page_size;
    int32_t n = a.L;
    if (a.n_new) n = min(max(a.n_new[b], 0), a.L);
    const int64_t last = min(first + n, cap);
    first = max(first, (int64_t)0);
    if (first >= last) return;
    const int64_t page0 = (first / a.pg.page_size + i) * a.pg.page_size;
    if (page0 >= last) return;
    const int32_t id = a.table.ids[b * a.table.stride + page0 / a.pg.page_size];
    if ((uint32_t)id >= (uint32_t)a.pg.n_pages) return;
    const int held = (int)min(last - page0, (int64_t)a.pg.page_size);
    const int64_t row0 = ((int64_t)id * a.pg.H + h) * a.pg.page_size;
    const char* keys = a.pg.k + row0 * RB;
    float lo[N], hi[N];
#pragma unroll
    for (int j = 0; j < N; j++) lo[j] = INFINITY, hi[j] = -INFINITY;
    constexpr int U = 8;  // rows a lane has in flight
    for (int r0 = lane / LPR; r0 < held; r0 += U * ROWS) {
        u4 w[U];
        uint32_t e[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int r = min(r0 + u * ROWS, held - 1);  // (a row again where there are no more)
            w[u] = __builtin_nontemporal_load((const u4*)(keys + (int64_t)r * RB + 16 * chunk));
            e[u] = k16 ? 0 : a.pg.k_exp[row0 + r];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            float x[N];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t v = w[u][j];
                if (FMT == FKV_PAGES_F16) {
                    x[2 * j] = h2f((uint16_t)v), x[2 * j + 1] = h2f((uint16_t)(v >> 16));
                } else if (FMT == FKV_PAGES_BF16) {
                    x[2 * j] = __uint_as_float(v << 16), x[2 * j + 1] = __uint_as_float(v & 0xFFFF0000u);
                } else {
                    const float s = exp_byte(e[u]);
                    const fkv_h2 p = e4m3x2_to_h2(v, false), q = e4m3x2_to_h2(v, true);
                    x[(4 * j) % N] = (float)p.x * s, x[(4 * j + 1) % N] = (float)p.y * s;
                    x[(4 * j + 2) % N] = (float)q.x * s, x[(4 * j + 3) % N] = (float)q.y * s;
                }
            }
            // (a NaN key counts as none)
#pragma unroll
            for (int j = 0; j < N; j++) lo[j] = fminf(lo[j], x[j]), hi[j] = fmaxf(hi[j], x[j]);
        }
    }
#pragma unroll
    for (int o = LPR; o < 64; o <<= 1)
#pragma unroll
        for (int j = 0; j < N; j++) lo[j] = fminf(lo[j], wave_xor(lo[j], o)), hi[j] = fmaxf(hi[j], wave_xor(hi[j], o));
    if (lane < 2 * LPR) {
        // lanes of the first row write the least keys, those of the second the largest
        uint16_t* out = a.bounds + (((int64_t)id * a.pg.H + h) * 2 + lane / LPR) * D + N * chunk;
#pragma unroll
        for (int j = 0; j < N; j += 8) {
            u4 w;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int x = j + 2 * k;
                w[k] = lane < LPR ? outward<false>(lo[x]) | outward<false>(lo[x + 1]) << 16
                                  : outward<true>(hi[x]) | outward<true>(hi[x + 1]) << 16;
            }
            *(u4*)(out + j) = w;
        }
    }
}

// ---------------------------------------------------------------------------
// scores
// ---------------------------------------------------------------------------

struct SparseArgs {
    PageView pg;
    TableView table;
    const uint16_t* bounds;
    const char* q;
    int64_t q_sb, q_sh;
    const int32_t* lens;
    float2* scores;     // workspace: (B, H, table.n) scores in 32 bits, sums of the terms' magnitudes
    uint64_t* exact;    // workspace: (B, H, table.n) scores in 64 bits, as numbers of the same order
    int32_t* chosen;    // workspace: (B * H, n_select) pages of the table for the attention, id * H + h
    int32_t* len;       // workspace: (B * H) tokens in them
    int32_t* selected;  // result (B, H, n_result) or NULL
    int32_t lens_add, Hq, G, n_select, n_result;
};

__device__ inline int32_t length_of(const SparseArgs& a, int b) {
    const int64_t n = (int64_t)a.lens[b] + a.lens_add, cap = (int64_t)a.table.n * a.pg.page_size;
    return (int32_t)(n < 0 ? 0 : n > cap ? cap : n);
}
// Pages that hold a sequence's tokens.
__device__ inline int32_t pages_of(const SparseArgs& a, int32_t len) {
    return (int32_t)(((int64_t)len + a.pg.page_size - 1) >> (31 - __builtin_clz((unsigned)a.pg.page_size)));
}

__device__ inline f4 mfma16(u4 x, u4 y, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), c, 0, 0, 0);
}
// Signs and magnitudes of two bf16 numbers: those that are positive, those that are
// negative (0 in the others' place).
__device__ inline uint32_t positive(uint32_t w) {
    const uint32_t s = (w >> 15) & 0x00010001u;
    return w & ~((s << 16) - s);
}
__device__ inline uint32_t negative(uint32_t w) {
    const uint32_t s = (w >> 15) & 0x00010001u;
    return w & ((s << 16) - s);
}

// The largest over a row of 16 lanes, in all of them.
__device__ inline float row_max(float v) {
    v = fmaxf(v, dpp_f32<kDppXor1>(v));
    v = fmaxf(v, dpp_f32<kDppXor2>(v));
    v = fmaxf(v, dpp_f32<0x141>(v));     // row_half_mirror
    return fmaxf(v, dpp_f32<0x140>(v));  // row_mirror
}

// Bounds of 16 pages' scores with 16 query heads, by v_mfma_f32_16x16x32: rows are
// pages, columns heads.  An fp16 query is the sum of two bf16 numbers, of which the
// second is in the column eight to the right: 8 heads at a time.
// Bound by a wave's latencies: the length and ids, 8 KB of bounds, some 200 vector
// instructions.  35 MB in 12 us (16 ragged sequences, 8 KV heads), 8 MB in 5 us.
template <int D, bool BF>
__global__ void __launch_bounds__(256) page_score_kernel(SparseArgs a) {
    constexpr int NJ = D / 32, NH = BF ? 16 : 8;
    const int lane = threadIdx.x & 63, c = lane & 15, kq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.z, h = blockIdx.x;
    int32_t p0 = ((int32_t)blockIdx.y * 4 + wave) * 16;
    const int32_t* ids = a.table.ids + b * a.table.stride;
    int32_t id = ids[min(p0 + c, a.table.n - 1)];        // (asked for together with the length)
    const int32_t n = pages_of(a, length_of(a, b)) - 1;  // (the newest page needs no score)
    if (n < a.n_select) return;                          // (all pages are taken)
    u4 up[NJ], down[NJ];  // the queries' positive and negative elements
    auto queries = [&](int g0) {
        const int g = g0 + (c & (NH - 1));
        const char* row = a.q + 2 * (b * a.q_sb + (int64_t)(h * a.G + (g < a.G ? g : 0)) * a.q_sh + 8 * kq);
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const u4 q = *(const u4*)(row + 64 * j);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t part = q[i];
                if (!BF) {
                    const float x = h2f((uint16_t)q[i]), y = h2f((uint16_t)(q[i] >> 16));
                    const uint32_t u = __float_as_uint(x) & 0xFFFF0000u, v = __float_as_uint(y) & 0xFFFF0000u;
                    const float x2 = x - __uint_as_float(u), y2 = y - __uint_as_float(v);
                    part = c < NH ? u >> 16 | v : __float_as_uint(x2) >> 16 | (__float_as_uint(y2) & 0xFFFF0000u);
                }
                up[j][i] = positive(part), down[j][i] = negative(part);
            }
        }
    };
    if (a.G <= NH) queries(0);
    for (const int32_t hop = (int32_t)gridDim.y * 64; p0 < n; p0 += hop) {
        const bool held = (uint32_t)id < (uint32_t)a.pg.n_pages;
        const uint16_t* box = a.bounds + ((int64_t)(held ? id : 0) * a.pg.H + h) * 2 * D + 8 * kq;
        u4 mn[NJ], mx[NJ];
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            mn[j] = *(const u4*)(box + 32 * j);
            mx[j] = *(const u4*)(box + D + 32 * j);
        }
        id = ids[min(p0 + hop + c, a.table.n - 1)];
        // the largest over the heads (NaN counts as above all), and of the magnitudes' sums
        f4 best = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, size = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int g0 = 0; g0 < a.G; g0 += NH) {
            if (a.G > NH) queries(g0);
            f4 s = {0.0f, 0.0f, 0.0f, 0.0f}, m = s;
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                s = mfma16(mx[j], up[j], s);
                m = mfma16(mx[j] & 0x7FFF7FFFu, up[j], m);
                s = mfma16(mn[j], down[j], s);
                m = mfma16(mn[j] & 0x7FFF7FFFu, down[j] & 0x7FFF7FFFu, m);
            }
            if (!BF) {
#pragma unroll
                for (int i = 0; i < 4; i++) s[i] += dpp_f32<0x128>(s[i]), m[i] += dpp_f32<0x128>(m[i]);  // row_ror:8
            }
            if (g0 + (c & (NH - 1)) < a.G) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    best[i] = s[i] != s[i] ? INFINITY : fmaxf(best[i], s[i]);
                    size[i] = m[i] != m[i] ? INFINITY : fmaxf(size[i], m[i]);
                }
            }
        }
        // s[i] is page p0 + 4 (lane / 16) + i with head lane % 16
        const uint64_t none = __ballot(!held);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            best[i] = row_max(best[i]), size[i] = row_max(size[i]);
            const int32_t page = p0 + 4 * kq + i;
            if (c == i && page < n)
                a.scores[((int64_t)b * a.pg.H + h) * a.table.n + page] =
                    (none >> (4 * kq + i)) & 1 ? make_float2(-INFINITY, 0.0f) : make_float2(best[i], size[i]);
        }
    }
}

// ---------------------------------------------------------------------------
// choice
// ---------------------------------------------------------------------------

// A score as an unsigned number of the same order (-0 as 0).
__device__ inline uint64_t order_of(double s) {
    const uint64_t u = __builtin_bit_cast(uint64_t, s + 0.0);
    return u >> 63 ? ~u : u | 1ull << 63;
}
// Is key below, at or above the prefix in its bits from `shift` on?
__device__ inline int compare_from(uint64_t key, uint64_t prefix, int shift) {
    if (shift > 63) return 0;
    const uint64_t k = key >> shift, p = prefix >> shift;
    return k < p ? -1 : k > p ? 1 : 0;
}

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kHeld = 8192;  // pages whose scores and ids are held in the LDS
constexpr int kBins = 512, kFew = 64;
constexpr int kList = 1024;  // undecided pages that are ranked one against all

struct ChoiceLds {
    uint32_t bins[kBins];
    float ends[3][kWaves];
    uint64_t keys[2][kWaves];
    int32_t digit, above, inside, counts[2][kWaves];
};

// Of 64 lanes, each with N counts that follow the ones of the lane below: the place
// in whose count the need-th lies, by the lane that has it.
template <int N, typename FOUND>
__device__ inline void find_place(const uint32_t (&own)[N], int lane, uint32_t need, FOUND found) {
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < N; i++) mine += own[i];
    uint32_t before = sum_up_to(mine) - mine;
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (before < need && before + own[i] >= need) found(N * lane + i, before, own[i]);
        before += own[i];
    }
}

// The bits of the need-th largest of the keys key(i), i < n, of which in(i) says
// whether it is one, from the first bit in which they differ, eight a round: keys
// above prefix from bit `shift` on are among the largest, and of those equal to it
// `need` are.
template <typename KEY, typename IN>
__device__ inline void find_largest(ChoiceLds& lds, int32_t n, KEY key, IN in, uint64_t& prefix, int& shift, int32_t& need) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint64_t lo = ~0ull, hi = 0;
    for (int32_t i = tid; i < n; i += kThreads)
        if (in(i)) lo = min(lo, key(i)), hi = max(hi, key(i));
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        lo = min(lo, (uint64_t)wave_xor((unsigned long long)lo, o));
        hi = max(hi, (uint64_t)wave_xor((unsigned long long)hi, o));
    }
    if (lane == 0) lds.keys[0][wave] = lo, lds.keys[1][wave] = hi;
    if (tid < 256) lds.bins[tid] = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; w++) lo = min(lo, lds.keys[0][w]), hi = max(hi, lds.keys[1][w]);
    shift = lo >= hi ? 0 : 64 - __builtin_clzll(lo ^ hi);
    prefix = hi;  // (the bits from `shift` on are all keys')
    while (shift > 0) {
        const int next = max(0, shift - 8);
        for (int32_t i = tid; i < n; i += kThreads)
            if (in(i)) {
                const uint64_t k = key(i);
                if (compare_from(k, prefix, shift) == 0) atomicAdd(&lds.bins[(k >> next) & ((1u << (shift - next)) - 1)], 1u);
            }
        __syncthreads();
        if (wave == 0) {
            // from the largest digit down; lane l has digits 255 - 4 l to 252 - 4 l
            uint32_t own[4];
#pragma unroll
            for (int i = 0; i < 4; i++) own[i] = lds.bins[255 - 4 * lane - i], lds.bins[255 - 4 * lane - i] = 0;
            find_place(own, lane, (uint32_t)need, [&](int at, uint32_t above, uint32_t inside) {
                lds.digit = 255 - at, lds.above = (int32_t)above, lds.inside = (int32_t)inside;
            });
        }
        __syncthreads();
        const uint64_t mask = ((1ull << (shift - next)) - 1) << next;
        prefix = (prefix & ~mask) | (uint64_t)lds.digit << next;
        need -= lds.above;
        shift = next;
        if (lds.inside == need) break;  // (all that have these bits are taken)
    }
    __syncthreads();
}

// One workgroup per (sequence, KV head): its n_select - 1 pages with the largest
// scores, and the newest one, in order.  A chain of latencies, whatever the number
// of rows: for 2047 pages some 9 us, of which the loads are 2, the part of the
// scores that has the last page 1.5, what is undecided 2, the result 1.  (A search
// of the last score's bits, eight at a time, and then of the undecided ones: 16.)
template <int D, bool BF>
__global__ void __launch_bounds__(kThreads) page_choice_kernel(SparseArgs a) {
    __shared__ ChoiceLds lds;
    __shared__ float held[kHeld];
    __shared__ int32_t held_ids[kHeld], list[kList], listed;
    __shared__ uint64_t ranks[kList];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row = blockIdx.x, b = row / a.pg.H, h = row - b * a.pg.H;
    float2* scores = a.scores + (int64_t)row * a.table.n;
    uint64_t* exact = a.exact + (int64_t)row * a.table.n;
    const int32_t* ids = a.table.ids + b * a.table.stride;
    // (a first page of each thread, asked for together with the length)
    const int32_t first = min(tid, a.table.n - 1);
    const float2 score0 = first >= 0 ? scores[first] : make_float2(0.0f, 0.0f);
    const int32_t id0 = first >= 0 ? ids[first] : 0;
    const int32_t len = length_of(a, b), pages = pages_of(a, len), n = pages - 1;
    const int32_t want = min(a.n_select - 1, max(n, 0));
    const bool all = want >= n, in_lds = n <= kHeld;
    // pages above `over` are taken, those below `under` are not, others are undecided
    float over = INFINITY, under = -INFINITY;
    bool exactly = false;    // if all are taken, or else those whose exact scores are above
    uint64_t prefix = 0;     // this from bit `shift` on, and the first `need` that are equal to it
    int shift = 0;
    int32_t need = 0;
    auto score = [&](int32_t i) { return in_lds ? held[i] : scores[i].x; };
    auto undecided = [&](float s) { return !(s > over) && !(s < under); };
    if (!all && want > 0) {
        // a score or a size that is not finite says nothing of any page: all in 64 bits then
        float size = 0.0f, hi = -INFINITY, lo = INFINITY;
        int32_t there = 0;  // pages that have a score (those that are not there have -inf; lane 0 counts the wave's)
        for (int32_t i = tid; i < n; i += kThreads) {
            const float2 s = i == tid ? score0 : scores[i];
            there += __popcll(__ballot(s.x > -INFINITY));
            if (in_lds) held[i] = s.x, held_ids[i] = i == tid ? id0 : ids[i];
            size = fmaxf(size, s.x < INFINITY ? s.y : INFINITY);
            hi = fmaxf(hi, s.x);
            if (s.x > -INFINITY) lo = fminf(lo, s.x);
        }
        size = row_max(size), hi = row_max(hi), lo = -row_max(-lo);
#pragma unroll
        for (int o = 16; o <= 32; o <<= 1)
            size = fmaxf(size, wave_xor(size, o)), hi = fmaxf(hi, wave_xor(hi, o)), lo = fminf(lo, wave_xor(lo, o));
        if (lane == 0) lds.ends[0][wave] = size, lds.ends[1][wave] = hi, lds.ends[2][wave] = lo, lds.counts[1][wave] = there;
        if (tid < kBins) lds.bins[tid] = 0;
        if (tid == 0) listed = 0;
        __syncthreads();
        {
            const int w = lane & 15;
            size = row_max(lds.ends[0][w]), hi = row_max(lds.ends[1][w]), lo = -row_max(-lds.ends[2][w]);
            there = (int32_t)row_sum((uint32_t)lds.counts[1][w]);
        }
        if (size < INFINITY) {
            // A score in 32 bits is a sum of 4 D exact products at most: off by 2^-14 of
            // their magnitudes' sum (4 D roundings of 2^-23), and of what flushed denormals
            // leave.  Pages further apart than twice that are in order.
            const float off = 2.0f * (size * 1.01f * 0x1p-14f + 1e-25f);
            // The last one taken lies in [lo, hi], or is below all of it (a page that is
            // not there): 510 parts of it, until few pages are in the part that has it.
            // (The first bin is what is above, the last what is below; no page is in either at
            // the first round.)  A part's ends are off by some 2^-22 of hi - lo and of hi, which
            // the slack of 2^-6 of `off` holds: hi - lo and |hi| are 2 sizes at most.
            int32_t inside = n;
            while (inside > kFew && hi - lo > off) {
                const float step = (hi - lo) * (1.0f / (kBins - 2)), inv = (kBins - 2) / (hi - lo);
                for (int32_t i = tid; i < n; i += kThreads) {
                    const float s = score(i);
                    if (s >= lo) atomicAdd(&lds.bins[s > hi ? 0 : 1 + min((int)((hi - s) * inv), kBins - 3)], 1u);
                }
                __syncthreads();
                if (wave == 0) {
                    uint32_t own[kBins / 64];
#pragma unroll
                    for (int i = 0; i < kBins / 64; i++) own[i] = lds.bins[kBins / 64 * lane + i], lds.bins[kBins / 64 * lane + i] = 0;
                    if (lane == 63) own[kBins / 64 - 1] = 0x40000000;  // (all that are left)
                    find_place(own, lane, (uint32_t)want, [&](int at, uint32_t, uint32_t in) { lds.digit = at, lds.inside = (int32_t)in; });
                }
                __syncthreads();
                const int at = __builtin_amdgcn_readfirstlane(lds.digit);
                const float slack = off * 0x1p-6f, top = hi;
                over = at == 0 ? INFINITY : top - (at - 1) * step + (off + slack);
                under = at == kBins - 1 ? -INFINITY : top - at * step - (off + slack);
                if (at == 0 || at == kBins - 1) break;
                inside = lds.inside;
                hi = top - (at - 1) * step + slack, lo = top - at * step - slack;
            }
            // Few pages, or all within `off`: undecided, and with them those that are not there
            // where the others are not enough.
            if (over == INFINITY && under == -INFINITY) over = hi + 1.02f * off, under = there >= want ? lo - 1.02f * off : -INFINITY;
        }
        // how many are above, and the undecided ones
        int32_t up = 0, at = 0;
        for (int32_t i = tid; i < n; i += kThreads) {
            const float s = score(i);
            up += __popcll(__ballot(s > over));
            if (undecided(s)) {
                const int32_t slot = atomicAdd(&listed, 1);
                if (slot < kList) list[slot] = i, ranks[slot] = 0;
            }
        }
        if (lane == 0) lds.counts[0][wave] = up;
        __syncthreads();
        up = (int32_t)row_sum((uint32_t)lds.counts[0][lane & 15]), at = listed;
        need = want - up;
        if (at != need) {
            // the score of a page with one of the heads in 64 bits, by 16 lanes
            const int c = lane & 15;
            auto score64 = [&](int32_t page, int g) {
                const int32_t id = in_lds ? held_ids[page] : ids[page];
                const bool there = (uint32_t)id < (uint32_t)a.pg.n_pages, mine = c < D / 8;
                const uint16_t* box = a.bounds + ((int64_t)(there ? id : 0) * a.pg.H + h) * 2 * D + 8 * c;
                const u4 none = {0, 0, 0, 0}, mn = mine ? *(const u4*)box : none, mx = mine ? *(const u4*)(box + D) : none;
                const u4 x = mine ? *(const u4*)(a.q + 2 * (b * a.q_sb + (int64_t)(h * a.G + g) * a.q_sh) + 16 * c) : none;
                double s = 0.0, t = 0.0;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint16_t e = (uint16_t)(x[i / 2] >> 16 * (i & 1));
                    const double y = BF ? bf2f(e) : h2f(e);
                    s += fmin(y, 0.0) * (double)bf2f((uint16_t)(mn[i / 2] >> 16 * (i & 1)));
                    t += fmax(y, 0.0) * (double)bf2f((uint16_t)(mx[i / 2] >> 16 * (i & 1)));
                }
                s = row_sum(s + t);
                return order_of(!there ? -(double)INFINITY : s != s ? (double)INFINITY : s);
            };
            if (at <= kList) {
                // (the list is in any order; what is made of it is not)
                for (int i = tid >> 4; i < at * a.G; i += kThreads / 16) {
                    const int slot = i / a.G;
                    const uint64_t s = score64(list[slot], i - slot * a.G);
                    if (c == 0) atomicMax((unsigned long long*)&ranks[slot], (unsigned long long)s);
                }
                __syncthreads();
                for (int i = tid; i < at; i += kThreads) {
                    const uint64_t s = ranks[i];
                    const int32_t page = list[i];
                    int32_t better = 0;
                    for (int k = 0; k < at; k++) better += ranks[k] > s || (ranks[k] == s && list[k] < page);
                    const float settled = better < need ? INFINITY : -INFINITY;
                    if (in_lds) held[page] = settled;
                    else scores[page].x = settled;
                }
                over = fminf(over, 3e38f), under = INFINITY;
            } else {
                exactly = true;
                for (int32_t i = tid >> 4; i < n; i += kThreads / 16)
                    if (undecided(score(i))) {
                        uint64_t best = 0;
                        for (int g = 0; g < a.G; g++) best = max(best, score64(i, g));
                        if (c == 0) exact[i] = best;
                    }
            }
            __syncthreads();
            if (exactly)
                find_largest(lds, n, [&](int32_t i) { return exact[i]; },
                             [&](int32_t i) { return undecided(score(i)); }, prefix, shift, need);
        }
    }
    int32_t* chosen = a.chosen + (int64_t)row * a.n_select;
    int32_t* selected = a.selected ? a.selected + (int64_t)row * a.n_result : nullptr;
    auto take = [&](int32_t slot, int32_t page) {
        const int32_t id = !all && in_lds && page < n ? held_ids[page] : ids[page];
        chosen[slot] = (uint32_t)id < (uint32_t)a.pg.n_pages ? id * a.pg.H + h : -1;
        if (selected) selected[slot] = page;
    };
    if (all) {
        for (int32_t i = tid; i < n; i += kThreads) take(i, i);
    } else if (want > 0) {
        // each wave has neighbouring pages: counted first, then in their places
        const int32_t per = (n + kThreads - 1) / kThreads * 64, p1 = min(n, (wave + 1) * per);
        auto verdict = [&](int32_t i) {
            if (i >= p1) return -1;
            const float s = score(i);
            if (s > over) return 1;
            if (!undecided(s)) return -1;
            return exactly ? compare_from(exact[i], prefix, shift) : 1;
        };
        int32_t ups = 0, ats = 0;
        for (int32_t p0 = wave * per; p0 < p1; p0 += 64) {
            const int cmp = verdict(p0 + lane);
            ups += __popcll(__ballot(cmp > 0)), ats += __popcll(__ballot(cmp == 0));
        }
        if (lane == 0) lds.counts[0][wave] = ups, lds.counts[1][wave] = ats;
        __syncthreads();
        ups = (int32_t)row_sum((lane & 15) < wave ? (uint32_t)lds.counts[0][lane & 15] : 0);
        ats = (int32_t)row_sum((lane & 15) < wave ? (uint32_t)lds.counts[1][lane & 15] : 0);
        for (int32_t p0 = wave * per; p0 < p1; p0 += 64) {
            const int cmp = verdict(p0 + lane);
            const uint64_t up = __ballot(cmp > 0), at = __ballot(cmp == 0), below = (1ull << lane) - 1;
            const int32_t u = ups + __popcll(up & below), t = ats + __popcll(at & below);
            // (of equal scores the first `need`)
            if (cmp > 0 || (cmp == 0 && t < need)) take(u + min(t, need), p0 + lane);
            ups += __popcll(up), ats += __popcll(at);
        }
    }
    if (tid == 0) {
        if (pages > 0) take(want, n);
        a.len[row] = pages > 0 ? want * a.pg.page_size + len - n * a.pg.page_size : 0;
    }
    if (selected)
        for (int32_t i = (pages > 0 ? want + 1 : 0) + tid; i < a.n_result; i += kThreads) selected[i] = -1;
}

// ---------------------------------------------------------------------------
// launch
// ---------------------------------------------------------------------------

struct SparsePlan {
    int64_t exact_at, chosen_at, len_at, attn_at, attn_bytes, bytes;
};
// The chosen pages as the one-token attention sees them: a sequence of one KV
// head for each (sequence, head), and a page of one head for each (page, head).
static fkv_pages by_head(const fkv_pages* p) {
    fkv_pages r = *p;
    r.n_pages = p->n_pages * p->H;
    r.H = 1;
    return r;
}

static int check_sparse(const char* who, const fkv_pages* p, int32_t Hq, int32_t B, int32_t n_table, int32_t n_select) {
    const std::string w = who;
    if (int e = check_pages(who, p)) return e;
    if (B < 0 || (int64_t)B * p->H > 4096) return set_error(w + ": at most 4096 sequences times KV heads");
    if (Hq < 1 || Hq % p->H) return set_error(w + ": query heads must be a multiple of the KV heads");
    if (n_table < 0 || (int64_t)n_table * p->page_size > kMostTokens)
        return set_error(w + ": more than 2^31 tokens a sequence");
    if (n_select < 1 || (int64_t)n_select * p->page_size > kMostTokens)
        return set_error(w + ": at least one page must be selected, and less than 2^31 tokens");
    if ((int64_t)p->n_pages * p->H > 0x7FFFFFFF) return set_error(w + ": more than 2^31 pages times KV heads");
    // (the limits of the attention, whose tiles are 128 tokens of 16 heads)
    const int64_t rows = (int64_t)B * p->H * cdiv(Hq / p->H, 16);
    if (rows >= 1 << 24 || rows * (cdiv((int64_t)n_select * p->page_size, 128) + 1) > 0x7FFFFFFF)
        return set_error(w + ": the selected pages hold more than 2^31 tiles of 128 tokens over all heads");
    return FKV_OK;
}

// (n_select pages at most, whatever the lengths are)
static int64_t most_tokens(const fkv_pages* p, int32_t n_select, int64_t max_len) {
    return std::min<int64_t>((int64_t)n_select * p->page_size, max_len);
}

// A sequence has no more pages than its table's row.
static int32_t pages_to_select(int32_t n_table, int32_t n_select) { return std::min(n_select, std::max(n_table, 1)); }

static SparsePlan plan_sparse(const fkv_pages* p, int32_t Hq, int32_t B, int32_t n_table, int32_t n_select, int64_t max_len) {
    SparsePlan r;
    n_select = pages_to_select(n_table, n_select);
    const fkv_pages one = by_head(p);
    const int64_t rows = (int64_t)B * p->H;
    r.exact_at = round_up(8 * rows * n_table, 256);
    r.chosen_at = 2 * r.exact_at;
    r.len_at = r.chosen_at + round_up(4 * rows * n_select, 256);
    r.attn_at = r.len_at + round_up(4 * rows, 256);
    r.attn_bytes = fkv_paged_attn_workspace(&one, Hq / p->H, (int32_t)rows, most_tokens(p, n_select, max_len));
    r.bytes = r.attn_at + std::max<int64_t>(r.attn_bytes, 0);
    return r;
}

}  // namespace fkv

using namespace fkv;

extern "C" {

int fkv_paged_bounds(const fkv_pages* pages, void* bounds, int32_t B, int32_t L, const int32_t* table, int32_t n_table,
                     int64_t table_stride, const fkv_positions* start, const int32_t* n_new, void* stream) {
    const char* w = "fkv_paged_bounds";
    if (int e = check_pages(w, pages)) return e;
    if (int e = check_table(w, table, n_table, table_stride, B)) return e;
    if (L < 0) return set_error(std::string(w) + ": negative count of tokens");
    if (!start || start->per_token) return set_error(std::string(w) + ": start is one position per sequence");
    if (!bounds || (uintptr_t)bounds & 15) return set_error(std::string(w) + ": bounds must be 16-byte aligned device memory");
    if (B == 0 || L == 0 || n_table == 0) return FKV_OK;
    BoundArgs a;
    a.pg = page_view(pages);
    a.table = TableView{table, table_stride, n_table};
    a.start = PositionsView{start->data, start->stride_b, start->stride_l, start->base, start->is64, 0};
    a.n_new = n_new;
    a.bounds = (uint16_t*)bounds;
    a.L = L;
    // (L tokens that begin at a page's last one)
    a.touched = (int32_t)std::min<int64_t>(((int64_t)L + pages->page_size - 2) / pages->page_size + 1, n_table);
    const int64_t units = (int64_t)B * a.touched * pages->H;
    if (units > 0x7FFFFFF0) return set_error(std::string(w) + ": more than 2^31 pages times KV heads");
    a.units = (uint32_t)units;
    hipStream_t s = (hipStream_t)stream;
    auto go = [&](auto kernel) { return start_kernel(w, kernel, (uint32_t)cdiv(units, 4), 256, s, a); };
    if (pages->D == 64) {
        if (pages->format == FKV_PAGES_F16) return go(paged_bound_kernel<64, FKV_PAGES_F16>);
        if (pages->format == FKV_PAGES_BF16) return go(paged_bound_kernel<64, FKV_PAGES_BF16>);
        return go(paged_bound_kernel<64, FKV_PAGES_FP8>);
    }
    if (pages->format == FKV_PAGES_F16) return go(paged_bound_kernel<128, FKV_PAGES_F16>);
    if (pages->format == FKV_PAGES_BF16) return go(paged_bound_kernel<128, FKV_PAGES_BF16>);
    return go(paged_bound_kernel<128, FKV_PAGES_FP8>);
}

int64_t fkv_paged_attn_sparse_workspace(const fkv_pages* pages, int32_t Hq, int32_t B, int32_t n_table, int32_t n_select,
                                        int64_t max_len) {
    if (int e = check_sparse("fkv_paged_attn_sparse_workspace", pages, Hq, B, n_table, n_select)) return e;
    if (max_len < 0) return set_error("fkv_paged_attn_sparse_workspace: negative max_len");
    return plan_sparse(pages, Hq, B, n_table, n_select, max_len).bytes;
}

int fkv_paged_attn_sparse(const fkv_pages* pages, const void* bounds, const fkv_rows* query, int32_t q_dtype, int32_t Hq,
                          int32_t B, const int32_t* table, int32_t n_table, int64_t table_stride, const int32_t* lens,
                          int32_t lens_add, int64_t max_len, int32_t n_select, float scale, void* out, float* lse,
                          int32_t* selected, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* w = "fkv_paged_attn_sparse";
    if (int e = check_sparse(w, pages, Hq, B, n_table, n_select)) return e;
    if (int e = check_table(w, table, n_table, table_stride, B)) return e;
    if (max_len < 0) return set_error(std::string(w) + ": negative max_len");
    if (!(std::isfinite(scale) && scale >= 0.0f))
        return set_error(std::string(w) + ": scale must be finite and not negative (pages are chosen by their largest scores)");
    if (q_dtype != FKV_F16 && q_dtype != FKV_BF16) return set_error(std::string(w) + ": queries must be fp16 or bf16");
    if (pages->format <= FKV_PAGES_BF16 && (q_dtype == FKV_BF16) != (pages->format == FKV_PAGES_BF16))
        return set_error(std::string(w) + ": queries must have the 16-bit pages' type");
    if (B == 0) return FKV_OK;
    if (!query || !query->data || !out || !lens) return set_error(std::string(w) + ": NULL argument");
    if (!bounds || (uintptr_t)bounds & 15) return set_error(std::string(w) + ": bounds must be 16-byte aligned device memory");
    if (((uintptr_t)query->data | (uintptr_t)out | (uintptr_t)workspace) & 15 || (query->stride_b | query->stride_h) & 7)
        return set_error(std::string(w) + ": query, out and workspace must be 16-byte aligned, query strides multiples of 8");
    // (the attention takes each KV head's queries as a sequence's, a stride apart)
    if (B > 1 && pages->H > 1 && query->stride_b != Hq * query->stride_h)
        return set_error(std::string(w) + ": heads of neighbouring sequences must follow one another");
    const SparsePlan p = plan_sparse(pages, Hq, B, n_table, n_select, max_len);
    if (p.attn_bytes < 0) return FKV_EINVAL;
    if (!workspace || workspace_bytes < p.bytes)
        return set_error(std::string(w) + ": workspace of " + std::to_string(p.bytes) + " bytes needed");
    SparseArgs a;
    a.pg = page_view(pages);
    a.table = TableView{table, table_stride, n_table};
    a.bounds = (const uint16_t*)bounds;
    a.q = (const char*)query->data;
    a.q_sb = query->stride_b;
    a.q_sh = query->stride_h;
    a.lens = lens;
    a.scores = (float2*)workspace;
    a.exact = (uint64_t*)((char*)workspace + p.exact_at);
    a.chosen = (int32_t*)((char*)workspace + p.chosen_at);
    a.len = (int32_t*)((char*)workspace + p.len_at);
    a.selected = selected;
    a.lens_add = lens_add;
    a.Hq = Hq;
    a.G = Hq / pages->H;
    a.n_result = n_select;
    a.n_select = n_select = pages_to_select(n_table, n_select);
    hipStream_t s = (hipStream_t)stream;
    const fkv_pages one = by_head(pages);
    const int32_t rows = B * pages->H;
    fkv_rows q = *query;
    if (pages->H > 1) q.stride_b = (int64_t)a.G * query->stride_h;
    auto attend = [&](int32_t seqs) {
        return fkv_paged_attn(&one, &q, q_dtype, a.G, seqs, a.chosen, n_select, n_select, a.len, 0,
                              most_tokens(pages, n_select, max_len), scale, out, lse, (char*)workspace + p.attn_at,
                              std::max<int64_t>(p.attn_bytes, 0), stream);
    };
    const RowsShape heads{B, Hq, 1, pages->D, 2};
    const fkv_rows result{out, (int64_t)Hq * pages->D, pages->D, 0};
    if (int e = check_apart(w, "out, which is not the query, and the query", &result, heads, query, heads, true)) return e;
    const int64_t most = std::min<int64_t>(max_len, (int64_t)n_table * pages->page_size);
    const int64_t scored = cdiv(most, pages->page_size) - 1;
    // (about 768 workgroups, three a CU, of 64 pages at a time, neighbours of other heads,
    // which have as many pages to score; for 16 sequences of up to 1024
    // pages 512 take 0.9 us more, 1024 2)
    const int64_t groups = std::max<int64_t>(1, std::min<int64_t>(cdiv(scored, 64), cdiv(768, rows)));
    const dim3 grid(pages->H, (uint32_t)groups, B);
    auto choose = [&](auto score, auto choice) {
        if (n_table > n_select)  // (else all pages are taken)
            if (int e = start_kernel(w, score, grid, 256, s, a)) return e;
        return start_kernel(w, choice, (uint32_t)rows, kThreads, s, a);
    };
    auto by_dims = [&](auto d) {
        constexpr int D = decltype(d)::value;
        if (q_dtype == FKV_BF16) return choose(page_score_kernel<D, true>, page_choice_kernel<D, true>);
        return choose(page_score_kernel<D, false>, page_choice_kernel<D, false>);
    };
    const int e = pages->D == 64 ? by_dims(std::integral_constant<int, 64>{}) : by_dims(std::integral_constant<int, 128>{});
    if (e) return e;
    return attend(rows);
}

}  // extern "C"
