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
// Scores are computed in 64 bits: products of 16-bit numbers are exact there and
// their sums nearly so, so the choice does not depend on the order of evaluation,
// and equal bounds (pages that hold the same keys) go to the lower page.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "fkv_paged.h"

namespace fkv {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef double d4 __attribute__((ext_vector_type(4)));

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
// each, 16 bytes a lane.
template <int D, int FMT>
__global__ void __launch_bounds__(256) paged_bound_kernel(BoundArgs a) {
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
    constexpr int U = 4;  // rows a lane has in flight
    for (int r0 = lane / LPR; r0 < held; r0 += U * ROWS) {
        u4 w[U];
        uint32_t e[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int r = min(r0 + u * ROWS, held - 1);  // (a row again where there are no more)
            w[u] = *(const u4*)(keys + (int64_t)r * RB + 16 * chunk);
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
    double* scores;     // workspace: (B, H, table.n)
    int32_t* chosen;    // workspace: (B * H, n_select) pages of the table for the attention, id * H + h
    int32_t* len;       // workspace: (B * H) tokens in them
    int32_t* selected;  // result (B, H, n_select) or NULL
    int32_t lens_add, Hq, G, n_select;
};

__device__ inline int32_t length_of(const SparseArgs& a, int b) {
    const int64_t n = (int64_t)a.lens[b] + a.lens_add, cap = (int64_t)a.table.n * a.pg.page_size;
    return (int32_t)(n < 0 ? 0 : n > cap ? cap : n);
}
// Pages that hold a sequence's tokens.
__device__ inline int32_t pages_of(const SparseArgs& a, int32_t len) {
    return (int32_t)(((int64_t)len + a.pg.page_size - 1) >> (31 - __builtin_clz((unsigned)a.pg.page_size)));
}

// Bounds of 16 pages' scores with 16 query heads, by v_mfma_f64_16x16x4: rows are
// pages, columns heads, four dims a step.  A lane has 8 neighbouring dims of its
// page in a load, and takes the steps in an order in which these are its own.
template <int D, bool BF>
__global__ void __launch_bounds__(256) page_score_kernel(SparseArgs a) {
    const int lane = threadIdx.x & 63, c = lane & 15, kq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.z, h = blockIdx.y;
    const int32_t n = pages_of(a, length_of(a, b)) - 1;  // (the newest page needs no score)
    if (n < a.n_select) return;                          // (all pages are taken)
    for (int32_t p0 = ((int32_t)blockIdx.x * 4 + wave) * 16; p0 < n; p0 += (int32_t)gridDim.x * 64) {
        const int32_t at = min(p0 + c, n - 1);
        const int32_t id = a.table.ids[b * a.table.stride + at];
        const bool held = (uint32_t)id < (uint32_t)a.pg.n_pages;
        const uint16_t* box = a.bounds + ((int64_t)(held ? id : 0) * a.pg.H + h) * 2 * D + 8 * kq;
        u4 mn[D / 32], mx[D / 32];
#pragma unroll
        for (int j = 0; j < D / 32; j++) {
            mn[j] = *(const u4*)(box + 32 * j);
            mx[j] = *(const u4*)(box + D + 32 * j);
        }
        double best[4];
#pragma unroll
        for (int i = 0; i < 4; i++) best[i] = -INFINITY;
        for (int g0 = 0; g0 < a.G; g0 += 16) {
            const bool real = g0 + c < a.G;
            const char* row = a.q + 2 * (b * a.q_sb + (int64_t)(h * a.G + g0 + (real ? c : 0)) * a.q_sh + 8 * kq);
            d4 s = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < D / 32; j++) {
                const u4 q = *(const u4*)(row + 64 * j);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint16_t w = (uint16_t)(q[e / 2] >> (16 * (e & 1)));
                    const float x = BF ? bf2f(w) : h2f(w);
                    const float lo = bf2f((uint16_t)(mn[j][e / 2] >> (16 * (e & 1))));
                    const float hi = bf2f((uint16_t)(mx[j][e / 2] >> (16 * (e & 1))));
                    s = __builtin_amdgcn_mfma_f64_16x16x4f64((double)lo, (double)fminf(x, 0.0f), s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f64_16x16x4f64((double)hi, (double)fmaxf(x, 0.0f), s, 0, 0, 0);
                }
            }
            // (a page whose bounds are not finite comes first)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const double x = s[i] != s[i] ? (double)INFINITY : s[i];
                best[i] = real && x > best[i] ? x : best[i];
            }
        }
        // s[i] is page p0 + 4 i + lane / 16 with head lane % 16
        const uint64_t none = __ballot(!held);
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) {
                const double x = wave_xor(best[i], o);
                best[i] = x > best[i] ? x : best[i];
            }
            const int32_t page = p0 + 4 * i + kq;
            if (c == 0 && page < n)
                a.scores[((int64_t)b * a.pg.H + h) * a.table.n + page] =
                    (none >> (4 * i + kq)) & 1 ? -(double)INFINITY : best[i];
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

// One workgroup per (sequence, KV head): the n_select - 1 largest scores, by a
// search of the last one's bits from the first in which scores differ, eight a
// round, and the pages in order.
constexpr int kChoiceThreads = 1024;
__global__ void __launch_bounds__(kChoiceThreads) page_choice_kernel(SparseArgs a) {
    __shared__ uint32_t bins[256];
    __shared__ uint64_t ends[2][kChoiceThreads / 64];
    __shared__ int32_t digit, above, inside, counts[2][kChoiceThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = blockIdx.x, b = row / a.pg.H, h = row - b * a.pg.H;
    const int32_t len = length_of(a, b), pages = pages_of(a, len), n = pages - 1;
    const double* scores = a.scores + (int64_t)row * a.table.n;
    const int32_t want = min(a.n_select - 1, max(n, 0));
    uint64_t prefix = 0;
    int shift = 64;         // bits of the prefix that are not decided yet
    int32_t need = want;    // pages still to be taken among those that have its decided bits
    const bool all = want >= n;
    if (!all && want > 0) {
        uint64_t lo = ~0ull, hi = 0;
        for (int32_t i = tid; i < n; i += kChoiceThreads) {
            const uint64_t k = order_of(scores[i]);
            lo = min(lo, k), hi = max(hi, k);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) {
            lo = min(lo, (uint64_t)wave_xor((unsigned long long)lo, o));
            hi = max(hi, (uint64_t)wave_xor((unsigned long long)hi, o));
        }
        if (lane == 0) ends[0][wave] = lo, ends[1][wave] = hi;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kChoiceThreads / 64; w++) lo = min(lo, ends[0][w]), hi = max(hi, ends[1][w]);
        shift = lo == hi ? 0 : 64 - __builtin_clzll(lo ^ hi);
        prefix = hi;  // (the bits from `shift` on are all scores')
        while (shift > 0) {
            const int next = max(0, shift - 8);
            for (int i = tid; i < 256; i += kChoiceThreads) bins[i] = 0;
            __syncthreads();
            for (int32_t i = tid; i < n; i += kChoiceThreads) {
                const uint64_t k = order_of(scores[i]);
                if (compare_from(k, prefix, shift) == 0) atomicAdd(&bins[(k >> next) & ((1u << (shift - next)) - 1)], 1u);
            }
            __syncthreads();
            if (wave == 0) {
                // from the largest digit down; lane l has digits 255 - 4 l to 252 - 4 l
                uint32_t own[4], mine = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) own[i] = bins[255 - 4 * lane - i], mine += own[i];
                uint32_t before = mine;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const uint32_t x = __shfl_up(before, o, 64);
                    if (lane >= o) before += x;
                }
                before -= mine;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (before < (uint32_t)need && before + own[i] >= (uint32_t)need)
                        digit = 255 - 4 * lane - i, above = (int32_t)before, inside = (int32_t)own[i];
                    before += own[i];
                }
            }
            __syncthreads();
            const uint64_t mask = ((1ull << (shift - next)) - 1) << next;
            prefix = (prefix & ~mask) | (uint64_t)digit << next;
            need -= above;
            shift = next;
            const bool done = inside == need;  // (all that have these bits are taken)
            __syncthreads();
            if (done) break;
        }
    }
    int32_t* chosen = a.chosen + (int64_t)row * a.n_select;
    int32_t* selected = a.selected ? a.selected + (int64_t)row * a.n_select : nullptr;
    auto take = [&](int32_t slot, int32_t page) {
        const int32_t id = a.table.ids[b * a.table.stride + page];
        chosen[slot] = (uint32_t)id < (uint32_t)a.pg.n_pages ? id * a.pg.H + h : -1;
        if (selected) selected[slot] = page;
    };
    if (all) {
        for (int32_t i = tid; i < n; i += kChoiceThreads) take(i, i);
    } else if (want > 0) {
        int32_t above_before = 0, at_before = 0;
        for (int32_t p0 = 0; p0 < n; p0 += kChoiceThreads) {
            const int32_t i = p0 + tid;
            const int cmp = i < n ? compare_from(order_of(scores[i]), prefix, shift) : -1;
            const uint64_t up = __ballot(cmp > 0), at = __ballot(cmp == 0);
            if (lane == 0) counts[0][wave] = __popcll(up), counts[1][wave] = __popcll(at);
            __syncthreads();
            int32_t ups = above_before, ats = at_before;
#pragma unroll
            for (int w = 0; w < kChoiceThreads / 64; w++) {
                if (w < wave) ups += counts[0][w], ats += counts[1][w];
                above_before += counts[0][w], at_before += counts[1][w];
            }
            const uint64_t below = (1ull << lane) - 1;
            ups += __popcll(up & below), ats += __popcll(at & below);
            // (of equal scores the first `need`)
            if (cmp > 0 || (cmp == 0 && ats < need)) take(ups + min(ats, need), i);
            __syncthreads();
        }
    }
    if (tid == 0) {
        if (pages > 0) take(want, n);
        a.len[row] = pages > 0 ? want * a.pg.page_size + len - n * a.pg.page_size : 0;
    }
    if (selected)
        for (int32_t i = (pages > 0 ? want + 1 : 0) + tid; i < a.n_select; i += kChoiceThreads) selected[i] = -1;
}

// ---------------------------------------------------------------------------
// launch
// ---------------------------------------------------------------------------

struct SparsePlan {
    int64_t chosen_at, len_at, attn_at, attn_bytes, bytes;
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
    if (n_table < 0 || (int64_t)n_table * p->page_size > 0x7FFFFFFF - 4096)
        return set_error(w + ": more than 2^31 tokens a sequence");
    if (n_select < 1 || (int64_t)n_select * p->page_size > 0x7FFFFFFF - 4096)
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

static SparsePlan plan_sparse(const fkv_pages* p, int32_t Hq, int32_t B, int32_t n_table, int32_t n_select, int64_t max_len) {
    SparsePlan r;
    const fkv_pages one = by_head(p);
    const int64_t rows = (int64_t)B * p->H;
    r.chosen_at = round_up(8 * rows * n_table, 256);
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
    if (B > 1 && query->stride_b != Hq * query->stride_h)
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
    a.scores = (double*)workspace;
    a.chosen = (int32_t*)((char*)workspace + p.chosen_at);
    a.len = (int32_t*)((char*)workspace + p.len_at);
    a.selected = selected;
    a.lens_add = lens_add;
    a.Hq = Hq;
    a.G = Hq / pages->H;
    a.n_select = n_select;
    hipStream_t s = (hipStream_t)stream;
    const fkv_pages one = by_head(pages);
    const int32_t rows = B * pages->H;
    fkv_rows q = *query;
    q.stride_b = (int64_t)a.G * query->stride_h;
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
    if (n_table > n_select) {  // (else all pages are taken)
        const dim3 grid((uint32_t)std::max<int64_t>(1, std::min<int64_t>(cdiv(scored, 64), 4096)), pages->H, B);
        auto go = [&](auto kernel) { return start_kernel(w, kernel, grid, 256, s, a); };
        const bool bf = q_dtype == FKV_BF16;
        int e;
        if (pages->D == 64) e = bf ? go(page_score_kernel<64, true>) : go(page_score_kernel<64, false>);
        else e = bf ? go(page_score_kernel<128, true>) : go(page_score_kernel<128, false>);
        if (e) return e;
    }
    if (int e = start_kernel(w, page_choice_kernel, (uint32_t)rows, kChoiceThreads, s, a)) return e;
    return attend(rows);
}

}  // extern "C"
