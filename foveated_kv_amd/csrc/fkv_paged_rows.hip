// Attention of several new tokens per sequence over a paged KV cache, and of
// sequences whose first pages are the same.
//
// A row is one query head at one new token.  Row (b, l, g) of KV head h attends
// to the first lim = len_b - n_b + l + 1 tokens of its sequence (n_b new ones, of
// which it is the l-th), as the one-token kernel does:
//   s_t = scale * q . k_t,   out = sum_t exp(s_t) v_t / sum_t exp(s_t).
// Tokens below `shared` lie in the same pages for all sequences: the rows of all
// of them attend to these together, so that they are read once per 256 rows, and
// each sequence's rows to its own tokens.  Every part leaves a record (maximum,
// sum, numerators) per row, which a second kernel joins in a fixed order; a call
// that is not split writes its results at once.
//
// Matrix products, 32 rows a wave, 32 tokens a step:
//   S^T (32 tokens x 32 rows) = K (32 x 16 dims) Q^T,   v_mfma_f32_32x32x16
//   O^T (32 dims x 32 rows)  += V^T (32 x 16 tokens) P^T
// A lane of S^T holds 16 tokens of one row, the lane 32 further the other 16; in
// groups of 8 they are P^T's operand as they stand, since the order of the 16
// tokens within a product is free as long as V^T's is the same: tokens 4 h + i
// and 8 + 4 h + i of lanes' half h.  V^T comes out of the LDS by transposing
// reads, which hand a lane four tokens of one dim.
//
// A workgroup has NW waves, four (64 tokens a tile, two workgroups a CU) for few rows
// on a KV head, eight (128) for many; its threads decode a tile to 16 bits once into
// the LDS, the next tile's loads being in flight meanwhile.  WR waves stand for 32 rows
// each and WT = min(NW / 2, NW / WR) for parts of the tile's tokens: few rows (drafted
// tokens) are bound by the cache's bytes and take one wave each for their rows, many (a
// prompt's chunk, a shared beginning) by the products.
//
// Within a step the next 32 tokens' scores are computed between this one's weights: a
// wave issues a vector instruction every six cycles at most, a product takes 32, so
// each product is followed by some six of them.
//
// Measured, with what bounds it: 32 sequences of up to 8K tokens, five drafted tokens
// each, 32 / 8 heads of 128 dims in bf16: 125 us, the pages' 540 MB (4.3 TB/s).  2K
// tokens after 14K: 720 to 770 us, the products and the weights between them (a large
// library product would take 425 us for one number a weight, 640 for two).  64 sequences
// behind 16K shared tokens: 83 us, the shared tokens' products first.  (Comparisons
// below that do not say otherwise are of one 16-bit number a weight, see kParts, with
// which these took 101, 590 and 75.)
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "fkv_paged.h"

namespace fkv {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));

constexpr int kRowsMaxSeqs = 4096;
// More rows than this on a KV head: workgroups of eight waves and 128 tokens a tile
// in place of four and 64, of which a CU has two at once (see plan_rows()).
constexpr int64_t kFewRows = 256;
constexpr float kBegin = 6.0f, kJoin = 4.0f, kJoinPart = 0.12f;  // us, see plan_rows()
constexpr int kManyParts = 16;  // see paged_rows_join_kernel()
constexpr int kEvenSeqs = 256;  // sequences whose lengths even parts are made from
constexpr float kLowest = -3.402823466e38f;  // running maximum before the first token: no score lies below it
// As in the one-token kernel: the running maximum follows a score that exceeds it by
// more than 2^kRowSlack, and stays 2^kRowBias below the scores of fp16 pages, whose
// weights (2^15 at most) so keep away from the end of fp16's range.
template <int FMT>
constexpr float kRowSlack = FMT == FKV_PAGES_F16 ? 4.0f : 8.0f;
// Scores are scaled and the maximum taken off by one fma, whose product is not
// rounded as the maximum was: a difference of 2^-4 at most up to here; beyond,
// where it would be a power, in two steps.
constexpr float kWide = 1048576.0f;
template <int FMT>
constexpr float kRowBias = FMT == FKV_PAGES_F16 ? 11.0f : 0.0f;

// How one kind of part (the shared tokens, the sequences' own) is cut up.
struct RowParts {
    int32_t wr;      // waves of 32 rows per workgroup: 1, 2, 4 or 8
    int32_t tiles;   // workgroups of 32 * wr rows (per sequence, for the own tokens)
    int32_t splits;  // parts of the tokens
    int32_t chunk;   // tokens of a part; the last one of the own tokens takes what is left
};

struct RowsArgs {
    PageView pg;
    TableView table;
    RowsView q, out;
    const int32_t* lens;
    const int32_t* n_new;
    float* lse;
    float* records;  // workspace: per row and part D numerators, maximum, sum
    int32_t* chunk;  // workspace, of even parts: how many tokens they have
    RowParts common, own;
    int32_t lens_add, B, Hq, G, L, shared;
    int32_t tile;     // tokens of a tile
    int32_t even;     // != 0: as many parts of all sequences as this (see even_parts()), of
    int32_t least;    // this many tiles or more
    float scale;      // |scale| * log2(e)
    uint32_t q_sign, q_mask;  // its sign, for two 16-bit numbers; 0 where it is 0 (and |scale| 1)
};

typedef const __attribute__((address_space(4))) int32_t* scalar_ints;
__device__ inline int32_t scalar_load(const int32_t* p, int64_t i) { return ((scalar_ints)(uintptr_t)p)[i]; }

__device__ inline int32_t length_of(const RowsArgs& a, int32_t len) {
    const int64_t n = (int64_t)len + a.lens_add, cap = (int64_t)a.table.n * a.pg.page_size;  // (cap < 2^31)
    return (int32_t)(n < 0 ? 0 : n > cap ? cap : n);
}
// How many tokens row (b, l) attends to; -1 for a padded token's.
__device__ inline int32_t limit_of(const RowsArgs& a, int b, int l) {
    const int32_t n = a.n_new ? min(max(a.n_new[b], 0), a.L) : a.L;
    return l >= n ? -1 : max(length_of(a, a.lens[b]) - n + l + 1, 0);
}

// Parts of the sequences' own tokens from their lengths, which only the device has:
// the shortest parts of which there are `even` at most, that is, which the chip takes
// all at once.  -> tokens of a part; the sequence and the part that are number `unit`
// of all (seq -1: there are fewer).  Parts of max_len / n, whatever n, leave some of the
// chip idle where lengths differ, and empty workgroups among the others: 16 sequences of
// up to 32K tokens take 179 us and 183 to 313 so (n from 3 to 16), 32 of up to 8K 109 and
// 114 to 136, 32 of 8K each 177 and 173 to 231.
__device__ inline int32_t even_parts(const RowsArgs& a, int lane, uint32_t unit, int& seq, int& split) {
    uint32_t tiles[kEvenSeqs / 64], total = 0, longest = 0;
#pragma unroll
    for (int j = 0; j < kEvenSeqs / 64; j++) {
        const int b = 64 * j + lane;
        const int32_t n = b < a.B ? length_of(a, a.lens[b]) : 0;
        tiles[j] = ((uint32_t)n + a.tile - 1) / (uint32_t)a.tile;
        total += tiles[j], longest = max(longest, tiles[j]);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) longest = max(longest, wave_xor(longest, o));
    auto of_lane = [](uint32_t v, int i) { return (uint32_t)__builtin_amdgcn_readlane((int)v, i); };
    const uint32_t even = a.even, splits = a.own.splits;
    uint32_t chunk = max(max((of_lane(sum_up_to(total), 63) + even - 1) / even, (longest + splits - 1) / splits), (uint32_t)a.least);
    chunk = __builtin_amdgcn_readfirstlane(max(chunk, 1u));
    longest = __builtin_amdgcn_readfirstlane(longest);
    for (;;) {
        uint32_t before = 0;
        seq = -1;
#pragma unroll
        for (int j = 0; j < kEvenSeqs / 64; j++) {
            if (64 * j >= a.B) break;
            const uint32_t parts = (tiles[j] + chunk - 1) / chunk, upto = before + sum_up_to(parts);
            const uint64_t past = __ballot(upto > unit);
            if (past && seq < 0) {
                const int i = __builtin_ctzll(past);
                seq = 64 * j + i, split = (int)(unit - (of_lane(upto, i) - of_lane(parts, i)));
            }
            before = of_lane(upto, 63);
        }
        if (before <= even || chunk >= longest) break;
        chunk = min(chunk + chunk / 16 + 1, longest);
    }
    return (int32_t)(chunk * a.tile);
}

// A weight enters the products as the sum of two 16-bit numbers, whose error is a
// small part of what rounding the result costs, however far a weight lies below the
// row's largest:
//   bf16 pages   the upper half, and what that leaves, rounded: 2^-16 of the weight, where
//                a bf16 result is rounded by up to 2^-8.  (Both have the weight's sign, so
//                that an infinite value times both stays one.)
//   fp16 pages   the fp16 number nearest towards 0, and kUp times what that leaves, rounded:
//                2^-21 of the weight, or 2^-35, which is 2^-46 of the row's largest: times
//                the largest fp16 value 2^-30, where fp16 results have steps of 2^-24.  (One
//                fp16 number ends at 2^-24: a token 14 to 24 nats above the others, with a
//                value of zero, left 10 to no bits of theirs.)
//   quantised    bf16 numbers, which have the range of the values' scales, both rounded:
//                2^-18, where an fp16 result is rounded by up to 2^-11.
// One number, rounded, put results of bf16 and fp16 pages further from the exact ones by
// half of what their own rounding does (of the results' norm 2.5e-3 and 3.2e-4 off those
// of fp32 weights, with two 1.3e-4 and 2.4e-5).  The second costs least where the
// bytes bind: drafts of 32 ragged sequences to 8K tokens 125 us and 110 with one (bf16), 136
// and 110 (fp16), 111 and 98 (E4M3); 64 sequences behind 16K shared tokens 83 and 75; 2K
// tokens after 14K, bound by the products, 755 and 593 (bf16), 890 and 630 (fp16).  (A third,
// all 24 bits: 129, 191, 120; 91; 902, 1137.)
constexpr int kParts = 2;

template <bool BF>
__device__ inline f16v mfma32(u4 x, u4 y, f16v c) {
    if (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, x), __builtin_bit_cast(h8, y), c, 0, 0, 0);
}

// Two E4M3 codes (the chosen half of w) times a power of two, exact.
template <bool BF, bool HI>
__device__ inline uint32_t cvt_codes(uint32_t w, float scale) {
    if (BF) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
}
// 16 codes of a row with exponent byte e (0 stands for a factor of 0) as 16-bit numbers.
template <typename B>
__device__ inline void decode(u4 x, uint32_t e, B, uint32_t (&y)[8]) {
    const float scale = exp_byte(e);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t w = e ? x[j] : 0;
        y[2 * j] = cvt_codes<B::value, false>(w, scale);
        y[2 * j + 1] = cvt_codes<B::value, true>(w, scale);
    }
}
// Codes c of 0 to 15, a byte each, as the E4M3 numbers (c - 8) * 2^-9 (0 to 7 times
// that are subnormal numbers, 8 times the first normal one).
__device__ inline uint32_t less_eight(uint32_t c) {
    const uint32_t x = c ^ 0x08080808u, n = x & 0x08080808u;  // n: 8 where c < 8, and x is c + 8
    return ((x ^ ((n << 1) - (n >> 3))) + (n >> 3)) | n << 4;
}
__device__ inline uint32_t round_pair_bf16(float a, float b) {
    const b2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
}
__device__ inline uint32_t round_pair_fp16(float a, float b) {
    const h2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
}

// Pages that a call reads once are not kept in the caches: 32 sequences to 8K tokens,
// 540 MB, take 10 % less time so than by other loads.  Where several workgroups read them
// (a prompt's chunk 577 us and 597 so, shared tokens) the caches serve all but the first.
template <bool ONCE, typename T>
__device__ inline T read(const T* p) {
    return ONCE ? __builtin_nontemporal_load(p) : *p;
}

// A tile's tokens as a thread loads them: 16 (INT4 of 64 dims: 8) bytes of a row
// at a time, neighbouring threads a row.
template <int D, int FMT>
struct Rows {
    static constexpr bool k16 = FMT <= FKV_PAGES_BF16;
    static constexpr int KB = k16 ? 2 * D : D;                                 // bytes of a key row
    static constexpr int VB = k16 ? 2 * D : FMT == FKV_PAGES_FP8 ? D : D / 2;  // and of a value row
    static constexpr int KT = KB / 16, VT = VB == 32 ? 4 : VB / 16;            // threads a row
    static constexpr int KP = KT / 4, VP = VT / 4;                             // passes over a tile's rows
    u4 k[KP], v[VP];
    uint32_t kx[KP], vx[VP];  // exponent bytes of the rows (E4M3; of keys for bf16 queries)
    uint32_t ke;              // of run `wave`, token `lane`: the key's (for fp16 queries),
    float2 sz;                // an INT4 value's scale and minimum
};

template <int D, int NW>
struct RowsLds {
    static constexpr int kRow = 2 * D;                 // bytes of a row in 16 bits
    static constexpr int kTileBytes = 16 * NW * kRow;
    static constexpr int kNumerators = NW * 32 * (D + 4) * 4;
    static constexpr int kBytes = 4 * kTileBytes > kNumerators ? 4 * kTileBytes : kNumerators;
};

// Where 16-byte chunk `chunk` of row `row` lies in a tile of keys (eight
// neighbouring lanes read one chunk of eight rows: all banks) and of values (a
// transposing read takes 64 bytes of each of four rows).
template <int D>
__device__ inline uint32_t key_place(uint32_t row, uint32_t chunk) { return row * 2 * D + 16 * (chunk ^ (row & 7)); }
template <int D>
__device__ inline uint32_t value_turn(uint32_t row) { return D == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); }
template <int D>
__device__ inline uint32_t value_place(uint32_t row, uint32_t chunk) {
    return row * 2 * D + 16 * (chunk ^ value_turn<D>(row));
}

// Two packed 16-bit numbers times 0, added to s: NaN where one is infinite or NaN.
template <bool BF>
__device__ inline float times_zero(uint32_t w, float s) {
    if (BF) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, w), b2{}, s, false);
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w), h2{}, s, false);
}
// Are any of two packed 16-bit numbers infinite or NaN?
template <bool BF>
__device__ inline bool any_not_finite(uint32_t w) {
    const uint32_t e = BF ? 0x7F80u : 0x7C00u;
    return (w & e) == e || ((w >> 16) & e) == e;
}
template <bool BF>
__device__ inline uint32_t finite_or_zero(uint32_t w) {
    const uint32_t e = BF ? 0x7F80u : 0x7C00u;
    return ((w & e) == e ? 0 : w & 0xFFFFu) | (((w >> 16) & e) == e ? 0 : w & 0xFFFF0000u);
}

template <int D, int FMT, bool BF, int NW, bool ONCE>
__global__ void __launch_bounds__(64 * NW, 2) paged_rows_kernel(RowsArgs a) {
    using R = Rows<D, FMT>;
    constexpr int kRowWaves = NW, kTileTokens = 16 * NW, kSubs = NW / 2, kThreads = 64 * NW;
    constexpr bool kVB = FMT != FKV_PAGES_F16;  // values and weights are bf16 numbers
    // E4M3 keys as bf16 numbers hold their row's power of two; as fp16 numbers the
    // scores are multiplied by it
    constexpr bool kFactors = FMT >= FKV_PAGES_FP8 && !BF;
    constexpr int DT = D / 32;
    __shared__ __attribute__((aligned(16))) char tiles[RowsLds<D, NW>::kBytes];
    __shared__ __attribute__((aligned(16))) float key_factor[2][kTileTokens], value_scale[2][kTileTokens],
        value_min[2][kTileTokens];  // (the latter min + 8 scale)
    __shared__ float stat[kRowWaves][32][3];
    __shared__ int32_t least[kRowWaves], most[kRowWaves], run_tokens[2][kRowWaves], odd_tile[2];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sh = 31 - __builtin_clz((unsigned)a.pg.page_size);

    // the part: shared tokens (seq < 0) or sequence seq's own
    const int h = blockIdx.x % a.pg.H;
    int rest = blockIdx.x / a.pg.H, seq = -1, tile, split;
    RowParts p = a.common;
    if (rest < a.common.tiles * a.common.splits) {
        tile = rest / a.common.splits, split = rest - tile * a.common.splits;
    } else {
        rest -= a.common.tiles * a.common.splits;
        p = a.own;
        // (the last rows attend to the most tokens: they come first)
        const int per_tile = a.own.splits * a.B, t = ONCE && a.even ? 0 : rest / per_tile;
        tile = a.own.tiles - 1 - t;
        rest -= t * per_tile;
        if (ONCE && a.even) {
            p.chunk = even_parts(a, lane, rest, seq, split);
            if (blockIdx.x == 0 && tid == 0) *a.chunk = p.chunk;  // (for the join)
            if (seq < 0) return;
        } else {
            // (The first tokens of all sequences, then the next.  Later parts are empty where
            // sequences are short, and a sequence's long where it is: neither may come at a
            // step that is a power of two, which would put them on the same few CUs.)
            split = rest / a.B, seq = (rest + split * 5) % a.B;
        }
    }
    const int rows = seq < 0 ? a.B * a.L * a.G : a.L * a.G;
    const int wr = p.wr, wt = min(kSubs, kRowWaves / wr), rg = wave & (wr - 1), tg = wave / wr;
    const int row0 = tile * 32 * wr;
    // row r of the part -> (b, l, query head); -1: none
    auto place = [&](int r, int& b, int& l, int& hq) {
        const int token = r / a.G;
        b = seq < 0 ? token / a.L : seq;
        l = seq < 0 ? token - b * a.L : token;
        hq = h * a.G + r - token * a.G;
        return r < rows ? limit_of(a, b, l) : -1;
    };
    // (even parts may begin beyond 2^31, where no tokens are)
    const int32_t begin = (int32_t)min((seq < 0 ? 0 : a.shared) + (int64_t)split * p.chunk, (int64_t)0x7FFFFFFF);
    const int parts = a.common.splits + a.own.splits;
    // The ends of rows [first, last): the most tokens that one attends to (-1: none
    // is real) and the least that a real one does.  A sequence's own rows come by
    // their tokens, so these are its length and their numbers; the shared tokens'
    // rows are looked at one by one.
    int32_t wave_most, wave_least, end, all_least;
    int b, l, hq;
    int32_t lim;
    if (seq >= 0) {
        const int32_t len = length_of(a, scalar_load(a.lens, seq));
        const int32_t n = a.n_new ? min(max(scalar_load(a.n_new, seq), 0), a.L) : a.L;
        auto ends = [&](int first, int last, int32_t& most, int32_t& least) {
            last = min(last, rows);
            const int l0 = first / a.G, l1 = min((last - 1) / a.G, n - 1);
            most = first < last && l0 < n ? max(len - n + l1 + 1, 0) : -1;
            least = first < last && l0 < n ? max(len - n + l0 + 1, 0) : 0x7FFFFFFF;
        };
        ends(row0, row0 + 32 * wr, end, all_least);
        if (end <= begin && parts > 1) return;
        ends(row0 + 32 * rg, row0 + 32 * rg + 32, wave_most, wave_least);
        lim = place(row0 + 32 * rg + c, b, l, hq);
    } else {
        lim = min(place(row0 + 32 * rg + c, b, l, hq), a.shared);
        wave_most = lim, wave_least = lim >= 0 ? lim : 0x7FFFFFFF;
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) {
            wave_most = max(wave_most, wave_xor(wave_most, o));
            wave_least = min(wave_least, wave_xor(wave_least, o));
        }
        wave_most = __builtin_amdgcn_readfirstlane(wave_most);
        wave_least = __builtin_amdgcn_readfirstlane(wave_least);
        if (lane == 0) least[wave] = wave_least, most[wave] = wave_most;
        __syncthreads();
        end = most[0], all_least = least[0];
#pragma unroll
        for (int w = 1; w < kRowWaves; w++) end = max(end, most[w]), all_least = min(all_least, least[w]);
        end = __builtin_amdgcn_readfirstlane(end);
        all_least = __builtin_amdgcn_readfirstlane(all_least);
    }
    const bool real = lim >= 0;
    if (seq < 0 || split + 1 < p.splits) end = (int32_t)min((int64_t)end, (int64_t)begin + p.chunk);
    const int nt = end > begin ? (end - begin + kTileTokens - 1) / kTileTokens : 0;
    if (nt == 0 && parts > 1) return;
    if (tid < 2) odd_tile[tid] = -1;
    __syncthreads();  // (before the first store may set it)

    u4 q[D / 16];
    {
        const char* at = a.q.data + 2 * (b * a.q.sb + hq * a.q.sh + l * a.q.sl);
        const u4 none = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < D / 16; i++) q[i] = real ? (*(const u4*)(at + 32 * i + 16 * hf) & a.q_mask) ^ a.q_sign : none;
    }

    const int32_t* ids = a.table.ids + (seq < 0 ? 0 : seq) * a.table.stride;
    R st;
    // Runs of 16 tokens lie in one page.  A wave's loads are rows of KP runs of keys,
    // VP of values (the same ones where rows have as many bytes) and, for the rows'
    // scales, run `wave`; their pages' ids are loaded a tile ahead.
    constexpr bool kSame = R::KT == R::VT;
    constexpr int kIds = R::KP + (kSame ? 0 : R::VP) + 1;
    int32_t id[kIds];
    auto run_at = [&](int i) {
        return i < R::KP ? (kThreads / R::KT * i + (64 / R::KT) * wave) / 16
               : i < kIds - 1 ? (kThreads / R::VT * (i - R::KP) + (64 / R::VT) * wave) / 16 : wave;
    };
    auto fetch = [&](int32_t tok) {
#pragma unroll
        for (int i = 0; i < kIds; i++) id[i] = scalar_load(ids, min(tok + 16 * run_at(i), end - 1) >> sh);
    };
    // -> the run's first row in the pages (any that is there, where the run has none), how many of its tokens take part
    auto run_of = [&](int32_t tok, int i, int& n) {
        const int32_t at = tok + 16 * run_at(i);
        const bool in = (uint32_t)id[i] < (uint32_t)a.pg.n_pages;
        n = in ? min(max(end - at, 0), 16) : 0;
        return (((int64_t)(in ? id[i] : 0) * a.pg.H + h) << sh) + (at & (a.pg.page_size - 1));
    };
    // A tile's loads, as they are (what waits for them is store()).  `taken`: tokens
    // of each run that take part; `whole`: all 16 of all.
    bool whole = true;
    int taken[kIds];
    auto load = [&](int32_t tok) {
        int64_t first[kIds];
        whole = true;
#pragma unroll
        for (int i = 0; i < kIds; i++) {
            first[i] = run_of(tok, i, taken[i]);
            whole = whole && taken[i] == 16;
        }
        if (tok + kTileTokens < end) fetch(tok + kTileTokens);
#pragma unroll
        for (int i = 0; i < R::KP; i++) {
            st.k[i] = read<ONCE>((const u4*)(a.pg.k + first[i] * R::KB + (uint32_t)(((tid / R::KT) & 15) * R::KB + 16 * (tid % R::KT))));
            if (FMT >= FKV_PAGES_FP8 && !kFactors) st.kx[i] = (a.pg.k_exp + first[i])[(tid / R::KT) & 15];
        }
#pragma unroll
        for (int i = 0; i < R::VP; i++) {
            const int64_t row = first[kSame ? i : R::KP + i];
            const uint32_t r = (tid / R::VT) & 15;
            const char* at = a.pg.v + row * R::VB;
            if (R::VB == 32) {
                const u2 x = read<ONCE>((const u2*)(at + r * R::VB + 8 * (tid % R::VT)));
                st.v[i] = u4{x.x, x.y, 0, 0};
            } else {
                st.v[i] = read<ONCE>((const u4*)(at + r * R::VB + 16 * (tid % R::VT)));
            }
            if (FMT == FKV_PAGES_FP8) st.vx[i] = ((const uint8_t*)a.pg.v_scale)[row + r];
        }
        if (FMT >= FKV_PAGES_FP8 && lane < 16) {
            if (kFactors) st.ke = a.pg.k_exp[first[kIds - 1] + lane];
            if (FMT == FKV_PAGES_FP8_INT4) st.sz = ((const float2*)a.pg.v_scale)[first[kIds - 1] + lane];
        }
    };
    // Zeros in the place of what takes no part (of a tile that is not whole).
    auto blank = [&]() {
#pragma unroll
        for (int i = 0; i < R::KP; i++)
            if ((int)((tid / R::KT) & 15) >= taken[i]) st.k[i] = u4{0, 0, 0, 0}, st.kx[i] = 0;
#pragma unroll
        for (int i = 0; i < R::VP; i++)
            if ((int)((tid / R::VT) & 15) >= taken[kSame ? i : R::KP + i]) st.v[i] = u4{0, 0, 0, 0}, st.vx[i] = 0;
        if (lane >= taken[kIds - 1]) st.ke = 0, st.sz = make_float2(0.0f, 0.0f);
    };
    // ... and into the LDS, in 16 bits.
    auto store = [&](int32_t tok, int t, int buf) {
        if (!whole) blank();
        char* keys = tiles + buf * 2 * RowsLds<D, NW>::kTileBytes;
        char* values = keys + RowsLds<D, NW>::kTileBytes;
        const bool look = tok + kTileTokens > all_least;  // (tokens that not all rows attend to)
        bool odd = false;
        float seen = 0.0f;  // NaN where a 16-bit value is infinite or NaN
#pragma unroll
        for (int i = 0; i < R::KP; i++) {
            const int r = (kThreads / R::KT) * i + tid / R::KT, ch = tid % R::KT;
            const u4 x = st.k[i];
            if (R::k16) {
                *(u4*)(keys + key_place<D>(r, ch)) = x;
            } else {
                uint32_t y[8];
                decode(x, kFactors ? 127 : st.kx[i], std::integral_constant<bool, BF>{}, y);
                *(u4*)(keys + key_place<D>(r, 2 * ch)) = u4{y[0], y[1], y[2], y[3]};
                *(u4*)(keys + key_place<D>(r, 2 * ch + 1)) = u4{y[4], y[5], y[6], y[7]};
            }
        }
#pragma unroll
        for (int i = 0; i < R::VP; i++) {
            const int r = (kThreads / R::VT) * i + tid / R::VT, ch = tid % R::VT;
            const u4 x = st.v[i];
            if (R::k16) {
                *(u4*)(values + value_place<D>(r, ch)) = x;
#pragma unroll
                for (int j = 0; j < 4; j++) seen = times_zero<kVB>(x[j], seen);
            } else if (FMT == FKV_PAGES_FP8) {
                uint32_t y[8];
                decode(x, st.vx[i], std::true_type{}, y);
                *(u4*)(values + value_place<D>(r, 2 * ch)) = u4{y[0], y[1], y[2], y[3]};
                *(u4*)(values + value_place<D>(r, 2 * ch + 1)) = u4{y[4], y[5], y[6], y[7]};
                if (look) {
#pragma unroll
                    for (int j = 0; j < 8; j++) odd = odd || any_not_finite<true>(y[j]);
                }
            } else {
                // code - 8 in place of the code and min + 8 scale in place of min: both
                // are then of the values' size, and so is what rounding a weight costs
                constexpr int kWords = R::VB == 32 ? 2 : 4;  // dwords of eight codes: a chunk each
#pragma unroll
                for (int j = 0; j < kWords; j++) {
                    const uint32_t even = less_eight(x[j] & 0x0F0F0F0Fu), other = less_eight((x[j] >> 4) & 0x0F0F0F0Fu);
                    const uint32_t lo = __builtin_amdgcn_perm(other, even, 0x05010400u);
                    const uint32_t hi = __builtin_amdgcn_perm(other, even, 0x07030602u);
                    *(u4*)(values + value_place<D>(r, kWords * ch + j)) =
                        u4{cvt_codes<true, false>(lo, 512.0f), cvt_codes<true, true>(lo, 512.0f),
                           cvt_codes<true, false>(hi, 512.0f), cvt_codes<true, true>(hi, 512.0f)};
                }
            }
        }
        if (FMT >= FKV_PAGES_FP8 && lane < 16) {
            if (kFactors) key_factor[buf][16 * wave + lane] = exp_byte(st.ke);
            if (FMT == FKV_PAGES_FP8_INT4) {
                const float low = fmaf(8.0f, st.sz.x, st.sz.y);
                value_scale[buf][16 * wave + lane] = st.sz.x, value_min[buf][16 * wave + lane] = low;
                if (look) odd = odd || !(fabsf(low) < INFINITY);
            }
        }
        if (R::k16) odd = seen != seen;
        if (lane == 0) run_tokens[buf][wave] = taken[kIds - 1];
        if (__any(odd)) odd_tile[buf] = t;
    };

    f16v acc[DT];
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[d][i] = 0.0f;
    float m = kLowest, sum = 0.0f, z = 0.0f;
    bool wide = false;  // (of any of the wave's rows)

    // Lane constants of the LDS reads.  Keys: 16-byte chunk 2 i + hf of token c,
    // the chunk's upper bit a constant offset; values: of each 32 dims the rows and
    // bytes of a transposing read (tokens 8 and 16 further lie a constant further).
    constexpr int kKeys = 4, kRow = RowsLds<D, NW>::kRow;
    uint32_t key_lane[kKeys], value_lane[DT];
    {
        const uint32_t tr_row = 4 * hf + ((lane & 15) >> 2), tr_byte = 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
#pragma unroll
        for (int i = 0; i < kKeys; i++) key_lane[i] = key_place<D>(c, 2 * i + hf);
#pragma unroll
        for (int d = 0; d < DT; d++) value_lane[d] = value_place<D>(tr_row, 4 * d + (tr_byte >> 4)) + (tr_byte & 15);
    }
    // Matrix products take their pipe 32 cycles and the issue of vector
    // instructions 9 of these, so a wave's stream is one product, then about six
    // vector instructions, and so on: the weights of these tokens beside the next
    // ones' scores and their own products.  (A wave by itself issues a vector
    // instruction every 6.4 cycles, and two that each do one kind at a time mostly
    // wait for each other.)  The fences keep the order.
#define FENCE __builtin_amdgcn_sched_barrier(0)
    auto key_of = [&](const char* keys, int i) { return *(const u4*)(keys + key_lane[i % kKeys] + i / kKeys * 128); };
    // Scores (not scaled) of the tile's 32 tokens `sub`; the lane's are 8 (i / 4) + 4 hf + i % 4.
    auto score = [&](int buf, int sub) {
        const char* keys = tiles + buf * 2 * RowsLds<D, NW>::kTileBytes + 32 * sub * kRow;
        f16v s;
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 16; i++) s = mfma32<BF>(key_of(keys, i), q[i], s);
        return s;
    };
    // Keys' factors, and the largest score.
    auto factors = [&](f16v& s, int buf, int sub, int j) {
        if (kFactors) {
            const f4 f = *(const f4*)&key_factor[buf][32 * sub + 8 * j + 4 * hf];
#pragma unroll
            for (int i = 0; i < 4; i++) s[4 * j + i] *= f[i];
        }
    };
    auto largest = [](float x, float y) { return __builtin_elementwise_maximum(x, y); };  // (NaN where one is)
    auto max4 = [&](const f16v& s, int j) {
        return largest(largest(s[4 * j], s[4 * j + 1]), largest(s[4 * j + 2], s[4 * j + 3]));
    };
    // What takes no part, and the running maximum.
    bool masked = false;
    auto settle_scores = [&](f16v& s, float top, int32_t tok, int buf, int sub) {
        const int n0 = __builtin_amdgcn_readfirstlane(run_tokens[buf][2 * sub]);
        const int n1 = __builtin_amdgcn_readfirstlane(run_tokens[buf][2 * sub + 1]);
        masked = tok + 32 > wave_least || n0 < 16 || n1 < 16;
        if (masked) {
            const int left = lim - tok - 4 * hf, left0 = n0 - 4 * hf, left1 = n1 - 4 * hf;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int at = 8 * (i >> 2) + (i & 3);
                if (at >= left || (at & 15) >= (i < 8 ? left0 : left1)) s[i] = -INFINITY;
            }
            top = largest(largest(max4(s, 0), max4(s, 1)), largest(max4(s, 2), max4(s, 3)));
        }
        top *= a.scale;  // (not negative: the queries carry its sign)
        if (__any(top > m + (kRowSlack<FMT> + kRowBias<FMT>))) {
            top = fmaxf(top, wave_xor(top, 32));
            // (Before a row's first weight that is not 0 the numerators are 0, or infinite values
            // of this tile that settle() added: these stay.)
            const float up = fmaxf(m, top - kRowBias<FMT>);
            const float f = sum + wave_xor(sum, 32) == 0.0f ? 1.0f : __builtin_amdgcn_exp2f(m - up);
            m = up;
            wide = __any(fabsf(m) > kWide && m != kLowest);
            sum *= f;
            z *= f;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) acc[d][i] *= f;
        }
        if (wide) {
#pragma clang fp contract(off)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float x = s[i] * a.scale;
                s[i] = x - m;
            }
        }
    };
    // Weights of the scores s (whose tokens begin at tok), O^T += V^T P^T, and the
    // scores of the tokens `next` of the tile in next_buf, whose largest is returned
    // (of whatever lies there where these were the last ones).
    auto step = [&](f16v& s, int32_t tok, int buf, int sub, int next_buf, int next) {
        const char* values = tiles + (buf * 2 + 1) * RowsLds<D, NW>::kTileBytes + 32 * sub * kRow;
        const char* keys = tiles + next_buf * 2 * RowsLds<D, NW>::kTileBytes + 32 * next * kRow;
        const float by = wide ? 1.0f : a.scale, off = wide ? 0.0f : m;
        float w[16], part_sum = 0.0f;
        u4 part_of[2][kParts];  // [16 tokens][part]
        f4 v_scale[2], v_low[2];
        auto constants = [&](int g) {
            if (FMT != FKV_PAGES_FP8_INT4) return;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                v_scale[j] = *(const f4*)&value_scale[buf][32 * sub + 16 * g + 8 * j + 4 * hf];
                v_low[j] = *(const f4*)&value_min[buf][32 * sub + 16 * g + 8 * j + 4 * hf];
            }
        };
        auto weigh = [&](int i) {
            w[i] = __builtin_amdgcn_exp2f(fmaf(s[i], by, -off));
            part_sum += w[i];
            if (FMT == FKV_PAGES_FP8_INT4) {
                z = fmaf(w[i], v_low[(i >> 2) & 1][i & 3], z);
                w[i] *= v_scale[(i >> 2) & 1][i & 3];
            }
        };
        auto halve = [&](int j) {
            float x = w[2 * j], y = w[2 * j + 1];
            u4* part = part_of[j >> 2];
            if (!kVB) {
                part[0][j & 3] = take_fp16(x, y);
                part[1][j & 3] = round_pair_fp16(x, y);
            } else if (FMT == FKV_PAGES_BF16) {
                part[0][j & 3] = take_bf16(x, y);
                part[1][j & 3] = round_pair_bf16(x, y);
            } else {
                const uint32_t p = round_pair_bf16(x, y);
                part[0][j & 3] = p;
                part[1][j & 3] = round_pair_bf16(x - __uint_as_float(p << 16), y - __uint_as_float(p & 0xFFFF0000u));
            }
        };
        auto value_of = [&](int g, int d) {
            u4 v;
#pragma unroll
            for (int jj = 0; jj < 2; jj++) {
                const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s4*)(values + value_lane[d] + (16 * g + 8 * jj) * kRow));
                const u2 y = __builtin_bit_cast(u2, x);
                v[2 * jj] = y.x, v[2 * jj + 1] = y.y;
            }
            return v;
        };
        f16v after;
        u4 v[DT];
        // AHEAD: operands in flight; EARLY: weights that are made beside the scores
        constexpr int NQ = D / 16, AHEAD = kVB ? 3 : 2, EARLY = kVB ? 8 : 16;
        constants(0);
#pragma unroll
        for (int i = 0; i < 16; i++) after[i] = 0.0f;
        u4 k[NQ];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) k[i] = key_of(keys, i);
        FENCE;
#pragma unroll
        for (int i = 0; i < NQ; i++) {
            const int later = i + AHEAD - NQ;
            if (later < 0) k[i + AHEAD] = key_of(keys, i + AHEAD);
            else if (kVB && later < DT) v[later] = value_of(0, later);
            else if (!kVB && later < 2) v[later] = value_of(later, 0);
            after = mfma32<BF>(k[i], q[i], after);
#pragma unroll
            for (int j = EARLY / NQ * i; j < EARLY / NQ * (i + 1); j++) {
                weigh(j);
                if (j & 1) halve(j >> 1);
            }
            FENCE;
        }
        float top = -INFINITY;
        // the next scores' factors and maximum, a quarter at a time
        auto look_ahead = [&](int j) {
            if (j >= 4) return;
            factors(after, next_buf, next, j);
            top = largest(top, max4(after, j));
        };
        if constexpr (kVB) {
            constants(1);
            // two blocks of 32 dims at a time, so that no product waits for the one before
#pragma unroll
            for (int g = 0; g < 2; g++) {
#pragma unroll
                for (int d0 = 0; d0 < DT; d0 += 2)
#pragma unroll
                    for (int e = 0; e < 2 * kParts; e++) {
                        const int d = d0 + (e & 1), n = kParts * d0 + e;  // product n of kParts * DT
                        if (e < 2 && g == 0 && d + AHEAD < DT) v[d + AHEAD] = value_of(g, d + AHEAD);
                        acc[d] = mfma32<kVB>(v[d], part_of[g][e >> 1], acc[d]);
                        if (e >= 2 * kParts - 2 && g == 0) v[d] = value_of(1, d);  // (its last use was the product above)
                        if (g == 0) {
                            constexpr int PER = 8 / (kParts * DT);
#pragma unroll
                            for (int j = 8 + PER * n; j < 8 + PER * (n + 1); j++) {
                                weigh(j);
                                if (j & 1) halve(j >> 1);
                            }
                        } else {
                            look_ahead(n);
                        }
                        FENCE;
                    }
            }
        } else {
            // one block of 32 dims at a time: the smaller parts' sum has a scale of its own
#pragma unroll
            for (int d = 0; d < DT; d++) {
                f16v low;
#pragma unroll
                for (int i = 0; i < 16; i++) low[i] = 0.0f;
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    low = mfma32<kVB>(v[g], part_of[g][1], low);
                    look_ahead(2 * d + g);
                    FENCE;
                }
#pragma unroll
                for (int i = 0; i < 16; i++) acc[d][i] = fmaf(low[i], 1.0f / kUp, acc[d][i]);
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    acc[d] = mfma32<kVB>(v[g], part_of[g][0], acc[d]);
                    if (d + 1 < DT) v[g] = value_of(g, d + 1);
                    FENCE;
                }
            }
        }
        sum += part_sum;
        s = after;
        return top;
    };
    // Infinite or NaN values: a weight of 0 would carry them into rows that do not attend
    // to them, and a weight whose second number is 0 makes NaN of an infinite one.  So they
    // join the rows that attend to them here, and the products find zeros in their place.
    // (Looking for them in every tile, not in those alone that some row ends in, costs drafts
    // of ragged sequences 125 us, not 118, others 0 to 3 %.  Looking again, at all, where a
    // row is NaN at the end, costs more: its loop spills registers, 0 to 13 %.)
    // (Quantised values are looked at where not all rows attend to them: E4M3 ones are finite
    // or NaN, INT4 ones infinite by their row's minimum, which the products do not take.)
    auto settle = [&](int32_t tok, int buf) {
        char* values = tiles + (buf * 2 + 1) * RowsLds<D, NW>::kTileBytes;
        if (tg < wt)
            for (int r = 0; r < kTileTokens; r++) {
                if (((r >> 5) & (wt - 1)) != tg) continue;
                const bool in = r < lim - tok && (r & 15) < run_tokens[buf][r >> 4];
                if (FMT == FKV_PAGES_FP8_INT4) {
                    const float low = value_min[buf][r];
                    z += in && !(fabsf(low) < INFINITY) ? low : 0.0f;
                    continue;
                }
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const u2 w = *(const u2*)(values + value_place<D>(r, 4 * d + j) + 8 * hf);
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const uint32_t x = (w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu;
                            acc[d][4 * j + i] += in && any_not_finite<kVB>(x) ? (kVB ? bf2f(x) : h2f(x)) : 0.0f;
                        }
                    }
            }
        __syncthreads();
        if (FMT == FKV_PAGES_FP8_INT4) {
            if (tid < kTileTokens && !(fabsf(value_min[buf][tid]) < INFINITY)) value_scale[buf][tid] = value_min[buf][tid] = 0.0f;
        } else {
            for (int i = tid; i < RowsLds<D, NW>::kTileBytes / 8; i += 64 * kRowWaves) {
                const u2 w = *(const u2*)(values + 8 * i);
                *(u2*)(values + 8 * i) = u2{finite_or_zero<kVB>(w.x), finite_or_zero<kVB>(w.y)};
            }
        }
        __syncthreads();
    };

    // A tile's last step takes the next tile's first scores, so this is stored
    // before it; the other buffer is free once all waves are that far.
    f16v s;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; i++) s[i] = 0.0f;
    if (nt > 0) {
        fetch(begin);
        load(begin);
        store(begin, 0, 0);
        if (nt > 1) load(begin + kTileTokens);
        __syncthreads();
        if (tg < wt) {
            s = score(0, tg);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                factors(s, 0, tg, j);
                top = largest(top, max4(s, j));
            }
        }
    }
    for (int t = 0; t < nt; t++) {
        const int32_t tok = begin + t * kTileTokens;
        const int buf = t & 1;
        if (__builtin_amdgcn_readfirstlane(odd_tile[buf]) == t) settle(tok, buf);
        for (int j = wt; j <= kSubs; j += wt) {
            const bool last = j == kSubs;
            if (last && t + 1 < nt) {
                __syncthreads();
                store(tok + kTileTokens, t + 1, buf ^ 1);
                if (t + 2 < nt) load(tok + 2 * kTileTokens);
                __syncthreads();
            }
            const int sub = tg + j - wt;
            if (tg < wt && tok + 32 * sub < wave_most) {
                settle_scores(s, top, tok + 32 * sub, buf, sub);
                top = step(s, tok + 32 * sub, buf, sub, last ? buf ^ 1 : buf, last ? tg : sub + wt);
            }
        }
    }

    // The waves' sums meet in the LDS: 16 threads a row, D / 16 dims a thread.
    sum += wave_xor(sum, 32);
    z += wave_xor(z, 32);
    __syncthreads();
    float* num = (float*)tiles;
    if (tg < wt) {
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                *(f4*)(num + (wave * 32 + c) * (D + 4) + 32 * d + 8 * j + 4 * hf) =
                    f4{acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]};
        if (hf == 0) stat[wave][c][0] = m, stat[wave][c][1] = sum, stat[wave][c][2] = z;
    }
    __syncthreads();
    constexpr int N = D / 16;
    for (int r = tid >> 4; r < 32 * wr; r += kThreads / 16) {
        const int i = r >> 5, rr = r & 31, d0 = (tid & 15) * N;
        int b, l, hq;
        const int32_t lim = place(row0 + r, b, l, hq);
        const int64_t at = ((int64_t)b * a.Hq + hq) * a.L + l;
        if (lim < 0) {
            if (parts == 1 && a.lse && (tid & 15) == 0 && row0 + r < rows) a.lse[at] = -INFINITY;
            continue;
        }
        float top = kLowest, all = 0.0f, low = 0.0f, x[N] = {};
        for (int w = 0; w < wt; w++) top = fmaxf(top, stat[w * wr + i][rr][0]);
        for (int w = 0; w < wt; w++) {
            const float* s = stat[w * wr + i][rr];
            const float f = __builtin_amdgcn_exp2f(s[0] - top);
            all = fmaf(f, s[1], all);
            low = fmaf(f, s[2], low);
            const float* n = num + ((w * wr + i) * 32 + rr) * (D + 4) + d0;
#pragma unroll
            for (int j = 0; j < N; j++) x[j] = fmaf(f, n[j], x[j]);
        }
        if (FMT == FKV_PAGES_FP8_INT4) {
#pragma unroll
            for (int j = 0; j < N; j++) x[j] += low;
        }
        if (parts > 1) {
            float* out = a.records + (at * parts + (seq < 0 ? split : a.common.splits + split)) * (D + 4);
#pragma unroll
            for (int j = 0; j < N; j += 4) *(f4*)(out + d0 + j) = f4{x[j], x[j + 1], x[j + 2], x[j + 3]};
            if ((tid & 15) == 0) *(float2*)(out + D) = make_float2(top, all);
        } else {
            const float inv = all == 0.0f ? 0.0f : 1.0f / all;
            uint32_t o[N / 2];
#pragma unroll
            for (int j = 0; j < N / 2; j++) {
                const float u = x[2 * j] * inv, v = x[2 * j + 1] * inv;
                o[j] = BF ? round_pair_bf16(u, v) : (uint32_t)f2h(u) | ((uint32_t)f2h(v) << 16);
            }
            char* dst = a.out.data + 2 * (b * a.out.sb + hq * a.out.sh + l * a.out.sl + d0);
            if (N == 8) *(uint4*)dst = make_uint4(o[0], o[1], o[2 % (N / 2)], o[3 % (N / 2)]);
            else *(uint2*)dst = make_uint2(o[0], o[1]);
            if (a.lse && (tid & 15) == 0) a.lse[at] = (top + __builtin_amdgcn_logf(all)) * 0.69314718055994531f;
        }
    }
}

// The records of a row, in order: a wave a row, or four waves, each every fourth eight
// records, where there are more than kManyParts (65 records of 768 rows: 10.6 us and 7.6).
template <int D, bool BF, int WAVES>
__global__ void __launch_bounds__(256) paged_rows_join_kernel(RowsArgs a, int64_t n_rows) {
    constexpr int N = D / 64;
    __shared__ float part[WAVES][D + 2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t at = WAVES == 4 ? blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
    if (at >= n_rows) return;
    const int64_t bh = at / a.L;
    const int l = (int)(at - bh * a.L), b = (int)(bh / a.Hq), hq = (int)(bh - (int64_t)b * a.Hq);
    const int32_t lim = limit_of(a, b, l);
    if (lim < 0) {
        if (a.lse && threadIdx.x % (64 * WAVES) == 0) a.lse[at] = -INFINITY;
        return;
    }
    const int parts = a.common.splits + a.own.splits;
    const uint32_t own_chunk = a.even ? scalar_load(a.chunk, 0) : a.own.chunk, chunk = a.common.chunk;
    // (parts whose tokens begin below the row's end have a record)
    const int n_common = a.common.splits ? (int)min((uint32_t)a.common.splits, ((uint32_t)min(lim, a.shared) + chunk - 1) / chunk) : 0;
    const int n_own = lim > a.shared ? (int)min((uint32_t)a.own.splits, ((uint32_t)(lim - a.shared) + own_chunk - 1) / own_chunk) : 0;
    const int n = n_common + n_own;
    const float* rec = a.records + at * parts * (D + 4);
    float m = kLowest, sum = 0.0f, x[N] = {};
    constexpr int U = 8;  // records a step, their loads in flight together
    for (int i = WAVES == 4 ? wave * U : 0; i < n; i += WAVES * U) {
        float2 st[U];
        float v[U][N];
#pragma unroll
        for (int k = 0; k < U; k++) {
            const int r = min(i + k, n - 1);
            const float* p = rec + (r < n_common ? r : a.common.splits + r - n_common) * (D + 4);
            st[k] = *(const float2*)(p + D);
#pragma unroll
            for (int j = 0; j < N; j++) v[k][j] = p[64 * j + lane];
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < U; k++) top = fmaxf(top, st[k].x);
        const float f = __builtin_amdgcn_exp2f(m - top);
        m = top;
        sum *= f;
#pragma unroll
        for (int j = 0; j < N; j++) x[j] *= f;
#pragma unroll
        for (int k = 0; k < U; k++) {
            if (i + k < n) {
                const float w = __builtin_amdgcn_exp2f(st[k].x - m);
                sum = fmaf(w, st[k].y, sum);
#pragma unroll
                for (int j = 0; j < N; j++) x[j] = fmaf(w, v[k][j], x[j]);
            }
        }
    }
    if (WAVES == 4) {
        float* mine = part[wave];
        if (lane == 0) mine[D] = m, mine[D + 1] = sum;
#pragma unroll
        for (int j = 0; j < N; j++) mine[64 * j + lane] = x[j];
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int w = 0; w < WAVES; w++) m = fmaxf(m, part[w][D]);
        sum = 0.0f;
#pragma unroll
        for (int j = 0; j < N; j++) x[j] = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float f = __builtin_amdgcn_exp2f(part[w][D] - m);
            sum = fmaf(f, part[w][D + 1], sum);
#pragma unroll
            for (int j = 0; j < N; j++) x[j] = fmaf(f, part[w][64 * j + lane], x[j]);
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint16_t* out = (uint16_t*)a.out.data + b * a.out.sb + hq * a.out.sh + l * a.out.sl;
#pragma unroll
    for (int j = 0; j < N; j++) {
        const float y = x[j] * inv;
        out[64 * j + lane] = BF ? __builtin_bit_cast(uint16_t, (__bf16)y) : f2h(y);
    }
    if (a.lse && lane == 0) a.lse[at] = (m + __builtin_amdgcn_logf(sum)) * 0.69314718055994531f;
}

// ---------------------------------------------------------------------------
// launch
// ---------------------------------------------------------------------------

struct RowsPlan {
    RowParts common, own;
    int32_t shared, even, least;  // see even_parts()
    int waves;  // of a workgroup
    int64_t blocks, bytes;
};

// Workgroups and workspace of a call (a function of sizes alone).  How many parts
// the tokens are cut into is what a model of the time finds best: a workgroup
// takes kBegin for its beginning and end and a time per tile of tokens that grows
// with its rows (the cache's bytes, then the products) and where two share a CU, the
// chip has `slots` of them at once, and parts cost their join.  It knows of the rows and
// the format, not of the dims.  Against the best of 15 counts of parts its own takes 0 to
// 6 % more in 21 of 25 calls (one to 128 sequences, 64 and 128 dims, each format, with and
// without shared tokens, lengths equal and at random) and 12 to 23 % in 4: 20 sequences of
// fp16 pages behind 4K shared tokens 42 us, not 38; 32 of 64 dims in E4M3 behind 8K 40, not
// 32; 40 new tokens of 16 sequences to 4K 126, not 103 (bf16), 159, not 140 (INT4).
static RowsPlan plan_waves(const fkv_pages* p, int32_t Hq, int32_t B, int32_t L, int64_t shared, int64_t max_len, int waves,
                           float& best) {
    RowsPlan r;
    r.shared = (int32_t)shared;
    const int64_t G = Hq / p->H, own_rows = L * G, all_rows = B * own_rows;
    r.waves = waves;
    best = INFINITY;
    const int64_t tile = 16 * r.waves, slots = r.waves == 8 ? 256 : 512;
    auto part = [&](int64_t rows) {
        RowParts q;
        q.wr = rows > 128 && r.waves == 8 ? 8 : rows > 64 ? 4 : rows > 32 ? 2 : 1;
        q.tiles = (int32_t)cdiv(rows, 32 * q.wr);
        return q;
    };
    // us for a tile, of a workgroup of four waves as one of two on a CU or alone on it
    auto time = [&](const RowParts& q) {
        if (q.wr == 8) return 4.9f;
        if (q.wr == 4) return r.waves == 8 ? 3.7f : p->format == FKV_PAGES_FP8_INT4 ? 3.5f : 4.3f;
        return 2.8f;
    };
    auto time_alone = [&](const RowParts& q) {
        if (r.waves == 8) return time(q);
        if (q.wr == 4) return p->format == FKV_PAGES_FP8_INT4 ? 2.4f : 2.15f;
        return 1.6f;
    };
    r.own = part(own_rows);
    r.common = part(all_rows);
    if (!shared) r.common.tiles = 0;
    const int64_t own_tiles = cdiv(std::max<int64_t>(1, max_len - shared), tile), common_tiles = cdiv(shared, tile);
    const int64_t own_pieces = (int64_t)B * p->H * r.own.tiles, common_pieces = (int64_t)p->H * r.common.tiles;
    // a record of each row, written and read
    const float join = (float)((double)all_rows * p->H * (p->D + 4) * 8 / 4e6) + kJoinPart;
    r.common.splits = 0;
    r.even = r.least = 0;
    if (!shared && B > 4 && B <= kEvenSeqs && r.own.tiles == 1 && waves == 4 && own_pieces * 4 <= slots * 3) {
        // Few sequences, whose lengths differ: see even_parts().  Parts are not so short
        // that their records cost more than they gain
        r.even = (int32_t)(slots / p->H);
        r.least = std::max(1, (int32_t)std::sqrt((float)own_tiles * join / time(r.own)));
        r.own.splits = (int32_t)std::min<int64_t>(std::min(cdiv(own_tiles, r.least), cdiv(4 * r.even, B)), 64);
        // (short ones are not cut: 32 sequences of up to 128 tokens 11 us, cut 18; of up to 512 20 and 23)
        const float gain = (own_tiles - cdiv(own_tiles, r.own.splits)) * time_alone(r.own);
        if (gain <= kJoin + r.own.splits * join) r.even = 0, r.own.splits = 1;
    } else {
        const int64_t cut = shared ? common_tiles : own_tiles, most = std::min<int64_t>(cut, 64);
        for (int64_t n = 1, last = 0; n <= most; n++) {
            const int64_t of = cdiv(cut, n);  // tiles of a part
            if (of == last) continue;         // (fewer parts are as long)
            last = of;
            int64_t own_parts = n, common_parts = 0;
            float t, longest = 0;
            double work = 0;
            if (shared) {
                common_parts = cdiv(common_tiles, of);
                const int64_t blocks = common_pieces * common_parts;
                longest = kBegin + of * (blocks > 256 ? time(r.common) : time_alone(r.common));
                work = blocks * (kBegin + of * time(r.common));
                // (no longer than those; but no more than fill the chip, whose records cost more)
                own_parts = std::max<int64_t>(1, (int64_t)(own_tiles * time(r.own) / longest + 0.999f));
                own_parts = std::min(own_parts, std::max<int64_t>(16, cdiv(2 * slots, own_pieces)));
            }
            own_parts = cdiv(own_tiles, cdiv(own_tiles, own_parts));
            const float own_time = kBegin + cdiv(own_tiles, own_parts) * time(r.own);
            // (many sequences have lengths of their own: six tenths of max_len, say)
            work = (work + 0.6 * own_pieces * own_parts * own_time) / slots;
            if (shared) t = std::max(longest, (float)work);
            else if (B <= 4) t = cdiv(own_pieces * own_parts, slots) * own_time;
            else t = std::max((float)work, kBegin + cdiv(own_tiles, own_parts) * time_alone(r.own));
            if (common_parts + own_parts > 1) t += kJoin + (common_parts + own_parts) * join;
            if (t < best) {
                best = t;
                r.common.splits = (int32_t)common_parts;
                r.own.splits = (int32_t)own_parts;
            }
        }
    }
    r.common.chunk = (int32_t)(shared ? cdiv(common_tiles, r.common.splits) * tile : tile);
    r.own.chunk = (int32_t)(cdiv(own_tiles, r.own.splits) * tile);
    r.blocks = common_pieces * r.common.splits + (r.even ? (int64_t)p->H * r.even : own_pieces * r.own.splits);
    const int64_t parts = r.common.splits + r.own.splits;
    r.bytes = parts > 1 ? (int64_t)B * Hq * L * parts * (p->D + 4) * 4 + 16 : 0;
    return r;
}

// Many rows take workgroups of eight waves (100 new tokens of 4 heads over 16K: 59 us,
// with four 65; 64 of them the same).  Where many rows share tokens and few have their
// own, either may be better, and the model, which sees four waves 15 % slower than they
// are, decides: 128 sequences of up to 1K tokens of their own take 90 us with four and
// 110 with eight behind 4K shared tokens, 197 and 184 behind 32K.
static RowsPlan plan_rows(const fkv_pages* p, int32_t Hq, int32_t B, int32_t L, int64_t shared, int64_t max_len) {
    if (B == 1) shared = 0;  // (with nobody)
    max_len = std::min(max_len, kMostTokens);
    const int64_t own_rows = (int64_t)L * (Hq / p->H);
    float four, eight;
    if (own_rows > kFewRows) return plan_waves(p, Hq, B, L, shared, max_len, 8, eight);
    const RowsPlan r = plan_waves(p, Hq, B, L, shared, max_len, 4, four);
    if (!shared || B * own_rows <= kFewRows) return r;
    const RowsPlan wide = plan_waves(p, Hq, B, L, shared, max_len, 8, eight);
    return four <= 1.15f * eight ? r : wide;
}

static int check_rows(const char* who, const fkv_pages* p, int32_t Hq, int32_t B, int32_t L, int64_t shared, int64_t max_len) {
    const std::string w = who;
    if (int e = check_pages(who, p)) return e;
    if (B < 0 || B > kRowsMaxSeqs) return set_error(w + ": at most " + std::to_string(kRowsMaxSeqs) + " sequences");
    if (Hq < 1 || Hq % p->H) return set_error(w + ": query heads must be a multiple of the KV heads");
    if (L < 0 || (int64_t)B * L * Hq >= 1 << 28) return set_error(w + ": at most 2^28 rows of queries");
    if (max_len < 0) return set_error(w + ": negative max_len");
    if (shared < 0 || shared % p->page_size || shared > kMostTokens)
        return set_error(w + ": shared tokens must fill whole pages");
    return FKV_OK;
}

template <int D, int FMT, bool BF>
static int launch_rows(const RowsArgs& a, const RowsPlan& p, hipStream_t s) {
    const char* w = "fkv_paged_attn_rows";
    const bool once = a.shared == 0 && a.own.tiles == 1;  // (each token is read by one workgroup)
    if (int e = p.waves == 8 ? start_kernel(w, paged_rows_kernel<D, FMT, BF, 8, false>, (uint32_t)p.blocks, 512, s, a)
                : once       ? start_kernel(w, paged_rows_kernel<D, FMT, BF, 4, true>, (uint32_t)p.blocks, 256, s, a)
                             : start_kernel(w, paged_rows_kernel<D, FMT, BF, 4, false>, (uint32_t)p.blocks, 256, s, a)) return e;
    if (p.bytes == 0) return FKV_OK;
    const int64_t rows = (int64_t)a.B * a.Hq * a.L;
    if (a.common.splits + a.own.splits > kManyParts && rows < 1 << 24)  // (2^32 threads)
        return start_kernel(w, paged_rows_join_kernel<D, BF, 4>, (uint32_t)rows, 256, s, a, rows);
    return start_kernel(w, paged_rows_join_kernel<D, BF, 1>, (uint32_t)cdiv(rows, 4), 256, s, a, rows);
}

template <int D>
static int launch_rows_d(const RowsArgs& a, const RowsPlan& p, int format, bool bf, hipStream_t s) {
    if (format == FKV_PAGES_F16) return launch_rows<D, FKV_PAGES_F16, false>(a, p, s);
    if (format == FKV_PAGES_BF16) return launch_rows<D, FKV_PAGES_BF16, true>(a, p, s);
    if (format == FKV_PAGES_FP8 && bf) return launch_rows<D, FKV_PAGES_FP8, true>(a, p, s);
    if (format == FKV_PAGES_FP8) return launch_rows<D, FKV_PAGES_FP8, false>(a, p, s);
    if (bf) return launch_rows<D, FKV_PAGES_FP8_INT4, true>(a, p, s);
    return launch_rows<D, FKV_PAGES_FP8_INT4, false>(a, p, s);
}

}  // namespace fkv

using namespace fkv;

extern "C" {

int64_t fkv_paged_attn_rows_workspace(const fkv_pages* pages, int32_t Hq, int32_t B, int32_t L, int64_t shared,
                                      int64_t max_len) {
    if (int e = check_rows("fkv_paged_attn_rows_workspace", pages, Hq, B, L, shared, max_len)) return e;
    return plan_rows(pages, Hq, B, L, shared, max_len).bytes;
}

int fkv_paged_attn_rows(const fkv_pages* pages, const fkv_rows* query, int32_t q_dtype, int32_t Hq, int32_t B, int32_t L,
                        const int32_t* table, int32_t n_table, int64_t table_stride, const int32_t* lens,
                        int32_t lens_add, const int32_t* n_new, int64_t shared, int64_t max_len, float scale,
                        const fkv_rows* out, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* w = "fkv_paged_attn_rows";
    if (int e = check_rows(w, pages, Hq, B, L, shared, max_len)) return e;
    if (int e = check_table(w, table, n_table, table_stride, B)) return e;
    const int64_t cap = (int64_t)n_table * pages->page_size;
    if (cap > kMostTokens) return set_error(std::string(w) + ": more than 2^31 tokens a sequence");
    if (shared > cap) return set_error(std::string(w) + ": more shared tokens than the table holds");
    if (q_dtype != FKV_F16 && q_dtype != FKV_BF16) return set_error(std::string(w) + ": queries must be fp16 or bf16");
    if (pages->format <= FKV_PAGES_BF16 && (q_dtype == FKV_BF16) != (pages->format == FKV_PAGES_BF16))
        return set_error(std::string(w) + ": queries must have the 16-bit pages' type");
    if (!std::isfinite(scale)) return set_error(std::string(w) + ": scale must be finite");
    if (B == 0 || L == 0) return FKV_OK;
    if (!query || !query->data || !out || !out->data || !lens) return set_error(std::string(w) + ": NULL argument");
    for (const fkv_rows* r : {query, out})
        if ((uintptr_t)r->data & 15 || (r->stride_b | r->stride_h | r->stride_l) & 7)
            return set_error(std::string(w) + ": query and out must be 16-byte aligned, their strides multiples of 8");
    if ((uintptr_t)workspace & 15) return set_error(std::string(w) + ": workspace must be 16-byte aligned");
    const RowsPlan p = plan_rows(pages, Hq, B, L, shared, max_len);
    if (p.blocks > 0x7FFFFFFF / 512) return set_error(std::string(w) + ": more than 2^22 workgroups of rows");
    if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes))
        return set_error(std::string(w) + ": workspace of " + std::to_string(p.bytes) + " bytes needed");
    const RowsShape shape{B, Hq, L, pages->D, 2};
    if (int e = check_result_rows(w, "out", out, shape)) return e;
    // (a workgroup reads its rows' queries before it writes their results)
    if (int e = check_apart(w, "out, which is not the query, and the query", out, shape, query, shape, true)) return e;
    RowsArgs a;
    a.pg = page_view(pages);
    a.table = TableView{table, table_stride, n_table};
    a.q = RowsView{(char*)query->data, query->stride_b, query->stride_h, query->stride_l};
    a.out = RowsView{(char*)out->data, out->stride_b, out->stride_h, out->stride_l};
    a.lens = lens;
    a.n_new = n_new;
    a.lse = lse;
    a.records = (float*)workspace;
    a.chunk = p.even ? (int32_t*)((char*)workspace + p.bytes - 16) : nullptr;
    a.common = p.common;
    a.own = p.own;
    a.lens_add = lens_add;
    a.B = B;
    a.Hq = Hq;
    a.G = Hq / pages->H;
    a.L = L;
    a.shared = p.shared;
    a.tile = 16 * p.waves;
    a.even = p.even;
    a.least = p.least;
    a.scale = std::fabs(scale) * 1.4426950408889634f;
    a.q_sign = std::signbit(scale) ? 0x80008000u : 0;
    a.q_mask = ~0u;
    if (a.scale < 1e-37f) a.scale = 1.0f, a.q_mask = a.q_sign = 0;  // (scores that are all 0: -inf times 0 would not be)
    const bool bf = q_dtype == FKV_BF16;
    if (pages->D == 64) return launch_rows_d<64>(a, p, pages->format, bf, (hipStream_t)stream);
    return launch_rows_d<128>(a, p, pages->format, bf, (hipStream_t)stream);
}

}  // extern "C"
