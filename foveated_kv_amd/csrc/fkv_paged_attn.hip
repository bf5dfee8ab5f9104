// Attention of one new token per sequence over a paged KV cache.
//
// For each sequence b and KV head h, with the group's queries q_g and the
// cached rows k_t, v_t (t < len_b):
//   s_t = scale * q_g . k_t,   out_g = sum_t exp(s_t) v_t / sum_t exp(s_t),
// in one pass over the rows with the running maximum m and sum l of the
// softmax (in powers of two: exp(s) = 2^(s log2 e)).
//
// Bound: the cache's bytes.  Each row is read once for up to 16 query heads, or
// 32 of a long row (plan_of); the products run on the matrix cores, whose 16
// columns are heads:
//   S^T (16 tokens x 16 heads) = K (16 x 32 dims) Q^T,  v_mfma_f32_16x16x32
//   O^T (16 dims x 16 heads)  += V^T (16 x 32 tokens) P^T
// A lane of S^T holds four tokens of one head, which is where P^T's operand
// wants them once two 16-token tiles are taken as one 32-token step (the
// order of the 32 tokens within the product is free as long as V^T has the
// same), so the weights never cross lanes.  V^T's operand is made in
// registers: a lane loads 16 (8, 4) bytes of D / 16 neighbouring dims of its
// eight tokens -- 16 lanes a row, coalesced -- and pairs tokens by byte
// permutes.  Keys of 128 bytes a row and more go through the LDS, into which
// they are loaded whole lines at a time; the rest of it holds the waves' results
// at a row's end.
//
// Work: every (sequence, KV head) row is cut into tiles of 128 tokens (32 per
// wave), and all tiles (with a unit per row for its beginning and end) are
// dealt in equal runs to a fixed number of workgroups, whatever the lengths
// are; they are read on the device, so a captured launch serves a growing
// cache.  A row that ends up in several workgroups leaves one record (maximum,
// sum, numerators) per workgroup, joined by a second kernel in a fixed order.
//
// Measured: 4096 tokens of 64 sequences, 8 KV heads, bf16, 1.07 GB, 167 us with
// the join, 6.4 TB/s, over layers of 1.5 GB in turn, so that no cache holds one,
// as all times below; 16K tokens of 8 sequences, 537 MB, 88.  With three sets of
// 537 MB in turn, of which the last-level cache keeps a part, the kernel alone
// takes 81 us (6.6 TB/s).  64K tokens, fp8 / INT4, 105 MB: 21 us alone, of which
// about 5 are the chain lengths -> page ids -> first rows, and the rows' ends; the
// join 4 to 5 us.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "fkv_paged.h"

namespace fkv {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kMaxSeqs = 4096;
constexpr float kNegBig = -3.402823466e38f;  // running maximum before the first token: no score lies below it
// The running maximum follows a new one only when that exceeds it by more
// than 2^8: weights then reach 2^8 at most, which fp32 sums and 16-bit
// weights hold alike, and most steps need no rescaling and no reduction
// across lanes.
constexpr float kSlack = 8.0f;
// What the running maximum of fp16 pages stays below the scores': their largest
// weight is 2^7 to 2^15, so that small ones are as far as may be from the end of
// fp16's range.
template <int FMT>
constexpr float kBias = FMT == FKV_PAGES_F16 ? 7.0f : 0.0f;

struct AttnArgs {
    PageView pg;
    TableView table;
    const char* q;
    int64_t q_sb, q_sh;
    const int32_t* lens;
    char* out;
    float* lse;
    float* records;   // workspace: per workgroup two records
    int4* joins;      // workspace: per row (first workgroup, count, first slot, 0); count 0: nothing to join
    int32_t lens_add, B, Hq, G, HT, GT;  // HT passes of GT heads per KV head
    float scale;      // scale * log2(e)
};

// Lengths and page ids are the same for a whole wave: scalar loads, which do
// not wait behind the rows' vector loads.
typedef const __attribute__((address_space(4))) int32_t* scalar_ints;
__device__ inline int32_t scalar_load(const int32_t* p, int64_t i) { return ((scalar_ints)(uintptr_t)p)[i]; }

__device__ inline int32_t clamp_length(const AttnArgs& a, int32_t len) {
    const int64_t n = (int64_t)len + a.lens_add, cap = (int64_t)a.table.n * a.pg.page_size;  // (cap < 2^31)
    return (int32_t)(n < 0 ? 0 : n > cap ? cap : n);
}
__device__ inline int32_t length_of(const AttnArgs& a, int b) { return clamp_length(a, scalar_load(a.lens, b)); }
template <int NW>
__device__ inline int32_t tiles_of(int32_t len) { return (int32_t)(((uint32_t)len + 32 * NW - 1) / (32 * NW)); }

template <bool BF>
__device__ inline f4 mfma(u4 x, u4 y, f4 c) {
    if (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, x), __builtin_bit_cast(h8, y), c, 0, 0, 0);
}

// Two E4M3 codes (the chosen half of w) as two 16-bit numbers, exact.
template <bool BF>
__device__ inline uint32_t cvt_fp8(uint32_t w, bool hi) {
    if (BF) return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)
                                                   : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
    return as_u32(e4m3x2_to_h2(w, hi));
}

__device__ inline uint32_t bf16_pair(float a, float b) {
    const b2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
}

// Registers of one step: 32 tokens of a wave, as they were loaded.
template <int D, int FMT>
struct Step {
    static constexpr int RB = FMT <= FKV_PAGES_BF16 ? 2 * D : D;  // bytes of a key row
    static constexpr int KL = RB / 64;                            // 16-byte key loads per 16-token tile
    static constexpr bool LDS = RB >= 128;                        // keys go to the wave's part of the LDS
    // value bytes of a lane per token: D / 16 dims
    static constexpr int VB = FMT <= FKV_PAGES_BF16 ? D / 8 : FMT == FKV_PAGES_FP8 ? D / 16 : D / 32;
    u4 k[2][LDS ? 1 : KL];
    uint32_t v[8][VB < 4 ? 1 : VB / 4];
    uint32_t kx[2], vx[2];  // exponent bytes of the lane's four tokens per tile
    f4 sz[2][2];            // INT4: (scale, min) of the lane's four tokens
};

// Where the step's two 16-token tiles lie: row of the pages, and how many of
// the tile's tokens take part.
struct Place {
    int64_t row[2];
    int32_t n[2];
};

// Page ids of the two tiles that begin at tok and tok + 16 (0 past the end).
__device__ inline int2 ids_of(const int32_t* ids, int sh, int32_t tok, int32_t len) {
    int2 r = make_int2(0, 0);
    if (tok < len) r.x = scalar_load(ids, tok >> sh);
    if (tok + 16 < len) r.y = scalar_load(ids, (tok + 16) >> sh);
    return r;
}

__device__ inline Place place_of(const AttnArgs& a, int2 ids, int sh, int32_t tok, int32_t len, int h) {
    Place p;
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const int32_t left = len - tok - 16 * t;
        int32_t id = t ? ids.y : ids.x, n = left < 0 ? 0 : left > 16 ? 16 : left;
        if ((uint32_t)id >= (uint32_t)a.pg.n_pages) id = 0, n = 0;
        // a tile without tokens reads the first page, which is there
        const int32_t off = n > 0 ? (tok + 16 * t) & (a.pg.page_size - 1) : 0;
        p.row[t] = (((int64_t)id * a.pg.H + h) << sh) + off;
        p.n[t] = n;
    }
    return p;
}

// 16, 8, 4 or 2 bytes at a uniform base plus a lane's offset.  The cache is
// read once, so its lines are not kept.
template <typename T>
__device__ inline T load_at(const char* base, uint32_t off) {
    return __builtin_nontemporal_load((const T*)(base + off));
}

// Keys: the matrix instruction wants 16 bytes of each of 16 rows from 16
// neighbouring lanes, which a load into registers fetches as 64 lookups of 16
// bytes, and a row of 128 bytes or more line by line twice and more (INT4, D =
// 128: 2.0 requests to the L2 for a line, and loads that keep lines only moved
// others out).  A load into the LDS takes whole rows by neighbouring lanes, and
// leaves 16 to 64 registers free: 4096 tokens of 64 sequences 83.5 -> 71.7 us
// (INT4), 90.6 -> 88.4 (fp8), 168 -> 167 (bf16); 11003 tokens of 3 sequences,
// 4 KV heads, 15.1 -> 14.1, 15.1 -> 14.2 and 20.6 -> 19.0.  Rows of 64 bytes
// (E4M3, D = 64), 16 of which are neighbours anyway, keep to registers: 50.0 and
// 50.9 through the LDS (INT4), 50.6 and 50.4 (fp8).

// Where 16-byte chunk `chunk` of row `row` of a tile lies in the LDS: eight
// neighbouring lanes' reads of one chunk of eight rows fall on all banks.
template <int RB>
__device__ inline uint32_t key_at(int row, int chunk) { return row * RB + 16 * (chunk ^ (row & 7)); }

// 16 bytes a lane from a uniform base (of `size` bytes) plus a lane's and a
// uniform offset into 1024 bytes of LDS, streamed past the caches (2: nt).  (A
// buffer load: beside global loads into the LDS the compiler waits for all loads
// wherever it waits for one.)
__device__ inline void load_to_lds(char* lds, const char* base, int size, uint32_t off, int uniform_off) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, size, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, off, uniform_off, 0, 2);
}

template <int D, int FMT>
__device__ inline void load_keys(Step<D, FMT>& st, const AttnArgs& a, const Place& p, int g, int c, char* keys) {
    constexpr int RB = Step<D, FMT>::RB, KL = Step<D, FMT>::KL;
    if (FMT >= FKV_PAGES_FP8) {
#pragma unroll
        for (int t = 0; t < 2; t++) st.kx[t] = load_at<uint32_t>((const char*)a.pg.k_exp + p.row[t], 4 * g);
    }
    if constexpr (Step<D, FMT>::LDS) {
        constexpr int CHUNKS = RB / 16, ROWS = 64 / CHUNKS;  // of a row, and rows of a load
        const int lane = 16 * g + c, row = lane / CHUNKS, chunk = lane % CHUNKS;
        asm volatile("" ::: "memory");
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < KL; i++)
                load_to_lds(keys + 16 * RB * t + 1024 * i, a.pg.k + p.row[t] * RB, 16 * RB,
                            key_at<RB>(row + ROWS * i % 8, chunk) - ROWS * i % 8 * RB, 1024 * i);
        asm volatile("" ::: "memory");  // (the values' loads, which read_keys() counts, come behind these)
    } else {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < KL; i++) st.k[t][i] = load_at<u4>(a.pg.k + p.row[t] * RB, c * RB + 16 * g + 64 * i);
    }
}

template <int D, int FMT>
__device__ inline void load_values(Step<D, FMT>& st, const AttnArgs& a, const Place& p, int g, int c) {
    constexpr int VB = Step<D, FMT>::VB, RB = 16 * VB, VW = VB < 4 ? 1 : VB / 4;
    const uint32_t off = 4 * g * RB + VB * c;
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const char* base = a.pg.v + p.row[t] * RB;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t* w = st.v[4 * t + j];
            if (VB == 16) {
                const u4 x = load_at<u4>(base, off + j * RB);
                w[0] = x.x, w[1 % VW] = x.y, w[2 % VW] = x.z, w[3 % VW] = x.w;
            } else if (VB == 8) {
                const fkv_u2 x = load_at<fkv_u2>(base, off + j * RB);
                w[0] = x.x, w[1 % VW] = x.y;
            } else if (VB == 4) {
                w[0] = load_at<uint32_t>(base, off + j * RB);
            } else {
                w[0] = load_at<uint16_t>(base, off + j * RB);
            }
        }
        if (FMT == FKV_PAGES_FP8) st.vx[t] = load_at<uint32_t>(a.pg.v_scale + p.row[t], 4 * g);
        if (FMT == FKV_PAGES_FP8_INT4) {
            st.sz[t][0] = load_at<f4>(a.pg.v_scale + 8 * p.row[t], 32 * g);
            st.sz[t][1] = load_at<f4>(a.pg.v_scale + 8 * p.row[t], 32 * g + 16);
        }
    }
}

// The step's keys out of the LDS, once they are there.  Loads end in the order of
// their issue, so all but load_values()'s, which come next and are counted here,
// must be done; what else was issued since only makes the wait longer.
template <int D, int FMT>
__device__ inline void read_keys(const char* keys, u4 (&k)[2][Step<D, FMT>::KL], int g, int c) {
    constexpr int RB = Step<D, FMT>::RB;
    constexpr int kBehind = 2 * (4 + (FMT == FKV_PAGES_FP8 ? 1 : FMT == FKV_PAGES_FP8_INT4 ? 2 : 0));
    const uint32_t base = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)keys;
    const uint32_t a0 = base + key_at<RB>(c, g), a1 = base + key_at<RB>(c, g + 4);
    if constexpr (RB == 128) {
        asm volatile("s_waitcnt vmcnt(%6)\n\t"
                     "ds_read_b128 %0, %4\n\t"
                     "ds_read_b128 %1, %5\n\t"
                     "ds_read_b128 %2, %4 offset:2048\n\t"
                     "ds_read_b128 %3, %5 offset:2048\n\t"
                     "s_waitcnt lgkmcnt(0)"
                     : "=&v"(k[0][0]), "=&v"(k[0][1]), "=&v"(k[1][0]), "=&v"(k[1][1])
                     : "v"(a0), "v"(a1), "n"(kBehind)
                     : "memory");
    } else {
        asm volatile("s_waitcnt vmcnt(%10)\n\t"
                     "ds_read_b128 %0, %8\n\t"
                     "ds_read_b128 %1, %9\n\t"
                     "ds_read_b128 %2, %8 offset:128\n\t"
                     "ds_read_b128 %3, %9 offset:128\n\t"
                     "ds_read_b128 %4, %8 offset:4096\n\t"
                     "ds_read_b128 %5, %9 offset:4096\n\t"
                     "ds_read_b128 %6, %8 offset:4224\n\t"
                     "ds_read_b128 %7, %9 offset:4224\n\t"
                     "s_waitcnt lgkmcnt(0)"
                     : "=&v"(k[0][0]), "=&v"(k[0][1]), "=&v"(k[0][2]), "=&v"(k[0][3]), "=&v"(k[1][0]), "=&v"(k[1][1]),
                       "=&v"(k[1][2]), "=&v"(k[1][3])
                     : "v"(a0), "v"(a1), "n"(kBehind)
                     : "memory");
    }
}

// The wave's sums over its tokens.
template <int D>
struct Sums {
    f4 acc[D / 16];  // O^T: acc[dt][i] is dim_of(dt, 4 g + i) of head c
    float m, l, z;   // maximum of the head, the lane's part of the sum and of INT4's minima
};

// Scores of a step's 32 tokens, T tiles of 16 heads.
template <int D, int FMT, bool BF, int T>
__device__ inline void scores(const Step<D, FMT>& st, const u4 (&keys)[2][Step<D, FMT>::KL],
                              const u4 (&q)[T][D / 32], const Place& p, float scale, int g, float (&s)[T][8]) {
#pragma unroll
    for (int t = 0; t < 2; t++) {
        f4 r[T];
#pragma unroll
        for (int n = 0; n < T; n++) r[n] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
            u4 k;
            if (FMT <= FKV_PAGES_BF16) {
                k = keys[t][i % Step<D, FMT>::KL];
            } else {
                const u4 w = keys[t][i / 2 % Step<D, FMT>::KL];
                const uint32_t w0 = i & 1 ? w.z : w.x, w1 = i & 1 ? w.w : w.y;
                k = u4{cvt_fp8<BF>(w0, false), cvt_fp8<BF>(w0, true), cvt_fp8<BF>(w1, false), cvt_fp8<BF>(w1, true)};
            }
#pragma unroll
            for (int n = 0; n < T; n++) r[n] = mfma<BF>(k, q[n][i], r[n]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float f = scale;
            if (FMT >= FKV_PAGES_FP8) f = exp_byte((st.kx[t] >> (8 * i)) & 0xFF);
#pragma unroll
            for (int n = 0; n < T; n++) s[n][4 * t + i] = (FMT >= FKV_PAGES_FP8 ? r[n][i] * scale : r[n][i]) * f;
        }
    }
    if (p.n[0] < 16 || p.n[1] < 16) {  // (the same in all lanes)
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
            for (int n = 0; n < T; n++)
                if (4 * g + (j & 3) >= p.n[j >> 2]) s[n][j] = -INFINITY;
    }
}

template <int D, int FMT>
__device__ inline void mask_values(Step<D, FMT>& st, const Place& p, int g) {
    constexpr int VW = Step<D, FMT>::VB < 4 ? 1 : Step<D, FMT>::VB / 4;
    // a token that takes no part has weight 0, but its row may hold anything,
    // NaN among it
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const bool in = 4 * g + (j & 3) < p.n[j >> 2];
#pragma unroll
        for (int w = 0; w < VW; w++) st.v[j][w] = in ? st.v[j][w] : 0;
        if (FMT == FKV_PAGES_FP8 && !in) st.vx[j >> 2] &= ~(0xFFu << (8 * (j & 3)));
        if (FMT == FKV_PAGES_FP8_INT4 && !in) {
            st.sz[j >> 2][(j & 3) >> 1][2 * (j & 1)] = 0.0f;
            st.sz[j >> 2][(j & 3) >> 1][2 * (j & 1) + 1] = 0.0f;
        }
    }
}

// A weight enters as three 16-bit numbers, for which there are matrix
// instructions.
// bf16: their sum is the weight, all 24 bits of it, each being the upper half of
// what is left; they have the range that rows' scales need.  (Two, rounded, hold
// 16 bits; the third product costs 0 to 2 %: 64 sequences of 4096 tokens 167.1 us
// with either (bf16, D = 128), 88.5 and 88.6 (fp8), 71.8 and 72.3 (INT4), 50.2 and
// 51.4 (INT4, D = 64).)
// fp16, the type of the values that it is for: the weight cut off to fp16, and
// 2^10 times what that leaves, twice.  Large weights have 24 bits and small ones
// steps of 2^-44, which is 2^-51 of the row's largest; fp16 alone ends at 2^-24,
// and a token 14 to 24 nats above the others, with a value of zero, left 10 to
// no bits of theirs.  (Beside two parts of one scale: 64 sequences of 4096 tokens
// 167.0 us and 167.8, 11003 tokens of 3 19.0 and 19.6, 512 of one 7.6 and 8.0;
// D = 64 85.8, 86.2; 13.2, 13.5; 5.7, 5.9.  Values taken apart into bf16, for which
// weights are as above, cost 1 % and, 512 tokens of one sequence, 2.1 to 2.7 us.)
constexpr int kParts = 3;

// A tile's running maximum and the step's weights.
template <int D, int FMT>
__device__ inline void weigh(const Step<D, FMT>& st, const float (&s)[8], Sums<D>& u, u4 (&part)[kParts]) {
    float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    if (__any(top > u.m + (kSlack + kBias<FMT>))) {
        top = fmaxf(top, wave_xor(top, 16));
        top = fmaxf(top, wave_xor(top, 32));
        const float m = fmaxf(u.m, top - kBias<FMT>), f = __builtin_amdgcn_exp2f(u.m - m);
        u.m = m;
        u.l *= f;
        u.z *= f;
#pragma unroll
        for (int d = 0; d < D / 16; d++) u.acc[d] *= f;
    }
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        w[j] = __builtin_amdgcn_exp2f(s[j] - u.m);
        u.l += w[j];
    }
    if (FMT == FKV_PAGES_FP8) {
#pragma unroll
        for (int j = 0; j < 8; j++) w[j] *= exp_byte((st.vx[j >> 2] >> (8 * (j & 3))) & 0xFF);
    }
    if (FMT == FKV_PAGES_FP8_INT4) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            u.z = fmaf(w[j], st.sz[j >> 2][(j & 3) >> 1][2 * (j & 1) + 1], u.z);
            w[j] *= st.sz[j >> 2][(j & 3) >> 1][2 * (j & 1)];
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
#pragma unroll
        for (int i = 0; i < kParts; i++)
            part[i][j] = FMT == FKV_PAGES_F16 ? take_fp16(w[2 * j], w[2 * j + 1]) : take_bf16(w[2 * j], w[2 * j + 1]);
    }
}

// Weights, and O^T += V^T P^T.
template <int D, int FMT, int T>
__device__ inline void accumulate(const Step<D, FMT>& st, const float (&s)[T][8], Sums<D> (&u)[T]) {
    constexpr int DT = D / 16, VW = Step<D, FMT>::VB < 4 ? 1 : Step<D, FMT>::VB / 4;
    constexpr bool kBF = FMT != FKV_PAGES_F16;
    u4 part[T][kParts];
#pragma unroll
    for (int n = 0; n < T; n++) weigh<D, FMT>(st, s[n], u[n], part[n]);
    auto add = [&](int d, u4 v) {
#pragma unroll
        for (int n = 0; n < T; n++) {
            f4& acc = u[n].acc[d];
            if (kBF) {
#pragma unroll
                for (int i = 0; i < kParts; i++) acc = mfma<kBF>(v, part[n][i], acc);
            } else {
                f4 low = mfma<kBF>(v, part[n][2], f4{0.0f, 0.0f, 0.0f, 0.0f});
                low = mfma<kBF>(v, part[n][1], low * (1.0f / kUp));
#pragma unroll
                for (int i = 0; i < 4; i++) acc[i] = fmaf(low[i], 1.0f / kUp, acc[i]);
                acc = mfma<kBF>(v, part[n][0], acc);
            }
        }
    };
    if (FMT <= FKV_PAGES_BF16) {
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const uint32_t sel = d & 1 ? 0x07060302u : 0x05040100u;
            u4 v;
#pragma unroll
            for (int j = 0; j < 4; j++)
                v[j] = __builtin_amdgcn_perm(st.v[2 * j + 1][(d / 2) % VW], st.v[2 * j][(d / 2) % VW], sel);
            add(d, v);
        }
    } else {
        // E4M3 bytes: INT4 codes 0..15 are the E4M3 numbers code * 2^-9 (its
        // smallest eight are subnormal, the next eight have the same step)
#pragma unroll
        for (int q = 0; q < DT / 4; q++) {  // four dims: one dword of bytes per token
            uint32_t e[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (FMT == FKV_PAGES_FP8) e[j] = st.v[j][q % VW];
                else if (D == 128) e[j] = (st.v[j][0] >> (4 * q)) & 0x0F0F0F0Fu;
                else e[j] = (st.v[j][0] & 0x0F0Fu) | ((st.v[j][0] & 0xF0F0u) << 12);
            }
#pragma unroll
            for (int half = 0; half < 2; half++) {  // bytes 0, 1 and bytes 2, 3
                uint32_t pair[4];
#pragma unroll
                for (int j = 0; j < 4; j++)
                    pair[j] = __builtin_amdgcn_perm(e[2 * j + 1], e[2 * j], half ? 0x07030602u : 0x05010400u);
#pragma unroll
                for (int w2 = 0; w2 < 2; w2++) {
                    const u4 v = {cvt_fp8<true>(pair[0], w2), cvt_fp8<true>(pair[1], w2), cvt_fp8<true>(pair[2], w2),
                                  cvt_fp8<true>(pair[3], w2)};
                    add(4 * q + 2 * half + w2, v);
                }
            }
        }
    }
}

// LDS of a row's end: the waves' numerators, rows of D + 4 floats (the 16
// heads fall on different banks), and their statistics.
template <int D, int NW>
struct RowLds {
    float num[NW][16][D + 4];
    float stat[NW][16][3];
};

// Joins the waves' sums of one tile of heads in the LDS and writes the row's
// result (whole) or its record.  Every wave of the workgroup calls it.
template <int D, int FMT, bool BF, int NW>
__device__ inline void finish_row(const AttnArgs& a, Sums<D>& u, RowLds<D, NW>& lds, int b, int hrow, int tile,
                                  float* record) {
    constexpr int DT = D / 16;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    u.l += wave_xor(u.l, 16);
    u.l += wave_xor(u.l, 32);
    if (FMT == FKV_PAGES_FP8_INT4) {
        u.z += wave_xor(u.z, 16);
        u.z += wave_xor(u.z, 32);
    }
    if (g == 0) lds.stat[wave][c][0] = u.m, lds.stat[wave][c][1] = u.l, lds.stat[wave][c][2] = u.z;
    // acc[.][i] are the D / 16 dims of the lane's row 4 g + i, in the order in
    // which accumulate() takes them
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int d = 0; d < DT; d += 4)
            *(f4*)&lds.num[wave][c][DT * (4 * g + i) + d] = f4{u.acc[d][i], u.acc[d + 1][i], u.acc[d + 2][i], u.acc[d + 3][i]};
    __syncthreads();
    // 16 threads a head, D / 16 dims a thread
    const int head = threadIdx.x >> 4, of_row = 16 * tile + head, r = threadIdx.x & 15, d0 = r * DT;
    const int h = hrow / a.HT, g0 = (hrow - h * a.HT) * a.GT;
    if (head < 16 && of_row < a.GT && g0 + of_row < a.G) {
        float m = kNegBig, l = 0.0f, z = 0.0f, y[DT] = {}, x[DT];
#pragma unroll
        for (int w = 0; w < NW; w++) m = fmaxf(m, lds.stat[w][head][0]);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float* st = lds.stat[w][head];
            const float f = __builtin_amdgcn_exp2f(st[0] - m);
            l = fmaf(f, st[1], l);
            z = fmaf(f, st[2], z);
#pragma unroll
            for (int i = 0; i < DT; i += 4) {
                const f4 n = *(const f4*)&lds.num[w][head][d0 + i];
#pragma unroll
                for (int k = 0; k < 4; k++) y[i + k] = fmaf(f, n[k], y[i + k]);
            }
        }
#pragma unroll
        for (int i = 0; i < DT; i++) {
            // INT4: the even dims' nibbles (low) come first, then the odd ones'
            const int from = FMT == FKV_PAGES_FP8_INT4 ? (i >> 1) + (i & 1) * (DT / 2) : i;
            x[i] = FMT == FKV_PAGES_FP8_INT4 ? fmaf(y[from], 512.0f, z) : y[from];
        }
        if (record) {
            float* out = record + of_row * (D + 4);
#pragma unroll
            for (int i = 0; i < DT; i += 4) *(f4*)(out + d0 + i) = f4{x[i], x[i + 1], x[i + 2], x[i + 3]};
            if (r == 0) *(float2*)(out + D) = make_float2(m, l);
        } else {
            const int64_t at = (int64_t)b * a.Hq + h * a.G + g0 + of_row;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            uint32_t o[DT / 2];
#pragma unroll
            for (int i = 0; i < DT / 2; i++) {
                const float p = x[2 * i] * inv, q = x[2 * i + 1] * inv;
                o[i] = BF ? bf16_pair(p, q) : (uint32_t)f2h(p) | ((uint32_t)f2h(q) << 16);
            }
            char* dst = a.out + 2 * (at * D + d0);
            if (DT == 8) *(uint4*)dst = make_uint4(o[0], o[1], o[2 % (DT / 2)], o[3 % (DT / 2)]);
            else *(uint2*)dst = make_uint2(o[0], o[1]);
            if (a.lse && r == 0) a.lse[at] = (m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f;
        }
    }
    __syncthreads();
}

// Inclusive sums over the wave's lanes: by DPP within rows of 16, then from
// each row's last lane to the rows behind it.
__device__ inline int32_t wave_scan(int32_t v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1, 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2, 3
    return v;
}

// A row's units of work: its tiles, and kRowCost for what beginning and ending
// a row costs; they come first, unit kRowCost + t being tile t.
// (64 sequences of 0 to 8K tokens, 8 KV heads, fp8: 31.5 us with 1, 32.5 with
// 2, 39.9 with 0, where the workgroups with many short rows come last.)
constexpr int kRowCost = 1;
__device__ inline int32_t units_of(int32_t tiles) { return tiles > 0 ? tiles + kRowCost : 0; }

// The units dealt to the grid: the first `more` workgroups take base + 1 each,
// the others base, so that no two differ by more than one.
struct Deal {
    uint32_t base, more;
};
__device__ inline uint32_t first_unit(const Deal& d, uint32_t w) { return w * d.base + (w < d.more ? w : d.more); }
__device__ inline uint32_t owner_of(const Deal& d, uint32_t unit) {
    const uint32_t big = d.more * (d.base + 1);
    return unit < big ? unit / (d.base + 1) : d.more + (unit - big) / d.base;
}

// A workgroup's run of units: [begin, end) among all, beginning with unit u0 of
// row (b, hrow).  Every wave finds it by itself, 64 sequences a step.
struct Run {
    Deal deal;
    uint32_t begin, end;
    int32_t b, len, hrow, u0;
};

template <int NW>
__device__ inline Run run_of(const AttnArgs& a, uint32_t rows_per_seq) {
    const int lane = threadIdx.x & 63;
    auto length = [&](int b) { return b < a.B ? clamp_length(a, a.lens[b]) : 0; };
    auto units = [&](int32_t len) { return units_of(tiles_of<NW>(len)); };
    const int32_t len0 = length(lane), mine0 = units(len0), first = wave_scan(mine0);
    uint32_t total = __builtin_amdgcn_readlane(first, 63);
    for (int b = 64; b < a.B; b += 64) total += __builtin_amdgcn_readlane(wave_scan(units(length(b + lane))), 63);
    total *= rows_per_seq;  // (below 2^31, checked on the host)
    Run r;
    r.deal.base = total / gridDim.x;
    r.deal.more = total - r.deal.base * gridDim.x;
    r.begin = first_unit(r.deal, blockIdx.x);
    r.end = first_unit(r.deal, blockIdx.x + 1);
    r.b = r.len = r.hrow = r.u0 = 0;
    if (r.begin == r.end) return r;
    uint32_t before = 0;  // units per row of the sequences before the step's
    for (int b = 0; b < a.B; b += 64) {
        const int32_t len = b == 0 ? len0 : length(b + lane), mine = units(len);
        const int32_t sum = b == 0 ? first : wave_scan(mine);
        const uint64_t past = __ballot((before + sum) * rows_per_seq > r.begin);
        if (past) {
            const int at = __builtin_ctzll(past);
            const uint32_t n = __builtin_amdgcn_readlane(mine, at);
            const uint32_t in_seq = r.begin - (before + __builtin_amdgcn_readlane(sum, at) - n) * rows_per_seq;
            r.b = b + at;
            r.len = __builtin_amdgcn_readlane(len, at);
            r.hrow = (int32_t)(in_seq / n);
            r.u0 = (int32_t)(in_seq - r.hrow * n);
            break;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return r;
}

// NW waves of 32 tokens a step.  SPLIT: runs of tiles dealt to the grid's
// workgroups, see the file's head; else one workgroup per row.
template <int D, int FMT, bool BF, int NW, bool SPLIT, int T>
__global__ void __launch_bounds__(64 * NW) paged_attn_kernel(AttnArgs a) {
    constexpr int kStep = 32 * NW;
    __shared__ RowLds<D, NW> lds;
    __shared__ __attribute__((aligned(16))) char key_lds[NW][Step<D, FMT>::LDS ? 32 * Step<D, FMT>::RB : 16];
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    char* keys = key_lds[wave];
    const int rows_per_seq = a.pg.H * a.HT;
    const int sh = 31 - __builtin_clz((unsigned)a.pg.page_size);

    Run run;
    if (SPLIT) {
        run = run_of<NW>(a, rows_per_seq);  // (b = 0 of a table that may be empty where there is nothing to do)
    } else {
        run.b = blockIdx.x / rows_per_seq;
        run.hrow = blockIdx.x - run.b * rows_per_seq;
        run.begin = run.u0 = 0;
        run.len = length_of(a, run.b);
    }
    // the part of a row that is this workgroup's: units from u0 on, tiles
    // [t0, t1) of (b, hrow); none where the run ends before the first tile
    int b = run.b, hrow = run.hrow, u0 = run.u0, len = run.len, nt = tiles_of<NW>(len);
    uint32_t at = run.begin;
    int t0 = 0, t1 = nt;
    auto part = [&]() {
        t0 = u0 > kRowCost ? u0 - kRowCost : 0;
        const int left = (int)(run.end - at) + u0 - kRowCost;
        t1 = left < nt ? left : nt;
    };
    if (SPLIT) part();
    bool work = !SPLIT || (at < run.end && t0 < t1);
    int h = hrow / a.HT, g0 = (hrow - h * a.HT) * a.GT;
    const int32_t* ids = a.table.ids + b * a.table.stride;

    Step<D, FMT> st;
    int32_t tok = t0 * kStep + 32 * wave;
    // (one workgroup per row: the first ids are loaded beside the length)
    Place place = place_of(a, ids_of(ids, sh, tok, SPLIT ? len : a.table.n << sh), sh, tok, len, h);
    if (work) {
        load_keys(st, a, place, g, c, keys);
        load_values(st, a, place, g, c);
    }

    while (work) {
        u4 q[T][D / 32];
#pragma unroll
        for (int n = 0; n < T; n++) {
            const int of_row = 16 * n + c;
            const bool real = of_row < a.GT && g0 + of_row < a.G;
            const char* row = a.q + 2 * (b * a.q_sb + (int64_t)(h * a.G + g0 + (real ? of_row : 0)) * a.q_sh);
#pragma unroll
            for (int i = 0; i < D / 32; i++) {
                const int d = FMT <= FKV_PAGES_BF16 ? 32 * i + 8 * g : 64 * (i / 2) + 16 * g + 8 * (i & 1);
                const u4 x = *(const u4*)(row + 2 * d), none = {0, 0, 0, 0};
                q[n][i] = real ? x : none;
            }
        }
        Sums<D> u[T];
#pragma unroll
        for (int n = 0; n < T; n++) {
            u[n].m = kNegBig, u[n].l = 0.0f, u[n].z = 0.0f;
#pragma unroll
            for (int d = 0; d < D / 16; d++) u[n].acc[d] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        // One step; with `more`, the next one's ids first, its keys into the
        // same place once these are used, its values once these are: 8 KB to 16
        // KB of a wave in flight at D = 128 in 16 bits.  (The last step
        // stands apart: loads under a condition inside the loop made every wait
        // in it one for all loads, and read_keys() counts on those of the step.
        // Keys in registers then, 16K tokens of 8 sequences took 83.5 us, not 81.9,
        // and a second set of registers, loaded a step further ahead, gained 2 %
        // there and lost 7 to 20 % with quantised rows.)
        auto step = [&](bool more) {
            u4 k[2][Step<D, FMT>::KL];
            if constexpr (Step<D, FMT>::LDS) {
                read_keys<D, FMT>(keys, k, g, c);
            } else {
#pragma unroll
                for (int i = 0; i < 2 * Step<D, FMT>::KL; i++) k[i & 1][i / 2] = st.k[i & 1][i / 2];
            }
            tok += kStep;
            const int2 id = more ? ids_of(ids, sh, tok, len) : make_int2(0, 0);
            const Place p = place;
            float s[T][8];
            scores<D, FMT, BF, T>(st, k, q, p, a.scale, g, s);
            if (more) {
                place = place_of(a, id, sh, tok, len, h);
                load_keys(st, a, place, g, c, keys);
            }
            if (p.n[0] < 16 || p.n[1] < 16) mask_values(st, p, g);
            accumulate<D, FMT, T>(st, s, u);
            if (more) load_values(st, a, place, g, c);
        };
        for (int t = t0; t < t1 - 1; t++) step(true);
        if (t0 < t1) step(false);
        // a row that begins and ends here is done; of another one the record
        // goes to this workgroup's first slot, or to its second one where the
        // row begins after the run does
        const bool whole = t0 == 0 && t1 == nt;
        float* record = nullptr;
        if (SPLIT) {
            const int slot = at > run.begin ? 1 : 0;
            if (t0 == 0 && tid == 0) {
                // (no further than the records go, whatever was done to lens meanwhile)
                const uint32_t last = min(owner_of(run.deal, at - u0 + kRowCost + nt - 1), gridDim.x - 1);
                a.joins[(int64_t)b * rows_per_seq + hrow] =
                    make_int4(blockIdx.x, whole ? 0 : (int)(last - blockIdx.x + 1), slot, 0);
            }
            if (!whole) record = a.records + ((int64_t)blockIdx.x * 2 + slot) * a.GT * (D + 4);
        }
        const int done_b = b, done_row = hrow;
        if (SPLIT) {
            // the next row's first loads before this one's end
            at += t1 + kRowCost - u0;
            u0 = 0;
            work = at < run.end;
            if (work) {
                if (++hrow == rows_per_seq) {
                    hrow = 0;
                    // (units are left, so a sequence with tokens follows)
                    do len = ++b < a.B ? length_of(a, b) : 1; while (len == 0);
                    if (b >= a.B) break;  // (lens changed under the call)
                    nt = tiles_of<NW>(len);
                    ids = a.table.ids + b * a.table.stride;
                }
                part();
                work = t0 < t1;
                h = hrow / a.HT, g0 = (hrow - h * a.HT) * a.GT;
                tok = 32 * wave;
                place = place_of(a, ids_of(ids, sh, tok, len), sh, tok, len, h);
                load_keys(st, a, place, g, c, keys);
                load_values(st, a, place, g, c);
            }
        }
#pragma unroll
        for (int n = 0; n < T; n++) finish_row<D, FMT, BF, NW>(a, u[n], lds, done_b, done_row, n, record);
        if (!SPLIT) return;
    }

    // sequences without tokens: their result is written here
    for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
        if (length_of(a, b) > 0) continue;
        for (int i = tid; i < a.Hq * D / 2; i += 64 * NW) ((uint32_t*)a.out)[(int64_t)b * a.Hq * (D / 2) + i] = 0;
        if (a.lse)
            for (int i = tid; i < a.Hq; i += 64 * NW) a.lse[(int64_t)b * a.Hq + i] = -INFINITY;
        for (int i = tid; i < rows_per_seq; i += 64 * NW) a.joins[(int64_t)b * rows_per_seq + i] = make_int4(0, 0, 0, 0);
    }
}

// One row's records, in order: 4 / HPW waves a head.
template <int D, bool BF, int HPW>
__global__ void __launch_bounds__(256) paged_join_kernel(AttnArgs a, int n_rows) {
    constexpr int PARTS = 4 / HPW, N = D / 64;
    __shared__ float part[4][D + 2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = blockIdx.y * HPW + wave / PARTS, w0 = wave % PARTS;
    const int rows_per_seq = a.pg.H * a.HT;
    for (int row = blockIdx.x; row < n_rows; row += gridDim.x) {
        const int4 j = {((scalar_ints)(uintptr_t)a.joins)[4 * row], ((scalar_ints)(uintptr_t)a.joins)[4 * row + 1],
                        ((scalar_ints)(uintptr_t)a.joins)[4 * row + 2], 0};
        if (j.y == 0) continue;  // (the same for the whole workgroup)
        const int b = row / rows_per_seq, hrow = row - b * rows_per_seq;
        const int h = hrow / a.HT, g0 = (hrow - h * a.HT) * a.GT;
        const bool real = head < a.GT && g0 + head < a.G;
        const int64_t rec = (int64_t)a.GT * (D + 4);
        float m = kNegBig, l = 0.0f, x[N] = {};
        if (real) {
            auto record = [&](int i) {
                return a.records + ((int64_t)(j.x + i) * 2 + (i == 0 ? j.z : 0)) * rec + head * (D + 4);
            };
            // eight records a step, their loads in flight together
            for (int i = w0; i < j.y; i += 8 * PARTS) {
                float2 st[8];
                float v[8][N];
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const bool in = i + k * PARTS < j.y;
                    const float* r = record(in ? i + k * PARTS : i);
                    st[k] = *(const float2*)(r + D);
                    if (!in) st[k] = make_float2(kNegBig, 0.0f);
#pragma unroll
                    for (int n = 0; n < N; n++) v[k][n] = r[64 * n + lane];
                }
                float top = m;
#pragma unroll
                for (int k = 0; k < 8; k++) top = fmaxf(top, st[k].x);
                const float f = __builtin_amdgcn_exp2f(m - top);
                m = top;
                l *= f;
#pragma unroll
                for (int n = 0; n < N; n++) x[n] *= f;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    // (a record past the end has weight 0 by its count, not by its
                    // maximum, which may be the others' too)
                    const float w = i + k * PARTS < j.y ? __builtin_amdgcn_exp2f(st[k].x - m) : 0.0f;
                    l = fmaf(w, st[k].y, l);
#pragma unroll
                    for (int n = 0; n < N; n++) x[n] = fmaf(w, v[k][n], x[n]);
                }
            }
        }
        if (PARTS > 1) {
#pragma unroll
            for (int n = 0; n < N; n++) part[wave][64 * n + lane] = x[n];
            if (lane == 0) part[wave][D] = m, part[wave][D + 1] = l;
            __syncthreads();
            const int base = wave - w0;
            m = kNegBig;
#pragma unroll
            for (int i = 0; i < PARTS; i++) m = fmaxf(m, part[base + i][D]);
            l = 0.0f;
#pragma unroll
            for (int n = 0; n < N; n++) x[n] = 0.0f;
#pragma unroll
            for (int i = 0; i < PARTS; i++) {
                const float f = __builtin_amdgcn_exp2f(part[base + i][D] - m);
                l = fmaf(f, part[base + i][D + 1], l);
#pragma unroll
                for (int n = 0; n < N; n++) x[n] = fmaf(f, part[base + i][64 * n + lane], x[n]);
            }
            __syncthreads();
        }
        if (real && w0 == 0) {
            const int64_t at = (int64_t)b * a.Hq + h * a.G + g0 + head;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
            for (int n = 0; n < N; n++) {
                const float y = x[n] * inv;
                ((uint16_t*)a.out)[at * D + 64 * n + lane] =
                    BF ? __builtin_bit_cast(uint16_t, (__bf16)y) : f2h(y);
            }
            if (a.lse && lane == 0) a.lse[at] = (m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f;
        }
    }
}

// ---------------------------------------------------------------------------
// launch
// ---------------------------------------------------------------------------

struct AttnPlan {
    int G, tiles, HT, GT, blocks;
    bool split;
    int64_t rows, records_at, bytes;
};

// Waves of a workgroup.  (Eight waves and half the workgroups: 11003 tokens of
// 3 sequences 21 us, not 19; one row of 512 tokens 7.8 us, not 7.3: a row's
// time is what one CU can load.)
constexpr int kAttnWaves = 4;
// Two workgroups per CU, each with its part of all rows.  (Three: 4096 tokens of
// 64 sequences 173.8 us, not 167.6 (bf16), 75.8 and 71.8 (INT4); 11003 tokens of
// 3 sequences 23.3 and 18.9.)
constexpr int kAttnGroups = 512;
// Rows up to this long are not split: one launch, no records.  512 tokens of
// one sequence's 8 KV heads 7.6 us and split 9.1 (bf16, D = 128), 8.0 and 9.6
// (fp16), 6.0 and 8.0 (fp16, 2 heads of 64 dims), of 64 sequences 22.2 and 22.0;
// 1024 tokens of one sequence 11.7 us and split 9.3.
constexpr int64_t kWholeRows = 512;
// Twice as long with as many rows as this, which then keep enough of the chip
// busy: 1024 tokens of 16 sequences 15.6 us and split 19.0 (bf16), 12.8 and 13.8
// (fp8), of 24 sequences with 5 KV heads 15.7 and 18.2, lengths at random up to
// 1024 13.7 and 14.0; where one sequence has 1024 and the others 128, 12.6 and
// 11.4.  8 sequences: 13.9 and 13.5.  (2048 tokens of 32 sequences 43.1 and 48.8,
// but with one that is longer than the others 22.5 and 15.7.)
constexpr int64_t kManyRows = 96;

// Workgroups and workspace of a call (a function of sizes alone).
static AttnPlan plan_of(const fkv_pages* p, int32_t Hq, int32_t B, int64_t max_len) {
    AttnPlan r;
    r.G = Hq / p->H;
    max_len = std::min(max_len, kMostTokens);
    const int64_t rows16 = (int64_t)B * p->H * ((r.G + 15) / 16);
    r.split = max_len > (rows16 >= kManyRows ? 2 * kWholeRows : kWholeRows);
    // Groups of more than 16 heads: two tiles of heads a pass over the rows.  32
    // heads on each of 2 KV heads, 16K tokens of 16 sequences, D = 128: 53 us and
    // 81 with one (fp16), 36.5 and 43.5 (fp8), 35.3 and 39.3 (INT4; 17 heads, 2000
    // tokens, 4 KV heads 18.3 and 17.0).  Not for rows that are not split, whose
    // time is a workgroup's (64 heads, 400 tokens of 32 sequences 9.9 us, 7.7 with
    // one), nor for quantised rows of 64 dims, whose second pass costs what the
    // second tile does (71 heads, 8K tokens of 8 sequences 15.8, 14.9 with one).
    r.tiles = r.G > 16 && r.split && (p->D == 128 || p->format <= FKV_PAGES_BF16) ? 2 : 1;
    r.HT = (r.G + 16 * r.tiles - 1) / (16 * r.tiles);
    r.GT = (r.G + r.HT - 1) / r.HT;
    r.rows = (int64_t)B * p->H * r.HT;
    const int64_t tiles = r.rows * std::max<int64_t>(1, cdiv(max_len, 32 * kAttnWaves));
    r.blocks = (int)(r.split ? std::min<int64_t>(tiles, kAttnGroups) : r.rows);
    r.records_at = round_up(16 * r.rows, 256);
    r.bytes = r.split ? r.records_at + (int64_t)r.blocks * 2 * r.GT * (p->D + 4) * 4 : 0;
    return r;
}

static int check_attn(const char* who, const fkv_pages* p, int32_t Hq, int32_t B, int64_t max_len) {
    const std::string w = who;
    if (int e = check_pages(who, p)) return e;
    if (B < 0 || B > kMaxSeqs) return set_error(w + ": at most " + std::to_string(kMaxSeqs) + " sequences");
    if (Hq < 1 || Hq % p->H) return set_error(w + ": query heads must be a multiple of the KV heads");
    if (max_len < 0) return set_error(w + ": negative max_len");
    return FKV_OK;
}

template <int D, int FMT, bool BF>
static int launch_attn(const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
    const char* w = "fkv_paged_attn";
    constexpr int threads = 64 * kAttnWaves;
    if (!p.split)
        return start_kernel(w, paged_attn_kernel<D, FMT, BF, kAttnWaves, false, 1>, p.blocks, threads, s, a);
    auto kernel = paged_attn_kernel<D, FMT, BF, kAttnWaves, true, 1>;
    if constexpr (D == 128 || FMT <= FKV_PAGES_BF16) {
        if (p.tiles == 2) kernel = paged_attn_kernel<D, FMT, BF, kAttnWaves, true, 2>;
    }
    if (int e = start_kernel(w, kernel, p.blocks, threads, s, a)) return e;
    const int rows = (int)std::min<int64_t>(p.rows, 1024);
    if (p.rows * p.GT <= 1024)
        return start_kernel(w, paged_join_kernel<D, BF, 1>, dim3(rows, p.GT), 256, s, a, (int)p.rows);
    return start_kernel(w, paged_join_kernel<D, BF, 4>, dim3(rows, (p.GT + 3) / 4), 256, s, a, (int)p.rows);
}

template <int D>
static int launch_attn_d(const AttnArgs& a, const AttnPlan& p, int format, bool bf, hipStream_t s) {
    if (format == FKV_PAGES_F16) return launch_attn<D, FKV_PAGES_F16, false>(a, p, s);
    if (format == FKV_PAGES_BF16) return launch_attn<D, FKV_PAGES_BF16, true>(a, p, s);
    if (format == FKV_PAGES_FP8 && bf) return launch_attn<D, FKV_PAGES_FP8, true>(a, p, s);
    if (format == FKV_PAGES_FP8) return launch_attn<D, FKV_PAGES_FP8, false>(a, p, s);
    if (bf) return launch_attn<D, FKV_PAGES_FP8_INT4, true>(a, p, s);
    return launch_attn<D, FKV_PAGES_FP8_INT4, false>(a, p, s);
}

}  // namespace fkv

using namespace fkv;

extern "C" {

int64_t fkv_paged_attn_workspace(const fkv_pages* pages, int32_t Hq, int32_t B, int64_t max_len) {
    if (int e = check_attn("fkv_paged_attn_workspace", pages, Hq, B, max_len)) return e;
    return plan_of(pages, Hq, B, max_len).bytes;
}

int fkv_paged_attn(const fkv_pages* pages, const fkv_rows* query, int32_t q_dtype, int32_t Hq, int32_t B,
                   const int32_t* table, int32_t n_table, int64_t table_stride, const int32_t* lens,
                   int32_t lens_add, int64_t max_len, float scale, void* out, float* lse, void* workspace,
                   int64_t workspace_bytes, void* stream) {
    const char* w = "fkv_paged_attn";
    if (int e = check_attn(w, pages, Hq, B, max_len)) return e;
    if (int e = check_table(w, table, n_table, table_stride, B)) return e;
    if ((int64_t)n_table * pages->page_size > kMostTokens) return set_error(std::string(w) + ": more than 2^31 tokens a sequence");
    if (q_dtype != FKV_F16 && q_dtype != FKV_BF16) return set_error(std::string(w) + ": queries must be fp16 or bf16");
    if (pages->format <= FKV_PAGES_BF16 && (q_dtype == FKV_BF16) != (pages->format == FKV_PAGES_BF16))
        return set_error(std::string(w) + ": queries must have the 16-bit pages' type");
    if (!std::isfinite(scale)) return set_error(std::string(w) + ": scale must be finite");
    if (B == 0) return FKV_OK;
    if (!query || !query->data || !out || !lens) return set_error(std::string(w) + ": NULL argument");
    if (((uintptr_t)query->data | (uintptr_t)out | (uintptr_t)workspace) & 15 || (query->stride_b | query->stride_h) & 7)
        return set_error(std::string(w) + ": query, out and workspace must be 16-byte aligned, query strides multiples of 8");
    const AttnPlan p = plan_of(pages, Hq, B, max_len);
    if (p.rows >= 1 << 24) return set_error(std::string(w) + ": more than 2^24 rows of heads");
    if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes))
        return set_error(std::string(w) + ": workspace of " + std::to_string(p.bytes) + " bytes needed");
    if (p.rows * (cdiv((int64_t)n_table * pages->page_size, 32 * kAttnWaves) + 1) > 0x7FFFFFFF)
        return set_error(std::string(w) + ": the tables hold more than 2^31 tiles of 128 tokens over all heads");
    const RowsShape heads{B, Hq, 1, pages->D, 2};
    const fkv_rows result{out, (int64_t)Hq * pages->D, pages->D, 0};
    if (int e = check_apart(w, "out, which is not the query, and the query", &result, heads, query, heads, true)) return e;
    AttnArgs a;
    a.pg = page_view(pages);
    a.table = TableView{table, table_stride, n_table};
    a.q = (const char*)query->data;
    a.q_sb = query->stride_b;
    a.q_sh = query->stride_h;
    a.lens = lens;
    a.out = (char*)out;
    a.lse = lse;
    a.joins = (int4*)workspace;
    a.records = (float*)((char*)workspace + p.records_at);
    a.lens_add = lens_add;
    a.B = B;
    a.Hq = Hq;
    a.G = p.G;
    a.HT = p.HT;
    a.GT = p.GT;
    a.scale = scale * 1.4426950408889634f;
    const bool bf = q_dtype == FKV_BF16;
    if (pages->D == 64) return launch_attn_d<64>(a, p, pages->format, bf, (hipStream_t)stream);
    return launch_attn_d<128>(a, p, pages->format, bf, (hipStream_t)stream);
}

}  // extern "C"
