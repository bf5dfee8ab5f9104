// Attention of one new token per sequence over a paged KV cache.
//
// For each sequence b and KV head h, with the group's queries q_g and the
// cached rows k_t, v_t (t < len_b):
//   s_t = scale * q_g . k_t,   out_g = sum_t exp(s_t) v_t / sum_t exp(s_t),
// in one pass over the rows with the running maximum m and sum l of the
// softmax (in powers of two: exp(s) = 2^(s log2 e)).
//
// Bound: the cache's bytes.  Each row is read once for up to 16 query heads;
// the products run on the matrix cores, whose 16 columns are those heads:
//   S^T (16 tokens x 16 heads) = K (16 x 32 dims) Q^T,  v_mfma_f32_16x16x32
//   O^T (16 dims x 16 heads)  += V^T (16 x 32 tokens) P^T
// A lane of S^T holds four tokens of one head, which is where P^T's operand
// wants them once two 16-token tiles are taken as one 32-token step (the
// order of the 32 tokens within the product is free as long as V^T has the
// same), so the weights never cross lanes.  V^T's operand is made in
// registers: a lane loads 16 (8, 4) bytes of D / 16 neighbouring dims of its
// eight tokens -- 16 lanes a row, coalesced -- and pairs tokens by byte
// permutes.  The LDS holds nothing but the waves' results at a row's end.
//
// Work: every (sequence, head) row is cut into tiles of 128 tokens (32 per
// wave), all tiles are dealt in equal runs to a fixed number of workgroups,
// whatever the lengths are; they are read on the device, so a captured launch
// serves a growing cache.  A row that ends up in several workgroups leaves
// one record (maximum, sum, numerators) per workgroup, joined by a second
// kernel in a fixed order.
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

constexpr int kAttnWaves = 4;
constexpr int kAttnTile = 32 * kAttnWaves;  // tokens of a workgroup's step
constexpr int kMaxSeqs = 4096;
constexpr float kNegBig = -1e30f;  // running maximum before the first token
// The running maximum follows a new one only when that exceeds it by more
// than 2^8: weights then reach 2^8 at most, which fp32 sums and 16-bit
// weights hold alike, and most steps need no rescaling and no reduction
// across lanes.
constexpr float kSlack = 8.0f;

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
    int32_t lens_add, B, Hq, G, HT, GT;  // HT head tiles of GT heads per KV head
    float scale;      // scale * log2(e)
};

__device__ inline int64_t length_of(const AttnArgs& a, int b) {
    int64_t n = (int64_t)a.lens[b] + a.lens_add;
    const int64_t cap = (int64_t)a.table.n * a.pg.page_size;
    return n < 0 ? 0 : n > cap ? cap : n;
}
__device__ inline int32_t tiles_of(const AttnArgs& a, int b) {
    return (int32_t)((length_of(a, b) + kAttnTile - 1) / kAttnTile);
}

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
    static constexpr int KL = FMT <= FKV_PAGES_BF16 ? D / 32 : D / 64;  // 16-byte key loads per 16-token tile
    // value bytes of a lane per token: D / 16 dims
    static constexpr int VB = FMT <= FKV_PAGES_BF16 ? D / 8 : FMT == FKV_PAGES_FP8 ? D / 16 : D / 32;
    u4 k[2][KL];
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

__device__ inline Place place_of(const AttnArgs& a, const int32_t* ids, int64_t tok, int64_t len, int h) {
    Place p;
    const int sh = 31 - __builtin_clz((unsigned)a.pg.page_size);
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const int64_t first = tok + 16 * t;
        int32_t n = (int32_t)(len - first < 16 ? len - first : 16);
        int32_t id = 0;
        if (n > 0) {
            id = ids[first >> sh];
            if ((uint32_t)id >= (uint32_t)a.pg.n_pages) id = 0, n = 0;
        } else {
            n = 0;
        }
        // a tile without tokens reads the first page, which is there
        p.row[t] = (((int64_t)id * a.pg.H + h) << sh) + (n > 0 ? (first & (a.pg.page_size - 1)) : 0);
        p.n[t] = n;
    }
    return p;
}

template <int D, int FMT>
__device__ inline void load_keys(Step<D, FMT>& st, const AttnArgs& a, const Place& p, int g, int c) {
    constexpr int RB = FMT <= FKV_PAGES_BF16 ? 2 * D : D;  // bytes of a key row
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const char* row = a.pg.k + (p.row[t] + c) * RB + 16 * g;
#pragma unroll
        for (int i = 0; i < Step<D, FMT>::KL; i++) st.k[t][i] = *(const u4*)(row + 64 * i);
        if (FMT >= FKV_PAGES_FP8) st.kx[t] = *(const uint32_t*)(a.pg.k_exp + p.row[t] + 4 * g);
    }
}

template <int D, int FMT>
__device__ inline void load_values(Step<D, FMT>& st, const AttnArgs& a, const Place& p, int g, int c) {
    constexpr int VB = Step<D, FMT>::VB, RB = 16 * VB;
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const char* base = a.pg.v + (p.row[t] + 4 * g) * RB + VB * c;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t* w = st.v[4 * t + j];
            const char* at = base + j * RB;
            if (VB == 16) {
                const uint4 x = *(const uint4*)at;
                w[0] = x.x, w[1 % (VB < 4 ? 1 : VB / 4)] = x.y;
                w[2 % (VB < 4 ? 1 : VB / 4)] = x.z, w[3 % (VB < 4 ? 1 : VB / 4)] = x.w;
            } else if (VB == 8) {
                const uint2 x = *(const uint2*)at;
                w[0] = x.x, w[1 % (VB < 4 ? 1 : VB / 4)] = x.y;
            } else if (VB == 4) {
                w[0] = *(const uint32_t*)at;
            } else {
                w[0] = *(const uint16_t*)at;
            }
        }
        if (FMT == FKV_PAGES_FP8) st.vx[t] = *(const uint32_t*)((const uint8_t*)a.pg.v_scale + p.row[t] + 4 * g);
        if (FMT == FKV_PAGES_FP8_INT4) {
            const f4* s = (const f4*)((const float*)a.pg.v_scale + 2 * (p.row[t] + 4 * g));
            st.sz[t][0] = s[0];
            st.sz[t][1] = s[1];
        }
    }
}

// The wave's sums over its tokens.
template <int D>
struct Sums {
    f4 acc[D / 16];  // O^T: acc[dt][i] is dim_of(dt, 4 g + i) of head c
    float m, l, z;   // maximum of the head, the lane's part of the sum and of INT4's minima
};

// One step: 32 tokens.  The values' registers are read after the scores, so
// the caller may have their loads in flight until then.
template <int D, int FMT, bool BF>
__device__ inline void scores(const Step<D, FMT>& st, const u4 (&q)[D / 32], const Place& p, float scale, int g,
                              float (&s)[8]) {
#pragma unroll
    for (int t = 0; t < 2; t++) {
        f4 r = {0.0f, 0.0f, 0.0f, 0.0f};
        if (FMT <= FKV_PAGES_BF16) {
#pragma unroll
            for (int i = 0; i < D / 32; i++) r = mfma<BF>(st.k[t][i % Step<D, FMT>::KL], q[i], r);
        } else {
#pragma unroll
            for (int i = 0; i < D / 32; i++) {
                const u4 w = st.k[t][(i / 2) % Step<D, FMT>::KL];
                const uint32_t w0 = i & 1 ? w.z : w.x, w1 = i & 1 ? w.w : w.y;
                const u4 k = {cvt_fp8<BF>(w0, false), cvt_fp8<BF>(w0, true), cvt_fp8<BF>(w1, false), cvt_fp8<BF>(w1, true)};
                r = mfma<BF>(k, q[i], r);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float x = r[i] * scale;
            if (FMT >= FKV_PAGES_FP8) x *= exp_byte((st.kx[t] >> (8 * i)) & 0xFF);
            s[4 * t + i] = x;
        }
    }
    if (p.n[0] < 16 || p.n[1] < 16) {  // (the same in all lanes)
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (4 * g + (j & 3) >= p.n[j >> 2]) s[j] = -INFINITY;
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

// Running maximum, weights, and O^T += V^T P^T.
template <int D, int FMT, bool BF>
__device__ inline void accumulate(const Step<D, FMT>& st, const float (&s)[8], Sums<D>& u) {
    constexpr int DT = D / 16, VW = Step<D, FMT>::VB < 4 ? 1 : Step<D, FMT>::VB / 4;
    float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    if (__any(top > u.m + kSlack)) {
        top = fmaxf(top, wave_xor(top, 16));
        top = fmaxf(top, wave_xor(top, 32));
        const float m = fmaxf(u.m, top), f = __builtin_amdgcn_exp2f(u.m - m);
        u.m = m;
        u.l *= f;
        u.z *= f;
#pragma unroll
        for (int d = 0; d < DT; d++) u.acc[d] *= f;
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
    // fp16 rows: weights to fp16 (11 bits, as the rows; 2^-12 of a weight at
    // most).  Elsewhere: bf16 weights, which have the range that the rows'
    // scales need but 8 bits, so each is taken as the sum of two (16 bits).
    u4 hi, lo;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float x = w[2 * j], y = w[2 * j + 1];
        if (FMT == FKV_PAGES_F16) {
            hi[j] = (uint32_t)f2h(x) | ((uint32_t)f2h(y) << 16);
        } else {
            hi[j] = bf16_pair(x, y);
            lo[j] = bf16_pair(x - __uint_as_float(hi[j] << 16), y - __uint_as_float(hi[j] & 0xFFFF0000u));
        }
    }
    auto add = [&](int d, u4 v) {
        if (FMT == FKV_PAGES_F16) {
            u.acc[d] = mfma<false>(v, hi, u.acc[d]);
        } else {
            u.acc[d] = mfma<true>(v, hi, u.acc[d]);
            u.acc[d] = mfma<true>(v, lo, u.acc[d]);
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

// Dim of the lane's row r (0..15) in acc[dt]: D / 16 neighbouring dims a
// lane, in the order in which accumulate() takes them.
template <int D, int FMT>
__device__ inline int dim_of(int dt, int r) {
    constexpr int DT = D / 16;
    if (FMT != FKV_PAGES_FP8_INT4) return DT * r + dt;
    // INT4: the four low nibbles (even dims), then the high ones
    if (D == 128) return DT * r + 2 * (dt & 3) + (dt >> 2);
    return DT * r + 2 * (dt & 1) + (dt >> 1);
}

// Joins the four waves' sums in the LDS and writes the row's result (whole)
// or its record.  Every wave of the workgroup calls it.
template <int D, int FMT, bool BF>
__device__ inline void finish_row(const AttnArgs& a, Sums<D>& u, float* lds, int b, int hrow, float* record) {
    constexpr int DT = D / 16, RS = D + 4;  // (rows of D + 4 floats: the 16 heads fall on different banks)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    float* num = lds;                               // [wave][16][RS]
    float* stat = lds + kAttnWaves * 16 * RS;       // [wave][16][3]
    u.l += wave_xor(u.l, 16);
    u.l += wave_xor(u.l, 32);
    if (FMT == FKV_PAGES_FP8_INT4) {
        u.z += wave_xor(u.z, 16);
        u.z += wave_xor(u.z, 32);
    }
    if (g == 0) {
        float* st = stat + (wave * 16 + c) * 3;
        st[0] = u.m, st[1] = u.l, st[2] = u.z;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
            num[(wave * 16 + c) * RS + dim_of<D, FMT>(dt, 4 * g + i)] = u.acc[dt][i];
    __syncthreads();
    // 16 threads a head, D / 16 dims a thread
    const int head = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * DT;
    const int h = hrow / a.HT, g0 = (hrow - h * a.HT) * a.GT;
    if (head < a.GT && g0 + head < a.G) {
        float m = kNegBig, l = 0.0f, z = 0.0f, x[DT] = {};
#pragma unroll
        for (int w = 0; w < kAttnWaves; w++) m = fmaxf(m, stat[(w * 16 + head) * 3]);
#pragma unroll
        for (int w = 0; w < kAttnWaves; w++) {
            const float* st = stat + (w * 16 + head) * 3;
            const float f = __builtin_amdgcn_exp2f(st[0] - m);
            l = fmaf(f, st[1], l);
            z = fmaf(f, st[2], z);
#pragma unroll
            for (int i = 0; i < DT; i++) x[i] = fmaf(f, num[(w * 16 + head) * RS + d0 + i], x[i]);
        }
        if (FMT == FKV_PAGES_FP8_INT4) {
#pragma unroll
            for (int i = 0; i < DT; i++) x[i] = fmaf(x[i], 512.0f, z);
        }
        if (record) {
            float* r = record + head * (D + 2);
#pragma unroll
            for (int i = 0; i < DT; i += 2) *(float2*)(r + d0 + i) = make_float2(x[i], x[i + 1]);
            if ((threadIdx.x & 15) == 0) *(float2*)(r + D) = make_float2(m, l);
        } else {
            const int64_t at = (int64_t)b * a.Hq + h * a.G + g0 + head;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            uint32_t o[DT / 2];
#pragma unroll
            for (int i = 0; i < DT / 2; i++) {
                const float p = x[2 * i] * inv, q = x[2 * i + 1] * inv;
                o[i] = BF ? bf16_pair(p, q) : (uint32_t)f2h(p) | ((uint32_t)f2h(q) << 16);
            }
            uint32_t* dst = (uint32_t*)(a.out + 2 * (at * D + d0));
#pragma unroll
            for (int i = 0; i < DT / 2; i++) dst[i] = o[i];
            if (a.lse && (threadIdx.x & 15) == 0) a.lse[at] = (m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f;
        }
    }
    __syncthreads();
}

// Tiles of `b` dealt from `first` on; see the file's head.
template <int D, int FMT, bool BF>
__global__ void __launch_bounds__(64 * kAttnWaves) paged_attn_kernel(AttnArgs a) {
    constexpr int RS = D + 4;
    __shared__ float lds[kAttnWaves * 16 * (RS + 3)];
    __shared__ int64_t found[3];  // total tiles, then sequence and tile offset where this workgroup's run begins
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rows_per_seq = a.pg.H * a.HT;

    // sequences without tokens: their result is written here
    for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
        if (tiles_of(a, b) > 0) continue;
        for (int i = tid; i < a.Hq * D / 2; i += 64 * kAttnWaves) ((uint32_t*)a.out)[(int64_t)b * a.Hq * (D / 2) + i] = 0;
        if (a.lse)
            for (int i = tid; i < a.Hq; i += 64 * kAttnWaves) a.lse[(int64_t)b * a.Hq + i] = -INFINITY;
        if (a.joins)
            for (int i = tid; i < rows_per_seq; i += 64 * kAttnWaves) a.joins[(int64_t)b * rows_per_seq + i] = make_int4(0, 0, 0, 0);
    }

    // the tiles of all sequences, and the run's place among them
    int64_t* part = (int64_t*)lds;
    const int per = (a.B + 64 * kAttnWaves - 1) / (64 * kAttnWaves), b0 = tid * per;
    int64_t mine = 0;
    for (int i = 0; i < per; i++)
        if (b0 + i < a.B) mine += tiles_of(a, b0 + i);
    part[tid] = mine;
    __syncthreads();
    int64_t before = 0, total = 0;
    for (int i = 0; i < 64 * kAttnWaves; i++) {
        const int64_t n = part[i];
        before += i < tid ? n : 0;
        total += n;
    }
    total *= rows_per_seq;
    before *= rows_per_seq;
    const int64_t share = (total + gridDim.x - 1) / gridDim.x;
    const int64_t run0 = share * blockIdx.x, run1 = run0 + share < total ? run0 + share : total;
    if (run0 >= run1) return;
    if (run0 >= before && run0 < before + mine * rows_per_seq) {
        int64_t at = before;
        for (int i = 0; i < per; i++) {
            const int64_t n = b0 + i < a.B ? (int64_t)tiles_of(a, b0 + i) * rows_per_seq : 0;
            if (run0 < at + n) {
                found[0] = b0 + i;
                found[1] = run0 - at;
                break;
            }
            at += n;
        }
    }
    __syncthreads();
    int b = __builtin_amdgcn_readfirstlane((int)found[0]);
    const int64_t in_seq = found[1];
    int nt = tiles_of(a, b);
    int hrow = __builtin_amdgcn_readfirstlane((int)(in_seq / nt));
    int t0 = __builtin_amdgcn_readfirstlane((int)(in_seq - (int64_t)hrow * nt));
    int64_t at = run0;

    while (at < run1) {
        // row (b, hrow): its tiles [t0, t1) are this workgroup's
        const int64_t len = length_of(a, b);
        const int t1 = (int)(run1 - at < nt - t0 ? t0 + (run1 - at) : nt);
        const int h = hrow / a.HT, g0 = (hrow - h * a.HT) * a.GT;
        const int32_t* ids = a.table.ids + b * a.table.stride;

        u4 q[D / 32];
        {
            const bool real = c < a.GT && g0 + c < a.G;
            const char* row = a.q + 2 * (b * a.q_sb + (int64_t)(h * a.G + g0 + (real ? c : 0)) * a.q_sh);
#pragma unroll
            for (int i = 0; i < D / 32; i++) {
                const int d = FMT <= FKV_PAGES_BF16 ? 32 * i + 8 * g : 64 * (i / 2) + 16 * g + 8 * (i & 1);
                const u4 x = *(const u4*)(row + 2 * d), none = {0, 0, 0, 0};
                q[i] = real ? x : none;
            }
        }
        Sums<D> u;
        u.m = kNegBig, u.l = 0.0f, u.z = 0.0f;
#pragma unroll
        for (int d = 0; d < D / 16; d++) u.acc[d] = f4{0.0f, 0.0f, 0.0f, 0.0f};

        Step<D, FMT> st;
        int64_t tok = (int64_t)t0 * kAttnTile + 32 * wave;
        Place p = place_of(a, ids, tok, len, h);
        load_keys(st, a, p, g, c);
        load_values(st, a, p, g, c);
        for (int t = t0; t < t1; t++) {
            tok += kAttnTile;
            const Place next = place_of(a, ids, t + 1 < t1 ? tok : len, len, h);
            float s[8];
            scores<D, FMT, BF>(st, q, p, a.scale, g, s);
            load_keys(st, a, next, g, c);
            if (p.n[0] < 16 || p.n[1] < 16) mask_values(st, p, g);
            accumulate<D, FMT, BF>(st, s, u);
            load_values(st, a, next, g, c);
            p = next;
        }
        // a row that begins and ends here is done; of another one the record
        // goes to this workgroup's first slot, or to its second one where the
        // row begins after the run does
        const bool whole = t0 == 0 && t1 == nt;
        const int slot = at > run0 ? 1 : 0;
        if (a.joins && t0 == 0 && tid == 0) {
            const int64_t end = at + nt;  // of the row, among all tiles
            const int last = (int)((end - 1) / share);
            a.joins[(int64_t)b * rows_per_seq + hrow] =
                make_int4(blockIdx.x, whole ? 0 : last - (int)blockIdx.x + 1, slot, 0);
        }
        float* record = whole ? nullptr : a.records + ((int64_t)blockIdx.x * 2 + slot) * a.GT * (D + 2);
        __syncthreads();
        finish_row<D, FMT, BF>(a, u, lds, b, hrow, record);
        at += t1 - t0;
        t0 = 0;
        if (at < run1 && ++hrow == rows_per_seq) {
            hrow = 0;
            do b++; while (b < a.B && (nt = tiles_of(a, b)) == 0);
            b = __builtin_amdgcn_readfirstlane(b);
            nt = __builtin_amdgcn_readfirstlane(nt);
        }
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
        const int4 j = a.joins[row];
        if (j.y == 0) continue;  // (the same for the whole workgroup)
        const int b = row / rows_per_seq, hrow = row - b * rows_per_seq;
        const int h = hrow / a.HT, g0 = (hrow - h * a.HT) * a.GT;
        const bool real = head < a.GT && g0 + head < a.G;
        const int64_t rec = (int64_t)a.GT * (D + 2);
        float m = kNegBig, l = 0.0f, x[N] = {};
        if (real) {
            auto record = [&](int i) {
                return a.records + ((int64_t)(j.x + i) * 2 + (i == 0 ? j.z : 0)) * rec + head * (D + 2);
            };
            for (int i = w0 + PARTS * lane; i < j.y; i += PARTS * 64) m = fmaxf(m, record(i)[D]);
            m = wave_max(m);
#pragma unroll 8
            for (int i = w0; i < j.y; i += PARTS) {
                const float* r = record(i);
                const float f = __builtin_amdgcn_exp2f(r[D] - m);
                l = fmaf(f, r[D + 1], l);
#pragma unroll
                for (int n = 0; n < N; n++) x[n] = fmaf(f, r[64 * n + lane], x[n]);
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
    int G, HT, GT, blocks, join_rows;
    bool split;
    int64_t rows, records_at, bytes;
};

// Workgroups and workspace of a call (a function of sizes alone).
static AttnPlan plan_of(const fkv_pages* p, int32_t Hq, int32_t B, int64_t max_len) {
    AttnPlan r;
    r.G = Hq / p->H;
    r.HT = (r.G + 15) / 16;
    r.GT = (r.G + r.HT - 1) / r.HT;
    r.rows = (int64_t)B * p->H * r.HT;
    const int64_t tiles = r.rows * std::max<int64_t>(1, cdiv(max_len, kAttnTile));
    r.blocks = (int)std::min<int64_t>(tiles, 512);
    r.split = true;
    r.records_at = round_up(16 * r.rows, 256);
    r.bytes = r.records_at + (int64_t)r.blocks * 2 * r.GT * (p->D + 2) * 4;
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
static void launch_attn(const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
    paged_attn_kernel<D, FMT, BF><<<p.blocks, 64 * kAttnWaves, 0, s>>>(a);
    if (!p.split) return;
    const int rows = (int)std::min<int64_t>(p.rows, 1024);
    if (p.rows * p.GT <= 1024) paged_join_kernel<D, BF, 1><<<dim3(rows, p.GT), 256, 0, s>>>(a, (int)p.rows);
    else paged_join_kernel<D, BF, 4><<<dim3(rows, (p.GT + 3) / 4), 256, 0, s>>>(a, (int)p.rows);
}

template <int D>
static void launch_attn_d(const AttnArgs& a, const AttnPlan& p, int format, bool bf, hipStream_t s) {
    if (format == FKV_PAGES_F16) launch_attn<D, FKV_PAGES_F16, false>(a, p, s);
    else if (format == FKV_PAGES_BF16) launch_attn<D, FKV_PAGES_BF16, true>(a, p, s);
    else if (format == FKV_PAGES_FP8 && bf) launch_attn<D, FKV_PAGES_FP8, true>(a, p, s);
    else if (format == FKV_PAGES_FP8) launch_attn<D, FKV_PAGES_FP8, false>(a, p, s);
    else if (bf) launch_attn<D, FKV_PAGES_FP8_INT4, true>(a, p, s);
    else launch_attn<D, FKV_PAGES_FP8_INT4, false>(a, p, s);
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
    if ((int64_t)n_table * pages->page_size > 0x7FFFFFFF) return set_error(std::string(w) + ": more than 2^31 tokens a sequence");
    if (q_dtype != FKV_F16 && q_dtype != FKV_BF16) return set_error(std::string(w) + ": queries must be fp16 or bf16");
    if (pages->format <= FKV_PAGES_BF16 && (q_dtype == FKV_BF16) != (pages->format == FKV_PAGES_BF16))
        return set_error(std::string(w) + ": queries must have the 16-bit pages' type");
    if (!std::isfinite(scale)) return set_error(std::string(w) + ": scale must be finite");
    if (B == 0) return FKV_OK;
    if (!query || !query->data || !out || !lens) return set_error(std::string(w) + ": NULL argument");
    if (((uintptr_t)query->data | (uintptr_t)out | (uintptr_t)workspace) & 15 || (query->stride_b | query->stride_h) & 7)
        return set_error(std::string(w) + ": query, out and workspace must be 16-byte aligned, query strides multiples of 8");
    const AttnPlan p = plan_of(pages, Hq, B, max_len);
    if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes))
        return set_error(std::string(w) + ": workspace of " + std::to_string(p.bytes) + " bytes needed");
    if (p.rows > 0x7FFFFFFF) return set_error(std::string(w) + ": too many rows");
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
    if (pages->D == 64) launch_attn_d<64>(a, p, pages->format, bf, (hipStream_t)stream);
    else launch_attn_d<128>(a, p, pages->format, bf, (hipStream_t)stream);
    return check_hip(hipGetLastError(), w);
}

}  // extern "C"
