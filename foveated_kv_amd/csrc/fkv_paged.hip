// Paged KV cache: rotary positions, the write of new tokens (rotated and
// encoded on the way) and the read-back.  All three stream rows once: eight
// elements a lane, a row of D elements on D / 8 neighbouring lanes, so the
// row's reductions (largest magnitude, minimum and maximum) are DPP steps
// within 8 or 16 lanes.
// (Contraction would also merge the rounding of a 64-bit sum to fp32 with the
// one to 16 bits behind it; results are rounded to fp32 first, whatever
// follows.)
#pragma clang fp contract(off)
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "fkv_paged.h"

namespace fkv {

// ---------------------------------------------------------------------------
// eight elements of a row: four from `lo` and four from `hi` on
// ---------------------------------------------------------------------------

// In the half layout a lane holds four pairs, elements lo..lo + 3 and their
// partners hi = lo + rot / 2..; elsewhere eight neighbouring elements.
struct Place8 {
    int lo, hi;
};

// STREAM: results of a large call are stored past the caches: a 64K context
// out of 8-bit pages 76.8 us, not 85; a 16K prompt into 8-bit keys and 4-bit
// values 92, not 96.  (Loads past them as well gained nothing.)
template <bool STREAM, typename T>
__device__ inline void put(void* p, T v) {
    if (STREAM) __builtin_nontemporal_store(v, (T*)p);
    else *(T*)p = v;
}

// A lane's eight elements as they were loaded.
template <int DT>
struct Raw {
    uint32_t w[DT == FKV_F32 ? 8 : 4];
};

__device__ inline uint32_t pack_bf16(float a, float b) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    const bf2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
}
__device__ inline uint32_t pack_f16(float a, float b) { return (uint32_t)f2h(a) | ((uint32_t)f2h(b) << 16); }

template <int DT>
__device__ inline uint32_t pack16(float a, float b) {
    return DT == FKV_F16 ? pack_f16(a, b) : pack_bf16(a, b);
}

template <int DT, bool STREAM>
__device__ inline void store4f(char* row, int64_t elem, const float* x) {
    if (DT == FKV_F32) {
        put<STREAM>((float*)row + elem, fkv_u4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                                               __float_as_uint(x[3])});
        return;
    }
    const fkv_u2 w = {pack16<DT>(x[0], x[1]), pack16<DT>(x[2], x[3])};
    put<STREAM>((uint16_t*)row + elem, w);
}

// A lane's elements; PAIRS: hi may lie anywhere, else behind lo, and 16 bits an
// element take one access.
template <int DT, bool PAIRS>
__device__ inline Raw<DT> load8(const char* row, Place8 at) {
    Raw<DT> r;
    if constexpr (DT == FKV_F32) {
        const uint4 a = *(const uint4*)(row + 4 * at.lo), b = *(const uint4*)(row + 4 * at.hi);
        r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w, r.w[4] = b.x, r.w[5] = b.y, r.w[6] = b.z, r.w[7] = b.w;
    } else if constexpr (PAIRS) {
        const uint2 a = *(const uint2*)(row + 2 * at.lo), b = *(const uint2*)(row + 2 * at.hi);
        r.w[0] = a.x, r.w[1] = a.y, r.w[2] = b.x, r.w[3] = b.y;
    } else {
        const uint4 a = *(const uint4*)(row + 2 * at.lo);
        r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w;
    }
    return r;
}
template <int DT>
__device__ inline void unpack8(const Raw<DT>& r, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if (DT == FKV_F32) x[i] = __uint_as_float(r.w[i % (DT == FKV_F32 ? 8 : 4)]);
        else if (DT == FKV_F16) x[i] = h2f((uint16_t)(r.w[i / 2] >> (16 * (i & 1))));
        else x[i] = __uint_as_float(i & 1 ? r.w[i / 2] & 0xFFFF0000u : r.w[i / 2] << 16);
    }
}
template <int DT, bool PAIRS, bool STREAM>
__device__ inline void store8f(char* row, Place8 at, const float (&x)[8]) {
    if (DT != FKV_F32 && !PAIRS) {
        const fkv_u4 w = {pack16<DT>(x[0], x[1]), pack16<DT>(x[2], x[3]), pack16<DT>(x[4], x[5]), pack16<DT>(x[6], x[7])};
        put<STREAM>(row + 2 * at.lo, w);
    } else {
        store4f<DT, STREAM>(row, at.lo, x);
        store4f<DT, STREAM>(row, at.hi, x + 4);
    }
}

// ---------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------

struct RopeView {
    const float* table;
    int32_t n_pos, rot, interleaved;
};

// The elements of lane `lane_in_row`.
__device__ inline Place8 place8(const RopeView& r, int lane_in_row) {
    const int d0 = 8 * lane_in_row;
    if (r.interleaved || d0 >= r.rot) return Place8{d0, d0 + 4};
    return Place8{d0 >> 1, (d0 >> 1) + (r.rot >> 1)};
}

// cos and sin of a lane's four pairs at a position (NaN outside the table).
struct Angles {
    float c[4], s[4];
};
__device__ inline Angles angles_of(const RopeView& r, int64_t pos, int lane_in_row) {
    Angles a;
    const bool inside = pos >= 0 && pos < r.n_pos;
    const float* t = r.table + (inside ? pos : 0) * r.rot + (8 * lane_in_row < r.rot ? 4 * lane_in_row : 0);
    const float4 c = *(const float4*)t, s = *(const float4*)(t + (r.rot >> 1));
    const float nan = __builtin_nanf("");
    a.c[0] = inside ? c.x : nan, a.c[1] = inside ? c.y : nan, a.c[2] = inside ? c.z : nan, a.c[3] = inside ? c.w : nan;
    a.s[0] = s.x, a.s[1] = s.y, a.s[2] = s.z, a.s[3] = s.w;
    return a;
}

// a b - c d.  The products of two fp32 numbers are exact in 64 bits, so the only
// roundings are the sum's there and its own to fp32, and what a quantised key
// is decided from does not depend on the order of evaluation.  (In fp32 the
// 16K prompt's 32 + 8 heads took 65.3 us, so 66.0: memory is the bound.)
__device__ inline float cross(float a, float b, float c, float d) {
    return (float)fma((double)a, (double)b, -((double)c * (double)d));
}

// `inter`: the lane's elements are (a, b) pairs in turn, else four a, four b.
__device__ inline void rotate8(float (&x)[8], const RopeView& r, const Angles& t, int lane_in_row, bool inter) {
    if (8 * lane_in_row >= r.rot) return;
    float y[8];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float a = inter ? x[2 * j] : x[j], b = inter ? x[2 * j + 1] : x[4 + j];
        y[2 * j] = cross(a, t.c[j], b, t.s[j]);
        y[2 * j + 1] = cross(b, t.c[j], a, -t.s[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = inter ? y[j] : y[2 * (j & 3) + (j >> 2)];
}

// The table: one angle a thread.  Frequencies come with the launch, so that
// there is no copy to wait for.
struct Frequencies {
    double f[256];
};
__global__ void __launch_bounds__(256) rope_table_kernel(Frequencies freq, uint32_t pairs, double factor, int64_t n,
                                                         float* table) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t pos = i / pairs;
        const uint32_t pair = (uint32_t)(i - pos * pairs);
        double s, c;
        sincos((double)pos * freq.f[pair], &s, &c);
        table[pos * 2 * pairs + pair] = (float)(c * factor);
        table[(pos * 2 + 1) * pairs + pair] = (float)(s * factor);
    }
}

// One row of D elements on D / 8 lanes of one wave (each lane writes the
// elements that it read: out may be x), the wave's rows and then N times as
// many being consecutive heads of one token, which share the lane's angles.
template <int DT, int N, bool PAIRS>
__global__ void __launch_bounds__(256) rope_kernel(RowsView x, RowsView out, RopeView rope, PositionsView pos,
                                                   uint32_t n_units, uint32_t H, uint32_t L, uint32_t lanes,
                                                   uint32_t rows_per_wave) {
    constexpr int ES = DT == FKV_F32 ? 4 : 2;
    const uint32_t lane = threadIdx.x & 63, unit = blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t sub = lane / lanes, lr = lane - sub * lanes, step = rows_per_wave;
    if (sub >= step || unit >= n_units) return;
    const uint32_t chunks = (H + N * step - 1) / (N * step);
    const uint32_t tok = unit / chunks, h0 = (unit - tok * chunks) * N * step + sub, b = tok / L, l = tok - b * L;
    if (h0 >= H) return;
    const Place8 at = place8(rope, lr);
    const char* src = x.data + (b * x.sb + l * x.sl) * ES;
    char* dst = out.data + (b * out.sb + l * out.sl) * ES;
    const Angles t = angles_of(rope, position_of(pos, b, l), lr);
    Raw<DT> raw[N];
#pragma unroll
    for (int i = 0; i < N; i++) {  // (past the last head: loaded, not used)
        const uint32_t h = h0 + i * step < H ? h0 + i * step : h0;
        raw[i] = load8<DT, PAIRS>(src + h * x.sh * ES, at);
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        float v[8];
        unpack8<DT>(raw[i], v);
        rotate8(v, rope, t, lr, N > 1 ? !PAIRS : rope.interleaved);
        if (h0 + i * step < H) store8f<DT, PAIRS, (N > 1)>(dst + (h0 + i * step) * out.sh * ES, at, v);
    }
}

// ---------------------------------------------------------------------------
// row codecs
// ---------------------------------------------------------------------------

constexpr int kDppHalfMirror = 0x141, kDppMirror = 0x140;

// Reduction over the D / 8 lanes of a row (8 or 16, aligned).
template <int D, typename F>
__device__ inline float row_reduce(float v, F f) {
    v = f(v, dpp_f32<kDppXor1>(v));
    v = f(v, dpp_f32<kDppXor2>(v));
    v = f(v, dpp_f32<kDppHalfMirror>(v));
    if (D == 128) v = f(v, dpp_f32<kDppMirror>(v));
    return v;
}

// E4M3 codes of the row's eight elements; returns e + 127.
template <int D>
__device__ inline uint32_t encode_fp8(const float (&x)[8], uint32_t (&codes)[2]) {
    float y[8], amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const bool finite = fabsf(x[j]) <= 3.402823466e38f;
        y[j] = finite ? x[j] : __builtin_nanf("");
        amax = fmaxf(amax, finite ? fabsf(x[j]) : 0.0f);
    }
    amax = row_reduce<D>(amax, [](float a, float b) { return fmaxf(a, b); });
    // amax = 1.m * 2^(E - 127) <= 1.75 * 2^(8 + e)
    const uint32_t bits = __float_as_uint(amax);
    int byte = (int)(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u);
    byte = bits == 0 ? 127 : byte < 1 ? 1 : byte;
    const float inv = exp_byte(254 - byte);  // 2^-e
#pragma unroll
    for (int w = 0; w < 2; w++) {
        int c = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * w] * inv, y[4 * w + 1] * inv, 0, false);
        c = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * w + 2] * inv, y[4 * w + 3] * inv, c, true);
        codes[w] = (uint32_t)c;
    }
    return (uint32_t)byte;
}

// INT4 codes of the row's eight elements (even dim in the low nibble).  The
// quotient (x - min) / scale in fp32 is off by less than 4e-6 (four roundings
// of a number up to 15); where it comes within 1e-4 of the middle between two
// codes, or is no number, the sign of d - (k + 1/2) scale decides in 64 bits,
// whose fma rounds once: always the code that the exact quotient rounds to.
template <int D>
__device__ inline uint32_t encode_int4(const float (&x)[8], float& scale, float& zero) {
    float lo = x[0], hi = x[0], bad = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        lo = fminf(lo, x[j]);
        hi = fmaxf(hi, x[j]);
        bad += x[j] * 0.0f;  // NaN where an element is not finite
    }
    lo = row_reduce<D>(lo, [](float a, float b) { return fminf(a, b); });
    hi = row_reduce<D>(hi, [](float a, float b) { return fmaxf(a, b); });
    bad = row_reduce<D>(bad, [](float a, float b) { return a + b; });
    const float s = (float)(((double)hi - (double)lo) / 15.0);
    scale = bad == 0.0f ? s : __builtin_nanf("");
    zero = lo;
    const float inv = __builtin_amdgcn_rcpf(s);
    float k[8];
    bool close = false;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float t = (x[j] - lo) * inv;
        k[j] = floorf(t);
        const float past = t - k[j] - 0.5f;
        close |= !(fabsf(past) > 1e-4f);
        k[j] += past > 0.0f ? 1.0f : 0.0f;
    }
    if (close) {
        const double sd = s, rcp = 1.0 / sd;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const double d = (double)x[j] - (double)lo, f = floor(d * rcp), r = fma(-(f + 0.5), sd, d);
            k[j] = (float)f + (r > 0.0 || (r == 0.0 && ((int)f & 1)) ? 1.0f : 0.0f);
        }
    }
    uint32_t packed = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uint32_t c = s > 0.0f ? (uint32_t)__builtin_amdgcn_fmed3f(k[j], 0.0f, 15.0f) : 0;
        packed |= c << (4 * j);
    }
    return packed;
}

// A lane's elements of row `row` of K (or V), stored as the format has them.
// (Values lie at neighbouring elements.)  Pages stay in the caches, for the
// attention or the read that follows: read back at once a 16K prompt takes 16
// us, not 22.
template <int D, int FMT, bool VALUE, bool PAIRS>
__device__ inline void store_row(const PageView& pg, int64_t row, int lane_in_row, Place8 at, const float (&x)[8]) {
    char* base = VALUE ? pg.v : pg.k;
    if (FMT <= FKV_PAGES_BF16) {
        store8f<FMT == FKV_PAGES_F16 ? FKV_F16 : FKV_BF16, PAIRS, false>(base + row * (2 * D), at, x);
    } else if (FMT == FKV_PAGES_FP8 || !VALUE) {
        uint32_t codes[2];
        const uint32_t byte = encode_fp8<D>(x, codes);
        if (PAIRS) {
            *(uint32_t*)(base + row * D + at.lo) = codes[0];
            *(uint32_t*)(base + row * D + at.hi) = codes[1];
        } else {
            *(uint2*)(base + row * D + at.lo) = make_uint2(codes[0], codes[1]);
        }
        if (lane_in_row == 0) (VALUE ? (uint8_t*)pg.v_scale : pg.k_exp)[row] = (uint8_t)byte;
    } else {
        float scale, zero;
        const uint32_t codes = encode_int4<D>(x, scale, zero);
        *(uint32_t*)(base + row * (D / 2) + at.lo / 2) = codes;
        if (lane_in_row == 0) ((float2*)pg.v_scale)[row] = make_float2(scale, zero);
    }
}

// ---------------------------------------------------------------------------
// write
// ---------------------------------------------------------------------------

struct WriteArgs {
    PageView pg;
    TableView table;
    RowsView q, q_out, k, v;
    PositionsView start;
    RopeView rope;
    const int32_t* n_new;
    uint32_t n_units, n_tokens, L, Hq;
};

enum { kQueries, kKeys, kValues };

// N consecutive heads of the wave's tokens.
template <int D, int DT, int FMT, int N, bool PAIRS, int KIND>
__device__ inline void write_heads(const WriteArgs& a, uint32_t h0, uint32_t b, uint32_t l, int lr) {
    constexpr int ES = DT == FKV_F32 ? 4 : 2;
    const RowsView& in = KIND == kQueries ? a.q : KIND == kKeys ? a.k : a.v;
    const uint32_t heads = KIND == kQueries ? a.Hq : a.pg.H;
    const bool inter = N > 1 ? !PAIRS : a.rope.interleaved;
    const Place8 at = KIND == kValues ? Place8{8 * lr, 8 * lr + 4} : place8(a.rope, lr);
    const char* src = in.data + ((int64_t)b * in.sb + (int64_t)l * in.sl) * ES;
    Raw<DT> raw[N];
#pragma unroll
    for (int i = 0; i < N; i++)  // (past the last head: loaded, not used)
        raw[i] = load8<DT, PAIRS && KIND != kValues>(src + (h0 + i < heads ? h0 + i : heads - 1) * in.sh * ES, at);
    const int64_t pos = position_of(a.start, b, l);
    Angles t = {};
    if (KIND != kValues && a.rope.rot) t = angles_of(a.rope, pos, lr);
    int64_t row = 0;
    if (KIND != kQueries) {
        row = page_row(a.pg, a.table, b, pos, h0);
        if (row < 0) return;  // (all lanes of a row agree)
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (h0 + i >= heads) return;
        float x[8];
        unpack8<DT>(raw[i], x);
        if (KIND != kValues) rotate8(x, a.rope, t, lr, inter);
        if (KIND == kQueries)
            store8f<DT, PAIRS, (N > 1)>(a.q_out.data + ((int64_t)b * a.q_out.sb + (h0 + i) * a.q_out.sh + (int64_t)l * a.q_out.sl) * ES,
                                        at, x);
        else
            store_row<D, FMT, KIND == kValues, PAIRS && KIND != kValues>(a.pg, row + (int64_t)i * a.pg.page_size, lr, at, x);
    }
}

// One launch for a step's rotation and its cache write.  A wave takes 64 /
// (D / 8) neighbouring tokens, a row of each at a time, and N consecutive
// heads of them, queries, keys or values: its stores of a head are
// neighbouring rows, and exponents or scales, of a page.
template <int D, int DT, int FMT, int N, bool PAIRS>
__global__ void __launch_bounds__(256) paged_write_kernel(WriteArgs a) {
    constexpr int LPR = D / 8, TOKENS = 64 / LPR;
    const uint32_t unit = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), lane = threadIdx.x & 63;
    if (unit >= a.n_units) return;
    const uint32_t cq = (a.Hq + N - 1) / N, ck = (a.pg.H + N - 1) / N, chunks = cq + 2 * ck;
    const uint32_t group = unit / chunks, chunk = unit - group * chunks;
    const uint32_t tok = group * TOKENS + lane / LPR, b = tok / a.L, l = tok - b * a.L;
    if (tok >= a.n_tokens || (a.n_new && (int32_t)l >= a.n_new[b])) return;
    const int lr = lane % LPR;
    if (chunk < cq) write_heads<D, DT, FMT, N, PAIRS, kQueries>(a, chunk * N, b, l, lr);
    else if (chunk < cq + ck) write_heads<D, DT, FMT, N, PAIRS, kKeys>(a, (chunk - cq) * N, b, l, lr);
    else write_heads<D, DT, FMT, N, PAIRS, kValues>(a, (chunk - cq - ck) * N, b, l, lr);
}

// ---------------------------------------------------------------------------
// read
// ---------------------------------------------------------------------------

__device__ inline void decode_fp8(const uint2 w, float scale, float (&x)[8]) {
    const uint32_t u[2] = {w.x, w.y};
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const fkv_f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[i], false);
        const fkv_f2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[i], true);
        x[4 * i] = lo.x * scale, x[4 * i + 1] = lo.y * scale;
        x[4 * i + 2] = hi.x * scale, x[4 * i + 3] = hi.y * scale;
    }
}

template <int D, int FMT, bool VALUE>
__device__ inline void load_row(const PageView& pg, int64_t row, int lane_in_row, float (&x)[8]) {
    const int64_t at = row * D + 8 * lane_in_row;
    const char* base = VALUE ? pg.v : pg.k;
    if (FMT <= FKV_PAGES_BF16) {
        constexpr int DT = FMT == FKV_PAGES_F16 ? FKV_F16 : FKV_BF16;
        unpack8<DT>(load8<DT, false>(base + 2 * at, Place8{0, 4}), x);
    } else if (FMT == FKV_PAGES_FP8 || !VALUE) {
        const uint32_t byte = (VALUE ? (const uint8_t*)pg.v_scale : pg.k_exp)[row];
        decode_fp8(*(const uint2*)(base + at), exp_byte(byte), x);
    } else {
        const uint32_t w = *(const uint32_t*)(base + at / 2);
        const float2 sz = ((const float2*)pg.v_scale)[row];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = fmaf((float)((w >> (4 * j)) & 15u), sz.x, sz.y);
    }
}

struct ReadArgs {
    PageView pg;
    TableView table;
    const int32_t* lens;
    char *k, *v;
    uint32_t n_units, S;
};

// 16 tokens of a head, which one page holds, on each wave: N rows of K and of
// V a lane, all of their loads in flight together.
template <int D, int FMT, int DT>
__global__ void __launch_bounds__(256) paged_read_kernel(ReadArgs a) {
    constexpr int LPR = D / 8, STEP = 64 / LPR, N = 16 / STEP;
    const uint32_t unit = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (unit >= a.n_units) return;
    const uint32_t chunks = (a.S + 15) / 16, bh = unit / chunks, first = 16 * (unit - bh * chunks);
    const uint32_t b = bh / a.pg.H, h = bh - b * a.pg.H, s0 = first + lane / LPR;
    const int lr = lane % LPR;
    const int32_t len = a.lens[b];
    const int64_t row0 = (int32_t)first < len ? page_row(a.pg, a.table, b, first, h) : -1;
    float k[N][8] = {}, v[N][8] = {};
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (row0 < 0 || (int32_t)(s0 + i * STEP) >= len) break;
        load_row<D, FMT, false>(a.pg, row0 + lane / LPR + i * STEP, lr, k[i]);
        load_row<D, FMT, true>(a.pg, row0 + lane / LPR + i * STEP, lr, v[i]);
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (s0 + i * STEP >= a.S) break;
        const int64_t at = ((int64_t)bh * a.S + s0 + i * STEP) * D;
        const Place8 e = {8 * lr, 8 * lr + 4};
        store8f<DT, false, true>(a.k + at * (DT == FKV_F32 ? 4 : 2), e, k[i]);
        store8f<DT, false, true>(a.v + at * (DT == FKV_F32 ? 4 : 2), e, v[i]);
    }
}

// ---------------------------------------------------------------------------
// argument checks and launches
// ---------------------------------------------------------------------------

static bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }

int check_pages(const char* who, const fkv_pages* p) {
    const std::string w = who;
    if (!p) return set_error(w + ": NULL pages");
    if (p->D != 64 && p->D != 128) return set_error(w + ": head dim must be 64 or 128, got " + std::to_string(p->D));
    if (p->format < FKV_PAGES_F16 || p->format > FKV_PAGES_FP8_INT4) return set_error(w + ": unknown page format");
    if (p->page_size < 16 || p->page_size > 1024 || (p->page_size & (p->page_size - 1)))
        return set_error(w + ": page size must be a power of two from 16 to 1024, got " + std::to_string(p->page_size));
    if (p->n_pages < 1 || p->H < 1 || p->H > 1024) return set_error(w + ": bad page or head count");
    const bool q = p->format >= FKV_PAGES_FP8;
    if (!p->k || !p->v || (q && (!p->k_exp || !p->v_scale))) return set_error(w + ": a page array is NULL");
    if (misaligned(p->k) || misaligned(p->v) || (q && (misaligned(p->k_exp) || misaligned(p->v_scale))))
        return set_error(w + ": page arrays must be 16-byte aligned");
    return FKV_OK;
}

int check_table(const char* who, const int32_t* table, int32_t n_table, int64_t stride, int32_t B) {
    const std::string w = who;
    if (B < 0 || n_table < 0 || (B > 1 && stride < n_table)) return set_error(w + ": bad table shape");
    if (B > 0 && n_table > 0 && !table) return set_error(w + ": NULL table");
    return FKV_OK;
}

PageView page_view(const fkv_pages* p) {
    return PageView{(char*)p->k, (char*)p->v, p->k_exp, (char*)p->v_scale, p->n_pages, p->page_size, p->H};
}

static int check_rows(const std::string& w, const fkv_rows* r) {
    if (!r || !r->data) return set_error(w + ": NULL rows");
    if (misaligned(r->data) || (r->stride_b | r->stride_h | r->stride_l) & 7)
        return set_error(w + ": rows must be 16-byte aligned with strides that are multiples of 8");
    return FKV_OK;
}

// One dimension of the difference of two rows' addresses: k * stride for a k of
// [lo, hi].
struct Steps {
    int64_t stride, lo, hi;
};

// Whether numbers k of the steps [i, n) bring `from` (elements) within D of 0;
// with `moved` false, numbers that are not all 0.  `left` bounds the search, and
// the answer is yes where it ends: strides are nested in any layout of a tensor,
// which leaves two or three k of each dimension to look at.
static bool can_meet(const Steps* st, int n, int i, int64_t from, int64_t D, bool moved, int& left) {
    if (i == n) return moved && from < D && -from < D;
    if (--left <= 0) return true;
    int64_t reach = D - 1;
    for (int j = i + 1; j < n; j++) reach += st[j].stride * std::max(-st[j].lo, st[j].hi);
    const Steps s = st[i];
    // |from + k stride| <= reach
    const int64_t lo = std::max(s.lo, -((from + reach) / s.stride)), hi = std::min(s.hi, (reach - from) / s.stride);
    for (int64_t k = lo; k <= hi; k++)
        if (can_meet(st, n, i + 1, from + k * s.stride, D, moved || k != 0, left)) return true;
    return false;
}

static bool can_meet(Steps* st, int n, int64_t from, int64_t D, bool moved) {
    int m = 0;
    for (int i = 0; i < n; i++) {
        Steps s = st[i];
        if (s.stride < 0) s = Steps{-s.stride, -s.hi, -s.lo};
        if (s.lo == 0 && s.hi == 0) continue;
        if (s.stride == 0) {
            moved = true;
            continue;
        }
        st[m++] = s;
    }
    std::sort(st, st + m, [](const Steps& a, const Steps& b) { return a.stride > b.stride; });
    int left = 4096;
    return can_meet(st, m, 0, from, D, moved, left);
}

// Whether strides are nested: each passes all that the smaller ones cover, as in
// any slice of a tensor.  (Found without a division, which each call would notice.)
static bool nested(const fkv_rows* r, const RowsShape& s) {
    int64_t stride[3] = {r->stride_b, r->stride_h, r->stride_l}, n[3] = {s.B, s.H, s.L};
    auto order = [&](int i, int j) {
        if (stride[i] < stride[j]) std::swap(stride[i], stride[j]), std::swap(n[i], n[j]);
    };
    order(0, 1), order(1, 2), order(0, 1);
    int64_t covered = s.D;
    for (int d = 2; d >= 0; d--) {
        if (n[d] > 1 && stride[d] < covered) return false;
        covered += n[d] > 1 ? (n[d] - 1) * stride[d] : 0;
    }
    return true;
}

int check_result_rows(const char* who, const char* name, const fkv_rows* out, const RowsShape& s) {
    if (nested(out, s)) return FKV_OK;
    Steps st[3] = {{out->stride_b, 1 - s.B, s.B - 1}, {out->stride_h, 1 - s.H, s.H - 1}, {out->stride_l, 1 - s.L, s.L - 1}};
    if (!can_meet(st, 3, 0, s.D, false)) return FKV_OK;
    return set_error(std::string(who) + ": rows of " + name + " share memory");
}

int check_apart(const char* who, const char* what, const fkv_rows* out, const RowsShape& o, const fkv_rows* in,
                const RowsShape& r, bool in_place) {
    const int64_t so[3] = {out->stride_b, out->stride_h, out->stride_l}, no[3] = {o.B, o.H, o.L},
                  si[3] = {in->stride_b, in->stride_h, in->stride_l}, ni[3] = {r.B, r.H, r.L};
    int64_t lo = 0, hi = 0, first = 0, last = 0;  // elements that each covers, from its address on
    bool same = in_place && out->data == in->data;
    for (int d = 0; d < 3; d++) {
        (so[d] < 0 ? lo : hi) += (no[d] - 1) * so[d];
        (si[d] < 0 ? first : last) += (ni[d] - 1) * si[d];
        same = same && no[d] == ni[d] && (no[d] == 1 || so[d] == si[d]);
    }
    const int64_t bytes = (const char*)out->data - (const char*)in->data;
    if (same || bytes + (hi + o.D) * o.es <= first * o.es || (last + r.D) * o.es <= bytes + lo * o.es) return FKV_OK;
    const int64_t from = bytes / o.es;
    Steps st[6];
    int n = 0;
    for (int d = 0; d < 3; d++) {
        if (so[d] == si[d]) {
            st[n++] = Steps{so[d], 1 - ni[d], no[d] - 1};
        } else {
            st[n++] = Steps{so[d], 0, no[d] - 1};
            st[n++] = Steps{si[d], 1 - ni[d], 0};
        }
    }
    if (!can_meet(st, n, from, o.D, true)) return FKV_OK;
    return set_error(std::string(who) + ": " + what + " share memory");
}

static RowsView rows_view(const fkv_rows* r) {
    return RowsView{(char*)r->data, r->stride_b, r->stride_h, r->stride_l};
}

static int check_rope(const std::string& w, const fkv_rope* r, int32_t D) {
    if (!r->table || misaligned(r->table)) return set_error(w + ": the rotary table must be a 16-byte aligned array");
    if (r->rot_dim < 16 || r->rot_dim > D || r->rot_dim % 16)
        return set_error(w + ": rot_dim must be a multiple of 16 from 16 to the head dim, got " +
                         std::to_string(r->rot_dim));
    if (r->n_positions < 1) return set_error(w + ": the rotary table has no positions");
    return FKV_OK;
}

static int check_positions(const std::string& w, const fkv_positions* p) {
    if (!p) return set_error(w + ": NULL positions");
    if (p->data && ((uintptr_t)p->data & (p->is64 ? 7 : 3))) return set_error(w + ": misaligned positions");
    return FKV_OK;
}

static PositionsView positions_view(const fkv_positions* p) {
    return PositionsView{p->data, p->stride_b, p->stride_l, p->base, p->is64, p->per_token};
}

// Rows that a lane takes one after the other: with four, the angles, the
// position and the divisions serve four rows, whose loads are in flight
// together; with one, few rows spread over more of the chip.
// (98K rows, four prompts' chunks of 512 tokens: 14.8 us with four, 17 with
// one; 3K rows, a decode step of 64 sequences, 4.0 with one.)
constexpr int64_t kFewRows = 16384;

// A grid has fewer than 2^32 threads: waves, four to a workgroup, that a launch
// may have.
constexpr int64_t kMaxUnits = 4 * ((int64_t{1} << 24) - 1);

static int too_many(const char* who) { return set_error(std::string(who) + ": too many rows for one call"); }

template <int D, int DT, int FMT>
static int launch_write_f(WriteArgs& a, int64_t tokens, hipStream_t s) {
    const int64_t heads = a.Hq + 2 * (int64_t)a.pg.H;
    a.n_tokens = (uint32_t)tokens;
    auto go = [&](auto n, auto pairs) {
        constexpr int N = decltype(n)::value;
        const int64_t units = cdiv(tokens, 64 / (D / 8)) * (cdiv(a.Hq, N) + 2 * cdiv(a.pg.H, N));
        if (units > kMaxUnits) return too_many("fkv_paged_write");
        a.n_units = (uint32_t)units;
        return start_kernel("fkv_paged_write", paged_write_kernel<D, DT, FMT, N, decltype(pairs)::value>,
                            (uint32_t)cdiv(a.n_units, 4), 256, s, a);
    };
    if (tokens * heads <= kFewRows) return go(std::integral_constant<int, 1>{}, std::true_type{});
    if (a.rope.rot && !a.rope.interleaved) return go(std::integral_constant<int, 4>{}, std::true_type{});
    return go(std::integral_constant<int, 4>{}, std::false_type{});
}

template <int D, int DT>
static int launch_write(WriteArgs& a, int format, int64_t tokens, hipStream_t s) {
    switch (format) {
        case FKV_PAGES_F16: return launch_write_f<D, DT, FKV_PAGES_F16>(a, tokens, s);
        case FKV_PAGES_BF16: return launch_write_f<D, DT, FKV_PAGES_BF16>(a, tokens, s);
        case FKV_PAGES_FP8: return launch_write_f<D, DT, FKV_PAGES_FP8>(a, tokens, s);
        default: return launch_write_f<D, DT, FKV_PAGES_FP8_INT4>(a, tokens, s);
    }
}

template <int D, int FMT>
static int launch_read(const ReadArgs& a, int dtype, uint32_t blocks, hipStream_t s) {
    const char* w = "fkv_paged_read";
    switch (dtype) {
        case FKV_F16: return start_kernel(w, paged_read_kernel<D, FMT, FKV_F16>, blocks, 256, s, a);
        case FKV_BF16: return start_kernel(w, paged_read_kernel<D, FMT, FKV_BF16>, blocks, 256, s, a);
        default: return start_kernel(w, paged_read_kernel<D, FMT, FKV_F32>, blocks, 256, s, a);
    }
}

}  // namespace fkv

using namespace fkv;

extern "C" {

int fkv_rope_table(const double* frequencies, int32_t rot_dim, double factor, int32_t n_positions, float* table,
                   void* stream) {
    const std::string w = "fkv_rope_table";
    if (!frequencies || !table || misaligned(table)) return set_error(w + ": NULL argument or misaligned table");
    if (rot_dim < 16 || rot_dim > 512 || rot_dim % 16)
        return set_error(w + ": rot_dim must be a multiple of 16 from 16 to 512, got " + std::to_string(rot_dim));
    if (n_positions < 1) return set_error(w + ": the rotary table has no positions");
    Frequencies f = {};
    for (int i = 0; i < rot_dim / 2; i++) f.f[i] = frequencies[i];
    const int64_t n = (int64_t)n_positions * (rot_dim / 2);
    return start_kernel(w.c_str(), rope_table_kernel, (uint32_t)std::min<int64_t>(cdiv(n, 256), 65536), 256,
                        (hipStream_t)stream, f, rot_dim / 2, factor, n, table);
}

int fkv_rope_apply(const fkv_rope* rope, const fkv_rows* x, const fkv_rows* out, int32_t dtype, int32_t B,
                   int32_t H, int32_t L, int32_t D, const fkv_positions* positions, void* stream) {
    const char* w = "fkv_rope_apply";
    if (!rope) return set_error(std::string(w) + ": NULL rope");
    if (dtype < FKV_F16 || dtype > FKV_F32) return set_error(std::string(w) + ": unknown dtype");
    if (B < 0 || H < 0 || L < 0) return set_error(std::string(w) + ": negative size");
    if (D < 16 || D > 512 || D % 8) return set_error(std::string(w) + ": head dim must be a multiple of 8 from 16 to 512");
    if (int e = check_rope(w, rope, D)) return e;
    if (int e = check_positions(w, positions)) return e;
    const double n = (double)B * H * L;
    if (n == 0) return FKV_OK;
    if (n >= 2147483648.0) return set_error(std::string(w) + ": more than 2^31 rows");
    if (int e = check_rows(w, x)) return e;
    if (int e = check_rows(w, out)) return e;
    const RowsShape shape{B, H, L, D, dtype == FKV_F32 ? 4 : 2};
    if (int e = check_result_rows(w, "out", out, shape)) return e;
    if (int e = check_apart(w, "out, which is not x, and x", out, shape, x, shape, true)) return e;
    const uint32_t lanes = D / 8, rpw = 64 / lanes;
    const RopeView rv{rope->table, rope->n_positions, rope->rot_dim, rope->interleaved};
    const PositionsView pv = positions_view(positions);
    hipStream_t s = (hipStream_t)stream;
    auto go = [&](auto dt, auto n, auto pairs) {
        constexpr int DT = decltype(dt)::value, N = decltype(n)::value;
        const int64_t units = (int64_t)B * L * cdiv(H, N * (int64_t)rpw);
        if (units > kMaxUnits) return too_many(w);
        return start_kernel(w, rope_kernel<DT, N, decltype(pairs)::value>, (uint32_t)cdiv(units, 4), 256, s, rows_view(x),
                            rows_view(out), rv, pv, (uint32_t)units, H, L, lanes, rpw);
    };
    auto by_rows = [&](auto dt) {
        if ((int64_t)B * H * L <= kFewRows) return go(dt, std::integral_constant<int, 1>{}, std::true_type{});
        if (!rope->interleaved) return go(dt, std::integral_constant<int, 4>{}, std::true_type{});
        return go(dt, std::integral_constant<int, 4>{}, std::false_type{});
    };
    if (dtype == FKV_F16) return by_rows(std::integral_constant<int, FKV_F16>{});
    if (dtype == FKV_BF16) return by_rows(std::integral_constant<int, FKV_BF16>{});
    return by_rows(std::integral_constant<int, FKV_F32>{});
}

int fkv_paged_write(const fkv_pages* pages, const fkv_rows* k, const fkv_rows* v, int32_t dtype, int32_t B,
                    int32_t L, const int32_t* table, int32_t n_table, int64_t table_stride,
                    const fkv_positions* start, const int32_t* n_new, const fkv_rope* rope, const fkv_rows* q,
                    const fkv_rows* q_out, int32_t Hq, void* stream) {
    const char* w = "fkv_paged_write";
    if (int e = check_pages(w, pages)) return e;
    if (dtype < FKV_F16 || dtype > FKV_F32) return set_error(std::string(w) + ": unknown dtype");
    if (L < 0) return set_error(std::string(w) + ": negative size");
    if (int e = check_table(w, table, n_table, table_stride, B)) return e;
    if (int e = check_positions(w, start)) return e;
    if (start->per_token) return set_error(std::string(w) + ": start is one position per sequence");
    if (!q != !q_out) return set_error(std::string(w) + ": q and q_out come together");
    if (q && Hq < 1) return set_error(std::string(w) + ": bad query head count");
    if (rope)
        if (int e = check_rope(w, rope, pages->D)) return e;
    const int64_t heads = (q ? Hq : 0) + 2 * (int64_t)pages->H;
    const double n = (double)B * L * heads;
    if (n == 0) return FKV_OK;
    if (n >= 2147483648.0) return set_error(std::string(w) + ": more than 2^31 rows");
    if (int e = check_rows(w, k)) return e;
    if (int e = check_rows(w, v)) return e;
    if (q) {
        if (int e = check_rows(w, q)) return e;
        if (int e = check_rows(w, q_out)) return e;
        const RowsShape sq{B, Hq, L, pages->D, dtype == FKV_F32 ? 4 : 2}, sk{B, pages->H, L, pages->D, sq.es};
        if (int e = check_result_rows(w, "q_out", q_out, sq)) return e;
        if (int e = check_apart(w, "q_out, which is not q, and q", q_out, sq, q, sq, true)) return e;
        if (int e = check_apart(w, "q_out and k", q_out, sq, k, sk, false)) return e;
        if (int e = check_apart(w, "q_out and v", q_out, sq, v, sk, false)) return e;
    }
    WriteArgs a;
    a.pg = page_view(pages);
    a.table = TableView{table, table_stride, n_table};
    a.k = rows_view(k);
    a.v = rows_view(v);
    a.q = q ? rows_view(q) : RowsView{};
    a.q_out = q ? rows_view(q_out) : RowsView{};
    a.start = positions_view(start);
    a.rope = rope ? RopeView{rope->table, rope->n_positions, rope->rot_dim, rope->interleaved} : RopeView{};
    a.n_new = n_new;
    a.L = L;
    a.Hq = q ? Hq : 0;
    const int64_t tokens = (int64_t)B * L;
    hipStream_t s = (hipStream_t)stream;
    if (pages->D == 64) {
        if (dtype == FKV_F16) return launch_write<64, FKV_F16>(a, pages->format, tokens, s);
        if (dtype == FKV_BF16) return launch_write<64, FKV_BF16>(a, pages->format, tokens, s);
        return launch_write<64, FKV_F32>(a, pages->format, tokens, s);
    }
    if (dtype == FKV_F16) return launch_write<128, FKV_F16>(a, pages->format, tokens, s);
    if (dtype == FKV_BF16) return launch_write<128, FKV_BF16>(a, pages->format, tokens, s);
    return launch_write<128, FKV_F32>(a, pages->format, tokens, s);
}

int fkv_paged_read(const fkv_pages* pages, const int32_t* table, int32_t n_table, int64_t table_stride,
                   const int32_t* lens, int32_t B, int32_t S, void* out_k, void* out_v, int32_t out_dtype,
                   void* stream) {
    const char* w = "fkv_paged_read";
    if (int e = check_pages(w, pages)) return e;
    if (out_dtype < FKV_F16 || out_dtype > FKV_F32) return set_error(std::string(w) + ": unknown dtype");
    if (S < 0) return set_error(std::string(w) + ": negative size");
    if (int e = check_table(w, table, n_table, table_stride, B)) return e;
    const double n = (double)B * S * pages->H;
    if (n == 0) return FKV_OK;
    if (n >= 2147483648.0) return set_error(std::string(w) + ": more than 2^31 rows");
    if (!lens || !out_k || !out_v || misaligned(out_k) || misaligned(out_v))
        return set_error(std::string(w) + ": lens and 16-byte aligned results are needed");
    ReadArgs a;
    a.pg = page_view(pages);
    a.table = TableView{table, table_stride, n_table};
    a.lens = lens;
    a.k = (char*)out_k;
    a.v = (char*)out_v;
    const int64_t units = (int64_t)B * pages->H * cdiv(S, 16);
    if (units > kMaxUnits) return too_many(w);
    a.n_units = (uint32_t)units;
    a.S = S;
    const uint32_t blocks = (uint32_t)cdiv(a.n_units, 4);
    hipStream_t s = (hipStream_t)stream;
    auto go = [&](auto d) {
        constexpr int D = decltype(d)::value;
        switch (pages->format) {
            case FKV_PAGES_F16: return launch_read<D, FKV_PAGES_F16>(a, out_dtype, blocks, s);
            case FKV_PAGES_BF16: return launch_read<D, FKV_PAGES_BF16>(a, out_dtype, blocks, s);
            case FKV_PAGES_FP8: return launch_read<D, FKV_PAGES_FP8>(a, out_dtype, blocks, s);
            default: return launch_read<D, FKV_PAGES_FP8_INT4>(a, out_dtype, blocks, s);
        }
    };
    if (pages->D == 64) return go(std::integral_constant<int, 64>{});
    return go(std::integral_constant<int, 128>{});
}

}  // extern "C"
