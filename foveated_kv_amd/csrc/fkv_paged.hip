// Paged KV cache: rotary positions, the write of new tokens (rotated and
// encoded on the way) and the read-back.  All three stream rows once: eight
// elements a lane, a row of D elements on D / 8 neighbouring lanes, so the
// row's reductions (largest magnitude, minimum and maximum) are DPP steps
// within 8 or 16 lanes and every access is 16 bytes a lane.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "fkv_paged.h"

namespace fkv {

// ---------------------------------------------------------------------------
// eight elements of an activation row
// ---------------------------------------------------------------------------

template <int DT>
__device__ inline void load8f(const char* row, int64_t elem, float (&x)[8]) {
    if (DT == FKV_F32) {
        const float4 a = ((const float4*)((const float*)row + elem))[0];
        const float4 b = ((const float4*)((const float*)row + elem))[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        return;
    }
    const uint4 w = *(const uint4*)((const uint16_t*)row + elem);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = DT == FKV_F16 ? h2f((uint16_t)u[i]) : __uint_as_float(u[i] << 16);
        x[2 * i + 1] = DT == FKV_F16 ? h2f((uint16_t)(u[i] >> 16)) : __uint_as_float(u[i] & 0xFFFF0000u);
    }
}

__device__ inline uint32_t pack_bf16(float a, float b) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    const bf2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
}
__device__ inline uint32_t pack_f16(float a, float b) { return (uint32_t)f2h(a) | ((uint32_t)f2h(b) << 16); }

template <int DT>
__device__ inline void store8f(char* row, int64_t elem, const float (&x)[8]) {
    if (DT == FKV_F32) {
        ((float4*)((float*)row + elem))[0] = make_float4(x[0], x[1], x[2], x[3]);
        ((float4*)((float*)row + elem))[1] = make_float4(x[4], x[5], x[6], x[7]);
        return;
    }
    auto two = [](float a, float b) { return DT == FKV_F16 ? pack_f16(a, b) : pack_bf16(a, b); };
    *(uint4*)((uint16_t*)row + elem) =
        make_uint4(two(x[0], x[1]), two(x[2], x[3]), two(x[4], x[5]), two(x[6], x[7]));
}

// ---------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------

struct RopeView {
    const float* table;
    int32_t n_pos, rot, interleaved;
};

// Elements [d0, d0 + 8) of a row at `pos`, rotated in place; `partner` holds
// elements [d0 + rot/2, ..) or [d0 - rot/2, ..) of the row in the half layout.
// The products of two fp32 numbers are exact in 64 bits, so the only rounding
// before the result's own is the sum's, in 64 bits, and its rounding to fp32:
// what a quantised key is decided from does not depend on the order of
// evaluation.  Memory stays the bound (see the kernels below).
__device__ inline void rotate8(float (&x)[8], const float (&partner)[8], const RopeView& r, int64_t pos, int d0) {
    if (d0 >= r.rot) return;
    const int hd = r.rot >> 1;
    const bool inside = pos >= 0 && pos < r.n_pos;
    const float* t = r.table + (inside ? pos : 0) * r.rot;
    if (r.interleaved) {
        const float4 c4 = *(const float4*)(t + (d0 >> 1)), s4 = *(const float4*)(t + hd + (d0 >> 1));
        const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const double a = x[2 * j], b = x[2 * j + 1], cd = c[j], sd = s[j];
            x[2 * j] = (float)fma(a, cd, -(b * sd));
            x[2 * j + 1] = (float)fma(b, cd, a * sd);
        }
    } else {
        const bool second = d0 >= hd;
        const int i0 = second ? d0 - hd : d0;
        float c[8], s[8];
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
            const float4 c4 = *(const float4*)(t + i0 + j), s4 = *(const float4*)(t + hd + i0 + j);
            c[j] = c4.x, c[j + 1] = c4.y, c[j + 2] = c4.z, c[j + 3] = c4.w;
            s[j] = s4.x, s[j + 1] = s4.y, s[j + 2] = s4.z, s[j + 3] = s4.w;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const double ps = (double)partner[j] * (double)s[j];
            x[j] = (float)fma((double)x[j], (double)c[j], second ? ps : -ps);
        }
    }
    if (!inside) {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = __builtin_nanf("");
    }
}

// Where the half layout's partner of elements [d0, d0 + 8) begins (d0 itself
// where nothing is rotated, so that every lane loads inside its row).
__device__ inline int partner_of(const RopeView& r, int d0) {
    const int hd = r.rot >> 1;
    if (r.interleaved || d0 >= r.rot) return d0;
    return d0 < hd ? d0 + hd : d0 - hd;
}

// One row of D elements on D / 8 lanes of one wave (rows never straddle
// waves, and every lane has read its elements and its partner's before any
// lane writes: out may be x).  A wave takes 64 / (D / 8) rows of consecutive
// heads, which share the position's table row in the L1.
template <int DT>
__global__ void __launch_bounds__(256) rope_kernel(RowsView x, RowsView out, RopeView rope, PositionsView pos,
                                                   uint32_t n_rows, uint32_t H, uint32_t L, uint32_t lanes,
                                                   uint32_t rows_per_wave) {
    constexpr int ES = DT == FKV_F32 ? 4 : 2;
    const uint32_t lane = threadIdx.x & 63, wave = blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t in_wave = lane / lanes;
    const uint64_t row = (uint64_t)wave * rows_per_wave + in_wave;
    if (in_wave >= rows_per_wave || row >= n_rows) return;
    const uint32_t r = (uint32_t)row, tok = r / H, h = r - tok * H, b = tok / L, l = tok - b * L;
    const int d0 = 8 * (lane - in_wave * lanes);
    const char* src = x.data + (b * x.sb + h * x.sh + l * x.sl) * ES;
    float v[8], p[8];
    load8f<DT>(src, d0, v);
    load8f<DT>(src, partner_of(rope, d0), p);
    __builtin_amdgcn_wave_barrier();
    rotate8(v, p, rope, position_of(pos, b, l), d0);
    __builtin_amdgcn_wave_barrier();
    store8f<DT>(out.data + (b * out.sb + h * out.sh + l * out.sl) * ES, d0, v);
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
// quotient is decided exactly: floor(d / s) within one unit in 64 bits, then
// the sign of d - (k + 1/2) s, whose fma rounds once.
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
    const double sd = s, inv = 1.0 / sd;
    uint32_t packed = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const double d = (double)x[j] - (double)lo;
        double k = floor(d * inv);
        const double r = fma(-(k + 0.5), sd, d);
        int c = (int)k;
        c += r > 0.0 || (r == 0.0 && (c & 1));
        c = c < 0 ? 0 : c > 15 ? 15 : c;
        if (!(s > 0.0f)) c = 0;
        packed |= (uint32_t)c << (4 * j);
    }
    return packed;
}

// Eight elements of row `row` of K (or V), stored as the format has them.
template <int D, int FMT, bool VALUE>
__device__ inline void store_row(const PageView& pg, int64_t row, int lane_in_row, const float (&x)[8]) {
    const int64_t at = row * D + 8 * lane_in_row;
    char* base = VALUE ? pg.v : pg.k;
    if (FMT == FKV_PAGES_F16) {
        store8f<FKV_F16>(base, at, x);
    } else if (FMT == FKV_PAGES_BF16) {
        store8f<FKV_BF16>(base, at, x);
    } else if (FMT == FKV_PAGES_FP8 || !VALUE) {
        uint32_t codes[2];
        const uint32_t byte = encode_fp8<D>(x, codes);
        if (row >= 0) {
            *(uint2*)(base + at) = make_uint2(codes[0], codes[1]);
            if (lane_in_row == 0) (VALUE ? (uint8_t*)pg.v_scale : pg.k_exp)[row] = (uint8_t)byte;
        }
    } else {
        float scale, zero;
        const uint32_t codes = encode_int4<D>(x, scale, zero);
        if (row >= 0) {
            *(uint32_t*)(base + at / 2) = codes;
            if (lane_in_row == 0) ((float2*)pg.v_scale)[row] = make_float2(scale, zero);
        }
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
    uint32_t n_rows, B, L, Hq;
};

// Rows (b, l, head) with the token's queries first, then its keys and its
// values: one launch for a decode step's rotation and its cache write.
template <int D, int DT, int FMT>
__global__ void __launch_bounds__(256) paged_write_kernel(WriteArgs a) {
    constexpr int LPR = D / 8, ES = DT == FKV_F32 ? 4 : 2;
    const uint32_t r = blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    if (r >= a.n_rows) return;
    const uint32_t HT = a.Hq + 2 * a.pg.H;
    const uint32_t tok = r / HT, hh = r - tok * HT, b = tok / a.L, l = tok - b * a.L;
    if (a.n_new && (int32_t)l >= a.n_new[b]) return;
    const int lr = threadIdx.x % LPR, d0 = 8 * lr;
    const int64_t pos = position_of(a.start, b, l);
    const bool is_q = hh < a.Hq, is_v = hh >= a.Hq + a.pg.H;
    const uint32_t h = is_q ? hh : is_v ? hh - a.Hq - a.pg.H : hh - a.Hq;
    const RowsView& in = is_q ? a.q : is_v ? a.v : a.k;
    const char* src = in.data + ((int64_t)b * in.sb + h * in.sh + l * in.sl) * ES;
    float x[8], p[8];
    load8f<DT>(src, d0, x);
    if (!is_v && a.rope.rot) {
        load8f<DT>(src, partner_of(a.rope, d0), p);
        __builtin_amdgcn_wave_barrier();
        rotate8(x, p, a.rope, pos, d0);
    }
    __builtin_amdgcn_wave_barrier();
    if (is_q) {
        store8f<DT>(a.q_out.data + ((int64_t)b * a.q_out.sb + h * a.q_out.sh + l * a.q_out.sl) * ES, d0, x);
        return;
    }
    // (all lanes of a row agree on its place, so they leave together)
    const int64_t row = page_row(a.pg, a.table, b, pos, h);
    if (row < 0) return;
    if (is_v) store_row<D, FMT, true>(a.pg, row, lr, x);
    else store_row<D, FMT, false>(a.pg, row, lr, x);
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
    if (FMT == FKV_PAGES_F16) {
        load8f<FKV_F16>(base, at, x);
    } else if (FMT == FKV_PAGES_BF16) {
        load8f<FKV_BF16>(base, at, x);
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
    uint32_t n_rows, S;
};

// Rows (b, h, s): neighbouring rows of a wave are neighbouring tokens of a
// page and of the result.
template <int D, int FMT, int DT>
__global__ void __launch_bounds__(256) paged_read_kernel(ReadArgs a) {
    constexpr int LPR = D / 8;
    const uint32_t r = blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    if (r >= a.n_rows) return;
    const uint32_t bh = r / a.S, s = r - bh * a.S, b = bh / a.pg.H, h = bh - b * a.pg.H;
    const int lr = threadIdx.x % LPR;
    float k[8] = {}, v[8] = {};
    const int64_t row = (int32_t)s < a.lens[b] ? page_row(a.pg, a.table, b, s, h) : -1;
    if (row >= 0) {
        load_row<D, FMT, false>(a.pg, row, lr, k);
        load_row<D, FMT, true>(a.pg, row, lr, v);
    }
    const int64_t at = (int64_t)r * D + 8 * lr;
    store8f<DT>(a.k, at, k);
    store8f<DT>(a.v, at, v);
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

template <int D, int DT>
static void launch_write(const WriteArgs& a, int format, uint32_t blocks, hipStream_t s) {
    switch (format) {
        case FKV_PAGES_F16: paged_write_kernel<D, DT, FKV_PAGES_F16><<<blocks, 256, 0, s>>>(a); break;
        case FKV_PAGES_BF16: paged_write_kernel<D, DT, FKV_PAGES_BF16><<<blocks, 256, 0, s>>>(a); break;
        case FKV_PAGES_FP8: paged_write_kernel<D, DT, FKV_PAGES_FP8><<<blocks, 256, 0, s>>>(a); break;
        default: paged_write_kernel<D, DT, FKV_PAGES_FP8_INT4><<<blocks, 256, 0, s>>>(a); break;
    }
}

template <int D, int FMT>
static void launch_read(const ReadArgs& a, int dtype, uint32_t blocks, hipStream_t s) {
    switch (dtype) {
        case FKV_F16: paged_read_kernel<D, FMT, FKV_F16><<<blocks, 256, 0, s>>>(a); break;
        case FKV_BF16: paged_read_kernel<D, FMT, FKV_BF16><<<blocks, 256, 0, s>>>(a); break;
        default: paged_read_kernel<D, FMT, FKV_F32><<<blocks, 256, 0, s>>>(a); break;
    }
}

}  // namespace fkv

using namespace fkv;

extern "C" {

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
    const uint32_t rows = (uint32_t)((int64_t)B * H * L), lanes = D / 8, rpw = 64 / lanes;
    const uint32_t blocks = (uint32_t)cdiv(rows, 4 * (int64_t)rpw);
    const RopeView rv{rope->table, rope->n_positions, rope->rot_dim, rope->interleaved};
    const PositionsView pv = positions_view(positions);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == FKV_F16)
        rope_kernel<FKV_F16><<<blocks, 256, 0, s>>>(rows_view(x), rows_view(out), rv, pv, rows, H, L, lanes, rpw);
    else if (dtype == FKV_BF16)
        rope_kernel<FKV_BF16><<<blocks, 256, 0, s>>>(rows_view(x), rows_view(out), rv, pv, rows, H, L, lanes, rpw);
    else
        rope_kernel<FKV_F32><<<blocks, 256, 0, s>>>(rows_view(x), rows_view(out), rv, pv, rows, H, L, lanes, rpw);
    return check_hip(hipGetLastError(), w);
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
    a.n_rows = (uint32_t)((int64_t)B * L * heads);
    a.B = B;
    a.L = L;
    a.Hq = q ? Hq : 0;
    const uint32_t blocks = (uint32_t)cdiv(a.n_rows, 256 / (pages->D / 8));
    hipStream_t s = (hipStream_t)stream;
    if (pages->D == 64) {
        if (dtype == FKV_F16) launch_write<64, FKV_F16>(a, pages->format, blocks, s);
        else if (dtype == FKV_BF16) launch_write<64, FKV_BF16>(a, pages->format, blocks, s);
        else launch_write<64, FKV_F32>(a, pages->format, blocks, s);
    } else {
        if (dtype == FKV_F16) launch_write<128, FKV_F16>(a, pages->format, blocks, s);
        else if (dtype == FKV_BF16) launch_write<128, FKV_BF16>(a, pages->format, blocks, s);
        else launch_write<128, FKV_F32>(a, pages->format, blocks, s);
    }
    return check_hip(hipGetLastError(), w);
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
    a.n_rows = (uint32_t)((int64_t)B * S * pages->H);
    a.S = S;
    const uint32_t blocks = (uint32_t)cdiv(a.n_rows, 256 / (pages->D / 8));
    hipStream_t s = (hipStream_t)stream;
    auto go = [&](auto d) {
        constexpr int D = decltype(d)::value;
        switch (pages->format) {
            case FKV_PAGES_F16: launch_read<D, FKV_PAGES_F16>(a, out_dtype, blocks, s); break;
            case FKV_PAGES_BF16: launch_read<D, FKV_PAGES_BF16>(a, out_dtype, blocks, s); break;
            case FKV_PAGES_FP8: launch_read<D, FKV_PAGES_FP8>(a, out_dtype, blocks, s); break;
            default: launch_read<D, FKV_PAGES_FP8_INT4>(a, out_dtype, blocks, s); break;
        }
    };
    if (pages->D == 64) go(std::integral_constant<int, 64>{});
    else go(std::integral_constant<int, 128>{});
    return check_hip(hipGetLastError(), w);
}

}  // extern "C"
