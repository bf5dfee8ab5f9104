// Paged KV cache: page addressing, row codecs and argument checks shared by
// the write / read / rotary kernels (fkv_paged.hip) and the one-token
// attention (fkv_paged_attn.hip).
#pragma once

#include "fkv_common.h"

namespace fkv {

// Device view of a layer's pages.  Row (page, h, off) is row
// (page * H + h) * page_size + off of every array: K and V rows of D elements
// (16-bit formats), D codes (E4M3) or D / 2 bytes (INT4), one exponent byte
// per E4M3 row and one (scale, zero) pair per INT4 row.
struct PageView {
    char* k;
    char* v;
    uint8_t* k_exp;
    char* v_scale;
    int32_t n_pages, page_size, H;
};

// Which page holds each sequence's tokens: entry (b, i) is the page of
// tokens [i * page_size, (i + 1) * page_size).
struct TableView {
    const int32_t* ids;
    int64_t stride;
    int32_t n;  // entries per sequence
};

// Tokens that a table may hold for a sequence.  Launches are planned for no more,
// whatever bound of the lengths a caller names.
constexpr int64_t kMostTokens = 0x7FFFFFFF - 4096;

// Rows (b, h, l) of an activation tensor, strides in elements.
struct RowsView {
    char* data;
    int64_t sb, sh, sl;
};

struct PositionsView {
    const void* data;
    int64_t sb, sl, base;
    int32_t is64, per_token;
};

__device__ inline int64_t position_of(const PositionsView& p, int64_t b, int64_t l) {
    int64_t v = p.base + (p.per_token ? 0 : l);
    if (p.data) {
        const int64_t i = b * p.sb + l * p.sl;
        v += p.is64 ? ((const int64_t*)p.data)[i] : (int64_t)((const int32_t*)p.data)[i];
    }
    return v;
}

// Row of the pages that holds token `pos` of sequence b, or -1: a position
// outside the table or a page id outside the pool names no row.
__device__ inline int64_t page_row(const PageView& pg, const TableView& t, int64_t b, int64_t pos, int32_t h) {
    if (pos < 0 || pos >= (int64_t)t.n * pg.page_size) return -1;
    const int32_t i = (int32_t)(pos >> (31 - __builtin_clz((unsigned)pg.page_size)));  // (a power of two)
    const int32_t off = (int32_t)pos & (pg.page_size - 1);
    const int32_t id = t.ids[b * t.stride + i];
    if ((uint32_t)id >= (uint32_t)pg.n_pages) return -1;
    return ((int64_t)id * pg.H + h) * pg.page_size + off;
}

// 2^e of an exponent byte (e + 127).
__device__ inline float exp_byte(uint32_t byte) { return __uint_as_float(byte << 23); }

template <typename T>
struct AsDeclared {
    using type = T;
};
// Starts a kernel -> FKV_OK, or this launch's own error with nothing started.
// (hipGetLastError() after a launch also reports, and clears, what an earlier
// call of the program's left behind: a failure although the kernel runs.)
template <typename... P>
int start_kernel(const char* who, void (*kernel)(P...), dim3 grid, uint32_t threads, hipStream_t s,
                 typename AsDeclared<P>::type... args) {
    void* p[] = {&args...};
    const hipError_t e = hipLaunchKernel((const void*)kernel, grid, dim3(threads), p, 0, s);
    if (e != hipSuccess) (void)hipGetLastError();  // (reported here, not by the next one to ask)
    return check_hip(e, who);
}

// Rows of a call: (B, H, L) of D elements of es bytes.
struct RowsShape {
    int64_t B, H, L, D, es;
};
// Refuses a result whose rows share memory with one another, or with rows that
// the call reads elsewhere.  `in_place`: rows that are the very ones read (the
// same address and strides) may be written, each by the lanes that read it.
int check_result_rows(const char* who, const char* name, const fkv_rows* out, const RowsShape& shape);
int check_apart(const char* who, const char* what, const fkv_rows* out, const RowsShape& out_shape, const fkv_rows* in,
                const RowsShape& in_shape, bool in_place);

int check_pages(const char* who, const fkv_pages* p);
int check_table(const char* who, const int32_t* table, int32_t n_table, int64_t stride, int32_t B);
PageView page_view(const fkv_pages* p);

// 16-bit numbers that the matrix products take two weights as, one after the other: the
// upper half of each (bf16), or the fp16 number nearest towards 0 and, next, kUp times
// what that leaves (see fkv_paged_attn.hip).
constexpr float kUp = 1024.0f;
__device__ inline uint32_t take_bf16(float& x, float& y) {
    const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
    x -= __uint_as_float(a & 0xFFFF0000u);
    y -= __uint_as_float(b & 0xFFFF0000u);
    return __builtin_amdgcn_perm(b, a, 0x07060302u);
}
__device__ inline uint32_t take_fp16(float& x, float& y) {
    const fkv_h2 h = __builtin_bit_cast(fkv_h2, __builtin_amdgcn_cvt_pkrtz(x, y));
    x = fmaf(-kUp, (float)h.x, kUp * x);
    y = fmaf(-kUp, (float)h.y, kUp * y);
    return as_u32(h);
}

template <int CTRL, int ROWS = 15>
__device__ inline uint32_t dpp_or_0(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 15, false);
}
template <int CTRL, int ROWS = 15>
__device__ inline double dpp_or_0(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)dpp_or_0<CTRL, ROWS>((uint32_t)(u >> 32)) << 32 | dpp_or_0<CTRL, ROWS>((uint32_t)u));
}
// The sum over the lanes up to and with this one.
template <typename T>
__device__ inline T sum_up_to(T v) {
    v += dpp_or_0<0x111>(v);  // row_shr:1, 2, 4, 8
    v += dpp_or_0<0x112>(v);
    v += dpp_or_0<0x114>(v);
    v += dpp_or_0<0x118>(v);
    v += dpp_or_0<0x142, 10>(v);  // row_bcast:15 into the second and fourth row
    return v + dpp_or_0<0x143, 12>(v);  // row_bcast:31 into the upper half
}
// The sum over a row of 16 lanes, in all of them.
template <typename T>
__device__ inline T row_sum(T v) {
    v += dpp_or_0<kDppXor1>(v);
    v += dpp_or_0<kDppXor2>(v);
    v += dpp_or_0<0x141>(v);         // row_half_mirror
    return v + dpp_or_0<0x140>(v);   // row_mirror
}

}  // namespace fkv
