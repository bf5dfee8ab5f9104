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

}  // namespace fkv
