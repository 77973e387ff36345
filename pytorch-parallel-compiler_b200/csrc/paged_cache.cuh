// The paged key-value cache of N models as the kernels see it, and the small
// integer helpers its addressing needs.
//
// Pages: k, v [n, pages, hk, page, d] dense, in the model's type, int8 or
// e4m3; the 8-bit formats keep one fp32 scale per (token, head) in
// [n, pages, hk, page]. Token p of sequence (i, b) lives in page
// table[i, b, p / page] of model i's pool, at offset p % page.
#pragma once

#include "common.cuh"

#include <cuda_fp8.h>

namespace widek {

// Quotient by a fixed divisor, for dividends below 2^31: q = (hi(x m) + x) >> s
// with s = ceil(log2 d), m = floor(2^32 (2^s - d) / d) + 1 (Granlund and
// Montgomery, division by invariant integers using multiplication).
struct FastDiv {
    uint32_t d, m, s;
    __host__ static FastDiv make(uint32_t d) {
        FastDiv f{d, 0, 0};
        while (f.s < 32 && (1ull << f.s) < d) ++f.s;
        f.m = (uint32_t)((((1ull << f.s) - d) << 32) / d + 1);
        return f;
    }
    __device__ __forceinline__ uint32_t div(uint32_t x) const { return (__umulhi(x, m) + x) >> s; }
    __device__ __forceinline__ uint32_t divmod(uint32_t x, uint32_t& rem) const {
        const uint32_t q = div(x);
        rem = x - q * d;
        return q;
    }
};

struct PagedCache {
    void *k, *v;
    float *ks, *vs;               // null unless the format is 8-bit
    const int* table;
    int64_t table_n, table_b;     // element strides of the table over models and sequences
    int pages, page, cols;        // pages per model, tokens per page, table entries per sequence
    FastDiv page_div;

    // Row (token slot) of one head inside model i's pool, or -1 where the
    // position or its table entry lies outside the pool.
    __device__ __forceinline__ int row(int64_t i, int64_t b, int hk, int h, int pos) const {
        uint32_t off;
        const uint32_t col = page_div.divmod((uint32_t)pos, off);
        if (pos < 0 || col >= (uint32_t)cols) return -1;
        const int p = __ldg(table + i * table_n + b * table_b + col);
        if ((uint32_t)p >= (uint32_t)pages) return -1;
        return (p * hk + h) * page + (int)off;
    }
};

// Storage formats of the cache (the dtype codes, then the 8-bit ones).
inline bool cache_fmt_8bit(int fmt) { return fmt == WIDEK_I8 || fmt == WIDEK_E4M3; }
inline size_t cache_fmt_size(int fmt) { return cache_fmt_8bit(fmt) ? 1 : dtype_size(fmt); }

// Checks the cache arguments shared by the entry points and fills `c`.
// cgeom: pages, page, table columns, table strides over models / sequences;
// calls: how many rows or sequences touch the cache (0: it may be null).
int cache_args(PagedCache& c, const char* what, void* k, void* v, float* ks, float* vs, const void* table,
               const int64_t* cgeom, int64_t calls, int64_t hk, int64_t d, int fmt, int dtype);

// An index that is stored as int32 or int64; values outside int32 saturate
// (every range check rejects them).
__device__ __forceinline__ int load_index(const void* p, int64_t i, int is64) {
    if (!is64) return __ldg(static_cast<const int*>(p) + i);
    const long long v = __ldg(static_cast<const long long*>(p) + i);
    return v < -1 ? -1 : (v > 0x7fffffffll ? 0x7fffffff : (int)v);
}

// Codes of an 8-bit row: scale = max(max|x|, kRowFloor) / Q in fp32 (Q = 127
// or 448), code = x / scale rounded half to even (to an integer, or to e4m3).
// The floor keeps the scale a normal number for a row of zeros, whose codes
// are then 0; a row that holds an infinity or a NaN gets such a scale and
// reads back as NaN throughout.
constexpr float kRowFloor = 9.094947017729282e-13f;   // 2^-40

__device__ __forceinline__ float code_scale(float amax, bool is_i8) {
    // amax is NaN when the row holds one: fmaxf would drop it
    const float m = amax != amax ? amax : fmaxf(amax, kRowFloor);
    return __fdiv_rn(m, is_i8 ? 127.f : 448.f);
}

__device__ __forceinline__ uint8_t code_i8(float x, float scale) {
    const int q = __float2int_rn(__fdiv_rn(x, scale));
    return (uint8_t)(int8_t)(q > 127 ? 127 : (q < -127 ? -127 : q));
}

__device__ __forceinline__ uint8_t code_e4m3(float x, float scale) {
    return (uint8_t)__nv_cvt_float_to_fp8(__fdiv_rn(x, scale), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float value_e4m3(uint8_t c) {
    __nv_fp8_e4m3 f;
    f.__x = c;
    return (float)f;
}

}  // namespace widek
