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

// Two fp32 operations in one instruction, each rounded as usual.
__device__ __forceinline__ void fma2(float& d0, float& d1, float a0, float a1, float b0, float b1, float c0, float c1) {
    asm("{.reg .b64 a, b, c, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c; mov.b64 {%0, %1}, d;}"
        : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void mul2(float& d0, float& d1, float a0, float a1, float b0, float b1) {
    asm("{.reg .b64 a, b, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mul.rn.f32x2 d, a, b; mov.b64 {%0, %1}, d;}"
        : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ void add2(float& d0, float& d1, float a0, float a1, float b0, float b1) {
    asm("{.reg .b64 a, b, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; add.rn.f32x2 d, a, b; mov.b64 {%0, %1}, d;}"
        : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
// d = a b + c, d = a b and d = a b with one b, over VEC elements.
template <int VEC>
__device__ __forceinline__ void fma_vec(float* d, const float* a, const float* b, const float* c) {
    if constexpr (VEC == 1) d[0] = fmaf(a[0], b[0], c[0]);
#pragma unroll
    for (int j = 0; j + 1 < VEC; j += 2) fma2(d[j], d[j + 1], a[j], a[j + 1], b[j], b[j + 1], c[j], c[j + 1]);
}
template <int VEC>
__device__ __forceinline__ void mul_vec(float* d, const float* a, const float* b) {
    if constexpr (VEC == 1) d[0] = a[0] * b[0];
#pragma unroll
    for (int j = 0; j + 1 < VEC; j += 2) mul2(d[j], d[j + 1], a[j], a[j + 1], b[j], b[j + 1]);
}
template <int VEC>
__device__ __forceinline__ void scale_vec(float* d, const float* a, float b) {
    if constexpr (VEC == 1) d[0] = a[0] * b;
#pragma unroll
    for (int j = 0; j + 1 < VEC; j += 2) mul2(d[j], d[j + 1], a[j], a[j + 1], b, b);
}
// Sum of a b over VEC elements, two partial sums.
template <int VEC>
__device__ __forceinline__ float dot_vec(const float* a, const float* b) {
    if constexpr (VEC == 1) return a[0] * b[0];
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int j = 0; j + 1 < VEC; j += 2) fma2(s0, s1, a[j], a[j + 1], b[j], b[j + 1], s0, s1);
    return s0 + s1;
}

// The larger of two magnitudes, NaN if either is (fmaxf would drop it).
__device__ __forceinline__ float amax2(float x, float y) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(fabsf(x)), "f"(fabsf(y)));
    return m;
}

// x / scale rounded once, for a row's VEC values, from the row's 1 / scale:
// the product q = x inv is off by a unit or two in the last place, its
// remainder x - q scale is exact in one fused multiply-add, and adding
// remainder * inv rounds to the quotient (Markstein, Computation of elementary
// functions on the IBM RISC System/6000 processor, 1990). A division for each
// value took the int8 write of 268 M values 341 us.
template <int VEC>
__device__ __forceinline__ void quotients(const float* x, float scale, float inv, float* q) {
    float rem[VEC], ns[VEC], in[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) ns[j] = -scale, in[j] = inv;
    mul_vec<VEC>(q, x, in);
    fma_vec<VEC>(rem, q, ns, x);
    fma_vec<VEC>(q, rem, in, q);
}

// Codes of a row's VEC values; 0 in a row whose scale is not finite.
template <int VEC>
__device__ __forceinline__ void codes_i8(const float* x, float scale, uint8_t* out) {
    const bool finite = scale < 3e38f;
    float q[VEC];
    quotients<VEC>(x, scale, __fdiv_rn(1.f, scale), q);
    // 1.5 * 2^23: the sum's low bits are q rounded half to even
    if constexpr (VEC == 1) q[0] += 12582912.f;
#pragma unroll
    for (int j = 0; j + 1 < VEC; j += 2) add2(q[j], q[j + 1], q[j], q[j + 1], 12582912.f, 12582912.f);
    if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int j = 0; j < VEC; j += 4) {
            const uint32_t lo = __byte_perm(__float_as_uint(q[j]), __float_as_uint(q[j + 1]), 0x0040);
            const uint32_t hi = __byte_perm(__float_as_uint(q[j + 2]), __float_as_uint(q[j + 3]), 0x0040);
            reinterpret_cast<uint32_t*>(out)[j / 4] = finite ? __byte_perm(lo, hi, 0x5410) : 0;
        }
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) out[j] = finite ? (uint8_t)__float_as_uint(q[j]) : 0;
    }
}

template <int VEC>
__device__ __forceinline__ void codes_e4m3(const float* x, float scale, uint8_t* out) {
    const bool finite = scale < 3e38f;
    float q[VEC];
    quotients<VEC>(x, scale, __fdiv_rn(1.f, scale), q);
    if constexpr (VEC == 1) out[0] = finite ? (uint8_t)__nv_cvt_float_to_fp8(q[0], __NV_SATFINITE, __NV_E4M3) : 0;
#pragma unroll
    for (int j = 0; j + 1 < VEC; j += 2) {
        const uint16_t c = __nv_cvt_float2_to_fp8x2(make_float2(q[j], q[j + 1]), __NV_SATFINITE, __NV_E4M3);
        reinterpret_cast<uint16_t*>(out)[j / 2] = finite ? c : 0;
    }
}

// Values of VEC codes (unscaled). An int8 by way of the fp32 number
// 2^23 + (code + 128): integer conversions run at a quarter of that rate.
template <int VEC>
__device__ __forceinline__ void values_i8(const uint8_t* c, float* x) {
    if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int j = 0; j < VEC; j += 4) {
            const uint32_t w = reinterpret_cast<const uint32_t*>(c)[j / 4] ^ 0x80808080u;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[j + e] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540 | e));
        }
#pragma unroll
        for (int j = 0; j < VEC; j += 2) add2(x[j], x[j + 1], x[j], x[j + 1], -8388736.f, -8388736.f);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] = __uint_as_float(0x4b000000u | (uint32_t)(c[j] ^ 0x80)) - 8388736.f;
    }
}
template <int VEC>
__device__ __forceinline__ void values_e4m3(const uint8_t* c, float* x) {
    if constexpr (VEC == 1) {
        __nv_fp8_e4m3 f;
        f.__x = c[0];
        x[0] = (float)f;
    }
#pragma unroll
    for (int j = 0; j + 1 < VEC; j += 2) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c[j] | (c[j + 1] << 8)), __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        x[j] = f.x;
        x[j + 1] = f.y;
    }
}

}  // namespace widek
