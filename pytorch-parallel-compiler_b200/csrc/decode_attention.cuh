// Attention of one new token of every sequence over a paged key-value cache:
// the kernel and what its instantiations (one source file per cache format)
// and its dispatcher share.
//
//   z_p = scale q . k_p,  out = sum_p exp(z_p - m) v_p / sum_p exp(z_p - m),
//   m = max z, over the tokens max(0, len - window) <= p < len; zeros where
//   there is none.
//
// Bound by memory: every cached value is read once and serves the G = Hq / Hk
// query heads of its group, 2 G flops a value. At G = 8 and 8-bit values that
// is more than the CUDA cores give at the memory's rate, so both products run
// on the tensor pipe (warp-level MMA: with 8 columns of queries a tile of
// tcgen05 would be mostly padding, and the operands would have to pass through
// shared memory, which the layout below avoids).
//
// Mapping. A block takes one key head of one sequence and up to 8 NT of its
// query heads, over a range of tokens; its 4 warps take every 4th tile of
// 16 MT tokens each, with their own running maxima and sums. Both products put
// tokens or channels on the MMA's 16 rows and the query heads on its 8 columns:
//   S^T [tokens, heads] = K q^T, O^T [channels, heads] += V^T P^T.
// The channel order of a dot product is free, and so is the row order of O^T,
// so each lane's operands are whole 16-byte pieces of cached rows: for K rows g
// and g + 8 of the tile (g = lane / 4), 4 lanes side by side; for V 4 tokens, 8
// lanes side by side, token pairs joined by byte permutes. Each thread copies
// its own pieces into its own places of shared memory (cp.async, zeros for
// tokens and channels that are not there) and reads them back itself, so the
// ring needs no barrier and no swizzle: it only holds what is in flight, about
// 190 KB on an SM. Held in registers instead, one tile ahead, the same loop
// reached 3.5 of 6.5 TB/s: other instructions waited on the loads' scoreboards.
// The weights change layout (tokens from rows to the contraction) by 8x8
// transposes within the warp.
//
// Rounding. Scores, maxima, sums and outputs are fp32. Weights go into the
// second product as two pieces of the MMA's type (their sum has 16 bits or
// more; one piece alone would show in a bf16 result). fp32 caches split both
// operands in two tf32 pieces and drop the product of the low ones (2^-22).
// 8-bit codes are exact in f16 and in bf16. Against K, q is scaled by a power
// of two per head into f16's range, in two pieces when it is fp32 (16-bit
// queries stay exact, which bf16 would not give f16 ones). The scale of a key
// row multiplies its score; that of a value row goes into its weight, whose
// product p vs has no fixed range: V and the weights meet in bf16, which has
// fp32's.
#pragma once

#include "paged_cache.cuh"
#include "sm100_ptx.cuh"

#include <atomic>

namespace widek {

struct DecodeArgs {
    const void* q;
    const void* lengths;
    void* out;
    float* part_o;               // [n b hq, groups, d] partial outputs (relative to their own maximum)
    float2* part_ml;             // [n b hq, groups] maximum and sum
    int64_t q_n, q_b, q_h, len_n, len_b;
    int n, b, hq, hk, d, group, len64, window, dtype, fmt;
    int tiles, unit;             // query-head tiles of a group, tokens of a block's tiles
    int splits, cluster, groups; // ranges of a sequence, joined in clusters of blocks, groups = splits / cluster
    int q_vec;                   // query rows start at multiples of 16 bytes
    float scale_log2;            // scale * log2(e)
    PagedCache c;
    int* err;
};

constexpr int kDecodeWarps = 4;
constexpr int kMostCluster = 8;       // blocks of a cluster that any GPU of the architecture takes

// Visible tokens of a sequence and its cut into ranges: the same for the
// attention and the join.
struct DecodeRange {
    int start, len, chunk, active;
    __device__ __forceinline__ DecodeRange(const DecodeArgs& a, int64_t i, int64_t b) {
        len = load_index(a.lengths, i * a.len_n + b * a.len_b, a.len64);
        const int most = a.c.cols * a.c.page;
        if (len > most) {
            len = most;
            if (threadIdx.x == 0) raise_device_error(a.err, DEV_ERR_INDEX);
        }
        if (len < 0) len = 0;
        start = a.window > 0 && len > a.window ? len - a.window : 0;
        const int range = len - start;
        chunk = (range + a.splits - 1) / a.splits;
        chunk = max(1, (chunk + a.unit - 1) / a.unit) * a.unit;
        active = (range + chunk - 1) / chunk;
    }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void store_out(void* p, int64_t at, float v, int dtype) {
    if (dtype == WIDEK_F32) static_cast<float*>(p)[at] = v;
    else if (dtype == WIDEK_BF16) static_cast<__nv_bfloat16*>(p)[at] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[at] = __float2half_rn(v);
}

// N queries' channels from `at` on, in 16-byte loads.
template <int N>
__device__ __forceinline__ void load_in16(const void* p, int64_t at, int dtype, float (&x)[N]) {
    if (dtype == WIDEK_F32) {
#pragma unroll
        for (int e = 0; e < N; e += 4) load16<float>(static_cast<const float*>(p) + at + e, x + e);
    } else if constexpr (N % 8 == 0) {
#pragma unroll
        for (int e = 0; e < N; e += 8) {
            if (dtype == WIDEK_BF16) load16<__nv_bfloat16>(static_cast<const __nv_bfloat16*>(p) + at + e, x + e);
            else load16<__half>(static_cast<const __half*>(p) + at + e, x + e);
        }
    }
}

__device__ __forceinline__ float load_in(const void* p, int64_t at, int dtype) {
    if (dtype == WIDEK_F32) return __ldg(static_cast<const float*>(p) + at);
    const unsigned short u = __ldg(static_cast<const unsigned short*>(p) + at);
    return dtype == WIDEK_BF16 ? __bfloat162float(__ushort_as_bfloat16(u)) : __half2float(__ushort_as_half(u));
}

// ---------------------------------------------------------------------------
// MMA and register-layout helpers
// ---------------------------------------------------------------------------
enum DecodeKind : int { DK_BF16, DK_F16, DK_F32, DK_I8, DK_E4M3 };

template <int KIND>
struct Kind {
    static constexpr bool code = KIND == DK_I8 || KIND == DK_E4M3;
    static constexpr bool f32 = KIND == DK_F32;
    static constexpr int size = code ? 1 : (f32 ? 4 : 2);
    static constexpr int values = code ? DK_BF16 : KIND;     // type of the second product
    // f16 weights are held times 2^15, at the top of f16's range: two pieces
    // then keep 16 bits of a weight down to 2^-24 of the largest, and reach
    // to 2^-40 of it (bf16 and tf32 have fp32's exponents).
    static constexpr float lift = KIND == DK_F16 ? 15.f : 0.f;
};

// D (16 x 8) += A (16 x 16, or 16 x 8 of tf32) B, fp32 sums.
template <int KIND>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    if constexpr (KIND == DK_BF16) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else if constexpr (KIND == DK_F32) {
        asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
}

// x = hi + lo in tf32 pieces.
__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t& hi, uint32_t& lo) {
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(__uint_as_float(x)));
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(__uint_as_float(x) - __uint_as_float(hi)));
}

// Two fp32 as a pair of the MMA's 16-bit type, and what that rounding left.
template <int KIND>
__device__ __forceinline__ uint32_t pack2(float x, float y, float& rx, float& ry) {
    if constexpr (KIND == DK_BF16) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(x, y);
        rx = x - __low2float(p);
        ry = y - __high2float(p);
        return *reinterpret_cast<const uint32_t*>(&p);
    } else {
        const __half2 p = __floats2half2_rn(x, y);
        rx = x - __low2float(p);
        ry = y - __high2float(p);
        return *reinterpret_cast<const uint32_t*>(&p);
    }
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// Two 8-bit codes (the low or the high half of x) as f16. An int8 becomes
// the f16 number 1024 + (code + 128), less 1152: exact.
template <int KIND, int HALF>
__device__ __forceinline__ uint32_t code_pair(uint32_t x) {
    if constexpr (KIND == DK_I8) {          // x already holds code + 128
        const uint32_t u = prmt(x, 0x64646464u, HALF ? 0x4342 : 0x4140);
        const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __floats2half2_rn(1152.f, 1152.f));
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const uint16_t s = HALF ? (uint16_t)(x >> 16) : (uint16_t)x;
        uint32_t y;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(y) : "h"(s));
        return y;
    }
}

// The same as bf16: 0x4300 + (code & 127) is 128 + those bits, and
// 0x4300 + (code & 128) is 128 or 256, what they are too large by.
template <int KIND, int HALF>
__device__ __forceinline__ uint32_t code_pair_bf16(uint32_t x) {
    if constexpr (KIND == DK_I8) {
        const uint32_t u = prmt(x, 0x43434343u, HALF ? 0x4342 : 0x4140);
        const uint32_t bits = u & 0xff7fff7fu, more = u & 0xff80ff80u;
        const __nv_bfloat162 h = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&bits),
                                         *reinterpret_cast<const __nv_bfloat162*>(&more));
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const uint32_t y = code_pair<KIND, HALF>(x);
        const __nv_bfloat162 h = __float22bfloat162_rn(__half22float2(*reinterpret_cast<const __half2*>(&y)));
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

template <int KIND>
__device__ __forceinline__ uint32_t code_word(uint32_t w) {
    return KIND == DK_I8 ? w ^ 0x80808080u : w;
}

// How cached rows lie: of any size and place, of multiples of 16 bytes, or
// those with exactly the channels of the tiles.
enum RowsAre : int { ROWS_ANY, ROWS_16, ROWS_FULL };

// Copies W words at byte `off` of a cached row (of `bytes`) to shared memory
// without waiting; zeros past the row, or all of them unless `live`. Rows of
// 16 bytes' multiples have a piece inside or outside; others come as words
// (cp.async of 4 bytes) or, where even these are not aligned, as elements.
template <int W, int SIZE, int ROWS>
__device__ __forceinline__ void copy_piece(uint32_t dst, const uint8_t* row, int off, int bytes, bool words,
                                           bool live) {
    if constexpr (ROWS != ROWS_ANY) {
        const int n = live && (ROWS == ROWS_FULL || off < bytes) ? 4 * W : 0;
        if constexpr (W == 4)
            asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(row + off), "r"(n)
                         : "memory");
        else
            asm volatile("cp.async.ca.shared.global.L2::256B [%0], [%1], %2, %3;" ::"r"(dst), "l"(row + off),
                         "n"(4 * W), "r"(n) : "memory");
        return;
    }
    if (words) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const int n = live && off + 4 * w < bytes ? 4 : 0;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + 4 * w),
                         "l"(row + (n ? off + 4 * w : 0)), "r"(n) : "memory");
        }
    } else {
#pragma unroll
        for (int w = 0; w < W; ++w) {
            uint32_t x = 0;
#pragma unroll
            for (int e = 0; e < 4 / SIZE; ++e) {
                const int o = off + 4 * w + e * SIZE;
                if (live && o < bytes)
                    x |= (uint32_t)(SIZE == 1 ? __ldg(row + o) : __ldg(reinterpret_cast<const uint16_t*>(row + o)))
                         << (8 * SIZE * e);
            }
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst + 4 * w), "r"(x) : "memory");
        }
    }
}

template <int W>
__device__ __forceinline__ void read_piece(uint32_t (&r)[W], uint32_t src) {
    if constexpr (W == 4)
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(src) : "memory");
    else if constexpr (W == 2)
        asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(src) : "memory");
    else
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r[0]) : "r"(src) : "memory");
}

__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// ---------------------------------------------------------------------------
// The kernel
//   DP     channels the tiles cover (the head's are fewer or equal)
//   NT     tiles of 8 query heads
//   MT     tiles of 16 tokens a warp has in registers at a time
//   SPLITQ the queries need two f16 pieces (8-bit cache, fp32 queries)
// ---------------------------------------------------------------------------
template <int KIND, int DP, int NT, int ROWS, bool SPLITQ>
struct DecodeShape {
    static constexpr int size = Kind<KIND>::size;
    static constexpr int row_bytes = DP * size;
    // tiles of a warp: 4 KB of K and 4 KB of V, more where 16 tokens already are
    static constexpr int MT = row_bytes >= 256 ? 1 : 256 / row_bytes;
    static constexpr int TOK = 16 * MT;
    static constexpr int KD = 16 / size < DP / 4 ? 16 / size : DP / 4;      // channels of a lane's K piece
    static constexpr int VD = 16 / size < DP / 8 ? 16 / size : DP / 8;      // and of its V piece
    static constexpr int KP = DP / 4 / KD, VP = DP / 8 / VD;                // pieces of a row per lane
    static constexpr int KW = KD * size / 4, VW = VD * size / 4;            // words of a piece
    static constexpr int KR = Kind<KIND>::f32 ? KD : KD / 2;                // MMA registers of a K piece
    static constexpr int QR = KP * KR;                                      // MMA registers of a query row
    // pieces read back from the ring at a time: 32 words, so that their latencies overlap
    static constexpr int KB = 16 / (MT * KW) < KP ? 16 / (MT * KW) : KP;
    static constexpr int VB = 8 / (MT * VW) < 1 ? 1 : (8 / (MT * VW) < VP ? 8 / (MT * VW) : VP);
    static constexpr int NR = (TOK + 31) / 32;                              // token slots a lane looks up
    // Ring of `units` units, a unit being a tile of K or of V of each warp.
    // Unit 2 i is K of tile i, unit 2 i + 1 its V; unit j lies in place
    // j % units, and j + units is copied as soon as j has been read.
    static constexpr int unit = 32 * kDecodeWarps * TOK * row_bytes / 32;   // bytes
    static constexpr int units = row_bytes <= 256 ? 3 : 2;
    static constexpr int ring = units * unit;
    static constexpr int blocks =                                           // of an SM
        row_bytes > 512 ? 1 : (row_bytes > 256 || NT == 2 || SPLITQ || DP == 256 ? 2 : (Kind<KIND>::f32 ? 3 : 4));
    static constexpr int joined = kDecodeWarps * 8 * NT * (DP + 2) * 4;     // the warps' sums, over the ring
    static constexpr int smem = ring > joined ? ring : joined;
};

template <int KIND, int DP, int NT, int ROWS, bool SPLITQ>
__global__ void __launch_bounds__(32 * kDecodeWarps, DecodeShape<KIND, DP, NT, ROWS, SPLITQ>::blocks)
    decode_kernel(const __grid_constant__ DecodeArgs a) {
    using S = DecodeShape<KIND, DP, NT, ROWS, SPLITQ>;
    using K = Kind<KIND>;
    constexpr int MT = S::MT, TOK = S::TOK;
    extern __shared__ __align__(16) uint8_t decode_ring[];
    uint8_t* const ring = decode_ring;
    __shared__ float sm_m[kDecodeWarps][8 * NT], sm_l[kDecodeWarps][8 * NT];
    __shared__ float2 sm_ml[8 * NT], sm_all[kMostCluster][8 * NT];
    // scales of the key and value rows of a tile and the next
    __shared__ float sm_s[2][kDecodeWarps][2][K::code ? TOK : 1];
    float(*sm_o)[8 * NT][DP + 2] = reinterpret_cast<float(*)[8 * NT][DP + 2]>(ring);

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, c = lane & 3;
    const int tile = blockIdx.x % a.tiles;
    const int kh = blockIdx.x / a.tiles % a.hk;
    const int64_t nb = blockIdx.x / a.tiles / a.hk;
    const int64_t i = nb / a.b, b = nb % a.b;
    const DecodeRange rg(a, i, b);
    if (a.groups > 1) sm100::grid_dep_launch_dependents();     // the join waits for this grid's end by itself
    const int split = blockIdx.y;
    // ranges that a short sequence does not have: their blocks are needed only
    // by a cluster that has others
    if (split >= rg.active && split / a.cluster * a.cluster >= max(rg.active, 1)) return;
    const int first = rg.start + split * rg.chunk;
    const int end = min(rg.len, first + rg.chunk);
    const int h0 = tile * 8 * NT;                        // first query head of the group here
    const int heads = min(8 * NT, a.group - h0);
    const int bytes = a.d * S::size;
    const int64_t pool = i * a.c.pages * a.hk * a.c.page;     // first row of this model's pool
    const uint8_t* kbase = static_cast<const uint8_t*>(a.c.k) + pool * bytes;
    const uint8_t* vbase = static_cast<const uint8_t*>(a.c.v) + pool * bytes;
    const bool words = ((bytes | reinterpret_cast<uintptr_t>(a.c.k) | reinterpret_cast<uintptr_t>(a.c.v)) & 3) == 0;

    // --- token slots: lane holds those of tokens (lane + 32 r) of a tile; -1
    // past the end, -2 where the table names no page of the pool
    auto look_up = [&](int (&rows)[S::NR], int tb) {
#pragma unroll
        for (int r = 0; r < S::NR; ++r) {
            const int p = tb + (TOK < 32 ? lane & (TOK - 1) : lane + 32 * r);
            rows[r] = p < end ? a.c.row(i, b, a.hk, kh, p) : -1;
            if (p < end && rows[r] < 0) rows[r] = -2;
        }
    };
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(ring);
    auto k_place = [&](int place, int mt, int hf, int p) {
        return mine + place * S::unit + (((mt * 2 + hf) * S::KP + p) * 32 * kDecodeWarps + threadIdx.x) * S::KW * 4;
    };
    auto v_place = [&](int place, int mt, int t, int p) {
        return mine + place * S::unit + (((mt * 4 + t) * S::VP + p) * 32 * kDecodeWarps + threadIdx.x) * S::VW * 4;
    };
    // K pieces of tokens g and g + 8 of every 16, the tile's scales, and a bit for each token that is there
    auto copy_k = [&](int place, int turn, const int (&rows)[S::NR], uint32_t (&seen)[S::NR]) {
#pragma unroll
        for (int r = 0; r < S::NR; ++r) {
            seen[r] = __ballot_sync(0xffffffffu, rows[r] >= 0);
            if (rows[r] == -2) raise_device_error(a.err, DEV_ERR_INDEX);
            if constexpr (K::code) {
                const int64_t at = pool + (rows[r] < 0 ? 0 : rows[r]);
                const int n = rows[r] >= 0 ? 4 : 0, t = TOK < 32 ? lane & (TOK - 1) : lane + 32 * r;
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                                 (uint32_t)__cvta_generic_to_shared(&sm_s[turn][warp][0][t])),
                             "l"(a.c.ks + at), "r"(n) : "memory");
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                                 (uint32_t)__cvta_generic_to_shared(&sm_s[turn][warp][1][t])),
                             "l"(a.c.vs + at), "r"(n) : "memory");
            }
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                // token 16 mt + 8 hf + g: the register that holds it is known at compile time, the lane is not
                const int r = __shfl_sync(0xffffffffu, rows[S::NR == 1 ? 0 : mt >> 1], (16 * mt + 8 * hf + g) & 31);
                const uint8_t* row = kbase + (int64_t)max(r, 0) * bytes;
#pragma unroll
                for (int p = 0; p < S::KP; ++p)
                    copy_piece<S::KW, S::size, ROWS>(k_place(place, mt, hf, p), row, (p * 4 + c) * S::KD * S::size,
                                                        bytes, words, r >= 0);
            }
    };
    auto copy_v = [&](int place, const int (&rows)[S::NR]) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                // the k index of lane c: tokens 2c, 2c + 1, 2c + 8, 2c + 9; tf32 c, c + 4, c + 8, c + 12
                const int tok = K::f32 ? c + 4 * t : 2 * c + (t & 1) + 8 * (t >> 1);
                const int r = __shfl_sync(0xffffffffu, rows[S::NR == 1 ? 0 : mt >> 1], (16 * mt + tok) & 31);
                const uint8_t* row = vbase + (int64_t)max(r, 0) * bytes;
#pragma unroll
                for (int p = 0; p < S::VP; ++p)
                    copy_piece<S::VW, S::size, ROWS>(v_place(place, mt, t, p), row, (p * 8 + g) * S::VD * S::size,
                                                        bytes, words, r >= 0);
            }
    };

    constexpr int STEP = kDecodeWarps * TOK;
    int tb = first + warp * TOK;
    int r1[S::NR], r2[S::NR];                // slots of the next tile and of the one after it
    uint32_t seen[2][S::NR];                 // tokens that are there, of the current tile and the next
    {
        int r0[S::NR];
        look_up(r0, tb);
        look_up(r1, tb + STEP);
        if constexpr (S::units == 3) look_up(r2, tb + 2 * STEP);
        copy_k(0, 0, r0, seen[0]);
        copy_commit();
        copy_v(1, r0);
        copy_commit();
        if constexpr (S::units == 3) {
            copy_k(2, 1, r1, seen[1]);
            copy_commit();
        }
    }

    // --- query fragments: lane (g, c) holds head g's channels of its K pieces
    uint32_t q[NT][S::QR], ql[SPLITQ ? NT : 1][SPLITQ ? S::QR : 1];
    float zs[NT][2];                                     // what a score is multiplied by, heads 2c and 2c + 1
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int h = t * 8 + g;
        const int64_t at = i * a.q_n + b * a.q_b + (int64_t)(kh * a.group + h0 + (h < heads ? h : 0)) * a.q_h;
        float x[S::KP][S::KD];
        float top = 0.f;
#pragma unroll
        for (int p = 0; p < S::KP; ++p) {
            const int ch = (p * 4 + c) * S::KD;
#pragma unroll
            for (int e = 0; e < S::KD; ++e) x[p][e] = 0.f;
            if (ROWS != ROWS_ANY && a.q_vec) {
                if (h < heads && ch < a.d) load_in16<S::KD>(a.q, at + ch, a.dtype, x[p]);
            } else {
#pragma unroll
                for (int e = 0; e < S::KD; ++e)
                    if (h < heads && ch + e < a.d) x[p][e] = load_in(a.q, at + ch + e, a.dtype);
            }
#pragma unroll
            for (int e = 0; e < S::KD; ++e) top = fmaxf(top, fabsf(x[p][e]));
        }
        zs[t][0] = zs[t][1] = a.scale_log2;
        float up = 1.f;
        if constexpr (K::code) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^(14 - exponent): the largest magnitude lands in [2^14, 2^15)
            const int ex = (int)(__float_as_uint(top) >> 23);
            const bool sized = ex >= 16 && ex < 255;
            up = sized ? __uint_as_float((uint32_t)(268 - ex) << 23) : 1.f;
            const float down = sized ? __uint_as_float((uint32_t)(ex - 14) << 23) : 1.f;
            zs[t][0] *= __shfl_sync(0xffffffffu, down, 8 * c);
            zs[t][1] *= __shfl_sync(0xffffffffu, down, 8 * c + 4);
        }
#pragma unroll
        for (int p = 0; p < S::KP; ++p)
#pragma unroll
            for (int e = 0; e < S::KR; ++e) {
                if constexpr (K::f32) {
                    q[t][p * S::KR + e] = __float_as_uint(x[p][e]);
                } else {
                    float rx, ry;
                    q[t][p * S::KR + e] = pack2<KIND>(x[p][2 * e] * up, x[p][2 * e + 1] * up, rx, ry);
                    if constexpr (SPLITQ) ql[t][p * S::KR + e] = pack2<KIND>(rx, ry, rx, ry);
                }
            }
    }

    float acc[NT][DP / 16][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int j = 0; j < DP / 16; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[t][j][e] = 0.f;
        m[t][0] = m[t][1] = -INFINITY;
        l[t][0] = l[t][1] = 0.f;
    }

    // S^T += K q^T over the pieces in registers
    float s[NT][MT][4];
    auto scores = [&](int place) {
        uint32_t batch[MT][S::KB][2][S::KW];
#pragma unroll
        for (int p0 = 0; p0 < S::KP; p0 += S::KB) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int p = 0; p < S::KB; ++p)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) read_piece<S::KW>(batch[mt][p][hf], k_place(place, mt, hf, p0 + p));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int p = p0; p < p0 + S::KB; ++p) {
                const uint32_t(&kr)[2][S::KW] = batch[mt][p - p0];
                if constexpr (K::f32) {
                    // the tensor core's sums round towards zero: chains of 6, added up in fp32
                    float part[NT][4];
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int j = 0; j < 4; ++j) part[t][j] = 0.f;
#pragma unroll
                    for (int e = 0; e < S::KR; e += 2) {
                        uint32_t hi[4], lo[4];
                        split_tf32(kr[0][e], hi[0], lo[0]);
                        split_tf32(kr[1][e], hi[1], lo[1]);
                        split_tf32(kr[0][e + 1], hi[2], lo[2]);
                        split_tf32(kr[1][e + 1], hi[3], lo[3]);
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            uint32_t qh0, ql0, qh1, ql1;
                            split_tf32(q[t][p * S::KR + e], qh0, ql0);
                            split_tf32(q[t][p * S::KR + e + 1], qh1, ql1);
                            mma<KIND>(part[t], lo[0], lo[1], lo[2], lo[3], qh0, qh1);
                            mma<KIND>(part[t], hi[0], hi[1], hi[2], hi[3], ql0, ql1);
                            mma<KIND>(part[t], hi[0], hi[1], hi[2], hi[3], qh0, qh1);
                        }
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[t][mt][j] += part[t][j];
                } else {
                    uint32_t r0[S::KR], r1[S::KR];
                    if constexpr (K::code) {
#pragma unroll
                        for (int w = 0; w < S::KW; ++w) {
                            const uint32_t x0 = code_word<KIND>(kr[0][w]), x1 = code_word<KIND>(kr[1][w]);
                            r0[2 * w] = code_pair<KIND, 0>(x0);
                            r0[2 * w + 1] = code_pair<KIND, 1>(x0);
                            r1[2 * w] = code_pair<KIND, 0>(x1);
                            r1[2 * w + 1] = code_pair<KIND, 1>(x1);
                        }
                    } else {
#pragma unroll
                        for (int w = 0; w < S::KW; ++w) r0[w] = kr[0][w], r1[w] = kr[1][w];
                    }
#pragma unroll
                    for (int e = 0; e < S::KR; e += 2)
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            const int j = p * S::KR + e;
                            if constexpr (SPLITQ)
                                mma<KIND>(s[t][mt], r0[e], r1[e], r0[e + 1], r1[e + 1], ql[t][j], ql[t][j + 1]);
                            mma<KIND>(s[t][mt], r0[e], r1[e], r0[e + 1], r1[e + 1], q[t][j], q[t][j + 1]);
                        }
                }
            }
        }
    };
    // Running maxima and sums; s becomes the weights that meet V.
    auto softmax = [&](const uint32_t (&seen)[S::NR], const float (&kt)[MT][2], const float (&vt)[MT][2]) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    s[t][mt][e] *= K::code ? zs[t][e & 1] * kt[mt][e >> 1] : zs[t][e & 1];
        bool all = true;
#pragma unroll
        for (int r = 0; r < S::NR; ++r) all = all && seen[r] == 0xffffffffu;
        if (!all) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!((seen[S::NR == 1 ? 0 : mt >> 1] >> ((16 * mt + 8 * (e >> 1) + g) & 31)) & 1))
                            s[t][mt][e] = -INFINITY;
        }
        float f[NT][2];
        bool same = true;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float top = -INFINITY;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) top = fmaxf(top, fmaxf(s[t][mt][e], s[t][mt][2 + e]));
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                top = fmaxf(top, m[t][e]);
                const float ref = top == -INFINITY ? 0.f : top;
                f[t][e] = ex2(m[t][e] - ref);
                m[t][e] = top;
                float sum = 0.f;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const float w = ex2(s[t][mt][2 * hf + e] - ref);
                        sum += w;
                        s[t][mt][2 * hf + e] = K::code ? w * vt[mt][hf] : (K::lift > 0.f ? w * 32768.f : w);
                    }
                l[t][e] = l[t][e] * f[t][e] + sum;
                same = same && f[t][e] == 1.f;
            }
        if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < DP / 16; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[t][j][e] *= f[t][e & 1];
        }
    };
    // Weights as B operands: hi and lo pieces of tokens (k) by heads (n)
    uint32_t ph[NT][MT][K::f32 ? 4 : 2], pl[NT][MT][K::f32 ? 4 : 2];
    auto turn_weights = [&]() {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                if constexpr (K::f32) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {        // tokens c + 4 j
                        const int src = ((c + 4 * (j & 1)) << 2) + (g >> 1);
                        const float x0 = __shfl_sync(0xffffffffu, s[t][mt][2 * (j >> 1)], src);
                        const float x1 = __shfl_sync(0xffffffffu, s[t][mt][2 * (j >> 1) + 1], src);
                        split_tf32(__float_as_uint(g & 1 ? x1 : x0), ph[t][mt][j], pl[t][mt][j]);
                    }
                } else {
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        float rx, ry;
                        const uint32_t hi = pack2<K::values>(s[t][mt][2 * hf], s[t][mt][2 * hf + 1], rx, ry);
                        const uint32_t lo = pack2<K::values>(rx, ry, rx, ry);
                        ph[t][mt][hf] = transpose8x8(hi);
                        pl[t][mt][hf] = transpose8x8(lo);
                    }
                }
            }
    };
    // O^T += V^T P^T over the pieces in registers
    auto values = [&](int place) {
        uint32_t batch[MT][S::VB][4][S::VW];
#pragma unroll
        for (int p0 = 0; p0 < S::VP; p0 += S::VB) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int p = 0; p < S::VB; ++p)
#pragma unroll
                for (int t = 0; t < 4; ++t) read_piece<S::VW>(batch[mt][p][t], v_place(place, mt, t, p0 + p));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int p = p0; p < p0 + S::VB; ++p) {
                const uint32_t(&vr)[4][S::VW] = batch[mt][p - p0];
                if constexpr (K::f32) {
#pragma unroll
                    for (int e = 0; e < S::VD; e += 2) {
                        float part[NT][4];
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int j = 0; j < 4; ++j) part[t][j] = 0.f;
#pragma unroll
                        for (int k8 = 0; k8 < 2; ++k8) {
                            uint32_t hi[4], lo[4];
                            split_tf32(vr[2 * k8][e], hi[0], lo[0]);
                            split_tf32(vr[2 * k8][e + 1], hi[1], lo[1]);
                            split_tf32(vr[2 * k8 + 1][e], hi[2], lo[2]);
                            split_tf32(vr[2 * k8 + 1][e + 1], hi[3], lo[3]);
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
                                const uint32_t* bh = &ph[t][mt][2 * k8];
                                const uint32_t* bl = &pl[t][mt][2 * k8];
                                mma<KIND>(part[t], lo[0], lo[1], lo[2], lo[3], bh[0], bh[1]);
                                mma<KIND>(part[t], hi[0], hi[1], hi[2], hi[3], bl[0], bl[1]);
                                mma<KIND>(part[t], hi[0], hi[1], hi[2], hi[3], bh[0], bh[1]);
                            }
                        }
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int j = 0; j < 4; ++j) acc[t][(p * S::VD + e) / 2][j] += part[t][j];
                    }
                } else {
                    uint32_t av[S::VD / 2][4];
                    if constexpr (K::code) {
#pragma unroll
                        for (int w = 0; w < S::VW; ++w) {
                            uint32_t x[4];
#pragma unroll
                            for (int t = 0; t < 4; ++t) x[t] = vr[t][w];
#pragma unroll
                            for (int k = 0; k < 2; ++k) {            // token pairs
                                const uint32_t x01 = prmt(x[2 * k], x[2 * k + 1], 0x5140);
                                const uint32_t x23 = prmt(x[2 * k], x[2 * k + 1], 0x7362);
                                av[2 * w][2 * k] = code_pair_bf16<KIND, 0>(x01);
                                av[2 * w][2 * k + 1] = code_pair_bf16<KIND, 1>(x01);
                                av[2 * w + 1][2 * k] = code_pair_bf16<KIND, 0>(x23);
                                av[2 * w + 1][2 * k + 1] = code_pair_bf16<KIND, 1>(x23);
                            }
                        }
                    } else {
#pragma unroll
                        for (int w = 0; w < S::VW; ++w) {
                            av[w][0] = prmt(vr[0][w], vr[1][w], 0x5410);
                            av[w][1] = prmt(vr[0][w], vr[1][w], 0x7632);
                            av[w][2] = prmt(vr[2][w], vr[3][w], 0x5410);
                            av[w][3] = prmt(vr[2][w], vr[3][w], 0x7632);
                        }
                    }
#pragma unroll
                    for (int w = 0; w < S::VD / 2; ++w)
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            float(&o)[4] = acc[t][p * S::VD / 2 + w];
                            mma<K::values>(o, av[w][0], av[w][1], av[w][2], av[w][3], pl[t][mt][0], pl[t][mt][1]);
                            mma<K::values>(o, av[w][0], av[w][1], av[w][2], av[w][3], ph[t][mt][0], ph[t][mt][1]);
                        }
                }
            }
        }
    };
    auto clear_scores = [&]() {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][mt][e] = 0.f;
    };

    int place = 0, turn = 0;
    for (; tb < end; tb += STEP) {
        copy_wait<S::units - 1>();
        float kt[MT][2], vt[MT][2];
        if constexpr (K::code) {
            __syncwarp();
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    kt[mt][hf] = sm_s[turn][warp][0][16 * mt + 8 * hf + g];
                    vt[mt][hf] = sm_s[turn][warp][1][16 * mt + 8 * hf + g];
                }
            __syncwarp();
        }
        clear_scores();
        scores(place);
        const int second = S::units == 3 && place == 2 ? 0 : place + 1;
        uint32_t now[S::NR];
#pragma unroll
        for (int r = 0; r < S::NR; ++r) now[r] = seen[0][r], seen[0][r] = seen[1][r];
        if constexpr (S::units == 3) {
            if (tb + STEP < end) copy_v(place, r1);
            copy_commit();
        } else {
            if (tb + STEP < end) copy_k(place, 0, r1, seen[0]);
            copy_commit();
        }
        softmax(now, kt, vt);
        turn_weights();
        copy_wait<S::units - 1>();
        values(second);
        if constexpr (S::units == 3) {
            if (tb + 2 * STEP < end) copy_k(second, turn, r2, seen[1]);
            copy_commit();
#pragma unroll
            for (int r = 0; r < S::NR; ++r) r1[r] = r2[r];
            look_up(r2, tb + 3 * STEP);
            turn ^= 1;
            place = place == 0 ? 2 : place - 1;          // (place + 2) % 3
        } else {
            if (tb + STEP < end) copy_v(second, r1);
            copy_commit();
            look_up(r1, tb + 2 * STEP);
        }
    }
    copy_wait<0>();
    __syncthreads();             // the ring now takes the warps' sums

    // --- join the warps
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], o);
            if (g == 0) {
                const int h = t * 8 + 2 * c + e;
                sm_m[warp][h] = m[t][e];
                sm_l[warp][h] = l[t][e];
            }
#pragma unroll
            for (int j = 0; j < DP / 16; ++j) {
                const int ch = j / (S::VD / 2) * 8 * S::VD + g * S::VD + j % (S::VD / 2) * 2;
                *reinterpret_cast<float2*>(&sm_o[warp][t * 8 + 2 * c + e][ch]) = make_float2(acc[t][j][e], acc[t][j][e + 2]);
            }
        }
    __syncthreads();
    const int64_t row0 = (i * a.b + b) * a.hq + (int64_t)kh * a.group + h0;
    const bool last = a.cluster == 1;                 // nothing to join within a cluster
    const bool whole = rg.active <= a.cluster;        // nothing to join after it
    const int group = split / a.cluster;
    auto put = [&](int h, int ch, float o, float total) {
        if (whole) store_out(a.out, (row0 + h) * a.d + ch, total == 0.f ? 0.f : o / total, a.dtype);
        else a.part_o[((row0 + h) * a.groups + group) * a.d + ch] = o;
    };
    for (int h = warp; h < heads; h += kDecodeWarps) {
        float top = sm_m[0][h];
#pragma unroll
        for (int w = 1; w < kDecodeWarps; ++w) top = fmaxf(top, sm_m[w][h]);
        const float ref = top == -INFINITY ? 0.f : top;
        float total = 0.f, f[kDecodeWarps];
#pragma unroll
        for (int w = 0; w < kDecodeWarps; ++w) {
            total += ex2(sm_m[w][h] - ref) * sm_l[w][h];
            f[w] = ex2(sm_m[w][h] - ref - K::lift);
        }
        for (int ch = lane; ch < a.d; ch += 32) {
            float o = 0.f;
#pragma unroll
            for (int w = 0; w < kDecodeWarps; ++w) o += f[w] * sm_o[w][h][ch];
            if (last) put(h, ch, o, total);
            else sm_o[0][h][ch] = o;                  // in place: this thread alone reads and writes it
        }
        if (lane == 0) {
            if (last && !whole) a.part_ml[(row0 + h) * a.groups + group] = make_float2(top, total);
            sm_ml[h] = make_float2(top, total);
        }
    }
    if (last) return;
    __syncwarp();

    // --- join the cluster's ranges: each block reads its share of the
    // channels from all blocks' shared memory, in the order of the ranges
    sm100::cluster_sync_all();
    const int rank = split % a.cluster;
    const int ranks = min(a.cluster, rg.active - group * a.cluster);
    for (int e = threadIdx.x; e < ranks * 8 * NT; e += 32 * kDecodeWarps) {
        const uint32_t at = sm100::map_to_rank(sm100::smem_addr(&sm_ml[e % (8 * NT)]), e / (8 * NT));
        float x, y;
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x), "=f"(y) : "r"(at) : "memory");
        sm_all[e / (8 * NT)][e % (8 * NT)] = make_float2(x, y);
    }
    __syncthreads();
    for (int e = rank * 32 * kDecodeWarps + threadIdx.x; e < heads * a.d; e += a.cluster * 32 * kDecodeWarps) {
        const int h = e / a.d, ch = e - h * a.d;
        float top = -INFINITY;
        for (int r = 0; r < ranks; ++r) top = fmaxf(top, sm_all[r][h].x);
        const float ref = top == -INFINITY ? 0.f : top;
        const uint32_t at = sm100::smem_addr(&sm_o[0][h][ch]);
        float o = 0.f, total = 0.f;
#pragma unroll 4
        for (int r = 0; r < ranks; ++r) {
            float x;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(sm100::map_to_rank(at, r)) : "memory");
            const float f = ex2(sm_all[r][h].x - ref);
            o += f * x;
            total += f * sm_all[r][h].y;
        }
        put(h, ch, o, total);
        if (!whole && ch == 0) a.part_ml[(row0 + h) * a.groups + group] = make_float2(top, total);
    }
    __syncwarp();
    sm100::cluster_sync_all();           // no block leaves while others read its sums
}

template <int KIND, int DP, int NT, int ROWS, bool SPLITQ>
int launch_decode_shape(const DecodeArgs& a, cudaStream_t st) {
    using S = DecodeShape<KIND, DP, NT, ROWS, SPLITQ>;
    auto kernel = decode_kernel<KIND, DP, NT, ROWS, SPLITQ>;
    static std::atomic<uint64_t> allowed{0};      // devices whose limit is raised
    const uint64_t bit = 1ull << (current_device() & 63);
    if (!(allowed.load(std::memory_order_relaxed) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem);
        if (e != cudaSuccess)
            return set_error(WIDEK_ERR_CUDA, "widek_decode_attention_fwd: shared memory of %d bytes: %s", S::smem,
                             cudaGetErrorString(e));
        allowed.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((int64_t)a.n * a.b * a.hk * a.tiles), (unsigned)a.splits);
    cfg.blockDim = dim3(32 * kDecodeWarps);
    cfg.dynamicSmemBytes = S::smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = (unsigned)a.cluster;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.cluster > 1 ? 1 : 0;
    cudaLaunchKernelEx(&cfg, kernel, a);
    return check_launch("widek_decode_attention_fwd");
}

// Query-head tiles of 8 in one block: two of them where a group has more
// than 8 heads, so that its cache is read once for 16; at d > 128, or with the
// split operands of fp32, their sums would not fit in registers beside the tile.
inline int decode_nt(int group, int d, int fmt) { return group > 8 && d <= 128 && fmt != WIDEK_F32 ? 2 : 1; }

// Tokens that the 4 warps of a block have in registers at a time.
inline int decode_unit(int d, int fmt) {
    const int bytes = (d <= 64 ? 64 : (d <= 128 ? 128 : 256)) * (int)cache_fmt_size(fmt);
    return kDecodeWarps * 16 * (bytes >= 256 ? 1 : 256 / bytes);
}

// Blocks of an SM, as DecodeShape has them (fp32 queries over codes: 2, not 4).
inline int decode_places(int d, int fmt, int nt) {
    const int bytes = (d <= 64 ? 64 : (d <= 128 ? 128 : 256)) * (int)cache_fmt_size(fmt);
    return bytes > 512 ? 1 : (bytes > 256 || nt == 2 || d > 128 ? 2 : (fmt == WIDEK_F32 ? 3 : 4));
}

template <int KIND, bool SPLITQ>
int launch_decode(const DecodeArgs& a, cudaStream_t st) {
    const bool aligned = (a.d * Kind<KIND>::size) % 16 == 0 && aligned16(a.c.k) && aligned16(a.c.v);
    const int nt = decode_nt(a.group, a.d, a.fmt);
#define WIDEK_DECODE(DP, NT)                                                             \
    return !aligned    ? launch_decode_shape<KIND, DP, NT, ROWS_ANY, SPLITQ>(a, st)      \
           : a.d == DP ? launch_decode_shape<KIND, DP, NT, ROWS_FULL, SPLITQ>(a, st)     \
                       : launch_decode_shape<KIND, DP, NT, ROWS_16, SPLITQ>(a, st)
    if constexpr (KIND != DK_F32) {
        if (nt == 2 && a.d <= 64) WIDEK_DECODE(64, 2);
        if (nt == 2) WIDEK_DECODE(128, 2);
    }
    if (a.d <= 64) WIDEK_DECODE(64, 1);
    if (a.d <= 128) WIDEK_DECODE(128, 1);
    WIDEK_DECODE(256, 1);
#undef WIDEK_DECODE
}

// One instantiation per source file (decode_attention_*.cu).
extern template int launch_decode<DK_BF16, false>(const DecodeArgs&, cudaStream_t);
extern template int launch_decode<DK_F16, false>(const DecodeArgs&, cudaStream_t);
extern template int launch_decode<DK_F32, false>(const DecodeArgs&, cudaStream_t);
extern template int launch_decode<DK_I8, false>(const DecodeArgs&, cudaStream_t);
extern template int launch_decode<DK_I8, true>(const DecodeArgs&, cudaStream_t);
extern template int launch_decode<DK_E4M3, false>(const DecodeArgs&, cudaStream_t);
extern template int launch_decode<DK_E4M3, true>(const DecodeArgs&, cudaStream_t);

}  // namespace widek
