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
// Work. A segment is one key head of one sequence with up to 8 NT of its query
// heads; it is walked in steps, a step being a tile of 16 MT tokens for each of
// a block's 4 warps. All segments' steps stand in one line, which the blocks
// (as many as the GPU holds) divide evenly: a block walks through segments of
// any length without a pause, the copies running ahead of the products over
// their borders. A segment that lies in several blocks leaves partial results,
// at most two for each block, which a second kernel joins in their order. (One
// block for each segment or fixed range lost 6.5 us of every block's life to
// its start and end, 45 of 328 us at 1.6 GB of bf16 pages.) With more
// sequences than are worth adding up, blocks take whole segments in turn.
//
// Mapping. Both products put tokens or channels on the MMA's 16 rows and the
// query heads on its 8 columns, each warp with its own running maxima and sums:
//   S^T [tokens, heads] = K q^T, O^T [channels, heads] += V^T P^T.
// The channel order of a dot product is free, and so is the row order of O^T,
// so each lane's operands are whole 16-byte pieces of cached rows: for K rows g
// and g + 8 of the tile (g = lane / 4), 4 lanes side by side; for V 4 tokens, 8
// lanes side by side, token pairs joined by byte permutes: no ldmatrix, no
// transposed copy. Each warp copies its own tiles into its own part of a ring
// in shared memory (cp.async of whole lines, zeros for tokens and channels that
// are not there), so the ring needs no barrier beyond the warp; it holds what
// is in flight, 128 KB and more on an SM. (Held in registers, one tile ahead,
// the loop reached 3.5 of 6.5 TB/s: other instructions waited on the loads'
// scoreboards. Copied by each lane for itself, 64 bytes of a row in a request,
// it stopped at 4.4 to 5.2 TB/s: the SM's requests in flight ran out.)
// The weights change layout (tokens from rows to the contraction) by 8x8
// transposes within the warp.
//
// Rounding. Scores, maxima, sums and outputs are fp32. Weights go into the
// second product as two pieces of the MMA's type (their sum has 16 bits or
// more; one piece alone would show in a bf16 result). fp32 caches split both
// operands in two tf32 pieces and drop the product of the low ones (2^-22).
// 8-bit codes are exact in f16 and in bf16. Against K, q is scaled by a power
// of two per head to the top of f16's range, in two pieces when it is fp32. A
// 16-bit query stays exact in channels above 2^-31 of the head's largest and is
// off by 2^-39 of it at most below (bf16 would round every f16 query). The scale
// of a key row multiplies its score; that of a value row goes into its weight, whose
// product p vs has no fixed range: V and the weights meet in bf16, which has
// fp32's, in three pieces where the result is fp32. The tensor core's sums
// round towards zero: fp32 results take them in short chains, added in fp32,
// and 16-bit ones in chains of 1024 tokens a warp, whose totals lie in the
// workspace meanwhile. (In one chain, 131072 values of one sign lost 1.8e-4 of
// their sum; 6e-6 so. Short chains for 16-bit results, as the adds and the
// registers of more products under way, cost 4 to 9 % with 8-bit caches or two
// head tiles; totals in local memory 4 to 6 % even where no chain was full;
// totals in the workspace 0 to 2 %, with 64 channels of 8 bits up to 3 %.)
//
// Measured (B200; floor at the measured copy rate): 1.6 GB of bf16 pages, 128
// ragged sequences, 32 over 8 heads of 128: 275 us (245). 411 MB of e4m3 pages,
// 256 sequences, 16 over 4 heads: 89 us (63); bound by instructions, of which
// the codes' conversion for the second product is the largest part. One int8
// sequence of 131007 tokens, 16 over 2 heads: 24 us (10.6), bound by the chain
// of loads at a block's start and end. fp32, window 511, heads of 84: 17 us (2).
#pragma once

#include "paged_cache.cuh"
#include "sm100_ptx.cuh"

#include <atomic>

namespace widek {

struct DecodeArgs {
    const void* q;
    const void* lengths;
    void* out;
    float* part_o;               // [blocks, 2, 8 NT, d] partial outputs (relative to their own maximum)
    float2* part_ml;             // [blocks, 2, 8 NT] maximum and sum
    float* done;                 // [blocks, NT (channels / 4 + 2), threads] totals of chains that are done
    int64_t q_n, q_b, q_h, len_n, len_b;
    int n, b, hq, hk, d, group, len64, window, dtype, fmt;
    int nt, tiles, step;         // 8 nt query heads of a segment, tiles of a group, tokens of a step
    int blocks, in_turn;         // blocks of the launch; whole segments in turn
    int q_vec;                   // query rows start at multiples of 16 bytes
    float scale_log2;            // scale * log2(e)
    PagedCache c;
    int* err;
};

constexpr int kDecodeWarps = 4;
constexpr int kChainTokens = 1024;           // of a warp in one chain of tensor-core sums of a 16-bit result

// Visible tokens of sequence nb.
struct DecodeRange {
    int start, len;
    __device__ __forceinline__ DecodeRange(const DecodeArgs& a, int nb) {
        const int i = nb / a.b, b = nb - i * a.b;
        len = load_index(a.lengths, i * a.len_n + b * a.len_b, a.len64);
        const int most = a.c.cols * a.c.page;
        if (len > most) {
            len = most;
            raise_device_error(a.err, DEV_ERR_INDEX);
        }
        if (len < 0) len = 0;
        start = a.window > 0 && len > a.window ? len - a.window : 0;
    }
    // Steps of one of its segments; an empty one has one, which writes zeros.
    __device__ __forceinline__ int steps(int step) const { return max(1, (len - start + step - 1) / step); }
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
    // The running maximum follows the scores only when they pass it by more:
    // weights up to 2^8 cost nothing where the exponents are fp32's, and the
    // sums then are rescaled a few times in a segment, not in most tiles.
    static constexpr float slack = KIND == DK_F16 ? 0.f : 8.f;
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

// How cached rows lie: of any size and place, as bytes that start inside words
// (see copy_place), of multiples of 16 bytes, or those with exactly the
// channels of the tiles.
enum RowsAre : int { ROWS_ANY, ROWS_BYTES, ROWS_16, ROWS_FULL };

// Copies 16 bytes at byte `off` of a cached row (of `bytes`) to shared memory
// without waiting; zeros past the row, or all of them unless `live`. Rows of
// 16 bytes' multiples have the place inside or outside; others come 8 or 4
// bytes at a time (cp.async's other sizes), as `grain`, the alignment of all
// rows, allows (below 4 bytes: copy_elements). ROWS_BYTES are rows of such
// sizes in a pool that starts on a word: they come as the words that they lie
// in, so that channel 0 is up to 3 bytes into the first place (`off` then
// counts from there), and the reader shifts. A 223 MB e4m3 cache with rows of
// 138 bytes takes 210 us so (a 265 MB one 221 us, 1150 us by elements); rows of
// 136 bytes take 163 us, of 128 bytes 57.
template <int ROWS>
__device__ __forceinline__ void copy_place(uint32_t dst, const uint8_t* row, int off, int bytes, int grain,
                                           bool live) {
    if constexpr (ROWS == ROWS_16 || ROWS == ROWS_FULL) {
        const int n = live && (ROWS == ROWS_FULL || off < bytes) ? 16 : 0;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(row + off), "r"(n) : "memory");
        return;
    }
    if constexpr (ROWS == ROWS_BYTES) {
        const int into = (int)(reinterpret_cast<uintptr_t>(row) & 3);
        const uint8_t* first = row - into;               // of the pool: the pool's own start is on a word
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int n = live ? max(0, min(4, into + bytes - off - 4 * w)) : 0;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + 4 * w),
                         "l"(first + (n ? off + 4 * w : 0)), "r"(n) : "memory");
        }
        return;
    }
    if (grain >= 8) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const int n = live && off + 8 * w < bytes ? 8 : 0;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst + 8 * w),
                         "l"(row + (n ? off + 8 * w : 0)), "r"(n) : "memory");
        }
    } else {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int n = live && off + 4 * w < bytes ? 4 : 0;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + 4 * w),
                         "l"(row + (n ? off + 4 * w : 0)), "r"(n) : "memory");
        }
    }
}

// The same by elements, for rows that cp.async cannot take.
template <int SIZE>
__device__ __forceinline__ void copy_elements(uint32_t dst, const uint8_t* row, int off, int bytes, bool live) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
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

template <int W>
__device__ __forceinline__ void read_piece(uint32_t (&r)[W], uint32_t src) {
    if constexpr (W == 4)
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(src) : "memory");
    else
        asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(src) : "memory");
}

// A piece that starts `bits` into its first word; the word after the piece is
// at `next`, or zero if negative.
template <int W>
__device__ __forceinline__ void read_piece(uint32_t (&r)[W], uint32_t src, int next, uint32_t bits) {
    uint32_t last;
    read_piece(r, src);
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(last) : "r"(next < 0 ? src : (uint32_t)next) : "memory");
    if (next < 0) last = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) r[w] = __funnelshift_r(r[w], w + 1 < W ? r[w + 1] : last, bits);
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
    // tiles of a warp: 8 KB of K and 8 KB of V where rows are 256 bytes or
    // more, 4 KB below (measured against twice and half as much)
    static constexpr int MT = row_bytes >= 512 ? 1 : (row_bytes == 256 ? 2 : 256 / row_bytes);
    static constexpr int TOK = 16 * MT;
    static constexpr int KD = 16 / size < DP / 4 ? 16 / size : DP / 4;      // channels of a lane's K piece
    static constexpr int VD = 16 / size < DP / 8 ? 16 / size : DP / 8;      // and of its V piece
    static constexpr int KP = DP / 4 / KD, VP = DP / 8 / VD;                // pieces of a row per lane
    static constexpr int KW = KD * size / 4, VW = VD * size / 4;            // words of a piece
    static_assert(KW == 4 && (VW == 4 || VW == 2), "pieces of 16 bytes, or halves");
    // A tile in shared memory: rows of row_bytes, their 16-byte places permuted
    // within every 128 bytes so that the 8 lanes of a quarter warp read from
    // different banks, for K (rows g, g + 1 side by side) as for V (4 tokens).
    static constexpr int places = row_bytes / 16;                           // of a row
    static constexpr int copies = TOK * places / 32;                        // of a lane for a tile
    static __device__ __forceinline__ int at(int row, int place) {
        if (row_bytes == 64) {               // two rows in 128 bytes
            const int p = ((row & 1) * 4 + place) ^ (((row >> 1) & 3) << 1);
            return (row >> 1) * 128 + p * 16;
        }
        return row * row_bytes + ((place ^ (((row >> 1) & 3) << 1) ^ ((row & 1) << 2)) * 16);
    }
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
        row_bytes > 512 ? 1 : (row_bytes >= 256 || NT == 2 || SPLITQ || DP == 256 ? 2 : 3);
    static constexpr int JC = DP > 64 ? 2 : 1;                              // 16-channel tiles joined at a time
    static constexpr bool chains = !Kind<KIND>::f32 && !SPLITQ;             // sums in long chains
    static constexpr int chain = kChainTokens / TOK;                        // and their steps
};

template <int KIND, int DP, int NT, int ROWS, bool SPLITQ>
__global__ void __launch_bounds__(32 * kDecodeWarps, DecodeShape<KIND, DP, NT, ROWS, SPLITQ>::blocks)
    decode_kernel(const __grid_constant__ DecodeArgs a) {
    using S = DecodeShape<KIND, DP, NT, ROWS, SPLITQ>;
    using K = Kind<KIND>;
    constexpr int MT = S::MT, TOK = S::TOK;
    extern __shared__ __align__(16) uint8_t decode_ring[];
    __shared__ float sm_m[kDecodeWarps][8 * NT], sm_l[kDecodeWarps][8 * NT];
    __shared__ float2 sm_t[8 * NT];
    __shared__ float2 sm_o[kDecodeWarps][8 * NT][8 * S::JC + 1];      // channels in pairs
    // scales of the key and value rows of a tile and the next
    __shared__ float sm_s[2][kDecodeWarps][2][K::code ? TOK : 1];
    __shared__ int sm_into[2][kDecodeWarps][ROWS == ROWS_BYTES ? TOK : 1];       // bytes from a word to a row's start
    __shared__ long long sm_sum[kDecodeWarps];
    __shared__ int sm_at[3];

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, c = lane & 3;
    constexpr int STEP = kDecodeWarps * TOK;
    const int bytes = ROWS == ROWS_FULL ? S::row_bytes : a.d * S::size;
    const int64_t pool_rows = (int64_t)a.c.pages * a.hk * a.c.page;      // rows of one model's pool
    const int lowest = (bytes | (int)reinterpret_cast<uintptr_t>(a.c.k) | (int)reinterpret_cast<uintptr_t>(a.c.v)) & 7;
    const int grain = lowest == 0 ? 8 : (lowest == 4 ? 4 : 1);           // alignment of every row
    // ROWS_ANY, ROWS_BYTES: the places that rows reach into; 65536 / live_places, rounded up
    const int live_places = (bytes + (ROWS == ROWS_BYTES ? (bytes % 2 ? 3 : 2) : 0) + 15) / 16;
    const int per_place = (65535 + live_places) / live_places;
    const int sequences = a.n * a.b, per_seq = a.hk * a.tiles;           // per_seq: segments of a sequence
    if (!a.in_turn) sm100::grid_dep_launch_dependents();                 // the join waits for this grid's end by itself

    // --- where this block's steps begin
    struct Walk {
        int nb, hp, pos, start, len, left;       // segment (nb, hp), token of the step, its range; steps still to do
        const int* table;                        // of the sequence
    };
    Walk front;
    if (a.in_turn) {
        front.nb = blockIdx.x / per_seq;
        front.hp = blockIdx.x - front.nb * per_seq;
        front.left = front.nb < sequences ? 0x7fffffff : 0;
    } else {
        const int each = (sequences + 32 * kDecodeWarps - 1) / (32 * kDecodeWarps);
        const int s0 = min(sequences, (int)threadIdx.x * each), s1 = min(sequences, s0 + each);
        long long mine = 0;
        for (int s = s0; s < s1; ++s) mine += DecodeRange(a, s).steps(STEP);
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        if (lane == 31) sm_sum[warp] = upto;
        __syncthreads();
        long long all = 0;
#pragma unroll
        for (int w = 0; w < kDecodeWarps; ++w) {
            if (w < warp) upto += sm_sum[w];
            all += sm_sum[w];
        }
        all *= per_seq;
        const long long per = (all + a.blocks - 1) / a.blocks, begin = per * blockIdx.x;
        long long before = (upto - mine) * per_seq;
        if (begin >= before && begin < upto * per_seq) {
            for (int s = s0; s < s1; ++s) {
                const int n = DecodeRange(a, s).steps(STEP);
                if (begin < before + (long long)n * per_seq) {
                    const int off = (int)(begin - before);
                    sm_at[0] = s, sm_at[1] = off / n, sm_at[2] = off % n;
                    break;
                }
                before += (long long)n * per_seq;
            }
        }
        __syncthreads();
        front.left = (int)max(0ll, min(per, all - begin));
        front.nb = sm_at[0], front.hp = sm_at[1];
    }
    if (front.left <= 0) return;
    auto enter = [&](Walk& w) {
        const DecodeRange r(a, w.nb);
        const int i = w.nb / a.b;
        w.start = w.pos = r.start;
        w.len = r.len;
        w.table = a.c.table + i * a.c.table_n + (w.nb - i * a.b) * a.c.table_b;
    };
    enter(front);
    if (!a.in_turn) front.pos += sm_at[2] * STEP;
    Walk at = front;                             // the step whose products are next; `front` the one to look up
    auto next_segment = [&](Walk& w) {
        w.hp += a.in_turn ? a.blocks : 1;
        if (w.hp >= per_seq) {
            w.nb += w.hp / per_seq;
            w.hp %= per_seq;
        }
        if (w.nb >= sequences) w.left = 0;
        if (w.left > 0) enter(w);
    };

    // --- token slots: lane holds those of tokens (lane + 32 r) of a tile.
    // look_up only asks for the pages; `resolve`, an iteration later, waits for them.
    struct Slots {
        int row[S::NR];                      // the page, then the row; -1 past the end, -2 where the pool has no such page
        int off[S::NR];                      // of the token in a page's rows of all heads, -1 past the end
        int model;
        bool run;                            // all there and one after the other
    };
    auto look_up = [&](Slots& x) {               // the step at `front`, which moves on
        const int kh = front.hp / a.tiles;
        x.model = front.left > 0 ? front.nb / a.b : 0;
#pragma unroll
        for (int r = 0; r < S::NR; ++r) {
            const int p = front.pos + warp * TOK + (TOK < 32 ? lane & (TOK - 1) : lane + 32 * r);
            x.row[r] = x.off[r] = -1;
            if (front.left > 0 && p < front.len) {       // the length never passes the table's columns
                uint32_t off;
                const uint32_t col = a.c.page_div.divmod((uint32_t)p, off);
                x.row[r] = __ldg(front.table + col);
                x.off[r] = kh * a.c.page + (int)off;
            }
        }
        if (front.left > 0) {
            --front.left;
            front.pos += STEP;
            if (front.pos >= front.len) next_segment(front);
        }
    };
    auto resolve = [&](Slots& x) {
#pragma unroll
        for (int r = 0; r < S::NR; ++r) {
            const bool there = (uint32_t)x.row[r] < (uint32_t)a.c.pages;
            x.row[r] = x.off[r] < 0 ? -1 : (there ? x.row[r] * (a.hk * a.c.page) + x.off[r] : -2);
        }
    };
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(decode_ring) + warp * (S::unit / kDecodeWarps);
    // One unit: the rows of a tile, whole rows side by side in each instruction
    // (every memory request is a full line); from one address on where the
    // slots follow one another, as they do inside a page.
    auto copy_rows = [&](int place, const void* pages, const Slots& x) {
        const uint8_t* base = static_cast<const uint8_t*>(pages) + x.model * pool_rows * bytes;
        const uint32_t dst = mine + place * S::unit;
        if constexpr (ROWS < ROWS_16) {
            auto one = [&](int n, auto copy) {
                const int row = n * per_place >> 16, p = n - row * live_places;
                int r = __shfl_sync(0xffffffffu, x.row[0], row & 31);
                if constexpr (S::NR > 1) {
                    const int r1 = __shfl_sync(0xffffffffu, x.row[1], row & 31);
                    if (row >= 32) r = r1;
                }
                if (row < TOK) copy(dst + S::at(row, p), base + (int64_t)max(r, 0) * bytes, p * 16, r >= 0);
            };
            // loops, as their unrolled code was more than the instruction cache holds
            if (ROWS == ROWS_ANY && S::size < 4 && grain < 4) {
#pragma unroll 1
                for (int n = lane; n < TOK * live_places + lane; n += 32)
                    one(n, [&](uint32_t to, const uint8_t* row, int off, bool live) {
                        if constexpr (S::size < 4) copy_elements<S::size>(to, row, off, bytes, live);
                    });
            } else {
#pragma unroll 4
                for (int n = lane; n < TOK * live_places + lane; n += 32)
                    one(n, [&](uint32_t to, const uint8_t* row, int off, bool live) {
                        copy_place<ROWS>(to, row, off, bytes, grain, live);
                    });
            }
        } else if (x.run) {
            const uint8_t* from = base + (int64_t)__shfl_sync(0xffffffffu, x.row[0], 0) * bytes;
#pragma unroll
            for (int j = 0; j < S::copies; ++j) {
                const int n = j * 32 + lane, row = n / S::places, p = n % S::places;
                copy_place<ROWS>(dst + S::at(row, p), from + row * bytes, p * 16, bytes, grain, true);
            }
        } else {
#pragma unroll
            for (int j = 0; j < S::copies; ++j) {
                const int n = j * 32 + lane, row = n / S::places, p = n % S::places;
                // the register that holds the row's slot is known at compile time, its lane is not
                const int r = __shfl_sync(0xffffffffu, x.row[S::NR == 1 ? 0 : (j * 32 / S::places) >> 5], row & 31);
                copy_place<ROWS>(dst + S::at(row, p), base + (int64_t)max(r, 0) * bytes, p * 16, bytes, grain,
                                          r >= 0);
            }
        }
    };
    // K of a tile with its scales, and a bit for each token that is there
    auto copy_k = [&](int place, int turn, Slots& x, uint32_t (&seen)[S::NR]) {
        resolve(x);
        const int64_t pool = x.model * pool_rows;
        const int first = __shfl_sync(0xffffffffu, x.row[0], 0);
        bool run = first >= 0;
#pragma unroll
        for (int r = 0; r < S::NR; ++r) {
            const int t = TOK < 32 ? lane & (TOK - 1) : lane + 32 * r;
            seen[r] = __ballot_sync(0xffffffffu, x.row[r] >= 0);
            run = run && x.row[r] == first + t;
            if (x.row[r] == -2) raise_device_error(a.err, DEV_ERR_INDEX);
            if constexpr (ROWS == ROWS_BYTES)
                sm_into[turn][warp][t] = (int)(((uint32_t)pool + (uint32_t)max(x.row[r], 0)) * (uint32_t)bytes & 3);
            if constexpr (K::code) {
                const int64_t at = pool + (x.row[r] < 0 ? 0 : x.row[r]);
                const int n = x.row[r] >= 0 ? 4 : 0;
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                                 (uint32_t)__cvta_generic_to_shared(&sm_s[turn][warp][0][t])),
                             "l"(a.c.ks + at), "r"(n) : "memory");
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                                 (uint32_t)__cvta_generic_to_shared(&sm_s[turn][warp][1][t])),
                             "l"(a.c.vs + at), "r"(n) : "memory");
            }
        }
        x.run = __all_sync(0xffffffffu, run);
        copy_rows(place, a.c.k, x);
    };
    auto copy_v = [&](int place, const Slots& x) { copy_rows(place, a.c.v, x); };

    if constexpr (ROWS < ROWS_16) {          // zeros in the places that no row reaches
#pragma unroll 1
        for (int u = 0; u < S::units; ++u)
#pragma unroll 1
            for (int o = 16 * lane; o < S::unit / kDecodeWarps; o += 512)
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(mine + u * S::unit + o), "r"(0) : "memory");
        __syncwarp();
    }

    Slots x1, x2;                            // slots of the next step and of the one after it
    uint32_t seen[2][S::NR];                 // tokens that are there, of the current step and the next
    {
        Slots x0;
        look_up(x0);
        look_up(x1);
        if constexpr (S::units == 3) look_up(x2);
        copy_k(0, 0, x0, seen[0]);
        copy_commit();
        copy_v(1, x0);
        copy_commit();
        if constexpr (S::units == 3) {
            copy_k(2, 1, x1, seen[1]);
            copy_commit();
        }
    }

    // --- query fragments of a segment: lane (g, c) holds head g's channels of its K pieces
    uint32_t q[NT][S::QR], ql[SPLITQ ? NT : 1][SPLITQ ? S::QR : 1];
    float zs[NT][2];                                     // what a score is multiplied by, heads 2c and 2c + 1
    auto load_queries = [&]() {
        const int i = at.nb / a.b, kh = at.hp / a.tiles, h0 = (at.hp - kh * a.tiles) * 8 * NT;
        const int heads = min(8 * NT, a.group - h0);
        const int64_t base = i * a.q_n + (at.nb - i * a.b) * a.q_b + (int64_t)(kh * a.group + h0) * a.q_h;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int h = t * 8 + g;
            const int64_t at = base + (h < heads ? h : 0) * a.q_h;
            float x[S::KP][S::KD];
            float top = 0.f;
#pragma unroll
            for (int p = 0; p < S::KP; ++p) {
                const int ch = (p * 4 + c) * S::KD;
#pragma unroll
                for (int e = 0; e < S::KD; ++e) x[p][e] = 0.f;
                if (ROWS >= ROWS_16 && a.q_vec) {
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
    };

    float acc[NT][DP / 16][4];
    float m[NT][2], l[NT][2];

    // acc += the totals of the segment's chains before (none if `first`), which
    // are relative to the maximum they had; `keep`: as the new totals.
    auto add_done = [&](bool first, bool keep) {
        constexpr int threads = 32 * kDecodeWarps;
        float* held = a.done + (int64_t)blockIdx.x * (NT * (DP / 4 + 2) * threads) + threadIdx.x;
#pragma unroll
        for (int t = 0; t < NT; ++t, held += (DP / 4 + 2) * threads) {
            float f[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                f[e] = first ? 0.f : ex2(held[(DP / 4 + e) * threads] - (m[t][e] == -INFINITY ? 0.f : m[t][e]));
                if (keep) held[(DP / 4 + e) * threads] = m[t][e];
            }
#pragma unroll
            for (int j = 0; j < DP / 16; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float* at = held + (4 * j + e) * threads;
                    const float x = first ? acc[t][j][e] : fmaf(*at, f[e & 1], acc[t][j][e]);
                    if (keep) *at = x;
                    acc[t][j][e] = keep ? 0.f : x;
                }
        }
    };

    // ROWS_BYTES: bytes into a word at which the lane's rows of K and V start, 2 bits each
    uint32_t k_into = 0, v_into = 0;

    // S^T += K q^T over the pieces in registers
    float s[NT][MT][4];
    auto scores = [&](int place) {
        const uint32_t from = mine + place * S::unit;
        uint32_t batch[MT][S::KB][2][S::KW];
#pragma unroll
        for (int p0 = 0; p0 < S::KP; p0 += S::KB) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int p = 0; p < S::KB; ++p)
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const int row = 16 * mt + 8 * hf + g, at = (p0 + p) * 4 + c;
                        if constexpr (ROWS == ROWS_BYTES)
                            read_piece(batch[mt][p][hf], from + S::at(row, at),
                                       at + 1 < S::places ? (int)(from + S::at(row, at + 1)) : -1,
                                       8 * (k_into >> 2 * (2 * mt + hf) & 3));
                        else read_piece(batch[mt][p][hf], from + S::at(row, at));
                    }
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
                        for (int t = 0; t < NT; ++t) {
                            float part[4] = {0.f, 0.f, 0.f, 0.f};
                            float(&o)[4] = SPLITQ ? part : s[t][mt];
#pragma unroll
                            for (int e = 0; e < S::KR; e += 2) {
                                const int j = p * S::KR + e;
                                if constexpr (SPLITQ)
                                    mma<KIND>(o, r0[e], r1[e], r0[e + 1], r1[e + 1], ql[t][j], ql[t][j + 1]);
                                mma<KIND>(o, r0[e], r1[e], r0[e + 1], r1[e + 1], q[t][j], q[t][j + 1]);
                            }
#pragma unroll
                            for (int e = 0; e < (SPLITQ ? 4 : 0); ++e) s[t][mt][e] += part[e];
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
                top = top > m[t][e] + K::slack ? top : m[t][e];
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
    // Weights as B operands: hi and lo pieces of tokens (k) by heads (n), and
    // a third where the result is fp32
    uint32_t ph[NT][MT][K::f32 ? 4 : 2], pl[NT][MT][K::f32 ? 4 : 2], pr[SPLITQ ? NT : 1][SPLITQ ? MT : 1][2];
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
                        if constexpr (SPLITQ) pr[t][mt][hf] = transpose8x8(pack2<K::values>(rx, ry, rx, ry));
                    }
                }
            }
    };
    // O^T += V^T P^T over the pieces in registers
    auto values = [&](int place) {
        const uint32_t from = mine + place * S::unit;
        uint32_t batch[MT][S::VB][4][S::VW];
#pragma unroll
        for (int p0 = 0; p0 < S::VP; p0 += S::VB) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int p = 0; p < S::VB; ++p)
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        // the k index of lane c: tokens 2c, 2c + 1, 2c + 8, 2c + 9; tf32 c, c + 4, c + 8, c + 12
                        const int row = 16 * mt + (K::f32 ? c + 4 * t : 2 * c + (t & 1) + 8 * (t >> 1));
                        // the 16-byte place, and the half in it
                        const int at = S::VW == 4 ? (p0 + p) * 8 + g : (p0 + p) * 4 + g / 2;
                        const int half = S::VW == 4 ? 0 : g % 2 * 8;
                        const uint32_t src = from + S::at(row, at) + half;
                        if constexpr (ROWS == ROWS_BYTES)
                            read_piece(batch[mt][p][t], src,
                                       S::VW == 2 && half == 0 ? (int)(src + 8)
                                       : at + 1 < S::places    ? (int)(from + S::at(row, at + 1))
                                                               : -1,
                                       8 * (v_into >> 2 * (4 * mt + t) & 3));
                        else read_piece(batch[mt][p][t], src);
                    }
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
                                float part[4] = {0.f, 0.f, 0.f, 0.f};
                                float(&o)[4] = SPLITQ ? part : acc[t][p * S::VD / 2 + w];
                                if constexpr (SPLITQ)
                                    mma<K::values>(o, av[w][0], av[w][1], av[w][2], av[w][3], pr[t][mt][0],
                                                   pr[t][mt][1]);
                                mma<K::values>(o, av[w][0], av[w][1], av[w][2], av[w][3], pl[t][mt][0], pl[t][mt][1]);
                                mma<K::values>(o, av[w][0], av[w][1], av[w][2], av[w][3], ph[t][mt][0], ph[t][mt][1]);
#pragma unroll
                                for (int e = 0; e < (SPLITQ ? 4 : 0); ++e) acc[t][p * S::VD / 2 + w][e] += part[e];
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

    // --- the end of a segment (or of this block's part of it): join the warps
    auto finish = [&](bool whole, int part) {
        const int kh = at.hp / a.tiles, h0 = (at.hp - kh * a.tiles) * 8 * NT;
        const int heads = min(8 * NT, a.group - h0);
        const int64_t row0 = (int64_t)at.nb * a.hq + kh * a.group + h0;
        const int64_t part0 = ((int64_t)blockIdx.x * 2 + part) * 8 * NT;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], o);
                if (g == 0) {
                    sm_m[warp][t * 8 + 2 * c + e] = m[t][e];
                    sm_l[warp][t * 8 + 2 * c + e] = l[t][e];
                }
            }
        __syncthreads();
        float f[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < kDecodeWarps; ++w) top = fmaxf(top, sm_m[w][t * 8 + 2 * c + e]);
                f[t][e] = ex2(m[t][e] - (top == -INFINITY ? 0.f : top) - K::lift);
            }
        if (threadIdx.x < heads) {
            float top = -INFINITY, total = 0.f;
#pragma unroll
            for (int w = 0; w < kDecodeWarps; ++w) top = fmaxf(top, sm_m[w][threadIdx.x]);
#pragma unroll
            for (int w = 0; w < kDecodeWarps; ++w)
                total += ex2(sm_m[w][threadIdx.x] - (top == -INFINITY ? 0.f : top)) * sm_l[w][threadIdx.x];
            sm_t[threadIdx.x] = make_float2(top, total);
            if (!whole) a.part_ml[part0 + threadIdx.x] = make_float2(top, total);
        }
#pragma unroll
        for (int j0 = 0; j0 < DP / 16; j0 += S::JC) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int jj = 0; jj < S::JC; ++jj)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        sm_o[warp][t * 8 + 2 * c + e][jj * 8 + g] =
                            make_float2(acc[t][j0 + jj][e] * f[t][e], acc[t][j0 + jj][e + 2] * f[t][e]);
            __syncthreads();
            for (int e = threadIdx.x; e < heads * 16 * S::JC; e += 32 * kDecodeWarps) {
                const int h = e / (16 * S::JC), x = e % (16 * S::JC), j = j0 + x / 16;
                const int ch = j / (S::VD / 2) * 8 * S::VD + x % 16 / 2 * S::VD + j % (S::VD / 2) * 2 + (x & 1);
                if (ROWS != ROWS_FULL && ch >= a.d) continue;
                float o = 0.f;
#pragma unroll
                for (int w = 0; w < kDecodeWarps; ++w) o += reinterpret_cast<const float*>(sm_o[w][h])[x];
                const float total = sm_t[h].y;
                if (whole) store_out(a.out, (row0 + h) * a.d + ch, total == 0.f ? 0.f : o / total, a.dtype);
                else a.part_o[(part0 + h) * a.d + ch] = o;
            }
            __syncthreads();
        }
    };

    int place = 0, turn = 0, part = 0;
    while (at.left > 0) {
        load_queries();
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int j = 0; j < DP / 16; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[t][j][e] = 0.f;
            m[t][0] = m[t][1] = -INFINITY;
            l[t][0] = l[t][1] = 0.f;
        }
        const int entered = at.pos;
        bool first = true;
        int stop = at.pos + S::chain * STEP;     // of the present chain of sums
        do {
                copy_wait<S::units - 1>();
                __syncwarp();                        // what the other lanes copied
                float kt[MT][2], vt[MT][2];
                if constexpr (K::code) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) {
                            kt[mt][hf] = sm_s[turn][warp][0][16 * mt + 8 * hf + g];
                            vt[mt][hf] = sm_s[turn][warp][1][16 * mt + 8 * hf + g];
                        }
                }
                if constexpr (ROWS == ROWS_BYTES) {
                    k_into = v_into = 0;
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf)
                            k_into |= (uint32_t)sm_into[turn][warp][16 * mt + 8 * hf + g] << 2 * (2 * mt + hf);
#pragma unroll
                        for (int t = 0; t < 4; ++t)
                            v_into |= (uint32_t)sm_into[turn][warp][16 * mt + 2 * c + (t & 1) + 8 * (t >> 1)]
                                      << 2 * (4 * mt + t);
                    }
                }
                uint32_t now[S::NR], any = 0;
#pragma unroll
                for (int r = 0; r < S::NR; ++r) now[r] = seen[0][r], any |= now[r], seen[0][r] = seen[1][r];
                const int second = S::units == 3 && place == 2 ? 0 : place + 1;
                if (any) {
                    clear_scores();
                    scores(place);
                }
                __syncwarp();                        // all lanes have read the unit
                if constexpr (S::units == 3) copy_v(place, x1);
                else copy_k(place, 0, x1, seen[0]);
                copy_commit();
                if (any) {
                    softmax(now, kt, vt);
                    turn_weights();
                }
                copy_wait<S::units - 1>();
                __syncwarp();
                if (any) values(second);
                __syncwarp();
                if constexpr (S::units == 3) {
                    copy_k(second, turn, x2, seen[1]);
                    copy_commit();
                    x1 = x2;
                    look_up(x2);
                    turn ^= 1;
                    place = place == 0 ? 2 : place - 1;          // (place + 2) % 3
                } else {
                    copy_v(second, x1);
                    copy_commit();
                    look_up(x1);
                }
                --at.left;
                at.pos += STEP;
            if constexpr (S::chains)
                if (at.pos >= stop && at.pos < at.len && at.left > 0) {
                    add_done(first, true);
                    first = false;
                    stop += S::chain * STEP;
                }
        } while (at.pos < at.len && at.left > 0);
        if (S::chains && !first) add_done(false, false);
        finish(entered == at.start && at.pos >= at.len, part);
        part = 1;
        if (at.left > 0) next_segment(at);
    }
    copy_wait<0>();
}

template <int KIND, int DP, int NT, int ROWS, bool SPLITQ>
int launch_decode_shape(const DecodeArgs& a, cudaStream_t st) {
    using S = DecodeShape<KIND, DP, NT, ROWS, SPLITQ>;
    auto kernel = decode_kernel<KIND, DP, NT, ROWS, SPLITQ>;
    static std::atomic<uint64_t> allowed{0};      // devices whose limit is raised
    const uint64_t bit = 1ull << (current_device() & 63);
    if (!(allowed.load(std::memory_order_relaxed) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::ring);
        if (e != cudaSuccess)
            return set_error(WIDEK_ERR_CUDA, "widek_decode_attention_fwd: shared memory of %d bytes: %s", S::ring,
                             cudaGetErrorString(e));
        allowed.fetch_or(bit, std::memory_order_relaxed);
    }
    kernel<<<(unsigned)a.blocks, 32 * kDecodeWarps, S::ring, st>>>(a);
    return check_launch("widek_decode_attention_fwd");
}

// Query-head tiles of 8 in one block: two of them where a group has more
// than 8 heads, so that its cache is read once for 16; at d > 128, or with the
// split operands of fp32, their sums would not fit in registers beside the tile.
inline int decode_nt(int group, int d, int fmt) { return group > 8 && d <= 128 && fmt != WIDEK_F32 ? 2 : 1; }

// Tokens of a step.
inline int decode_step(int d, int fmt) {
    const int bytes = (d <= 64 ? 64 : (d <= 128 ? 128 : 256)) * (int)cache_fmt_size(fmt);
    return kDecodeWarps * 16 * (bytes >= 512 ? 1 : (bytes == 256 ? 2 : 256 / bytes));
}

// Blocks of an SM, as DecodeShape has them (for fp32 queries over codes the
// entry takes 2).
inline int decode_places(int d, int fmt, int nt) {
    const int bytes = (d <= 64 ? 64 : (d <= 128 ? 128 : 256)) * (int)cache_fmt_size(fmt);
    return bytes > 512 ? 1 : (bytes >= 256 || nt == 2 || d > 128 ? 2 : 3);
}

template <int KIND, bool SPLITQ>
int launch_decode(const DecodeArgs& a, cudaStream_t st) {
    const int bytes = a.d * Kind<KIND>::size;
    const bool aligned = bytes % 16 == 0 && aligned16(a.c.k) && aligned16(a.c.v);
    // rows that start inside a word, with room for the bytes before them
    const int most = (a.d <= 64 ? 64 : (a.d <= 128 ? 128 : 256)) * Kind<KIND>::size - (bytes % 2 ? 3 : 2);
    const bool inside = bytes % 4 != 0 && bytes <= most &&
                        ((reinterpret_cast<uintptr_t>(a.c.k) | reinterpret_cast<uintptr_t>(a.c.v)) & 3) == 0;
#define WIDEK_DECODE(DP, NT)                                                                 \
    {                                                                                        \
        if constexpr (KIND != DK_F32)                                                        \
            if (inside) return launch_decode_shape<KIND, DP, NT, ROWS_BYTES, SPLITQ>(a, st); \
        return !aligned    ? launch_decode_shape<KIND, DP, NT, ROWS_ANY, SPLITQ>(a, st)      \
               : a.d == DP ? launch_decode_shape<KIND, DP, NT, ROWS_FULL, SPLITQ>(a, st)     \
                           : launch_decode_shape<KIND, DP, NT, ROWS_16, SPLITQ>(a, st);      \
    }
    if constexpr (KIND != DK_F32) {
        if (a.nt == 2 && a.d <= 64) WIDEK_DECODE(64, 2)
        if (a.nt == 2) WIDEK_DECODE(128, 2)
    }
    if (a.d <= 64) WIDEK_DECODE(64, 1)
    if (a.d <= 128) WIDEK_DECODE(128, 1)
    WIDEK_DECODE(256, 1)
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
