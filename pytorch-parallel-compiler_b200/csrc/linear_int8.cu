// Linear layers of n models on 8-bit codes, on the tensor cores (tcgen05 kind::i8):
//
//   y[i, m, o] = act((sum_k a[i, m, k] w[i, o, k]) sa[i, m] sw[i, o] + bias[i, o])
//
// The sum is exact in int32 (K <= 131071 keeps it below 2^31); the scales, the
// bias and the activation are fp32, rounded once to y's type.
//
// Two kernels. Both stream 128-code (one swizzle row) blocks of K by TMA into a
// ring, one thread issuing the MMAs into TMEM:
//   wide    many rows: a cluster of two CTAs holds a 256 x 256 tile (cta_group::2),
//           each SM half of both operands; persistent, the epilogue of one tile
//           under the products of the next. A single CTA's 128 x 256 tile would
//           move 96 KB through shared memory in the 512 clocks that its products
//           of one K block take, over the 128 bytes a clock that it has; half of
//           both operands is 64 KB. Bound by the tensor cores from K = 2048 on, under
//           the power cap (8 x 4096 rows of 4096 -> 4096: 377 us, 2919 TOP/s; 75 % of
//           the tensor cycles of an SM's time in ncu), by the results' bytes at K = 256
//           (77.6 us for 268 MB, a fill takes 70), between them by both; by the
//           epilogue's instructions where a GELU meets a short K (1024 -> 4096: 126 us
//           without, 150 with).
//   narrow  few rows: bound by the weights' bytes. The weights' rows are the MMA's
//           128 lanes and up to 128 tokens its columns, so that no tensor time goes
//           to rows that are not there; K is split over a cluster when there are
//           too few tiles for the device, and the parts (integers: any order gives
//           the same sum) are added through distributed shared memory. 8 models of
//           4096 -> 16384 for one token: 92 us, 5.9 TB/s; small ones are latency (33 MB
//           of weights 11.6 to 13.5 us, the least 5.4).
#include <algorithm>
#include <atomic>

#include "residual_norm.cuh"

namespace widek {
namespace {

using namespace sm100;

constexpr int kBK = 128;              // codes of K in a block: one 128-byte swizzle row
constexpr int64_t kMaxK = 131071;     // 128 * 128 * K < 2^31

// Instruction descriptor, kind::i8: int32 accumulators, signed operands, K-major.
constexpr uint32_t idesc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(smem_addr(src)), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}
// Arrives on another CTA's mbarrier without waiting for this thread's stores.
__device__ __forceinline__ void mbar_arrive_remote_relaxed(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ uint32_t load_cluster_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}


// max(x, 0), NaN kept.
__device__ __forceinline__ float relu_nan(float x) {
    float y;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(x));
    return y;
}

// Two fp32 values in a register pair, and arithmetic on both at once.
using F2 = uint64_t;
__device__ __forceinline__ F2 pair_of(float a, float b) {
    F2 p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ void halves(F2 p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) {
    F2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ F2 mul(F2 a, F2 b) {
    F2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// GELU of two values for a 16-bit result: max(x, 0) - a Q(a) with a = |x| and the
// normal tail Q(a) = 2^(-a^2 log2(e) / 2 + r(a)), r a polynomial (fit_gelu_tail.py:
// Q is off by 9e-6 of itself up to a = 8, where f16's half step is 2.4e-4; past 8,
// where a Q(a) < 5e-15, r and the factor a stay at 8). It takes 9 instructions a
// value; by way of erff the epilogue of a tile takes longer than its products. The
// constants are set up once, in registers.
struct Gelu2 {
    F2 r[9], half;
    __device__ __forceinline__ Gelu2() {
        constexpr float c[9] = {-0.9999924f, -1.1513219f, 0.26315188f, -0.05433736f, 0.008762172f, -0.0010219777f,
                                7.9574354e-05f, -3.6553492e-06f, 7.428467e-08f};
#pragma unroll
        for (int i = 0; i < 9; ++i) {             // r in powers of -a
            const float v = i % 2 ? -c[i] : c[i];
            asm volatile("mov.b64 %0, {%1, %1};" : "=l"(r[i]) : "f"(v));
        }
        asm volatile("mov.b64 %0, {%1, %1};" : "=l"(half) : "f"(-0.72134752f));
    }
    __device__ __forceinline__ F2 operator()(F2 x) const {
        float x0, x1, e0, e1;
        halves(x, x0, x1);
        const F2 b = pair_of(fmaxf(-fabsf(x0), -8.f), fmaxf(-fabsf(x1), -8.f));
        F2 p = r[8];
#pragma unroll
        for (int i = 7; i >= 0; --i) p = fma(p, b, r[i]);
        p = fma(mul(x, half), x, p);
        halves(p, e0, e1);
        asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e0));
        asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e1));
        return fma(b, pair_of(e0, e1), pair_of(relu_nan(x0), relu_nan(x1)));
    }
};

// The activation of N values (an even number), NaN kept.
template <typename T, int N>
__device__ __forceinline__ void activate(F2 (&v)[N / 2], int act, const Gelu2& gelu) {
    if (act == WIDEK_ACT_NONE) return;
    if (sizeof(T) == 2 && act == WIDEK_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < N / 2; ++j) v[j] = gelu(v[j]);
        return;
    }
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
        float a, b;
        halves(v[j], a, b);
        v[j] = act == WIDEK_ACT_RELU ? pair_of(relu_nan(a), relu_nan(b)) : pair_of(gelu_erf(a), gelu_erf(b));
    }
}

// N values as stored (N * sizeof(T) = 16 bytes).
template <typename T>
__device__ __forceinline__ uint4 store_form(const F2* v) {
    float f[16 / sizeof(T)];
#pragma unroll
    for (int j = 0; j < (int)(8 / sizeof(T)); ++j) halves(v[j], f[2 * j], f[2 * j + 1]);
    const rnorm::Pack<T, 16 / sizeof(T)> p = rnorm::pack<T, 16 / sizeof(T)>(f);
    return *reinterpret_cast<const uint4*>(&p);
}

// Two sums with their scales and biases.
__device__ __forceinline__ F2 finish(uint32_t acc0, uint32_t acc1, F2 sa, F2 sw, F2 bias) {
    return fma(mul(pair_of((float)(int)acc0, (float)(int)acc1), sa), sw, bias);
}

struct Int8Args {
    const float *sa, *sw;             // [n, m], [n, o]
    const void* bias;                 // [n, o] or null
    void* y;                          // [n, m, o]
    int n, m, k, o, act, vec_store;
    int* err;
};

// ---------------------------------------------------------------------------
// wide: 256 x 256 tiles by pairs of CTAs
// ---------------------------------------------------------------------------
constexpr int kGroups = 4;            // of 4 epilogue warps, each finishing a quarter of the columns
constexpr int kWideThreads = 64 + 128 * kGroups;     // and a TMA warp and an MMA warp
constexpr int kGroupCols = 256 / kGroups;

template <typename T>
struct WideSmem {
    static constexpr int STAGES = sizeof(T) == 4 ? 4 : 5;     // what 227 KB leave room for
    static constexpr uint32_t PART = 128 * kBK;                 // one CTA's half of an operand
    static constexpr uint32_t RING = STAGES * 2 * PART;
    static constexpr uint32_t OUT_CHUNK = 128 * 32 * sizeof(T);
    static constexpr uint32_t OUT_BYTES = kGroups * OUT_CHUNK;
    static constexpr uint32_t VEC_BYTES = 256 * 8;              // (scale, bias) of the columns
    static constexpr uint32_t TOTAL = 1024 + RING + OUT_BYTES + VEC_BYTES + 8 * (2 * STAGES + 5) + 16;
    static_assert(TOTAL <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ void group_sync(int wg) { asm volatile("bar.sync %0, 128;" ::"r"(1 + wg) : "memory"); }

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kWideThreads, 1)
    wide_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w,
                const __grid_constant__ CUtensorMap tm_y, const Int8Args p) {
    using S = WideSmem<T>;
    constexpr int STAGES = S::STAGES;
    constexpr uint32_t IDESC = idesc_i8(256, 256);
    constexpr uint32_t TMEM_COLS = 512;      // two accumulators of 256 columns

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sA = smem;
    uint8_t* sB = smem + STAGES * S::PART;
    uint8_t* sOut = smem + S::RING;
    float* sVec = reinterpret_cast<float*>(sOut + S::OUT_BYTES);
    uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(sVec) + S::VEC_BYTES);
    uint64_t* empty = full + STAGES;
    uint64_t* tfull = empty + STAGES;
    uint64_t* tempty = tfull + 2;
    uint64_t* done = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
    const int mt_count = (p.m + 255) / 256, nt_count = (p.o + 255) / 256, kb_count = (p.k + kBK - 1) / kBK;
    const int tiles = p.n * mt_count * nt_count;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tfull[a], 1);
            mbar_init(&tempty[a], 2 * 4 * kGroups);   // both CTAs' epilogue warps
        }
        mbar_init(done, 1);
        *abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&tm_a);
        tma_prefetch_desc(&tm_w);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, TMEM_COLS);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync_all();                      // barriers of both CTAs initialised, TMEM allocated
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        // TMA producer (both CTAs); bytes land on the leader's full barrier.
        const uint64_t pol_a = l2_policy_evict_last();
        const uint64_t pol_w = mt_count == 1 ? l2_policy_evict_first() : l2_policy_evict_normal();
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int tile = pair; tile < tiles && ok; tile += npairs) {
            const int mt = tile % mt_count, rest = tile / mt_count, nt = rest % nt_count, model = rest / nt_count;
            for (int kb = 0; kb < kb_count; ++kb) {
                if (!mbar_wait(&empty[s], ph ^ 1, abort_flag)) { ok = false; break; }
                if (lane == 0) {
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], 4 * S::PART);
                    const uint32_t leader_full = map_to_rank(smem_addr(&full[s]), 0);
                    tma_load_3d_pair(sA + s * S::PART, &tm_a, leader_full, kb * kBK, mt * 256 + (int)rank * 128, model,
                                     pol_a);
                    tma_load_3d_pair(sB + s * S::PART, &tm_w, leader_full, kb * kBK, nt * 256 + (int)rank * 128, model,
                                     pol_w);
                }
                __syncwarp();
                if (++s == STAGES) { s = 0; ph ^= 1; }
            }
        }
        if (!ok) {
            *abort_flag = 1;
            raise_device_error(p.err, DEV_ERR_GEMM_TIMEOUT);
        }
    } else if (warp == 1) {
        if (rank == 0 && lane == 0) {
            int s = 0, local = 0;
            uint32_t ph = 0;
            bool ok = true;
            const uint64_t a_desc0 = sdesc_kmajor_sw128(smem_addr(sA)), b_desc0 = sdesc_kmajor_sw128(smem_addr(sB));
            for (int tile = pair; tile < tiles && ok; tile += npairs, ++local) {
                const int acc = local & 1;
                if (!mbar_wait(&tempty[acc], ((local >> 1) & 1) ^ 1, abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + acc * 256;
                for (int kb = 0; kb < kb_count; ++kb) {
                    if (!mbar_wait(&full[s], ph, abort_flag)) { ok = false; break; }
                    tc_fence_after();
                    const uint64_t ad = a_desc0 + (uint64_t)((s * S::PART) >> 4), bd = b_desc0 + (uint64_t)((s * S::PART) >> 4);
#pragma unroll
                    for (int k = 0; k < kBK / 32; ++k) umma_i8_pair(d_tmem, ad + 2 * k, bd + 2 * k, IDESC, (kb | k) != 0);
                    umma_commit_pair_mc(&empty[s], 0x3);
                    if (++s == STAGES) { s = 0; ph ^= 1; }
                }
                if (!ok) break;
                umma_commit_pair_mc(&tfull[acc], 0x3);
            }
            if (!ok) {
                *abort_flag = 1;
                raise_device_error(p.err, DEV_ERR_GEMM_TIMEOUT);
            }
            umma_commit_pair_mc(done, 0x1);
            const volatile int never = 0;
            mbar_wait(done, 0, &never);
        }
        __syncwarp();
    } else {
        // Epilogue: group wg drains columns [64 wg, 64 wg + 64) of this CTA's 128
        // rows, 32 at a time through a staging buffer a warp; warp quarter q is
        // the TMEM lanes (rows) 32 q .. 32 q + 31. Four groups, as two left the
        // issue slots two thirds empty; a warp stores by itself (TMA). An arrival that
        // waited for the stores held a tile of K = 256 at 4.0 us, where it takes 2.8.
        const int q = warp & 3, wg = (warp - 2) >> 2, ep_tid = threadIdx.x - 64 - 128 * wg;
        uint8_t* buf = sOut + (wg * 4 + q) * (S::OUT_CHUNK / 4);
        float* vec = sVec + wg * 2 * kGroupCols;             // scales, then biases
        const Gelu2 gelu;
        const uint32_t leader_tempty0 = map_to_rank(smem_addr(&tempty[0]), 0);
        const T* bias = static_cast<const T*>(p.bias);
        // A tile's scales and biases are asked for while the last one is finished.
        float next_sa = 0.f, next_sw = 0.f, next_bias = 0.f;
        auto ask = [&](int tile) {
            const int mt = tile % mt_count, rest = tile / mt_count, nt = rest % nt_count, model = rest / nt_count;
            const int row = mt * 256 + (int)rank * 128 + q * 32 + lane, c = nt * 256 + wg * kGroupCols + ep_tid;
            next_sa = tile < tiles && row < p.m ? p.sa[(int64_t)model * p.m + row] : 0.f;
            const bool col = tile < tiles && ep_tid < kGroupCols && c < p.o;
            const int64_t at = (int64_t)model * p.o + c;
            next_sw = col ? p.sw[at] : 0.f;
            next_bias = col && bias ? to_f<T>(bias[at]) : 0.f;
        };
        ask(pair);
        int local = 0;
        for (int tile = pair; tile < tiles; tile += npairs, ++local) {
            const int mt = tile % mt_count, rest = tile / mt_count, nt = rest % nt_count, model = rest / nt_count;
            const int acc = local & 1, row0 = mt * 256 + (int)rank * 128, c0 = nt * 256 + wg * kGroupCols;
            group_sync(wg);                              // the group has read the last tile's
            if (ep_tid < kGroupCols) {
                vec[ep_tid] = next_sw;
                vec[kGroupCols + ep_tid] = next_bias;
            }
            const F2 sa = pair_of(next_sa, next_sa);
            group_sync(wg);
            ask(tile + npairs);
            if (!mbar_wait(&tfull[acc], (local >> 1) & 1, abort_flag)) {
                *abort_flag = 1;
                raise_device_error(p.err, DEV_ERR_GEMM_TIMEOUT);
                break;
            }
            tc_fence_after();
            // The accumulator is given back as soon as it is in registers; its stores are
            // not waited for.
            const int cols = min(kGroupCols, p.o - c0);
            auto release = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_remote_relaxed(leader_tempty0 + acc * 8);
            };
            if (cols <= 0) release();
#pragma unroll 1
            for (int c = 0; c < cols; c += 32) {
                uint32_t r[32];
                tmem_ld_32x32b_x32(tmem_base + (uint32_t)(acc * 256 + wg * kGroupCols + c) + ((uint32_t)(q * 32) << 16), r);
                tmem_ld_wait();
                if (c + 32 >= cols) release();
                F2 v[16];
                const ulonglong2* sw = reinterpret_cast<const ulonglong2*>(vec + c);
                const ulonglong2* sb = reinterpret_cast<const ulonglong2*>(vec + kGroupCols + c);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const ulonglong2 f = sw[j], g = sb[j];
                    v[2 * j] = finish(r[4 * j], r[4 * j + 1], sa, f.x, g.x);
                    v[2 * j + 1] = finish(r[4 * j + 2], r[4 * j + 3], sa, f.y, g.y);
                }
                activate<T, 32>(v, p.act, gelu);
                if (p.vec_store) {
                    // A warp stores its 32 rows by itself, through its staging buffer. Rows
                    // past m are clipped by the store; a warp whose rows all lie past m
                    // stores nothing.
                    if (lane == 0) bulk_wait_group_read<0>();
                    __syncwarp();
                    constexpr int PIECES = 32 * sizeof(T) / 16, PER = 16 / sizeof(T);
#pragma unroll
                    for (int j = 0; j < PIECES; ++j) {
                        const int phys = PIECES == 4 ? j ^ ((lane >> 1) & 3) : j ^ (lane & 7);
                        *reinterpret_cast<uint4*>(buf + lane * 32 * sizeof(T) + phys * 16) = store_form<T>(v + PER / 2 * j);
                    }
                    fence_async_shared();
                    __syncwarp();
                    if (lane == 0 && row0 + q * 32 < p.m) {
                        tma_store_3d(&tm_y, buf, c0 + c, row0 + q * 32, model);
                        bulk_commit_group();
                    }
                } else {
                    // Rows that start off the 16-byte borders: through this warp's part
                    // of the staging buffer (columns turned by the row: no bank twice), so that a
                    // store covers 32 neighbours (119544 rows of 404 results 88 us; each
                    // thread storing its own row 486).
                    T* stage = reinterpret_cast<T*>(buf);
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        float a, b;
                        halves(v[j / 2], a, b);
                        stage[lane * 32 + ((j + lane) & 31)] = from_f<T>(a);
                        stage[lane * 32 + ((j + 1 + lane) & 31)] = from_f<T>(b);
                    }
                    __syncwarp();
                    const int col = c0 + c + lane, rows = min(32, p.m - row0 - q * 32);
                    T* dst = static_cast<T*>(p.y) + ((int64_t)model * p.m + row0 + q * 32) * p.o + col;
                    if (col < p.o) {
#pragma unroll 8
                        for (int j = 0; j < rows; ++j, dst += p.o) *dst = stage[j * 32 + ((lane + j) & 31)];
                    }
                }
            }
        }
        if (lane == 0) bulk_wait_group_all();
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 0 && *abort_flag) {
        // A role failed. This CTA's copies count on the leader's barrier; give them time to
        // land (bounded) before the pair's shared memory is released.
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 1000000ull) { }
    }
    __syncwarp();
    cluster_sync_all();                      // no CTA leaves while its pair may still touch its smem / TMEM
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, TMEM_COLS);
    }
}

// ---------------------------------------------------------------------------
// narrow: 128 output channels x BN tokens, K split over a cluster
// ---------------------------------------------------------------------------
constexpr int kNarrowThreads = 128;

// Adds the S parts of this thread's channel for the tokens rank, rank + S, .., four
// at a time (their loads from the other CTAs in flight together), and finishes them.
template <typename T, int S>
__device__ __forceinline__ void add_parts(const uint32_t* part, int rank, int tokens, const float* sa, float sw,
                                          float bias, int act, bool live, T* y, int64_t ld) {
    const Gelu2 gelu;
    uint32_t from[S];
#pragma unroll
    for (int k = 0; k < S; ++k) from[k] = map_to_rank(smem_addr(part) + threadIdx.x * 4, k);
    for (int c = rank; c < tokens; c += 4 * S) {
        uint32_t acc[4] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i * S < tokens) {
#pragma unroll
                for (int k = 0; k < S; ++k) acc[i] += load_cluster_u32(from[k] + (c + i * S) * 512);
            }
        F2 v[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c0 = c + 2 * i * S, c1 = c0 + S;
            v[i] = finish(acc[2 * i], acc[2 * i + 1], pair_of(c0 < tokens ? sa[c0] : 0.f, c1 < tokens ? sa[c1] : 0.f),
                          pair_of(sw, sw), pair_of(bias, bias));
        }
        activate<T, 4>(v, act, gelu);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c0 = c + 2 * i * S, c1 = c0 + S;
            float a, b;
            halves(v[i], a, b);
            if (live && c0 < tokens) y[c0 * ld] = from_f<T>(a);
            if (live && c1 < tokens) y[c1 * ld] = from_f<T>(b);
        }
    }
}

template <typename T, int BN>
__global__ void __launch_bounds__(kNarrowThreads)
    narrow_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w, const Int8Args p,
                  int split, int stages) {
    constexpr uint32_t W_BYTES = 128 * kBK, A_BYTES = BN * kBK;
    constexpr uint32_t IDESC = idesc_i8(128, BN);
    constexpr uint32_t TMEM_COLS = BN < 32 ? 32 : BN;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[8], empty[8], tfull;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    __shared__ __align__(16) float s_sa[BN];
    volatile int* abort_flag = &abort_word;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sW = smem;
    uint8_t* sA = smem + stages * W_BYTES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int ot_count = (p.o + 127) / 128, mt_count = (p.m + BN - 1) / BN, kb_count = (p.k + kBK - 1) / kBK;
    const int rank = blockIdx.x % split, tile = blockIdx.x / split;
    const int mt = tile % mt_count, ot = tile / mt_count % ot_count, model = tile / mt_count / ot_count;
    const int kb0 = kb_count * rank / split, kbs = kb_count * (rank + 1) / split - kb0;

    // Thread = output channel in the end, columns = tokens.
    const int o = ot * 128 + threadIdx.x, tokens = min(BN, p.m - mt * BN);
    const int64_t wat = (int64_t)model * p.o + o;
    if (threadIdx.x < BN)
        s_sa[threadIdx.x] = threadIdx.x < tokens ? p.sa[(int64_t)model * p.m + mt * BN + threadIdx.x] : 0.f;
    const float sw = o < p.o ? p.sw[wat] : 0.f;
    const float bias = p.bias && o < p.o ? to_f<T>(static_cast<const T*>(p.bias)[wat]) : 0.f;
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tm_a);
        tma_prefetch_desc(&tm_w);
        for (int s = 0; s < stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&tfull, 1);
        *abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == 1) {
        tmem_alloc(&tmem_slot, TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_slot;

    int issued = 0;                          // blocks asked for, by thread 0
    if (warp == 0) {
        if (lane == 0) {
            const uint64_t pol_a = l2_policy_evict_last();
            const uint64_t pol_w = mt_count == 1 ? l2_policy_evict_first() : l2_policy_evict_normal();
            for (; issued < kbs; ++issued) {
                const int s = issued % stages;
                if (!mbar_wait(&empty[s], (uint32_t)(issued / stages & 1) ^ 1, abort_flag)) break;
                mbar_arrive_expect_tx(&full[s], W_BYTES + A_BYTES);
                tma_load_3d(sW + s * W_BYTES, &tm_w, &full[s], (kb0 + issued) * kBK, ot * 128, model, pol_w);
                tma_load_3d(sA + s * A_BYTES, &tm_a, &full[s], (kb0 + issued) * kBK, mt * BN, model, pol_a);
            }
            if (issued < kbs) {
                *abort_flag = 1;
                raise_device_error(p.err, DEV_ERR_GEMM_TIMEOUT);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint64_t w_desc0 = sdesc_kmajor_sw128(smem_addr(sW)), a_desc0 = sdesc_kmajor_sw128(smem_addr(sA));
            for (int i = 0; i < kbs; ++i) {
                const int s = i % stages;
                if (!mbar_wait(&full[s], (uint32_t)(i / stages & 1), abort_flag)) {
                    *abort_flag = 1;
                    raise_device_error(p.err, DEV_ERR_GEMM_TIMEOUT);
                    break;
                }
                tc_fence_after();
                const uint64_t wd = w_desc0 + (uint64_t)((s * W_BYTES) >> 4), ad = a_desc0 + (uint64_t)((s * A_BYTES) >> 4);
#pragma unroll
                for (int k = 0; k < kBK / 32; ++k) umma_i8(tmem_base, wd + 2 * k, ad + 2 * k, IDESC, (i | k) != 0);
                umma_commit(&empty[s]);
            }
            umma_commit(&tfull);             // also after a failure: the MMAs issued so far end before TMEM is freed
        }
    }
    __syncwarp();
    const volatile int never = 0;
    const bool ok = __all_sync(0xffffffffu, mbar_wait(&tfull, 0, &never));     // a warp reads TMEM as one
    if (!ok) {                               // stores nothing, and says so
        *abort_flag = 1;
        raise_device_error(p.err, DEV_ERR_GEMM_TIMEOUT);
    }
    tc_fence_after();

    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    T* y = static_cast<T*>(p.y) + ((int64_t)model * p.m + mt * BN) * p.o + o;
    constexpr int CH = BN < 32 ? BN : 32;
    auto load = [&](int c, uint32_t (&r)[CH]) {
        if constexpr (CH == 16) tmem_ld_32x32b_x16(tmem_base + lanes + c, r);
        else tmem_ld_32x32b_x32(tmem_base + lanes + c, r);
        tmem_ld_wait();
    };
    auto free_columns = [&]() {
        tc_fence_before();
        __syncthreads();
        if (warp == 1) {
            tc_fence_after();
            tmem_dealloc(tmem_base, TMEM_COLS);
        }
        // After a failure of any role: copies in flight land before the CTA's memory is released.
        if (threadIdx.x == 0 && *abort_flag)
            for (int j = max(issued - stages, 0); j < issued; ++j)
                mbar_wait_ns(&full[j % stages], (uint32_t)(j / stages & 1), &never, kWaitLimitNs / 8);
        __syncwarp();                        // the cluster's barriers take whole warps
    };
    if (split == 1) {
        const Gelu2 gelu;
#pragma unroll 1
        for (int c = 0; ok && c < tokens; c += CH) {
            uint32_t r[CH];
            load(c, r);
            F2 v[CH / 2];
#pragma unroll
            for (int j = 0; j < CH; j += 2)
                v[j / 2] = finish(r[j], r[j + 1], *reinterpret_cast<const F2*>(s_sa + c + j), pair_of(sw, sw),
                                  pair_of(bias, bias));
            activate<T, CH>(v, p.act, gelu);
#pragma unroll
            for (int j = 0; j < CH; j += 2) {
                float a, b;
                halves(v[j / 2], a, b);
                if (c + j < tokens && o < p.o) y[(int64_t)(c + j) * p.o] = from_f<T>(a);
                if (c + j + 1 < tokens && o < p.o) y[(int64_t)(c + j + 1) * p.o] = from_f<T>(b);
            }
        }
        free_columns();
    } else {
        // The parts as [token][channel] in the ring's memory (its copies have been
        // used up); CTA r adds and finishes the tokens r, r + split, ..
        uint32_t* part = reinterpret_cast<uint32_t*>(smem);
        if (ok) {
#pragma unroll 1
            for (int c = 0; c < tokens; c += CH) {
                uint32_t r[CH];
                load(c, r);
#pragma unroll
                for (int j = 0; j < CH; ++j) part[(c + j) * 128 + threadIdx.x] = r[j];
            }
        }
        // A CTA that waits for others holds no columns: a pair of CTAs (of any kernel) may
        // hold one SM's while it waits for its partner's, and the two would wait for ever.
        free_columns();
        cluster_sync_all();
        if (ok && split == 2) add_parts<T, 2>(part, rank, tokens, s_sa, sw, bias, p.act, o < p.o, y, p.o);
        else if (ok && split == 4) add_parts<T, 4>(part, rank, tokens, s_sa, sw, bias, p.act, o < p.o, y, p.o);
        else if (ok) add_parts<T, 8>(part, rank, tokens, s_sa, sw, bias, p.act, o < p.o, y, p.o);
        cluster_sync_all();                  // no CTA leaves while others read its part
    }
}

// A pair's kernel (wide_kernel; linear_tc_pair_kernel, 194 KB and the system's 1)
// leaves less of an SM's 228 KB than this and the 2 KB for alignment and the system.
constexpr int kBesidePair = 36 * 1024;
static_assert(WideSmem<float>::TOTAL + kBesidePair + 3 * 1024 > 228 * 1024, "a part of K beside a pair");
static_assert(WideSmem<__half>::TOTAL + kBesidePair + 3 * 1024 > 228 * 1024, "a part of K beside a pair");
static_assert(WideSmem<__nv_bfloat16>::TOTAL + kBesidePair + 3 * 1024 > 228 * 1024, "a part of K beside a pair");

int rows_map(CUtensorMap* map, const void* base, int64_t n, int64_t rows, int64_t k, int64_t ld, int64_t ms, uint32_t box) {
    const uint64_t dims[3] = {(uint64_t)k, (uint64_t)rows, (uint64_t)n};
    const uint64_t strides[2] = {(uint64_t)ld, (uint64_t)ms};
    const uint32_t boxes[3] = {kBK, box, 1};
    return encode_tmap_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, base, dims, strides, boxes, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename T>
CUtensorMapDataType out_type() {
    return sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                          : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

// Lets the kernel have `bytes` of shared memory; `had` is what it has, by device.
template <typename K>
int reserve(K kernel, size_t bytes, std::atomic<int> (&had)[64]) {
    std::atomic<int>& h = had[current_device() & 63];
    if (h.load(std::memory_order_relaxed) >= (int)bytes) return WIDEK_OK;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != cudaSuccess)
        return set_error(WIDEK_ERR_CUDA, "widek_linear_int8_fwd: %zu bytes of shared memory: %s", bytes, cudaGetErrorString(e));
    h.store((int)bytes, std::memory_order_relaxed);
    return WIDEK_OK;
}

struct Int8Launch {
    Int8Args p;
    const void *a, *w;
    int64_t a_ld, a_ms, w_ld, w_ms;
    cudaStream_t st;

    template <typename T>
    int wide() {
        using S = WideSmem<T>;
        CUtensorMap ta, tw;
        int rc = rows_map(&ta, a, p.n, p.m, p.k, a_ld, a_ms, 128);
        if (rc == WIDEK_OK) rc = rows_map(&tw, w, p.n, p.o, p.k, w_ld, w_ms, 128);
        p.vec_store = (int64_t)p.o * sizeof(T) % 16 == 0 && aligned16(p.y);
        CUtensorMap ty = ta;
        if (rc == WIDEK_OK && p.vec_store) {
            const uint64_t dims[3] = {(uint64_t)p.o, (uint64_t)p.m, (uint64_t)p.n};
            const uint64_t strides[2] = {(uint64_t)p.o * sizeof(T), (uint64_t)p.m * p.o * sizeof(T)};
            const uint32_t box[3] = {32, 32, 1};
            rc = encode_tmap_tiled(&ty, out_type<T>(), 3, p.y, dims, strides, box,
                                   sizeof(T) == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
        }
        static std::atomic<int> had[64];
        if (rc == WIDEK_OK) rc = reserve(wide_kernel<T>, S::TOTAL, had);
        if (rc != WIDEK_OK) return rc;
        const int64_t tiles = (int64_t)p.n * ((p.m + 255) / 256) * ((p.o + 255) / 256);
        const int grid = (int)std::min<int64_t>(2 * tiles, sm_count(current_device()) / 2 * 2);
        wide_kernel<T><<<grid, kWideThreads, S::TOTAL, st>>>(ta, tw, ty, p);
        return check_launch("widek_linear_int8_fwd (wide)");
    }

    int64_t narrow_tiles(int bn) const { return (int64_t)p.n * ((p.m + bn - 1) / bn) * ((p.o + 127) / 128); }
    // K is split where that fills the device and leaves each CTA four blocks of it:
    // (us, alone / in parts) 1 x 4096 -> 4096 for one token 18 / 9.4, 2 x 4176 ->
    // 4096 for 22 tokens 26 / 16; but 8 x 1024 -> 4096 for 4 tokens 11.9 / 12.9.
    int parts_of_k(int bn) const {
        const int sms = sm_count(current_device()), kb = (p.k + kBK - 1) / kBK;
        const int64_t tiles = narrow_tiles(bn);
        int split = 1;
        while (split < 8 && tiles * split <= (bn > 64 ? sms / 2 : sms) && kb >= 8 * split) split *= 2;
        return split;
    }

    template <typename T, int BN>
    int narrow() {
        CUtensorMap ta, tw;
        int rc = rows_map(&ta, a, p.n, p.m, p.k, a_ld, a_ms, BN);
        if (rc == WIDEK_OK) rc = rows_map(&tw, w, p.n, p.o, p.k, w_ld, w_ms, 128);
        const int sms = sm_count(current_device()), kb = (p.k + kBK - 1) / kBK;
        const int64_t tiles = narrow_tiles(BN);
        const int split = parts_of_k(BN);
        // The ring is as deep as lets the SM's share of CTAs (up to 5) be there at once.
        const int most = (kb + split - 1) / split, share = (int)std::min<int64_t>(5, (tiles * split + sms - 1) / sms);
        const int fit = 222 * 1024 / std::max(2, share) / ((128 + BN) * kBK);
        const int stages = std::min(most, std::max(2, std::min(8, fit)));
        size_t bytes = (size_t)stages * (128 + BN) * kBK;
        if (split > 1) bytes = std::max<size_t>({bytes, (size_t)BN * 512, (size_t)kBesidePair});
        // A CTA holds at least 456 bytes of an SM's 228 KB for each of its 512 TMEM
        // columns that it takes, so that an SM starts no CTA of this kernel that would wait
        // for the columns of others; and kBesidePair keeps parts of K, whose cluster
        // would wait along, off an SM where a pair of CTAs holds all columns to its end.
        bytes = std::max<size_t>(bytes + 1024, (BN < 32 ? 32 : BN) * 456);
        if (tiles * split > 0x7fffffff) return set_error(WIDEK_ERR_INVALID, "widek_linear_int8_fwd: over 2^31 tiles");
        static std::atomic<int> had[64];
        // (the most that any call asks for, so that calls on two threads cannot take it back)
        if (rc == WIDEK_OK) rc = reserve(narrow_kernel<T, BN>, 224 * 1024, had);
        if (rc != WIDEK_OK) return rc;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)(tiles * split));
        cfg.blockDim = dim3(kNarrowThreads);
        cfg.dynamicSmemBytes = bytes;
        cfg.stream = st;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim = {(unsigned)split, 1, 1};
        cfg.attrs = &attr;
        cfg.numAttrs = split > 1 ? 1 : 0;
        cudaLaunchKernelEx(&cfg, narrow_kernel<T, BN>, ta, tw, p, split, stages);
        return check_launch("widek_linear_int8_fwd (narrow)");
    }

    template <typename T>
    int run() {
        // Past 128 rows wide tiles where they fill a quarter of the device's pairs. Fewer of
        // them finish later than four times as many narrow ones when results are fp32 or rows
        // off the 16-byte borders (device times in us, wide / narrow: f32, 12 pairs, K = 64
        // 8.2 / 6.0, K = 1024 10.7 / 10.9; odd bf16 9.8 / 9.0 and 12.2 / 12.4), and else only
        // when those share out a long K, in four or more parts, or in two of 64 blocks: 129 rows
        // of 256 -> 128 6.8 / 8.4, 20 x 256 of 4096 -> 256 18.5 / 23.8; in parts 256 of 2048 ->
        // 256 11.6 / 9.9, 129 of 65536 -> 128 150 / 35; in two 16 x 130 of 4096 -> 256 17.5 / 18.9,
        // of 16384 48.3 / 47.7. From a quarter on: 4 x 129 of 1024 -> 2560 10.8 / 12.7, 8 x 256 of
        // 4096 -> 4096 35 / 64; but f32 of K = 64 8.7 / 8.4, odd bf16 of 80 pairs 15.3 / 11.2.
        if (p.m > 128) {
            const int64_t pairs = (int64_t)p.n * ((p.m + 255) / 256) * ((p.o + 255) / 256);
            const bool vectors = sizeof(T) == 2 && p.o % 8 == 0 && aligned16(p.y);
            const int parts = parts_of_k(128);
            const bool share = !vectors || parts >= 4 || (parts == 2 && p.k >= 128 * kBK);
            return pairs * 4 < sm_count(current_device()) && share ? narrow<T, 128>() : wide<T>();
        }
        if (p.m <= 16) return narrow<T, 16>();
        if (p.m <= 32) return narrow<T, 32>();
        if (p.m <= 64) return narrow<T, 64>();
        return narrow<T, 128>();
    }
};

}  // namespace
}  // namespace widek

using namespace widek;

extern "C" int widek_linear_int8_fwd(const void* a, const float* a_scale, const void* w, const float* w_scale,
                                     const void* bias, void* y, int64_t n, int64_t m, int64_t k, int64_t o, int64_t a_ld,
                                     int64_t a_ms, int64_t w_ld, int64_t w_ms, int act, int dtype, void* stream) {
    const char* what = "widek_linear_int8_fwd";
    if (n < 0 || m < 0 || o < 0 || k < 1 || k > kMaxK)
        return set_error(WIDEK_ERR_INVALID, "%s: bad sizes n=%lld m=%lld k=%lld o=%lld (k from 1 to %lld)", what,
                         (long long)n, (long long)m, (long long)k, (long long)o, (long long)kMaxK);
    if (act < WIDEK_ACT_NONE || act > WIDEK_ACT_GELU) return set_error(WIDEK_ERR_INVALID, "%s: unknown activation %d", what, act);
    if (dtype_size(dtype) == 0) return set_error(WIDEK_ERR_INVALID, "%s: unknown dtype code %d", what, dtype);
    if (n == 0 || m == 0 || o == 0) return WIDEK_OK;
    if (!a || !a_scale || !w || !w_scale || !y) return set_error(WIDEK_ERR_INVALID, "%s: null pointer", what);
    if (a_ld < 0 || w_ld < 0 || a_ld > (int64_t)1 << 32 || w_ld > (int64_t)1 << 32)
        return set_error(WIDEK_ERR_INVALID, "%s: bad strides", what);
    if (n > 0x7fffffff || m > 0x7fffff00 || o > 0x7fffff00 || n * ((m + 15) / 16) > 0x7fffffff / ((o + 127) / 128))
        return set_error(WIDEK_ERR_INVALID, "%s: too many tiles (n=%lld m=%lld o=%lld)", what, (long long)n, (long long)m,
                         (long long)o);
    if (n == 1) {                     // no second model to step to
        a_ms = m * a_ld;
        w_ms = o * w_ld;
    }
    if (!aligned16(a) || !aligned16(w) || a_ld % 16 != 0 || w_ld % 16 != 0 || a_ms % 16 != 0 || w_ms % 16 != 0 || a_ld < k ||
        w_ld < k || a_ms < (m - 1) * a_ld + k || w_ms < (o - 1) * w_ld + k)
        return set_error(WIDEK_ERR_INVALID, "%s: rows of codes must lie a multiple of 16 bytes apart, models behind one "
                         "another", what);
    if (a_ld >= (int64_t)1 << 40 || w_ld >= (int64_t)1 << 40 || a_ms >= (int64_t)1 << 40 || w_ms >= (int64_t)1 << 40)
        return set_error(WIDEK_ERR_INVALID, "%s: strides of 2^40 bytes or more", what);
    Int8Launch l{{a_scale, w_scale, bias, y, (int)n, (int)m, (int)k, (int)o, act, 0, device_error_ptr()},
                 a, w, a_ld, a_ms, w_ld, w_ms, static_cast<cudaStream_t>(stream)};
    return dispatch_dtype(dtype, l);
}
