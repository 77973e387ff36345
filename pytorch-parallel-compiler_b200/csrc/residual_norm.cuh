// Shared parts of the block-boundary row kernels (residual_norm.cu,
// residual_norm_bwd.cu): arguments, row vectors and reductions over a row.
#pragma once

#include "paged_cache.cuh"
#include "sm100_ptx.cuh"

#include <atomic>
#include <initializer_list>
#include <type_traits>

namespace widek {
namespace rnorm {

// A row is one token of one model: d channels, dense. Rows of a model follow
// one another; gate row of row r: r / gate_rows (0: no gate).
struct Args {
    const void *x, *y, *w, *wb, *pw, *pb, *gate;
    void *h, *z;                   // z: rows of the type, or codes with rows `ld` apart
    float* cscale;                 // scales of the codes
    float* stats;                  // [rows][4] mean and factor of y and of h, or null
    int64_t rows, ld;
    int d, center;
    uint32_t gate_rows;
    FastDiv gate_div;
    float scale, eps;
    int64_t n, model_rows;
    int teams;                     // of each model (Walk)
};

constexpr int kMaxChannels = 8192;

// VE channels as one load or store.
template <typename T, int VE>
struct alignas(sizeof(T) * VE) Pack {
    T v[VE];
};

// A thread holds K channels of a row as K / VE vectors: vector i of thread t is the
// VE channels from (t + threads i) VE on. The kernels walk over rows, so that a
// channel's weights and sums stay in its thread's registers.
template <typename T, int VE>
__device__ __forceinline__ Pack<T, VE> pack(const float* v) {
    Pack<T, VE> p;
    if constexpr (VE >= 2 && std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
        for (int j = 0; j < VE; j += 2) reinterpret_cast<__nv_bfloat162*>(p.v)[j / 2] = __floats2bfloat162_rn(v[j], v[j + 1]);
    } else if constexpr (VE >= 2 && std::is_same<T, __half>::value) {
#pragma unroll
        for (int j = 0; j < VE; j += 2) reinterpret_cast<__half2*>(p.v)[j / 2] = __floats2half2_rn(v[j], v[j + 1]);
    } else {
#pragma unroll
        for (int j = 0; j < VE; ++j) p.v[j] = from_f<T>(v[j]);
    }
    return p;
}

// Largest vector of T (16 bytes at most) that d channels and all the pointers allow.
template <typename T>
inline int vec_elems(int64_t d, std::initializer_list<const void*> ptrs) {
    for (int ve = 16 / (int)sizeof(T); ve > 1; ve /= 2) {
        bool ok = d % ve == 0;
        for (const void* p : ptrs) ok = ok && reinterpret_cast<uintptr_t>(p) % (ve * sizeof(T)) == 0;
        if (ok) return ve;
    }
    return 1;
}

// Two values an instruction: v += c, a += b, the sum of v.
template <int K>
__device__ __forceinline__ void shift_vec(float (&v)[K], float c) {
#pragma unroll
    for (int j = 0; j < K; j += 2) add2(v[j], v[j + 1], v[j], v[j + 1], c, c);
}
template <int K>
__device__ __forceinline__ void add_vec(float (&a)[K], const float (&b)[K]) {
#pragma unroll
    for (int j = 0; j < K; j += 2) add2(a[j], a[j + 1], a[j], a[j + 1], b[j], b[j + 1]);
}
template <int K>
__device__ __forceinline__ float sum_vec(const float (&v)[K]) {
    float s0 = v[0], s1 = v[1];
#pragma unroll
    for (int j = 2; j < K; j += 2) add2(s0, s1, s0, s1, v[j], v[j + 1]);
    return s0 + s1;
}

// Who shares a row: up to 32 lanes of a warp, a block, or the two blocks of a cluster.
enum Team : int { WARP = 0, BLOCK = 1, PAIR = 2 };

struct TeamShape {
    int team, threads, lanes;      // of a block; of a row, within a warp
    int rows() const { return team == WARP ? threads / lanes : 1; }     // rows of a block at a time
};
constexpr int kBlockThreads = 512; // at most: 128 registers a thread
// Lanes for d channels, k a thread, else a block, else a pair of them.
inline TeamShape team_shape(int d, int k) {
    if (d <= 32 * k) return {WARP, 128, d <= 4 * k ? 4 : d <= 8 * k ? 8 : d <= 16 * k ? 16 : 32};
    const int threads = (d + 32 * k - 1) / (32 * k) * 32;
    if (threads <= kBlockThreads) return {BLOCK, threads, 32};
    return {PAIR, (threads + 63) / 64 * 32, 32};
}

// Where a thread stands.
template <int TEAM>
struct Seat {
    int t, threads;                // in its team
    int64_t team;
    unsigned mask;                 // its team's lanes in its warp
    __device__ __forceinline__ Seat(int lanes) {
        if constexpr (TEAM == WARP) {
            t = threadIdx.x & (lanes - 1);
            threads = lanes;
            team = (int64_t)blockIdx.x * (blockDim.x / lanes) + threadIdx.x / lanes;
            mask = lanes == 32 ? 0xffffffffu : ((1u << lanes) - 1u) << (threadIdx.x & 31 & ~(lanes - 1));
        } else {
            t = TEAM == BLOCK ? threadIdx.x : sm100::cluster_ctarank() * blockDim.x + threadIdx.x;
            threads = TEAM == BLOCK ? blockDim.x : 2 * blockDim.x;
            team = TEAM == BLOCK ? blockIdx.x : blockIdx.x >> 1;
            mask = 0xffffffffu;
        }
    }
};

// Sums (or maxima of magnitudes, NaN kept) over the threads of a row. Beyond a
// warp they go through `slots`, one float a warp and value (zeros past the last
// warp); two sets that calls take in turn, so that one barrier each is enough:
// who writes a set again has passed the barrier of the call between, which
// everyone reaches after reading.
template <int TEAM, int N>
struct Reduce {
    float (*slots)[32];            // [2 N][32]
    int lanes;
    unsigned mask;
    int turn = 0;
    __device__ __forceinline__ Reduce(float (*s)[32], const Seat<TEAM>& seat)
        : slots(s), lanes(TEAM == WARP ? seat.threads : 32), mask(seat.mask) {
        if constexpr (TEAM != WARP) {
            for (int i = threadIdx.x; i < 2 * N * 32; i += blockDim.x) slots[i / 32][i % 32] = 0.f;
            if constexpr (TEAM == PAIR) sm100::cluster_sync_all();     // both blocks are there, their slots zero
            else __syncthreads();
        }
    }
    __device__ __forceinline__ int warps() const { return (blockDim.x >> 5) << (TEAM == PAIR ? 1 : 0); }
    // Puts this warp's values where everyone finds them; returns the set.
    __device__ __forceinline__ float (*exchange(const float (&v)[N]))[32] {
        float (*s)[32] = slots + turn * N;
        turn ^= 1;
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        if constexpr (TEAM == BLOCK) {
            if (lane == 0) {
#pragma unroll
                for (int k = 0; k < N; ++k) s[k][warp] = v[k];
            }
            __syncthreads();
        } else {
            if (lane < 2) {        // lane r writes into block r of the pair
                const int at = sm100::cluster_ctarank() * (blockDim.x >> 5) + warp;
#pragma unroll
                for (int k = 0; k < N; ++k)
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(
                                     sm100::map_to_rank(sm100::smem_addr(&s[k][at]), lane)), "f"(v[k]) : "memory");
            }
            sm100::cluster_sync_all();
        }
        return s;
    }
    __device__ __forceinline__ void sum(float (&v)[N]) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            if (TEAM == WARP && o >= lanes) continue;
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(mask, v[k], o);
        }
        if constexpr (TEAM != WARP) {
            float (*s)[32] = exchange(v);
            const int w = warps();
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const float4* q = reinterpret_cast<const float4*>(s[k]);
                float4 a = q[0];
                for (int i = 1; 4 * i < w; ++i) {
                    const float4 b = q[i];
                    a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
                }
                v[k] = (a.x + a.y) + (a.z + a.w);
            }
        }
    }
    __device__ __forceinline__ float amax(float v) {
        static_assert(N == 1, "one value");
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            if (TEAM == WARP && o >= lanes) continue;
            v = amax2(v, __shfl_xor_sync(mask, v, o));
        }
        if constexpr (TEAM != WARP) {
            const float one[1] = {v};
            const float4* q = reinterpret_cast<const float4*>(exchange(one)[0]);
            const int w = warps();
            v = 0.f;
            for (int i = 0; 4 * i < w; ++i) {
                const float4 b = q[i];
                v = amax2(amax2(v, b.x), amax2(amax2(b.y, b.z), b.w));
            }
        }
        return v;
    }
};

// The rows ahead: a ring of STAGES rows of TENSORS tensors in shared memory,
// every thread copying (without waiting) and reading back its own channels.
// Single 16-bit values, which are too small for such copies, wait in registers
// instead, one row ahead. Channels past the row's end read as zeros.
template <typename T, int VE, int K, int TENSORS>
struct Ring {
    static constexpr int V = K / VE;
    static constexpr int STAGES = TENSORS * K * sizeof(T) > 128 ? 2 : 3;      // 227 KB of 512 threads
    static constexpr bool REGS = sizeof(T) * VE < 4;
    using P = Pack<T, VE>;
    static constexpr int bytes(int threads) { return REGS ? 0 : STAGES * TENSORS * K * (int)sizeof(T) * threads; }

    P* own;                        // this thread's first pack
    int t, threads, nvec;
    P held[REGS ? TENSORS : 1][REGS ? V : 1];

    __device__ __forceinline__ Ring(uint8_t* smem, int t_, int threads_, int nvec_)
        : own(reinterpret_cast<P*>(smem) + threadIdx.x), t(t_), threads(threads_), nvec(nvec_) {
        P zero;
#pragma unroll
        for (int j = 0; j < VE; ++j) zero.v[j] = from_f<T>(0.f);
        if constexpr (REGS) {
#pragma unroll
            for (int k = 0; k < TENSORS; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) held[k][i] = zero;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (t + threads * i >= nvec)
                    for (int k = 0; k < STAGES * TENSORS; ++k) own[(k * V + i) * blockDim.x] = zero;
        }
    }
    // Zeros for a tensor that is not there.
    __device__ __forceinline__ void clear(int tensor) {
        P zero;
#pragma unroll
        for (int j = 0; j < VE; ++j) zero.v[j] = from_f<T>(0.f);
        if constexpr (!REGS) {
            for (int s = 0; s < STAGES; ++s)
#pragma unroll
                for (int i = 0; i < V; ++i) own[((s * TENSORS + tensor) * V + i) * blockDim.x] = zero;
        }
    }
    // One tensor's row (null: not copied) into a stage.
    __device__ __forceinline__ void fetch(int stage, int tensor, const void* base, int row, int d) {
        if (!base) return;
        const P* src = reinterpret_cast<const P*>(static_cast<const T*>(base) + (int64_t)row * d);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = t + threads * i;
            if (c >= nvec) continue;
            if constexpr (REGS) {
                held[tensor][i] = src[c];
            } else {
                P* dst = own + ((stage * TENSORS + tensor) * V + i) * blockDim.x;
                if constexpr (sizeof(P) == 16)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(sm100::smem_addr(dst)), "l"(src + c)
                                 : "memory");
                else
                    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(sm100::smem_addr(dst)), "l"(src + c),
                                 "n"(sizeof(P)) : "memory");
            }
        }
    }
    __device__ __forceinline__ void commit() {
        if constexpr (!REGS) asm volatile("cp.async.commit_group;" ::: "memory");
    }
    // Rows that are fetched before the first one is used; and the wait for the
    // oldest once the next one has been asked for.
    static constexpr int AHEAD = REGS ? 1 : STAGES - 1;
    __device__ __forceinline__ void wait() {
        if constexpr (!REGS) asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
    }
    __device__ __forceinline__ void finish() {
        if constexpr (!REGS) asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __device__ __forceinline__ void packs(int stage, int tensor, P (&out)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if constexpr (REGS) out[i] = held[tensor][i];
            else out[i] = own[((stage * TENSORS + tensor) * V + i) * blockDim.x];
        }
    }
    __device__ __forceinline__ void get(int stage, int tensor, float (&out)[K]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            P p;
            if constexpr (REGS) p = held[tensor][i];
            else p = own[((stage * TENSORS + tensor) * V + i) * blockDim.x];
#pragma unroll
            for (int j = 0; j < VE; ++j) out[i * VE + j] = to_f<T>(p.v[j]);
        }
    }
};

// A thread's channels of one row of weights (`fill` without them, 0 past the end).
template <typename T, int VE, int K>
__device__ __forceinline__ void load_weights(const void* base, int64_t row, int d, int t, int threads, float fill,
                                             float (&out)[K]) {
#pragma unroll
    for (int i = 0; i < K / VE; ++i) {
        const int c = t + threads * i;
        Pack<T, VE> p;
        const bool in = c < d / VE;
        if (base && in) p = *reinterpret_cast<const Pack<T, VE>*>(static_cast<const T*>(base) + row * d + c * VE);
#pragma unroll
        for (int j = 0; j < VE; ++j) out[i * VE + j] = !in ? 0.f : base ? to_f<T>(p.v[j]) : fill;
    }
}

template <typename T, int VE, int K>
__device__ __forceinline__ void store_row(void* base, int row, int d, int t, int threads, const float (&v)[K]) {
    Pack<T, VE>* dst = reinterpret_cast<Pack<T, VE>*>(static_cast<T*>(base) + (int64_t)row * d);
#pragma unroll
    for (int i = 0; i < K / VE; ++i) {
        const int c = t + threads * i;
        if (c < d / VE) dst[c] = pack<T, VE>(v + i * VE);
    }
}

// Rows first .. end - 1 of team `team` of `teams` teams a model: consecutive rows, evenly.
struct Walk {
    int model, first, end;
    __device__ __forceinline__ Walk(int64_t team, int teams, int64_t model_rows) {
        model = (int)(team / teams);
        const int64_t k = team - (int64_t)model * teams;
        first = (int)(model * model_rows + model_rows * k / teams);
        end = (int)(model * model_rows + model_rows * (k + 1) / teams);
    }
    // Whether the row `ahead` rows on is the walk's too; their sum may not fit in 32 bits.
    __device__ __forceinline__ bool has(int row, int ahead) const { return ahead < end - row; }
};

// Blocks of `kernel` that an SM holds at once, asked for once; the kernel may have as
// much shared memory as any launch of it takes from then on.
template <typename K>
inline int resident_blocks(std::atomic<int>& known, K kernel, int threads, int smem) {
    int per = known.load(std::memory_order_relaxed);
    if (per > 0) return per;
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024);
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, threads, smem) != cudaSuccess || per < 1) per = 1;
    known.store(per, std::memory_order_relaxed);
    return per;
}

// Checks the sizes and pointers that the entry points share and fills `a`.
// gate_rows: rows that share a row of the gate, -1 without one.
int make_args(Args& a, const char* what, const void* x, const void* y, const void* w, const void* wb, const void* pw,
              const void* pb, const void* gate, int64_t n, int64_t rows, int64_t d, int64_t gate_rows, double scale,
              double eps, int center, int dtype);

}  // namespace rnorm
}  // namespace widek
