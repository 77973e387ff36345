// Shared parts of the block-boundary row kernels (residual_norm.cu,
// residual_norm_bwd.cu): arguments, row vectors and reductions over a row.
#pragma once

#include "paged_cache.cuh"
#include "sm100_ptx.cuh"

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
    FastDiv model_div, gate_div;
    float scale, eps;
};

constexpr int kMaxChannels = 8192;

template <typename T, int VE>
struct alignas(sizeof(T) * VE) Pack {
    T v[VE];
};

// V vectors of VE channels a thread: vector i of thread t is channels
// (t + threads i) VE ...
template <typename T, int VE, int V>
struct Raw {
    Pack<T, VE> p[V];
    __device__ __forceinline__ void load(const T* row, int t, int threads, int nvec) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = t + threads * i;
            if (c < nvec) p[i] = *reinterpret_cast<const Pack<T, VE>*>(row + (int64_t)c * VE);
        }
    }
    __device__ __forceinline__ float get(int i, int j) const { return to_f<T>(p[i].v[j]); }
};

// Largest vector of T (16 bytes at most) that d channels and all the pointers allow.
template <typename T>
inline int vec_elems(int d, std::initializer_list<const void*> ptrs) {
    for (int ve = 16 / (int)sizeof(T); ve > 1; ve /= 2) {
        if (ve != 16 / (int)sizeof(T) && ve != 4) continue;
        bool ok = d % ve == 0;
        for (const void* p : ptrs) ok = ok && reinterpret_cast<uintptr_t>(p) % (ve * sizeof(T)) == 0;
        if (ok) return ve;
    }
    return 1;
}

// Who shares a row: a warp, a block, or the two blocks of a cluster.
enum Team : int { WARP = 0, BLOCK = 1, PAIR = 2 };

// Sums (or maxima of magnitudes, NaN kept) over the threads of a row. Beyond a
// warp they go through `slots`, one float a warp and value; two sets that calls
// take in turn, so that one barrier each is enough: who writes a set again has
// passed the barrier of the call between, which everyone reaches after reading.
template <int TEAM, int N>
struct Reduce {
    float (*slots)[32];            // [2 N][32]
    int turn;
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
    __device__ __forceinline__ int warps() const { return (blockDim.x >> 5) << (TEAM == PAIR ? 1 : 0); }
    __device__ __forceinline__ void sum(float (&v)[N]) {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = warp_sum(v[k]);
        if constexpr (TEAM != WARP) {
            float (*s)[32] = exchange(v);
            const int lane = threadIdx.x & 31;
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = warp_sum(lane < warps() ? s[k][lane] : 0.f);
        }
    }
    __device__ __forceinline__ float amax(float v) {
        static_assert(N == 1, "one value");
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = amax2(v, __shfl_xor_sync(0xffffffffu, v, o));
        if constexpr (TEAM != WARP) {
            const float one[1] = {v};
            float (*s)[32] = exchange(one);
            const int lane = threadIdx.x & 31;
            v = lane < warps() ? s[0][lane] : 0.f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v = amax2(v, __shfl_xor_sync(0xffffffffu, v, o));
        }
        return v;
    }
};

// Checks the sizes and pointers that the entry points share and fills `a`.
// gate_rows: rows that share a row of the gate, -1 without one.
int make_args(Args& a, const char* what, const void* x, const void* y, const void* w, const void* wb, const void* pw,
              const void* pb, const void* gate, int64_t n, int64_t rows, int64_t d, int64_t gate_rows, double scale,
              double eps, int center, int dtype);

}  // namespace rnorm
}  // namespace widek
