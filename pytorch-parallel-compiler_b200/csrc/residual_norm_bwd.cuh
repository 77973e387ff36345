// Gradients of the residual stream and its norms (the forward's formulas stand
// in residual_norm.cu). With un, hn the normalised rows, ru, rh their factors
// and gz = dz w:
//
//   dx = dh + rh (gz - hn mean(gz hn) - c mean(gz))
//   dw = sum dz hn, db = sum dz over a model's rows
//   t = scale dx;  dgate = sum of t u over the gate's rows
//   g = t gate pw;  dpw = sum t gate un, dpb = sum t gate
//   dy = ru (g - un mean(g un) - c mean(g)), or t gate without a norm of y
//
// A team (a warp, or a block for long rows) walks over consecutive rows of one
// model, each thread keeping its channels' weights and sums in registers, the
// next row's loads in flight while it works on one. Sums over rows go out once
// a team and are added in a fixed order by a second kernel. While a gate row
// stays the same, only A = sum t un and B = sum t are kept: dgate = pw A + pb B,
// dpw = gate A, dpb = gate B. A gate per sequence is finished whenever the walk
// leaves its rows: at once when all of them were this team's, else through the
// first or last partial sums of the teams that share it.
#include "residual_norm.cuh"

#include <initializer_list>

namespace widek {
namespace rnorm {

enum Mode : int { PLAIN = 0, MODEL = 1, SEQUENCE = 2, TOKEN = 3 };

struct BwdArgs {
    Args f;
    const void *dh, *dz;
    void *dx, *dy, *dw, *dwb, *dpw, *dpb, *dgate;
    float* part;                   // [teams][slots][d]
    int teams;                     // of each model
    int64_t n, model_rows;
};

__host__ __device__ constexpr int slot_count(int mode, bool center) {
    const int k = center ? 2 : 1;
    return mode == PLAIN ? k : mode == SEQUENCE ? 4 * k : 2 * k;
}

// Threads of a block for rows of d channels, 8 a thread: a warp, a block of up
// to 512 threads (128 registers each), or two such blocks in a cluster.
struct TeamShape {
    int team, threads;
};
inline TeamShape team_shape(int d) {
    if (d <= 256) return {WARP, 128};
    if (d <= 4096) return {BLOCK, (d + 255) / 256 * 32};
    return {PAIR, (d + 511) / 512 * 32};
}

// Teams of each model: one wave over the device, a few rows each.
int bwd_teams(int64_t n, int64_t rows, int d, int sms);
int bwd_mode(const Args& a, int64_t rows);

struct BwdLaunch {
    BwdArgs a;
    int mode;
    cudaStream_t st;
    template <typename T>
    int run();
};

extern template int BwdLaunch::run<float>();
extern template int BwdLaunch::run<__half>();
extern template int BwdLaunch::run<__nv_bfloat16>();

#ifdef WIDEK_RNORM_BWD_BODY
namespace {

// The rows ahead: a ring of kStages rows of x, y, dh and dz in shared memory,
// every thread copying (without waiting) and reading back its own channels.
constexpr int kStages = 3;

template <typename T, int VE>
__device__ __forceinline__ void copy_async(Pack<T, VE>* dst, const Pack<T, VE>* src) {
    if constexpr (sizeof(Pack<T, VE>) == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(sm100::smem_addr(dst)), "l"(src) : "memory");
    else if constexpr (sizeof(Pack<T, VE>) >= 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(sm100::smem_addr(dst)), "l"(src),
                     "n"(sizeof(Pack<T, VE>)) : "memory");
    else
        *dst = *src;
}

template <typename T, int VE, int V>
struct Ring {
    Pack<T, VE>* own;              // this thread's first pack
    int t, threads, nvec;
    __device__ __forceinline__ Pack<T, VE>* at(int stage, int tensor, int i) const {
        return own + ((stage * 4 + tensor) * V + i) * blockDim.x;
    }
    __device__ __forceinline__ void fetch(int stage, int tensor, const void* base, int64_t row, int d) const {
        if (!base) return;
        const Pack<T, VE>* src = reinterpret_cast<const Pack<T, VE>*>(static_cast<const T*>(base) + row * d);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (t + threads * i < nvec) copy_async<T, VE>(at(stage, tensor, i), src + t + threads * i);
    }
    __device__ __forceinline__ void fetch_row(int stage, const BwdArgs& a, int64_t row, bool live) const {
        if (live) {
            fetch(stage, 0, a.f.x, row, a.f.d);
            fetch(stage, 1, a.f.y, row, a.f.d);
            fetch(stage, 2, a.dh, row, a.f.d);
            fetch(stage, 3, a.dz, row, a.f.d);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    // One pack of the row (zeros where there is no such tensor).
    __device__ __forceinline__ void get(int stage, int tensor, const void* base, int i, float (&out)[VE]) const {
        if (base) {
            const Pack<T, VE> p = *at(stage, tensor, i);
#pragma unroll
            for (int j = 0; j < VE; ++j) out[j] = to_f<T>(p.v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < VE; ++j) out[j] = 0.f;
        }
    }
};

template <typename T, int VE, int V>
__device__ __forceinline__ void load_row(Raw<T, VE, V>& r, const void* base, int64_t row, int d, int t, int threads,
                                         int nvec, float fill) {
    if (base) {
        r.load(static_cast<const T*>(base) + row * d, t, threads, nvec);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int j = 0; j < VE; ++j) r.p[i].v[j] = from_f<T>(fill);
    }
}

template <int VE, int V>
__device__ __forceinline__ void put_part(float* dst, const float (&v)[V][VE], int t, int threads, int nvec) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = t + threads * i;
        if (c < nvec) {
#pragma unroll
            for (int j = 0; j < VE; ++j) dst[c * VE + j] = v[i][j];
        }
    }
}

template <typename T, int VE, int V, int MODE, bool CENTER, int TEAM>
__global__ void __launch_bounds__(TEAM == WARP ? 128 : 512) backward_kernel(const BwdArgs a) {
    constexpr int N = CENTER ? 2 : 1;
    constexpr int SLOTS = slot_count(MODE, CENTER);
    constexpr bool YSIDE = MODE != PLAIN;
    __shared__ float slots[2 * N][32];
    extern __shared__ uint8_t ring_bytes[];
    const int threads = TEAM == WARP ? 32 : TEAM == BLOCK ? blockDim.x : 2 * blockDim.x;
    const int t = TEAM == WARP ? threadIdx.x & 31 : TEAM == BLOCK ? threadIdx.x
                : sm100::cluster_ctarank() * blockDim.x + threadIdx.x;
    const int64_t team = TEAM == WARP ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5)
                       : TEAM == BLOCK ? blockIdx.x : blockIdx.x >> 1;
    if constexpr (TEAM == PAIR) sm100::cluster_sync_all();     // both blocks are there before one writes to the other
    if (team >= a.n * a.teams) return;
    Reduce<TEAM, N> red{slots, 0};
    const int d = a.f.d, nvec = d / VE;
    const float inv_d = 1.f / (float)d, scale = a.f.scale;
    const int64_t model = team / a.teams, j0 = team % a.teams;
    const int64_t base = model * a.model_rows;
    const int64_t first = base + a.model_rows * j0 / a.teams, end = base + a.model_rows * (j0 + 1) / a.teams;
    const Ring<T, VE, V> ring{reinterpret_cast<Pack<T, VE>*>(ring_bytes) + threadIdx.x, t, threads, nvec};
    const float4* stats = reinterpret_cast<const float4*>(a.f.stats);
#pragma unroll
    for (int k = 0; k < kStages - 1; ++k) ring.fetch_row(k, a, first + k, first + k < end);
    float4 st = stats[first];

    Raw<T, VE, V> w, pw, pb, gate;
    load_row<T, VE, V>(w, a.f.w, model, d, t, threads, nvec, 1.f);
    if constexpr (YSIDE) {
        load_row<T, VE, V>(pw, a.f.pw, model, d, t, threads, nvec, 1.f);
        if constexpr (CENTER) load_row<T, VE, V>(pb, a.f.pb, model, d, t, threads, nvec, 0.f);
        if constexpr (MODE == MODEL) load_row<T, VE, V>(gate, a.f.gate, model, d, t, threads, nvec, 1.f);
    }
    float P[V][VE] = {}, Q[V][VE] = {}, A[V][VE] = {}, B[V][VE] = {}, At[V][VE] = {}, Bt[V][VE] = {};
    float* part = a.part + team * SLOTS * d;

    int stage = 0;
    for (int64_t row = first; row < end; ++row) {
        const int ahead = stage == 0 ? kStages - 1 : stage - 1;
        ring.fetch_row(ahead, a, row + kStages - 1, row + kStages - 1 < end);
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        const float mu = st.x, ru = st.y, mh = st.z, rh = st.w;
        if (row + 1 < end) st = stats[row + 1];
        const int64_t at = row * d;
        uint32_t grow = 0;
        if constexpr (MODE == SEQUENCE || MODE == TOKEN) {
            grow = a.f.gate_div.div((uint32_t)row);
            if (MODE == TOKEN || row == first || row == (int64_t)grow * a.f.gate_rows)
                gate.load(static_cast<const T*>(a.f.gate) + (int64_t)grow * d, t, threads, nvec);
        }
        const bool post = YSIDE && a.f.pw;
        float un[V][VE], hn[V][VE], gz[V][VE];
        float s[N] = {};
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (t + threads * i >= nvec) continue;
            float x[VE], y[VE], dz[VE];
            ring.get(stage, 0, a.f.x, i, x);
            ring.get(stage, 1, a.f.y, i, y);
            ring.get(stage, 3, a.dz, i, dz);
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                float h;
                if constexpr (YSIDE) {
                    un[i][j] = post ? (y[j] - mu) * ru : y[j];
                    const float u = fmaf(un[i][j], pw.get(i, j), CENTER ? pb.get(i, j) : 0.f);
                    h = fmaf(scale * gate.get(i, j), u, x[j]);
                } else {
                    h = fmaf(scale, y[j], x[j]);
                }
                hn[i][j] = (h - mh) * rh;
                gz[i][j] = dz[j] * w.get(i, j);
                P[i][j] = fmaf(dz[j], hn[i][j], P[i][j]);
                s[0] = fmaf(gz[i][j], hn[i][j], s[0]);
                if constexpr (CENTER) {
                    Q[i][j] += dz[j];
                    s[N - 1] += gz[i][j];
                }
            }
        }
        red.sum(s);
        const float c1 = s[0] * inv_d, c2 = CENTER ? s[N - 1] * inv_d : 0.f;
        s[0] = s[N - 1] = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = t + threads * i;
            if (c >= nvec) continue;
            float dh[VE];
            ring.get(stage, 2, a.dh, i, dh);
            Pack<T, VE> ox, og;
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const float dx = fmaf(rh, gz[i][j] - fmaf(hn[i][j], c1, c2), dh[j]);
                ox.v[j] = from_f<T>(dx);
                float tt = scale * dx;
                if constexpr (YSIDE) {
                    if constexpr (MODE == TOKEN) {
                        og.v[j] = from_f<T>(tt * fmaf(un[i][j], pw.get(i, j), CENTER ? pb.get(i, j) : 0.f));
                        tt *= gate.get(i, j);
                    }
                    A[i][j] = fmaf(tt, un[i][j], A[i][j]);
                    if constexpr (CENTER) B[i][j] += tt;
                    if constexpr (MODE != TOKEN) tt *= gate.get(i, j);
                    gz[i][j] = tt * pw.get(i, j);       // now the gradient of un
                    s[0] = fmaf(gz[i][j], un[i][j], s[0]);
                    if constexpr (CENTER) s[N - 1] += gz[i][j];
                } else {
                    gz[i][j] = tt;
                }
            }
            if (a.dx) *reinterpret_cast<Pack<T, VE>*>(static_cast<T*>(a.dx) + at + (int64_t)c * VE) = ox;
            if constexpr (MODE == TOKEN)
                if (a.dgate) *reinterpret_cast<Pack<T, VE>*>(static_cast<T*>(a.dgate) + at + (int64_t)c * VE) = og;
        }
        if (a.dy) {
            float k1 = 0.f, k2 = 0.f, k0 = 1.f;
            if (post) {
                red.sum(s);
                k0 = ru;
                k1 = s[0] * inv_d;
                k2 = CENTER ? s[N - 1] * inv_d : 0.f;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = t + threads * i;
                if (c >= nvec) continue;
                Pack<T, VE> oy;
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    if constexpr (YSIDE) oy.v[j] = from_f<T>(k0 * (gz[i][j] - fmaf(un[i][j], k1, k2)));
                    else oy.v[j] = from_f<T>(gz[i][j]);
                }
                *reinterpret_cast<Pack<T, VE>*>(static_cast<T*>(a.dy) + at + (int64_t)c * VE) = oy;
            }
        }
        if constexpr (MODE == SEQUENCE) {
            const int64_t g0 = (int64_t)grow * a.f.gate_rows, g1 = g0 + a.f.gate_rows;
            if (row + 1 == end || row + 1 == g1) {
                const bool whole = g0 >= first && g1 <= end;
                const bool leading = g0 <= first;
                if (!whole) {
                    float* dst = part + (leading ? N : 2 * N) * d;
                    put_part<VE, V>(dst, A, t, threads, nvec);
                    if constexpr (CENTER) put_part<VE, V>(dst + d, B, t, threads, nvec);
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int c = t + threads * i;
                    if (c >= nvec) continue;
                    Pack<T, VE> og;
#pragma unroll
                    for (int j = 0; j < VE; ++j) {
                        const float g = gate.get(i, j);
                        og.v[j] = from_f<T>(fmaf(A[i][j], pw.get(i, j), CENTER ? B[i][j] * pb.get(i, j) : 0.f));
                        At[i][j] = fmaf(g, A[i][j], At[i][j]);
                        Bt[i][j] = fmaf(g, B[i][j], Bt[i][j]);
                        A[i][j] = B[i][j] = 0.f;
                    }
                    if (whole && a.dgate)
                        *reinterpret_cast<Pack<T, VE>*>(static_cast<T*>(a.dgate) + (int64_t)grow * d + (int64_t)c * VE) = og;
                }
            }
        }
        stage = stage == kStages - 1 ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    put_part<VE, V>(part, P, t, threads, nvec);
    if constexpr (CENTER) put_part<VE, V>(part + d, Q, t, threads, nvec);
    if constexpr (MODE == SEQUENCE) {
        put_part<VE, V>(part + 3 * N * d, At, t, threads, nvec);
        if constexpr (CENTER) put_part<VE, V>(part + (3 * N + 1) * d, Bt, t, threads, nvec);
    } else if constexpr (YSIDE) {
        put_part<VE, V>(part + N * d, A, t, threads, nvec);
        if constexpr (CENTER) put_part<VE, V>(part + (N + 1) * d, B, t, threads, nvec);
    }
    if constexpr (TEAM == PAIR) sm100::cluster_sync_all();     // the other block's sums are still written to this one
}

template <typename T>
__device__ __forceinline__ float at_or(const void* p, int64_t i, float other) {
    return p ? to_f<T>(static_cast<const T*>(p)[i]) : other;
}
template <typename T>
__device__ __forceinline__ void put(void* p, int64_t i, float v) {
    if (p) static_cast<T*>(p)[i] = from_f<T>(v);
}

// Sums of the teams' parts, 32 channels of a model a block: warp k takes the
// teams k, k + 32, .., then their sums are added in order.
template <typename T, int MODE, bool CENTER>
__global__ void __launch_bounds__(1024) finish_kernel(const BwdArgs a) {
    constexpr int N = CENTER ? 2 : 1;
    constexpr int SLOTS = slot_count(MODE, CENTER);
    constexpr int SUMS = MODE == PLAIN ? N : 2 * N;
    __shared__ float sums[SUMS][32][33];
    const int d = a.f.d, c = blockIdx.x * 32 + threadIdx.x;
    const int64_t model = blockIdx.y;
    float v[SUMS] = {};
    if (c < d) {
        const float* p = a.part + model * a.teams * SLOTS * d + c;
#pragma unroll 4
        for (int k = threadIdx.y; k < a.teams; k += 32) {
#pragma unroll
            for (int q = 0; q < SUMS; ++q) {
                const int slot = MODE == SEQUENCE && q >= N ? q + 2 * N : q;
                v[q] += p[((int64_t)k * SLOTS + slot) * d];
            }
        }
    }
#pragma unroll
    for (int q = 0; q < SUMS; ++q) sums[q][threadIdx.y][threadIdx.x] = v[q];
    __syncthreads();
    if (threadIdx.y != 0 || c >= d) return;
#pragma unroll
    for (int q = 0; q < SUMS; ++q) {
        v[q] = 0.f;
        for (int k = 0; k < 32; ++k) v[q] += sums[q][k][threadIdx.x];
    }
    const int64_t at = model * d + c;
    put<T>(a.dw, at, v[0]);
    if constexpr (CENTER) put<T>(a.dwb, at, v[1]);
    if constexpr (MODE != PLAIN) {
        float va = v[N], vb = CENTER ? v[SUMS - 1] : 0.f;
        if constexpr (MODE == MODEL) {
            const float g = at_or<T>(a.f.gate, at, 1.f);
            put<T>(a.dgate, at, fmaf(va, at_or<T>(a.f.pw, at, 1.f), vb * at_or<T>(a.f.pb, at, 0.f)));
            va *= g;
            vb *= g;
        }
        put<T>(a.dpw, at, va);
        if constexpr (CENTER) put<T>(a.dpb, at, vb);
    }
}

// Gate rows whose sequence was split between teams: their partial sums in
// order. Blocks of 256 channels, one gate row each.
template <typename T, bool CENTER>
__global__ void __launch_bounds__(256) finish_gate_kernel(const BwdArgs a) {
    constexpr int N = CENTER ? 2 : 1;
    constexpr int SLOTS = slot_count(SEQUENCE, CENTER);
    const int d = a.f.d, c = blockIdx.y * 256 + threadIdx.x;
    const int64_t g0 = (int64_t)blockIdx.x * a.f.gate_rows, model = g0 / a.model_rows;
    const int64_t r0 = g0 - model * a.model_rows, r1 = r0 + a.f.gate_rows;
    auto team_of = [&](int64_t r) { return ((r + 1) * a.teams - 1) / a.model_rows; };
    const int64_t k0 = team_of(r0), k1 = team_of(r1 - 1);
    if (k0 == k1 || c >= d) return;
    float va = 0.f, vb = 0.f;
    for (int64_t k = k0; k <= k1; ++k) {
        const bool leading = r0 <= a.model_rows * k / a.teams;
        const float* p = a.part + ((model * a.teams + k) * SLOTS + (leading ? N : 2 * N)) * d + c;
        va += p[0];
        if constexpr (CENTER) vb += p[d];
    }
    const int64_t at = model * d + c;
    static_cast<T*>(a.dgate)[(int64_t)blockIdx.x * d + c] =
        from_f<T>(fmaf(va, at_or<T>(a.f.pw, at, 1.f), vb * at_or<T>(a.f.pb, at, 0.f)));
}

template <typename T, int VE, int MODE, bool CENTER>
int bwd_go(const BwdArgs& a, cudaStream_t st) {
    constexpr int V = 8 / VE;
    const TeamShape shape = team_shape(a.f.d);
    const int64_t teams = a.n * a.teams;
    void (*kernel)(BwdArgs) = shape.team == WARP    ? backward_kernel<T, VE, V, MODE, CENTER, WARP>
                              : shape.team == BLOCK ? backward_kernel<T, VE, V, MODE, CENTER, BLOCK>
                                                    : backward_kernel<T, VE, V, MODE, CENTER, PAIR>;
    const size_t smem = (size_t)kStages * 4 * 8 * sizeof(T) * shape.threads;
    if (smem > 40 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess)
            return set_error(WIDEK_ERR_CUDA, "widek_residual_norm_bwd: %zu bytes of shared memory: %s", smem,
                             cudaGetErrorString(e));
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(shape.team == WARP ? (teams + 3) / 4 : shape.team == BLOCK ? teams : 2 * teams));
    cfg.blockDim = dim3(shape.threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute pair;
    pair.id = cudaLaunchAttributeClusterDimension;
    pair.val.clusterDim = {2, 1, 1};
    cfg.attrs = &pair;
    cfg.numAttrs = shape.team == PAIR ? 1 : 0;
    cudaLaunchKernelEx(&cfg, kernel, a);
    int rc = check_launch("widek_residual_norm_bwd");
    if (rc != WIDEK_OK) return rc;
    finish_kernel<T, MODE, CENTER><<<dim3((a.f.d + 31) / 32, a.n), dim3(32, 32), 0, st>>>(a);
    rc = check_launch("widek_residual_norm_bwd (sums)");
    if (MODE != SEQUENCE || !a.dgate || rc != WIDEK_OK) return rc;
    finish_gate_kernel<T, CENTER><<<dim3(a.f.rows / a.f.gate_rows, (a.f.d + 255) / 256), 256, 0, st>>>(a);
    return check_launch("widek_residual_norm_bwd (gates)");
}

template <typename T, int VE, bool CENTER>
int bwd_mode_of(const BwdArgs& a, int mode, cudaStream_t st) {
    switch (mode) {
        case PLAIN: return bwd_go<T, VE, PLAIN, CENTER>(a, st);
        case MODEL: return bwd_go<T, VE, MODEL, CENTER>(a, st);
        case SEQUENCE: return bwd_go<T, VE, SEQUENCE, CENTER>(a, st);
        default: return bwd_go<T, VE, TOKEN, CENTER>(a, st);
    }
}

template <typename T, int VE>
int bwd_center_of(const BwdArgs& a, int mode, cudaStream_t st) {
    return a.f.center ? bwd_mode_of<T, VE, true>(a, mode, st) : bwd_mode_of<T, VE, false>(a, mode, st);
}

}  // namespace

template <typename T>
int BwdLaunch::run() {
    const Args& f = a.f;
    const int ve = vec_elems<T>(f.d, {f.x, f.y, f.w, f.wb, f.pw, f.pb, f.gate, a.dh, a.dz, a.dx, a.dy, a.dgate});
    if constexpr (sizeof(T) == 2)
        if (ve == 8) return bwd_center_of<T, 8>(a, mode, st);
    return ve >= 4 ? bwd_center_of<T, 4>(a, mode, st) : bwd_center_of<T, 1>(a, mode, st);
}
#endif

}  // namespace rnorm
}  // namespace widek
