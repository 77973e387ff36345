// Gradients of the residual stream and its norms (the forward's formulas stand
// in residual_norm.cu). With un, hn the normalised rows, ru, rh their factors
// and gz = dz w:
//
//   dx = dh + rh (gz - hn mean(gz hn) - c mean(gz))
//   dw = sum dz hn, db = sum dz over a model's rows
//   dgate = scale sum of dx u over the gate's rows
//   g = scale dx gate;  dpw = sum g un, dpb = sum g
//   dy = ru (g pw - un mean(g pw un) - c mean(g pw)), or g without a norm of y
//
// The walk is the forward's. Sums over rows stay in the registers of the
// channels' threads, go out once a team and are added in a fixed order by a second
// kernel. While a gate row stays the same, A = sum dx un and B = sum dx are all
// that its gradient and those of y's norm need: dgate = scale (pw A + pb B), dpw =
// scale gate A, dpb = scale gate B. Where gates change (GROUPS) that is finished
// whenever the walk leaves a gate's rows: at once when all of them were this
// team's, else through the first or last partial sums of the teams that share it.
#include "residual_norm.cuh"

#include <algorithm>
#include <atomic>

namespace widek {
namespace rnorm {

// PLAIN: no norm or gate of y; MODEL: one gate a model (or none); GROUPS: one for
// each gate_rows rows.
enum Mode : int { PLAIN = 0, MODEL = 1, GROUPS = 2 };

struct BwdArgs {
    Args f;
    const void *dh, *dz;
    void *dx, *dy, *dw, *dwb, *dpw, *dpb, *dgate;
    float* part;                   // [teams][slots][d]
};

// Partial sums of a team: P and Q (dw, db); A and B, or their sums over gates;
// GROUPS: A and B of its first and of its last gate.
__host__ __device__ constexpr int slot_count(int mode, bool center) {
    const int k = center ? 2 : 1;
    return mode == PLAIN ? k : mode == GROUPS ? 4 * k : 2 * k;
}

constexpr int kBwdChannels = 8;    // a thread

// Teams of each model: one wave of `threads` threads an SM, a few rows each. The
// workspace has room for 1024.
int bwd_teams(int64_t n, int64_t rows, int d, int sms, int threads);
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

// This thread's channels of one slot of partial sums (fp32, dense).
template <int VE>
__device__ __forceinline__ void put_part(float* dst, const float (&v)[kBwdChannels], int t, int threads, int nvec) {
#pragma unroll
    for (int i = 0; i < kBwdChannels / VE; ++i) {
        const int c = t + threads * i;
        if (c < nvec) {
#pragma unroll
            for (int j = 0; j < VE; ++j) dst[c * VE + j] = v[i * VE + j];
        }
    }
}

template <typename T, int VE, int MODE, bool CENTER, int TEAM>
__global__ void __launch_bounds__(TEAM == WARP ? 128 : kBlockThreads) backward_kernel(const BwdArgs a, int lanes) {
    constexpr int K = kBwdChannels;
    constexpr int N = CENTER ? 2 : 1;
    constexpr int SLOTS = slot_count(MODE, CENTER);
    constexpr bool YSIDE = MODE != PLAIN;
    __shared__ __align__(16) float slots[2 * N][32];
    extern __shared__ __align__(16) uint8_t ring_bytes[];
    const Seat<TEAM> at(lanes);
    Reduce<TEAM, N> red(slots, at);
    if (at.team >= a.f.n * a.f.teams) return;
    const Walk walk(at.team, a.f.teams, a.f.model_rows);
    const int d = a.f.d, nvec = d / VE;
    const float inv_d = 1.f / (float)d;
    constexpr int TENSORS = MODE == GROUPS ? 5 : 4;
    Ring<T, VE, K, TENSORS> ring(ring_bytes, at.t, at.threads, nvec);
    if (!a.f.y) ring.clear(1);
    if (!a.dh) ring.clear(2);
    if (!a.dz) ring.clear(3);
    auto fetch = [&](int stage, int row) {
        if (row < walk.end) {
            ring.fetch(stage, 0, a.f.x, row, d);
            ring.fetch(stage, 1, a.f.y, row, d);
            ring.fetch(stage, 3, a.dz, row, d);
            ring.fetch(stage, 2, a.dh, row, d);
            if constexpr (MODE == GROUPS) {
                uint32_t in_gate;
                const uint32_t g = a.f.gate_div.divmod((uint32_t)row, in_gate);
                if (in_gate == 0 || row == walk.first) ring.fetch(stage, 4, a.f.gate, (int)g, d);
            }
        }
        ring.commit();
    };
    for (int k = 0; k < ring.AHEAD; ++k) fetch(k, walk.first + k);
    const float4* stats = reinterpret_cast<const float4*>(a.f.stats);
    float4 st = stats[walk.first];

    // k = scale gate pw, kb = scale gate pb of the present gate
    float w[K], k[K], kb[K], gate[K];
    load_weights<T, VE>(a.f.w, walk.model, d, at.t, at.threads, 1.f, w);
    auto weights_of_y = [&]() {
        load_weights<T, VE>(a.f.pw, walk.model, d, at.t, at.threads, 1.f, k);
        mul_vec<K>(k, k, gate);
        scale_vec<K>(k, k, a.f.scale);
        if constexpr (CENTER) {
            load_weights<T, VE>(a.f.pb, walk.model, d, at.t, at.threads, 0.f, kb);
            mul_vec<K>(kb, kb, gate);
            scale_vec<K>(kb, kb, a.f.scale);
        }
    };
    if constexpr (MODE == MODEL) {
        load_weights<T, VE>(a.f.gate, walk.model, d, at.t, at.threads, 1.f, gate);
        weights_of_y();
    }
    float P[K] = {}, Q[K] = {}, A[K] = {}, B[K] = {}, At[K] = {}, Bt[K] = {};
    float* part = a.part + at.team * SLOTS * d;
    const bool post = YSIDE && a.f.pw;
    uint32_t left = 0;                     // rows of the present gate
    int g0 = 0;                        // its first row

    int stage = 0;
    for (int row = walk.first; row < walk.end; ++row) {
        float x[K], y[K], dz[K], dh[K], hn[K], s[N];
        if constexpr (!ring.REGS) {
            fetch(stage == 0 ? ring.STAGES - 1 : stage - 1, row + ring.STAGES - 1);
            ring.wait();
        }
        const float mu = st.x, ru = st.y, mh = st.z, rh = st.w;
        if (row + 1 < walk.end) st = stats[row + 1];
        ring.get(stage, 0, x);
        ring.get(stage, 1, y);
        ring.get(stage, 3, dz);
        if constexpr (MODE == GROUPS) {
            if (left == 0) {
                uint32_t in_gate;
                a.f.gate_div.divmod((uint32_t)row, in_gate);
                left = a.f.gate_rows - in_gate;
                g0 = row - (int)in_gate;
                ring.get(stage, 4, gate);
                weights_of_y();
            }
        }
        if constexpr (ring.REGS) {
            ring.get(stage, 2, dh);
            fetch(0, row + 1);
        }
        // un in place of y, then hn
        if constexpr (YSIDE) {
            if (post) {
                if constexpr (CENTER) shift_vec<K>(y, -mu);
                scale_vec<K>(y, y, ru);
            }
            fma_vec<K>(hn, y, k, x);
            if constexpr (CENTER) add_vec<K>(hn, kb);
        } else {
#pragma unroll
            for (int j = 0; j < K; ++j) hn[j] = fmaf(y[j], a.f.scale, x[j]);
        }
        if constexpr (CENTER) shift_vec<K>(hn, -mh);
        scale_vec<K>(hn, hn, rh);
        fma_vec<K>(P, dz, hn, P);
        if constexpr (CENTER) add_vec<K>(Q, dz);
        mul_vec<K>(dz, dz, w);             // gz
        s[0] = dot_vec<K>(dz, hn);
        if constexpr (CENTER) s[N - 1] = sum_vec<K>(dz);
        red.sum(s);
        if constexpr (!ring.REGS) ring.get(stage, 2, dh);
        // dx in place of dh
        scale_vec<K>(hn, hn, -s[0] * inv_d);
        if constexpr (CENTER) shift_vec<K>(hn, -s[N - 1] * inv_d);
        add_vec<K>(dz, hn);
        {
            float r[K];
#pragma unroll
            for (int j = 0; j < K; ++j) r[j] = rh;
            fma_vec<K>(dh, dz, r, dh);
        }
        if (a.dx) store_row<T, VE>(a.dx, row, d, at.t, at.threads, dh);
        if constexpr (YSIDE) {
            fma_vec<K>(A, dh, y, A);
            if constexpr (CENTER) add_vec<K>(B, dh);
            mul_vec<K>(dz, dh, k);         // the gradient of un, or of y
        } else {
            scale_vec<K>(dz, dh, a.f.scale);
        }
        if (a.dy) {
            if (post) {
                s[0] = dot_vec<K>(dz, y);
                if constexpr (CENTER) s[N - 1] = sum_vec<K>(dz);
                red.sum(s);
                scale_vec<K>(y, y, -s[0] * inv_d);
                if constexpr (CENTER) shift_vec<K>(y, -s[N - 1] * inv_d);
                add_vec<K>(dz, y);
                scale_vec<K>(dz, dz, ru);
            }
            store_row<T, VE>(a.dy, row, d, at.t, at.threads, dz);
        }
        if constexpr (MODE == GROUPS) {
            if (--left == 0 || row + 1 == walk.end) {
                const bool whole = g0 >= walk.first && left == 0;
                if (!whole) {
                    float* dst = part + (g0 <= walk.first ? N : 2 * N) * d;
                    put_part<VE>(dst, A, at.t, at.threads, nvec);
                    if constexpr (CENTER) put_part<VE>(dst + d, B, at.t, at.threads, nvec);
                }
                fma_vec<K>(At, gate, A, At);
                if (whole && a.dgate) {
                    load_weights<T, VE>(a.f.pw, walk.model, d, at.t, at.threads, 1.f, dz);
                    mul_vec<K>(dz, dz, A);
                    if constexpr (CENTER) {
                        load_weights<T, VE>(a.f.pb, walk.model, d, at.t, at.threads, 0.f, y);
                        fma_vec<K>(dz, y, B, dz);
                    }
                    scale_vec<K>(dz, dz, a.f.scale);
                    store_row<T, VE>(a.dgate, (int)a.f.gate_div.div((uint32_t)row), d, at.t, at.threads, dz);
                }
                if constexpr (CENTER) fma_vec<K>(Bt, gate, B, Bt);
#pragma unroll
                for (int j = 0; j < K; ++j) A[j] = B[j] = 0.f;
            }
        }
        stage = stage == ring.STAGES - 1 ? 0 : stage + 1;
    }
    ring.finish();
    put_part<VE>(part, P, at.t, at.threads, nvec);
    if constexpr (CENTER) put_part<VE>(part + d, Q, at.t, at.threads, nvec);
    if constexpr (MODE == GROUPS) {
        put_part<VE>(part + 3 * N * d, At, at.t, at.threads, nvec);
        if constexpr (CENTER) put_part<VE>(part + (3 * N + 1) * d, Bt, at.t, at.threads, nvec);
    } else if constexpr (YSIDE) {
        put_part<VE>(part + N * d, A, at.t, at.threads, nvec);
        if constexpr (CENTER) put_part<VE>(part + (N + 1) * d, B, at.t, at.threads, nvec);
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

// Sums of the teams' parts, 32 (or 8) channels a block: row k of the block takes the
// teams k, k + blockDim.y, .., then the rows' sums are added in order. Blocks past
// the models' (GROUPS) finish the gates whose rows were split between teams.
template <typename T, int MODE, bool CENTER>
__global__ void __launch_bounds__(1024) finish_kernel(const BwdArgs a) {
    constexpr int N = CENTER ? 2 : 1;
    constexpr int SLOTS = slot_count(MODE, CENTER);
    constexpr int SUMS = MODE == PLAIN ? N : 2 * N;
    __shared__ float sums[SUMS][1024];
    const int d = a.f.d, c = blockIdx.y * blockDim.x + threadIdx.x;
    const int64_t slot = (int64_t)SLOTS * d;
    float v[SUMS] = {};
    int64_t model = blockIdx.x;
    const bool of_gate = MODE == GROUPS && model >= a.f.n;
    const int64_t gate = model - a.f.n;
    if (!of_gate) {
        if (c < d) {
            const float* p = a.part + model * a.f.teams * slot + c;
#pragma unroll 4
            for (int k = threadIdx.y; k < a.f.teams; k += blockDim.y) {
#pragma unroll
                for (int q = 0; q < SUMS; ++q) v[q] += p[k * slot + (MODE == GROUPS && q >= N ? q + 2 * N : q) * d];
            }
        }
    } else {
        const int64_t first = gate * a.f.gate_rows;
        model = first / a.f.model_rows;
        const int64_t r0 = first - model * a.f.model_rows, r1 = r0 + a.f.gate_rows;
        // the last team whose first row is not past r
        auto team_of = [&](int64_t r) { return ((r + 1) * a.f.teams - 1) / a.f.model_rows; };
        const int64_t k0 = team_of(r0), k1 = team_of(r1 - 1);
        if (k0 == k1) return;
        if (c < d) {
#pragma unroll 4
            for (int64_t k = k0 + threadIdx.y; k <= k1; k += blockDim.y) {
                const bool leading = r0 <= a.f.model_rows * k / a.f.teams;
                const float* p = a.part + (model * a.f.teams + k) * slot + (leading ? N : 2 * N) * d + c;
#pragma unroll
                for (int q = 0; q < N; ++q) v[N + q] += p[q * d];
            }
        }
    }
#pragma unroll
    for (int q = 0; q < SUMS; ++q) sums[q][threadIdx.y * blockDim.x + threadIdx.x] = v[q];
    __syncthreads();
    if (threadIdx.y != 0 || c >= d) return;
#pragma unroll
    for (int q = 0; q < SUMS; ++q) {
        v[q] = 0.f;
        for (int k = 0; k < blockDim.y; ++k) v[q] += sums[q][k * blockDim.x + threadIdx.x];
    }
    const int64_t at = model * d + c;
    if constexpr (MODE != PLAIN) {
        float va = v[N] * a.f.scale, vb = CENTER ? v[SUMS - 1] * a.f.scale : 0.f;
        if (of_gate || MODE == MODEL) {
            const float dg = fmaf(va, at_or<T>(a.f.pw, at, 1.f), vb * at_or<T>(a.f.pb, at, 0.f));
            put<T>(a.dgate, of_gate ? gate * d + c : at, dg);
            if (of_gate) return;
            const float g = at_or<T>(a.f.gate, at, 1.f);
            va *= g;
            vb *= g;
        }
        put<T>(a.dpw, at, va);
        if constexpr (CENTER) put<T>(a.dpb, at, vb);
    }
    put<T>(a.dw, at, v[0]);
    if constexpr (CENTER) put<T>(a.dwb, at, v[1]);
}

template <typename T, int VE, int MODE, bool CENTER>
int bwd_go(BwdArgs a, cudaStream_t st) {
    const TeamShape shape = team_shape(a.f.d, kBwdChannels);
    void (*kernel)(BwdArgs, int) = shape.team == WARP    ? backward_kernel<T, VE, MODE, CENTER, WARP>
                                   : shape.team == BLOCK ? backward_kernel<T, VE, MODE, CENTER, BLOCK>
                                                         : backward_kernel<T, VE, MODE, CENTER, PAIR>;
    const int smem = Ring<T, VE, kBwdChannels, MODE == GROUPS ? 5 : 4>::bytes(shape.threads);
    if (smem > 40 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess)
            return set_error(WIDEK_ERR_CUDA, "widek_residual_norm_bwd: %d bytes of shared memory: %s", smem,
                             cudaGetErrorString(e));
    }
    static std::atomic<int> resident[64][kBlockThreads / 32 + 1][2];       // asked for once a kernel, block and device
    const int dev = current_device() & 63;
    std::atomic<int>& known = resident[dev][shape.threads / 32][shape.team == PAIR];
    int per = known.load(std::memory_order_relaxed);
    if (per == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, shape.threads, smem) != cudaSuccess || per < 1) per = 1;
        known.store(per, std::memory_order_relaxed);
    }
    a.f.teams = bwd_teams(a.f.n, a.f.model_rows, a.f.d, sm_count(dev), std::min(1024, per * shape.threads));
    const int64_t teams = a.f.n * a.f.teams;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(shape.team == PAIR ? 2 * teams : (teams + shape.rows() - 1) / shape.rows()));
    cfg.blockDim = dim3(shape.threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute pair;
    pair.id = cudaLaunchAttributeClusterDimension;
    pair.val.clusterDim = {2, 1, 1};
    cfg.attrs = &pair;
    cfg.numAttrs = shape.team == PAIR ? 1 : 0;
    cudaLaunchKernelEx(&cfg, kernel, a, shape.lanes);
    int rc = check_launch("widek_residual_norm_bwd");
    if (rc != WIDEK_OK) return rc;
    // short rows: fewer channels a block, to add more teams at a time
    const int tx = a.f.d <= 64 ? 8 : 32;
    int ty = 1;
    while (ty < 1024 / tx && ty < a.f.teams) ty *= 2;
    // gates of more rows than one may be split between teams
    const int64_t gates = MODE == GROUPS && a.dgate && a.f.gate_rows > 1 && a.f.teams > 1 ? a.f.rows / a.f.gate_rows : 0;
    finish_kernel<T, MODE, CENTER>
        <<<dim3((unsigned)(a.f.n + gates), (a.f.d + tx - 1) / tx), dim3(tx, ty), 0, st>>>(a);
    return check_launch("widek_residual_norm_bwd (sums)");
}

template <typename T, int VE, bool CENTER>
int bwd_mode_of(const BwdArgs& a, int mode, cudaStream_t st) {
    if (mode == PLAIN) return bwd_go<T, VE, PLAIN, CENTER>(a, st);
    return mode == MODEL ? bwd_go<T, VE, MODEL, CENTER>(a, st) : bwd_go<T, VE, GROUPS, CENTER>(a, st);
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
    if constexpr (sizeof(T) == 2) {
        if (ve == 8) return bwd_center_of<T, 8>(a, mode, st);
        if (ve == 2) return bwd_center_of<T, 2>(a, mode, st);
    }
    return ve == 4 ? bwd_center_of<T, 4>(a, mode, st) : bwd_center_of<T, 1>(a, mode, st);
}
#endif

}  // namespace rnorm
}  // namespace widek
