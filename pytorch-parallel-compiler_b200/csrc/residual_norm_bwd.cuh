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
//
// Bound by memory latency: 33.6 M bf16 values (two RMS norms, a gate a model) take 71
// us (62 at the measured copy rate) and 6 for the sums, LayerNorms before blocks of 16.8
// M f16 values 47 (31). Weights folded together and two values an instruction took the
// first from 106 to 74 us, as many blocks as its 94 registers allow to 71. Without the
// ring in shared memory the loads ahead spill, and do so for 16-bit rows of an odd number
// of channels, which it cannot hold: past 256 channels with gates that change 0.3 to 1.8
// KB a thread. LayerNorms with such gates spill 30 to 110 bytes in vectors too.
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
    auto fetch = [&](int stage, int from, int ahead) {
        if (walk.has(from, ahead)) {
            const int row = from + ahead;
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
    for (int k = 0; k < ring.AHEAD; ++k) fetch(k, walk.first, k);
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
            fetch(stage == 0 ? ring.STAGES - 1 : stage - 1, row, ring.STAGES - 1);
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
            fetch(0, row, 1);
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

// How the blocks of finish_kernel go over the gates that were split between teams
// (GROUPS): by gates, a block for blockDim.x channels as for a model, where a gate has
// many teams; else a block for as many channels as threads, by gates or, where those
// are more, by the places between two teams of a model, of which a gate's first counts.
struct GateBlocks {
    int64_t items;
    int channels;                  // of a block
    bool by_gate, side_by_side;    // teams over blockDim.y
    __host__ __device__ GateBlocks(const BwdArgs& a, int tx, int ty) {
        const int64_t gates = (uint32_t)a.f.rows / a.f.gate_rows, places = a.f.n * (a.f.teams - 1);
        side_by_side = gates * 8 < places;
        by_gate = gates <= places;
        items = by_gate ? gates : places;
        channels = side_by_side ? tx : tx * ty;
    }
};

// Sums of the teams' parts: a block adds up blockDim.x channels of a model (or gate),
// its row k every blockDim.y-th team from k on, then the rows' sums in order.
template <typename T, int MODE, bool CENTER>
__global__ void __launch_bounds__(1024) finish_kernel(const BwdArgs a) {
    constexpr int N = CENTER ? 2 : 1;
    constexpr int SLOTS = slot_count(MODE, CENTER);
    constexpr int SUMS = MODE == PLAIN ? N : 2 * N;
    __shared__ float sums[SUMS][1024];
    const int d = a.f.d, per = (d + blockDim.x - 1) / blockDim.x;
    const int64_t slot = (int64_t)SLOTS * d;
    const bool of_gate = MODE == GROUPS && blockIdx.x >= (uint32_t)(a.f.n * per);
    float v[SUMS] = {};
    int64_t model = blockIdx.x / per, gate = 0;
    int c = (int)(blockIdx.x % per) * blockDim.x + threadIdx.x;
    bool side_by_side = true;
    if (!of_gate) {
        if (c < d) {
            const float* p = a.part + model * a.f.teams * slot + c;
#pragma unroll 8
            for (int k = threadIdx.y; k < a.f.teams; k += blockDim.y) {
#pragma unroll
                for (int q = 0; q < SUMS; ++q) v[q] += p[k * slot + (MODE == GROUPS && q >= N ? q + 2 * N : q) * d];
            }
        }
    } else if constexpr (MODE == GROUPS) {
        const GateBlocks g(a, blockDim.x, blockDim.y);
        const uint32_t block = blockIdx.x - (uint32_t)(a.f.n * per), gper = (d + g.channels - 1) / g.channels;
        side_by_side = g.side_by_side;
        c = (int)(block % gper) * g.channels + (side_by_side ? threadIdx.x : threadIdx.y * blockDim.x + threadIdx.x);
        // One thread finds the gate, its model and teams: the divisions of 64-bit
        // numbers by all of them took most of the kernel's time.
        __shared__ int64_t found[4];
        __shared__ int first_of_team;
        if (threadIdx.x == 0 && threadIdx.y == 0) {
            const int64_t item = block / gper, rows = a.f.model_rows, teams = a.f.teams;
            int64_t m, gt, place = 0;
            if (g.by_gate) {
                gt = item;
                m = gt * a.f.gate_rows / rows;
            } else {
                m = item / (teams - 1);
                place = item - m * (teams - 1) + 1;
                gt = (m * rows + rows * place / teams) / a.f.gate_rows;
            }
            const int64_t r0 = gt * a.f.gate_rows - m * rows;
            // the last team whose first row is not past r: ((r + 1) teams - 1) / rows
            const int64_t k0 = ((r0 + 1) * teams - 1) / rows, k1 = ((r0 + a.f.gate_rows) * teams - 1) / rows;
            found[0] = gt;
            found[1] = m;
            found[2] = k0;
            found[3] = place > 0 && place != k0 + 1 ? k0 : k1;      // k0: nothing to do here
            first_of_team = r0 <= rows * k0 / teams;
        }
        __syncthreads();
        gate = found[0];
        model = found[1];
        const int k0 = (int)found[2], k1 = (int)found[3];
        if (k0 == k1) return;
        if (c < d) {
            // it is its teams' first gate but, unless it starts where that team does, of
            // the one that it starts in
            const float* p = a.part + (model * a.f.teams + k0) * slot + (int64_t)N * d + c;
            const int step = side_by_side ? blockDim.y : 1;
#pragma unroll 4
            for (int k = side_by_side ? threadIdx.y : 0; k <= k1 - k0; k += step) {
                const float* pk = p + k * slot + (k > 0 || first_of_team ? 0 : N * d);
#pragma unroll
                for (int q = 0; q < N; ++q) v[N + q] += pk[q * d];
            }
        }
    }
    if (side_by_side) {
#pragma unroll
        for (int q = 0; q < SUMS; ++q) sums[q][threadIdx.y * blockDim.x + threadIdx.x] = v[q];
        __syncthreads();
        if (threadIdx.y != 0) return;
#pragma unroll
        for (int q = 0; q < SUMS; ++q) {
            v[q] = 0.f;
#pragma unroll 4
            for (int k = 0; k < blockDim.y; ++k) v[q] += sums[q][k * blockDim.x + threadIdx.x];
        }
    }
    if (c >= d) return;
    const int64_t at = model * d + c;
    if constexpr (MODE != PLAIN) {
        float va = v[N] * a.f.scale, vb = CENTER ? v[SUMS - 1] * a.f.scale : 0.f;
        if (of_gate || MODE == MODEL)
            put<T>(a.dgate, of_gate ? gate * d + c : at, fmaf(va, at_or<T>(a.f.pw, at, 1.f), vb * at_or<T>(a.f.pb, at, 0.f)));
        if (of_gate) return;
        if constexpr (MODE == MODEL) {
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
    // (by the kind of team too: how the sums are split may not depend on earlier calls)
    static std::atomic<int> resident[64][3][kBlockThreads / 32 + 1];
    const int dev = current_device() & 63;
    const int per = resident_blocks(resident[dev][shape.team][shape.threads / 32], kernel, shape.threads, smem);
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
    // Blocks of tx channels and up to `most` teams at a time. Device times in us:
    //  - many blocks, or few teams: 32 x 16 (8 models of 1024 channels, 92 teams: 5.7, with
    //    16 x 64 8.8; 2 of 4096, 74 teams: 5.4 and 17);
    //  - few blocks of many teams (short rows, few models): 16 x 64, from where both are
    //    equal (1 x 1024, 100 teams: 5.0, with 32 x 16 5.3; 150: 5.4 and 6.5; 740: 8.4 and 20;
    //    3 x 64, 3157 teams: 21 and 55);
    //  - where they finish gates, of which there may be many, 32 x 8 (144 gates of 131 teams a
    //    model: 11, with 16 teams at a time 18, with 32 51; 32 gates of 74 teams 8.8, 12, 29;
    //    but 24 gates of 276 teams 18, 11, 12), and 32 x 32 from 512 teams on, where each
    //    gate's sum is long (144 gates of 789 teams 17, with 16 25, with 8 47; 6 of 600 7.7,
    //    12, 22). Between 130 and 511 teams few gates would have 32 as well: 9 gates of 450
    //    teams take 17, with 32 6.5.
    const bool gates = MODE == GROUPS && a.dgate && a.f.gate_rows > 1;       // else a gate is one team's
    const bool few = a.f.n * ((a.f.d + 31) / 32) < sm_count(dev);
    const int tx = !gates && few && a.f.teams >= 128 ? 16 : 32, most = gates ? (a.f.teams >= 512 ? 32 : 8) : tx == 16 ? 64 : 16;
    int ty = 1;
    while (ty < most && ty < a.f.teams) ty *= 2;
    int64_t blocks = a.f.n * ((a.f.d + tx - 1) / tx);
    if (gates) {
        const GateBlocks g(a, tx, ty);
        blocks += g.items * ((a.f.d + g.channels - 1) / g.channels);
    }
    finish_kernel<T, MODE, CENTER><<<(unsigned)blocks, dim3(tx, ty), 0, st>>>(a);
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
    if constexpr (sizeof(T) == 2)
        if (ve == 8) return bwd_center_of<T, 8>(a, mode, st);
    if (ve == 2) return bwd_center_of<T, 2>(a, mode, st);
    return ve == 4 ? bwd_center_of<T, 4>(a, mode, st) : bwd_center_of<T, 1>(a, mode, st);
}
#endif

}  // namespace rnorm
}  // namespace widek
