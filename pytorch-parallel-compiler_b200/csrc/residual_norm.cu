// The residual stream at the border of two blocks, and rows as 8-bit codes.
//
//   u = norm(y; pw, pb) or y,   h = x + scale gate u,   z = norm(h; w, b)
//   norm(v) = (v - c mean(v)) rsqrt(mean((v - c mean(v))^2) + eps) w + b
// with c = 1 (LayerNorm) or 0 (RMS), per model and channel weights, a gate per
// model, sequence or token. z comes out in the rows' type, or as int8 codes with
// one scale a row (scale = max(max|z|, 2^-40) / 127, code = z / scale rounded
// half to even); quantize_rows makes such codes of any rows.
//
// A team (lanes of a warp, or a block) walks over consecutive rows of one model,
// 8 channels a thread: their weights, folded together, stay in registers, the next
// rows are on their way to shared memory meanwhile, and a row is read and written
// once. Statistics are sums over the values in registers (the variance around the
// mean that was taken first), in fp32; z is taken from the unrounded h.
#include "residual_norm.cuh"

#include <algorithm>
#include <atomic>

namespace widek {
namespace rnorm {

int make_args(Args& a, const char* what, const void* x, const void* y, const void* w, const void* wb, const void* pw,
              const void* pb, const void* gate, int64_t n, int64_t rows, int64_t d, int64_t gate_rows, double scale,
              double eps, int center, int dtype) {
    if (n < 0 || rows < 0 || d < 1 || d > kMaxChannels)
        return set_error(WIDEK_ERR_INVALID, "%s: bad sizes n=%lld rows=%lld d=%lld (1 to %d channels)", what,
                         (long long)n, (long long)rows, (long long)d, kMaxChannels);
    if (dtype_size(dtype) == 0) return set_error(WIDEK_ERR_INVALID, "%s: unknown dtype code %d", what, dtype);
    if (n > 0 && rows > 0x7fffffff / n)
        return set_error(WIDEK_ERR_INVALID, "%s: over 2^31 rows", what);
    const bool empty = n == 0 || rows == 0;                    // its tensors may have no storage
    if (empty) gate_rows = gate ? 1 : -1;
    if ((gate != nullptr) != (gate_rows > 0) || (gate && rows > 0 && rows % gate_rows != 0))
        return set_error(WIDEK_ERR_INVALID, "%s: a gate of one row for %lld of %lld", what, (long long)gate_rows,
                         (long long)rows);
    if (!empty && !y && (pw || pb || gate))
        return set_error(WIDEK_ERR_INVALID, "%s: a norm or gate of y, but no y", what);
    if (pb && !pw) return set_error(WIDEK_ERR_INVALID, "%s: a bias of y's norm without its weight", what);
    if (!center && (wb || pb))
        return set_error(WIDEK_ERR_INVALID, "%s: biases belong to LayerNorm (center), not to RMS norms", what);
    if (!empty && (!x || !w)) return set_error(WIDEK_ERR_INVALID, "%s: null pointer", what);
    a = Args{x, y, w, wb, pw, pb, gate, nullptr, nullptr, nullptr, nullptr, n * rows, d, (int)d, center ? 1 : 0,
             gate ? (uint32_t)gate_rows : 0, FastDiv::make(gate ? (uint32_t)gate_rows : 1), (float)scale, (float)eps, n, rows,
             1};
    return WIDEK_OK;
}

namespace {

// Takes the mean out of the row's values (center) and returns 1 / their rms.
template <int VE, int K, int TEAM, bool CENTER>
__device__ __forceinline__ float factor_of(float (&v)[K], Reduce<TEAM, 1>& red, const Seat<TEAM>& at, int nvec,
                                           float inv_d, float eps, float& mean) {
    float s[1];
    mean = 0.f;
    if constexpr (CENTER) {
        s[0] = sum_vec<K>(v);                            // zeros past the end
        red.sum(s);
        mean = s[0] * inv_d;
        shift_vec<K>(v, -mean);
        if (nvec < at.threads * (K / VE)) {              // and again
#pragma unroll
            for (int i = 0; i < K / VE; ++i)
#pragma unroll
                for (int j = 0; j < VE; ++j) v[i * VE + j] = at.t + at.threads * i < nvec ? v[i * VE + j] : 0.f;
        }
    }
    s[0] = dot_vec<K>(v, v);
    red.sum(s);
    return rsqrtf(fmaf(s[0], inv_d, eps));
}

template <typename T, int VE, int K, int TEAM, bool CENTER, bool CODES>
__global__ void __launch_bounds__(TEAM == WARP ? 128 : kBlockThreads, sizeof(T) * VE < 4 ? 1 : TEAM == WARP ? (K > 8 || CENTER ? 4 : 8) : K > 8 || CENTER ? 1 : 2)
    forward_kernel(const Args a, int lanes) {
    __shared__ __align__(16) float slots[2][32];
    extern __shared__ __align__(16) uint8_t ring_bytes[];
    const Seat<TEAM> at(lanes);
    Reduce<TEAM, 1> red(slots, at);
    if (at.team >= a.n * a.teams) return;
    const Walk walk(at.team, a.teams, a.model_rows);
    const int d = a.d, nvec = d / VE;
    const float inv_d = 1.f / (float)d;
    Ring<T, VE, K, 3> ring(ring_bytes, at.t, at.threads, nvec);
    // Gates that change on the way come along with the first of their rows (or of
    // the walk): the rows at which the next one is fetched, and used.
    const bool groups = a.gate && a.gate_rows < a.model_rows;
    int fetch_gate = groups ? walk.first : -1, use_gate = fetch_gate;
    auto next_gate = [&](int row, uint32_t& g) {
        uint32_t in_gate;
        g = a.gate_div.divmod((uint32_t)row, in_gate);
        return row - (int)in_gate + (int)a.gate_rows;
    };
    auto fetch = [&](int stage, int row) {
        if (row < walk.end) {
            ring.fetch(stage, 1, a.y, row, d);
            ring.fetch(stage, 0, a.x, row, d);
            if (row == fetch_gate) {
                uint32_t g;
                fetch_gate = next_gate(row, g);
                ring.fetch(stage, 2, a.gate, (int)g, d);
            }
        }
        ring.commit();
    };
    for (int k = 0; k < ring.AHEAD; ++k) fetch(k, walk.first + k);
    // k = scale gate pw, kb = scale gate pb
    float w[K], wb[K], k[K], kb[K];
    load_weights<T, VE>(a.w, walk.model, d, at.t, at.threads, 1.f, w);
    if constexpr (CENTER) load_weights<T, VE>(a.wb, walk.model, d, at.t, at.threads, 0.f, wb);
    auto weights_of_y = [&](float (&g)[K]) {
        load_weights<T, VE>(a.pw, walk.model, d, at.t, at.threads, 1.f, k);
        mul_vec<K>(k, k, g);
        scale_vec<K>(k, k, a.scale);
        if constexpr (CENTER) {
            load_weights<T, VE>(a.pb, walk.model, d, at.t, at.threads, 0.f, kb);
            mul_vec<K>(kb, kb, g);
            scale_vec<K>(kb, kb, a.scale);
        }
    };
    if (a.y && !groups) {
        float g[K];
        load_weights<T, VE>(a.gate, walk.model, d, at.t, at.threads, 1.f, g);
        weights_of_y(g);
    }
    int stage = 0;
    for (int row = walk.first; row < walk.end; ++row) {
        float v[K], x[K], mu = 0.f, ru = 1.f, mh;
        if constexpr (!ring.REGS) {
            fetch(stage == 0 ? ring.STAGES - 1 : stage - 1, row + ring.STAGES - 1);
            ring.wait();
        }
        if (row == use_gate) {
            uint32_t i;
            use_gate = next_gate(row, i);
            ring.get(stage, 2, v);
            weights_of_y(v);
        }
        ring.get(stage, 0, x);
        if (a.y) {
            ring.get(stage, 1, v);
            if constexpr (ring.REGS) fetch(0, row + 1);
            if (a.pw) {
                ru = factor_of<VE, K, TEAM, CENTER>(v, red, at, nvec, inv_d, a.eps, mu);
                scale_vec<K>(v, v, ru);
            }
            if constexpr (CENTER) add_vec<K>(x, kb);
            fma_vec<K>(v, v, k, x);
            store_row<T, VE>(a.h, row, d, at.t, at.threads, v);
        } else {
            if constexpr (ring.REGS) fetch(0, row + 1);
#pragma unroll
            for (int j = 0; j < K; ++j) v[j] = x[j];
        }
        const float rh = factor_of<VE, K, TEAM, CENTER>(v, red, at, nvec, inv_d, a.eps, mh);
        if (a.stats && at.t == 0) *reinterpret_cast<float4*>(a.stats + 4 * (int64_t)row) = make_float4(mu, ru, mh, rh);
        scale_vec<K>(v, v, rh);
        if constexpr (CENTER) fma_vec<K>(v, v, w, wb);
        else mul_vec<K>(v, v, w);
        if constexpr (CODES) {
            float top = 0.f;
#pragma unroll
            for (int j = 0; j < K; ++j) top = amax2(top, v[j]);     // w and wb are 0 past the end
            const float scale = code_scale(red.amax(top), true);
            if (at.t == 0) a.cscale[row] = scale;
#pragma unroll
            for (int i = 0; i < K / VE; ++i) {
                const int c = at.t + at.threads * i;
                Pack<uint8_t, VE> out;
                codes_i8<VE>(v + i * VE, scale, out.v);
                if (c < nvec) reinterpret_cast<Pack<uint8_t, VE>*>(static_cast<uint8_t*>(a.z) + row * a.ld)[c] = out;
            }
        } else {
            store_row<T, VE>(a.z, row, d, at.t, at.threads, v);
        }
        stage = stage == ring.STAGES - 1 ? 0 : stage + 1;
    }
    ring.finish();
    if constexpr (TEAM == PAIR) sm100::cluster_sync_all();     // the other block's sums are still written to this one
}

struct ForwardLaunch {
    Args a;
    bool codes;
    cudaStream_t st;

    template <typename T, int VE, int K, int TEAM, bool CENTER, bool CODES>
    int go(const TeamShape& shape) {
        void (*kernel)(Args, int) = forward_kernel<T, VE, K, TEAM, CENTER, CODES>;
        const int smem = Ring<T, VE, K, 3>::bytes(shape.threads);
        if (smem > 40 * 1024) {
            cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
            if (e != cudaSuccess)
                return set_error(WIDEK_ERR_CUDA, "widek_residual_norm_fwd: %d bytes of shared memory: %s", smem,
                                 cudaGetErrorString(e));
        }
        // One wave of teams (asked for once a kernel, block and device), a row each at least.
        static std::atomic<int> resident[64][kBlockThreads / 32 + 1];
        const int dev = current_device() & 63;
        int per = resident[dev][shape.threads / 32].load(std::memory_order_relaxed);
        if (per == 0) {
            if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, shape.threads, smem) != cudaSuccess || per < 1)
                per = 1;
            resident[dev][shape.threads / 32].store(per, std::memory_order_relaxed);
        }
        const int64_t wave = (int64_t)sm_count(dev) * per * shape.rows() / (TEAM == PAIR ? 2 : 1);
        a.teams = (int)std::max<int64_t>(1, std::min<int64_t>(wave / a.n, a.model_rows));
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)(TEAM == PAIR ? 2 * a.n * a.teams : (a.n * a.teams + shape.rows() - 1) / shape.rows()));
        cfg.blockDim = dim3(shape.threads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        cudaLaunchAttribute pair;
        pair.id = cudaLaunchAttributeClusterDimension;
        pair.val.clusterDim = {2, 1, 1};
        cfg.attrs = &pair;
        cfg.numAttrs = TEAM == PAIR ? 1 : 0;
        cudaLaunchKernelEx(&cfg, kernel, a, shape.lanes);
        return check_launch("widek_residual_norm_fwd");
    }
    template <typename T, int VE, int K, bool CODES>
    int team() {
        const TeamShape s = team_shape(a.d, K);
        if (s.team == WARP) return a.center ? go<T, VE, K, WARP, true, CODES>(s) : go<T, VE, K, WARP, false, CODES>(s);
        if (s.team == BLOCK) return a.center ? go<T, VE, K, BLOCK, true, CODES>(s) : go<T, VE, K, BLOCK, false, CODES>(s);
        return a.center ? go<T, VE, K, PAIR, true, CODES>(s) : go<T, VE, K, PAIR, false, CODES>(s);
    }
    template <typename T, int VE>
    int pick() {
        if constexpr (VE >= 4) {
            if (a.d > 4096 || (a.d > 256 && a.rows * a.d > (int64_t)sm_count(current_device()) * 16384)) return codes ? team<T, VE, 16, true>() : team<T, VE, 16, false>();
        }
        return codes ? team<T, VE, 8, true>() : team<T, VE, 8, false>();
    }
    template <typename T>
    int run() {
        const int ve = vec_elems<T>(a.d, {a.x, a.y, a.w, a.wb, a.pw, a.pb, a.gate, a.h, codes ? nullptr : a.z});
        if constexpr (sizeof(T) == 2) {
            if (ve == 8) return pick<T, 8>();
            if (ve == 2) return pick<T, 2>();
        }
        return ve == 4 ? pick<T, 4>() : pick<T, 1>();
    }
};

// Codes of rows of any length: 8 values a thread stay in registers; what is past
// them in longer rows is read twice (the second time from L2).
template <typename T, int VE, int V, int TEAM>
__global__ void __launch_bounds__(TEAM == WARP ? 128 : 1024)
    quantize_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes, float* __restrict__ scales, int64_t rows, int d,
                    int64_t ld, int64_t x_ld, int lanes) {
    __shared__ __align__(16) float slots[2][32];
    const Seat<TEAM> at(lanes);
    Reduce<TEAM, 1> red(slots, at);
    const int64_t row = at.team;
    if (row >= rows) return;
    const int nvec = d / VE;
    const T* xr = x + row * x_ld;
    uint8_t* out = codes + row * ld;
    using P = Pack<T, VE>;
    P p[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = at.t + at.threads * i;
        if (c < nvec) p[i] = *reinterpret_cast<const P*>(xr + (int64_t)c * VE);
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (at.t + at.threads * i < nvec) {
#pragma unroll
            for (int j = 0; j < VE; ++j) top = amax2(top, to_f<T>(p[i].v[j]));
        }
    for (int c = at.t + at.threads * V; c < nvec; c += at.threads) {
        const P q = *reinterpret_cast<const P*>(xr + (int64_t)c * VE);
#pragma unroll
        for (int j = 0; j < VE; ++j) top = amax2(top, to_f<T>(q.v[j]));
    }
    const float scale = code_scale(red.amax(top), true);
    if (at.t == 0) scales[row] = scale;
    auto put = [&](const P& q, int c) {
        float v[VE];
        Pack<uint8_t, VE> o;
#pragma unroll
        for (int j = 0; j < VE; ++j) v[j] = to_f<T>(q.v[j]);
        codes_i8<VE>(v, scale, o.v);
        *reinterpret_cast<Pack<uint8_t, VE>*>(out + (int64_t)c * VE) = o;
    };
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (at.t + at.threads * i < nvec) put(p[i], at.t + at.threads * i);
    for (int c = at.t + at.threads * V; c < nvec; c += at.threads)
        put(*reinterpret_cast<const P*>(xr + (int64_t)c * VE), c);
}

struct QuantizeLaunch {
    const void* x;
    void* codes;
    float* scales;
    int64_t rows;
    int d;
    int64_t ld, x_ld;
    cudaStream_t st;

    template <typename T, int VE, int V, int TEAM>
    int go(int threads, int lanes) {
        const int64_t per = TEAM == WARP ? threads / lanes : 1;
        quantize_kernel<T, VE, V, TEAM><<<(unsigned)((rows + per - 1) / per), threads, 0, st>>>(
            static_cast<const T*>(x), static_cast<uint8_t*>(codes), scales, rows, d, ld, x_ld, lanes);
        return check_launch("widek_quantize_rows_fwd");
    }
    template <typename T, int VE>
    int pick() {
        if (d <= 256) {
            const TeamShape s = team_shape(d < 1 ? 1 : d, 8);
            return go<T, VE, 8 / VE, WARP>(s.threads, s.lanes);
        }
        // Few rows: 8 values a thread, many threads. Many: 32 a thread, few reductions.
        if (d <= 8192 && rows * d < (int64_t)sm_count(current_device()) * 16384)
            return go<T, VE, 8 / VE, BLOCK>((d + 255) / 256 * 32, 32);
        if (d <= 1024) return go<T, VE, 32 / VE, WARP>(128, 32);
        return go<T, VE, 32 / VE, BLOCK>(std::min(1024, (d + 1023) / 1024 * 32), 32);
    }
    template <typename T>
    int run() {
        int ve = vec_elems<T>(d, {x});
        while (ve > 1 && x_ld % ve != 0) ve /= 2;
        if constexpr (sizeof(T) == 2) {
            if (ve == 8) return pick<T, 8>();
            if (ve == 2) return pick<T, 2>();
        }
        return ve == 4 ? pick<T, 4>() : pick<T, 1>();
    }
};

int forward(const char* what, Args& a, bool codes, int dtype, void* stream) {
    if (a.rows == 0) return WIDEK_OK;
    if (!a.z || (a.y && !a.h) || (codes && !a.cscale)) return set_error(WIDEK_ERR_INVALID, "%s: null pointer", what);
    return dispatch_dtype(dtype, ForwardLaunch{a, codes, static_cast<cudaStream_t>(stream)});
}

// Rows of codes start at multiples of 16 bytes.
int check_codes(const char* what, const void* codes, int64_t ld, int64_t d) {
    if (ld < d || ld % 16 != 0 || !aligned16(codes))
        return set_error(WIDEK_ERR_INVALID, "%s: rows of codes must lie a multiple of 16 bytes apart (%lld for %lld)", what,
                         (long long)ld, (long long)d);
    return WIDEK_OK;
}

}  // namespace
}  // namespace rnorm
}  // namespace widek

using namespace widek;

extern "C" int widek_residual_norm_fwd(const void* x, const void* y, const void* w, const void* wb, const void* pw,
                                       const void* pb, const void* gate, void* h, void* z, float* stats, int64_t n,
                                       int64_t rows, int64_t d, int64_t gate_rows, double scale, double eps, int center,
                                       int dtype, void* stream) {
    const char* what = "widek_residual_norm_fwd";
    rnorm::Args a;
    int rc = rnorm::make_args(a, what, x, y, w, wb, pw, pb, gate, n, rows, d, gate_rows, scale, eps, center, dtype);
    if (rc != WIDEK_OK) return rc;
    a.h = h;
    a.z = z;
    a.stats = stats;
    if (!aligned16(stats)) return set_error(WIDEK_ERR_INVALID, "%s: statistics off a 16-byte border", what);
    return rnorm::forward(what, a, false, dtype, stream);
}

extern "C" int widek_residual_norm_quantize_fwd(const void* x, const void* y, const void* w, const void* wb,
                                                const void* pw, const void* pb, const void* gate, void* h, void* codes,
                                                float* scales, int64_t ld, int64_t n, int64_t rows, int64_t d,
                                                int64_t gate_rows, double scale, double eps, int center, int dtype,
                                                void* stream) {
    const char* what = "widek_residual_norm_quantize_fwd";
    rnorm::Args a;
    int rc = rnorm::make_args(a, what, x, y, w, wb, pw, pb, gate, n, rows, d, gate_rows, scale, eps, center, dtype);
    if (rc == WIDEK_OK) rc = rnorm::check_codes(what, codes, ld, d);
    if (rc != WIDEK_OK) return rc;
    a.h = h;
    a.z = codes;
    a.cscale = scales;
    a.ld = ld;
    return rnorm::forward(what, a, true, dtype, stream);
}

extern "C" int widek_quantize_rows_fwd(const void* x, void* codes, float* scales, int64_t rows, int64_t d, int64_t x_ld,
                                       int64_t ld, int dtype, void* stream) {
    const char* what = "widek_quantize_rows_fwd";
    if (rows < 0 || d < 0 || rows > 0x7fffffff || d > 0x7fffffff || x_ld < 0)
        return set_error(WIDEK_ERR_INVALID, "%s: bad sizes rows=%lld d=%lld", what, (long long)rows, (long long)d);
    if (dtype_size(dtype) == 0) return set_error(WIDEK_ERR_INVALID, "%s: unknown dtype code %d", what, dtype);
    int rc = rnorm::check_codes(what, codes, ld, d);
    if (rc != WIDEK_OK) return rc;
    if (rows == 0) return WIDEK_OK;
    if (!scales || (d > 0 && (!x || !codes))) return set_error(WIDEK_ERR_INVALID, "%s: null pointer", what);
    return dispatch_dtype(dtype, rnorm::QuantizeLaunch{x, codes, scales, rows, (int)d, ld, x_ld,
                                                       static_cast<cudaStream_t>(stream)});
}
