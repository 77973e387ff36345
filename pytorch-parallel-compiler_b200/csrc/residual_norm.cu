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
//
// Bound by memory, not far from the instructions' bound: norm + residual of 134 M
// bf16 values (65536 rows of 2048) takes 187 us (floor at the measured copy rate 166);
// one row a block without a walk took 270, 8 channels a thread 244. Into codes 16.8 M
// f16 values 26 us (18), rows of 4096 bf16 values into codes 71 (62). Short rows cost
// their reductions: LayerNorms of 143208 rows of 152 f16 channels 70 us (27). Rows of an
// odd number of 16-bit channels go one channel at a time, through registers: 165188 rows
// of 105 bf16 channels 98 us (21).
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

// Blocks an SM that the registers are cut to: 64 a thread for RMS norms with 8
// channels, else 128 (the odd 16-bit rows, which wait in registers, as many as the block
// leaves them: 128 in blocks of 512, where RMS norms into codes by pairs of blocks spill
// 148 bytes). LayerNorms of 16 channels a thread spill 16 to 64 bytes in their cut.
constexpr int forward_blocks(int team, int k, bool center, bool regs) {
    const bool wide = k > 8 || center;
    return regs ? 1 : team == WARP ? (wide ? 4 : 8) : wide ? 1 : 2;
}

template <typename T, int VE, int K, int TEAM, bool CENTER, bool CODES>
__global__ void __launch_bounds__(TEAM == WARP ? 128 : kBlockThreads, forward_blocks(TEAM, K, CENTER, sizeof(T) * VE < 4))
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
    auto fetch = [&](int stage, int from, int ahead) {
        if (walk.has(from, ahead)) {
            const int row = from + ahead;
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
    for (int k = 0; k < ring.AHEAD; ++k) fetch(k, walk.first, k);
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
            fetch(stage == 0 ? ring.STAGES - 1 : stage - 1, row, ring.STAGES - 1);
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
            if constexpr (ring.REGS) fetch(0, row, 1);
            if (a.pw) {
                ru = factor_of<VE, K, TEAM, CENTER>(v, red, at, nvec, inv_d, a.eps, mu);
                scale_vec<K>(v, v, ru);
            }
            if constexpr (CENTER) add_vec<K>(x, kb);
            fma_vec<K>(v, v, k, x);
            store_row<T, VE>(a.h, row, d, at.t, at.threads, v);
        } else {
            if constexpr (ring.REGS) fetch(0, row, 1);
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
        static std::atomic<int> resident[64][kBlockThreads / 32 + 1];
        const int dev = current_device() & 63;
        const int per = resident_blocks(resident[dev][shape.threads / 32], kernel, shape.threads, smem);
        // one wave of teams, a row each at least
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
        if constexpr (VE < 4)            // wider vectors hold rows past 4096 in one block, 16 channels a thread
            if (s.team == PAIR) return a.center ? go<T, VE, K, PAIR, true, CODES>(s) : go<T, VE, K, PAIR, false, CODES>(s);
        return a.center ? go<T, VE, K, BLOCK, true, CODES>(s) : go<T, VE, K, BLOCK, false, CODES>(s);
    }
    template <typename T, int VE>
    int pick() {
        // 16 channels a thread where there are rows enough: half as many instructions a
        // value go to reductions and addresses (65536 rows of 2048 bf16 channels 244 /
        // 187 us); few rows are spread over more threads. Rows past 4096 would take
        // two blocks with 8.
        if constexpr (VE >= 4) {
            if (a.d > 4096 || a.rows * a.d > (int64_t)sm_count(current_device()) * 16384)
                return codes ? team<T, VE, 16, true>() : team<T, VE, 16, false>();
        }
        return codes ? team<T, VE, 8, true>() : team<T, VE, 8, false>();
    }
    template <typename T>
    int run() {
        const int ve = vec_elems<T>(a.d, {a.x, a.y, a.w, a.wb, a.pw, a.pb, a.gate, a.h, codes ? nullptr : a.z});
        if constexpr (sizeof(T) == 2)
            if (ve == 8) return pick<T, 8>();
        if (ve == 2) return pick<T, 2>();
        return ve == 4 ? pick<T, 4>() : pick<T, 1>();
    }
};

// The largest magnitude of a pack joined to `top`, NaN kept: magnitudes of 16-bit
// types as their bits, two at a time, of fp32 as numbers.
template <typename T, int VE>
struct Top {
    uint32_t bits = 0;
    float number = 0.f;
    __device__ __forceinline__ void take(const Pack<T, VE>& p) {
        if constexpr (sizeof(T) == 2 && VE >= 2) {
#pragma unroll
            for (int j = 0; j < VE / 2; ++j) bits = __vmaxu2(bits, reinterpret_cast<const uint32_t*>(p.v)[j] & 0x7fff7fffu);
        } else {
#pragma unroll
            for (int j = 0; j < VE; ++j) number = amax2(number, to_f<T>(p.v[j]));
        }
    }
    __device__ __forceinline__ float value() const {
        if constexpr (sizeof(T) == 2 && VE >= 2) {
            const uint16_t m = (uint16_t)max(bits & 0xffffu, bits >> 16);
            return to_f<T>(*reinterpret_cast<const T*>(&m));
        } else {
            return number;
        }
    }
};

template <typename T, int VE>
__device__ __forceinline__ void put_codes(uint8_t* row, int c, const Pack<T, VE>& p, float scale) {
    float v[VE];
    Pack<uint8_t, VE> o;
#pragma unroll
    for (int j = 0; j < VE; ++j) v[j] = to_f<T>(p.v[j]);
    codes_i8<VE>(v, scale, o.v);
    reinterpret_cast<Pack<uint8_t, VE>*>(row)[c] = o;
}

// Codes of rows: the walk of the norms, K values a thread.
template <typename T, int VE, int K, int TEAM>
__global__ void __launch_bounds__(TEAM == WARP ? 128 : kBlockThreads, TEAM == WARP ? 8 : 2)
    quantize_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes, float* __restrict__ scales, int64_t rows, int d,
                    int64_t ld, int teams, int lanes) {
    constexpr int V = K / VE;
    __shared__ __align__(16) float slots[2][32];
    extern __shared__ __align__(16) uint8_t ring_bytes[];
    const Seat<TEAM> at(lanes);
    Reduce<TEAM, 1> red(slots, at);
    if (at.team >= teams) return;
    const Walk walk(at.team, teams, rows);
    const int nvec = d / VE;
    Ring<T, VE, K, 1> ring(ring_bytes, at.t, at.threads, nvec);
    auto fetch = [&](int stage, int row, int ahead) {
        if (walk.has(row, ahead)) ring.fetch(stage, 0, x, row + ahead, d);
        ring.commit();
    };
    for (int k = 0; k < ring.AHEAD; ++k) fetch(k, walk.first, k);
    int stage = 0;
    for (int row = walk.first; row < walk.end; ++row) {
        if constexpr (!ring.REGS) {
            fetch(stage == 0 ? ring.STAGES - 1 : stage - 1, row, ring.STAGES - 1);
            ring.wait();
        }
        Pack<T, VE> p[V];
        ring.packs(stage, 0, p);
        if constexpr (ring.REGS) fetch(0, row, 1);
        Top<T, VE> top;
#pragma unroll
        for (int i = 0; i < V; ++i) top.take(p[i]);          // zeros past the end
        const float scale = code_scale(red.amax(top.value()), true);
        if (at.t == 0) scales[row] = scale;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (at.t + at.threads * i < nvec) put_codes<T, VE>(codes + row * ld, at.t + at.threads * i, p[i], scale);
        stage = stage == ring.STAGES - 1 ? 0 : stage + 1;
    }
    ring.finish();
}

// Rows that a block's registers do not hold: read twice, the second time from L2.
template <typename T, int VE>
__global__ void __launch_bounds__(1024)
    quantize_long_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes, float* __restrict__ scales, int d, int64_t ld) {
    __shared__ __align__(16) float slots[2][32];
    const Seat<BLOCK> at(32);
    Reduce<BLOCK, 1> red(slots, at);
    const int64_t row = blockIdx.x;
    const Pack<T, VE>* xr = reinterpret_cast<const Pack<T, VE>*>(x + row * d);
    const uint32_t nvec = d / VE;          // unsigned: a place past the end of a long row may pass 2^31
    Top<T, VE> top;
    for (uint32_t c = at.t; c < nvec; c += at.threads) top.take(xr[c]);
    const float scale = code_scale(red.amax(top.value()), true);
    if (at.t == 0) scales[row] = scale;
    for (uint32_t c = at.t; c < nvec; c += at.threads) put_codes<T, VE>(codes + row * ld, c, xr[c], scale);
}

struct QuantizeLaunch {
    const void* x;
    void* codes;
    float* scales;
    int64_t rows;
    int d;
    int64_t ld;
    cudaStream_t st;

    template <typename T, int VE, int K, int TEAM>
    int go(const TeamShape& shape) {
        auto kernel = quantize_kernel<T, VE, K, TEAM>;
        const int smem = Ring<T, VE, K, 1>::bytes(shape.threads);
        static std::atomic<int> resident[64][kBlockThreads / 32 + 1];
        const int dev = current_device() & 63;
        const int per = resident_blocks(resident[dev][shape.threads / 32], kernel, shape.threads, smem);
        const int64_t teams = std::min<int64_t>((int64_t)sm_count(dev) * per * shape.rows(), rows);
        kernel<<<(unsigned)((teams + shape.rows() - 1) / shape.rows()), shape.threads, smem, st>>>(
            static_cast<const T*>(x), static_cast<uint8_t*>(codes), scales, rows, d, ld, (int)teams, shape.lanes);
        return check_launch("widek_quantize_rows_fwd");
    }
    template <typename T, int VE, int K>
    int team() {
        const TeamShape s = team_shape(d < 1 ? 1 : d, K);
        if constexpr (K <= 16)           // 32 values a thread are for rows past 2048
            if (s.team == WARP) return go<T, VE, K, WARP>(s);
        return go<T, VE, K, BLOCK>(s);
    }
    // Few rows, 8 values a thread on many threads; many, more and fewer reductions, as
    // far as a row still has four warps (bf16, 8 / 16 / 32 a thread: 30000 rows of 512
    // 14.2 / 12.9 / 13.5 us, 68000 of 1024 51 / 42.5 / 44, 8192 of 2048 15.5 / 12.7 /
    // 13.8, 32768 of 4096 108 / 76 / 76; 16384 of 4096 with a cold cache - / 43 / 38).
    template <typename T, int VE>
    int pick() {
        constexpr int MOST = VE == 1 ? 16 : 32;
        if (d > MOST * kBlockThreads) {
            quantize_long_kernel<T, VE><<<(unsigned)rows, 1024, 0, st>>>(static_cast<const T*>(x), static_cast<uint8_t*>(codes),
                                                                     scales, d, ld);
            return check_launch("widek_quantize_rows_fwd");
        }
        if (d <= 8 * kBlockThreads && (d <= 256 || rows * d < (int64_t)sm_count(current_device()) * 16384))
            return team<T, VE, 8>();
        if (d <= 16 * 128) return team<T, VE, 16>();
        return team<T, VE, MOST>();
    }
    template <typename T>
    int run() {
        const int ve = vec_elems<T>(d, {x});
        if constexpr (sizeof(T) == 2)
            if (ve == 8) return pick<T, 8>();
        if (ve == 2) return pick<T, 2>();
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

extern "C" int widek_quantize_rows_fwd(const void* x, void* codes, float* scales, int64_t rows, int64_t d, int64_t ld,
                                       int dtype, void* stream) {
    const char* what = "widek_quantize_rows_fwd";
    if (rows < 0 || d < 0 || rows > 0x7fffffff || d > 0x7fffff00)
        return set_error(WIDEK_ERR_INVALID, "%s: bad sizes rows=%lld d=%lld", what, (long long)rows, (long long)d);
    if (dtype_size(dtype) == 0) return set_error(WIDEK_ERR_INVALID, "%s: unknown dtype code %d", what, dtype);
    int rc = rnorm::check_codes(what, codes, ld, d);
    if (rc != WIDEK_OK) return rc;
    if (rows == 0) return WIDEK_OK;
    if (!scales || (d > 0 && (!x || !codes))) return set_error(WIDEK_ERR_INVALID, "%s: null pointer", what);
    return dispatch_dtype(dtype, rnorm::QuantizeLaunch{x, codes, scales, rows, (int)d, ld,
                                                       static_cast<cudaStream_t>(stream)});
}
