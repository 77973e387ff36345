// The residual stream at the border of two blocks, and rows as 8-bit codes.
//
//   u = norm(y; pw, pb) or y,   h = x + scale gate u,   z = norm(h; w, b)
//   norm(v) = (v - c mean(v)) rsqrt(mean((v - c mean(v))^2) + eps) w + b
// with c = 1 (LayerNorm) or 0 (RMS), per model and channel weights, a gate per
// model, sequence or token. z comes out in the rows' type, or as int8 codes with
// one scale a row (scale = max(max|z|, 2^-40) / 127, code = z / scale rounded
// half to even); quantize_rows makes such codes of any rows.
//
// A row stays in registers from its one read to its one write: a warp, or a
// block, holds it, and the statistics are sums over the values themselves (the
// variance around the mean that was taken first), in fp32. z is taken from the
// unrounded h.
#include "residual_norm.cuh"

#include <initializer_list>

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
             gate ? (uint32_t)gate_rows : 0, FastDiv::make((uint32_t)(rows > 0 ? rows : 1)),
             FastDiv::make(gate ? (uint32_t)gate_rows : 1), (float)scale, (float)eps};
    return WIDEK_OK;
}

namespace {

// Normalises the row's values in place (without weights): mean and factor out.
template <int VE, int V, int TEAM>
__device__ __forceinline__ void normalise(float (&v)[V][VE], Reduce<TEAM, 1>& red, int t, int threads, int nvec,
                                          float inv_d, bool center, float eps, float& mean, float& factor) {
    float s[1];
    mean = 0.f;
    if (center) {
        s[0] = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int j = 0; j < VE; ++j) s[0] += v[i][j];
        red.sum(s);
        mean = s[0] * inv_d;
    }
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const bool in = t + threads * i < nvec;
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            v[i][j] = in ? v[i][j] - mean : 0.f;
            s[0] = fmaf(v[i][j], v[i][j], s[0]);
        }
    }
    red.sum(s);
    factor = rsqrtf(fmaf(s[0], inv_d, eps));
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
        for (int j = 0; j < VE; ++j) v[i][j] *= factor;
}

// One vector of a weight row, or `fill`.
template <typename T, int VE>
__device__ __forceinline__ void weights(const void* base, int64_t row, int d, int c, float fill, float (&out)[VE]) {
    if (base) {
        const Pack<T, VE> p = *reinterpret_cast<const Pack<T, VE>*>(static_cast<const T*>(base) + row * d + c * VE);
#pragma unroll
        for (int j = 0; j < VE; ++j) out[j] = to_f<T>(p.v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < VE; ++j) out[j] = fill;
    }
}

template <typename T, int VE, int V, int TEAM, bool CODES>
__global__ void __launch_bounds__(TEAM == TEAM == WARP ? 128 : 256) forward_kernel(const Args a) {
    __shared__ float slots[2][32];
    const int threads = TEAM == WARP ? 32 : blockDim.x;
    const int t = TEAM == WARP ? threadIdx.x & 31 : threadIdx.x;
    const int64_t row = TEAM == WARP ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.rows) return;
    Reduce<TEAM, 1> red{slots, 0};
    const int nvec = a.d / VE;
    const float inv_d = 1.f / (float)a.d;
    const uint32_t model = a.model_div.div((uint32_t)row);
    Raw<T, VE, V> rx, ry;
    if (a.y) ry.load(static_cast<const T*>(a.y) + row * a.d, t, threads, nvec);
    rx.load(static_cast<const T*>(a.x) + row * a.d, t, threads, nvec);

    float v[V][VE], mu = 0.f, ru = 0.f, mh, rh;
    if (a.y) {
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int j = 0; j < VE; ++j) v[i][j] = t + threads * i < nvec ? ry.get(i, j) : 0.f;
        if (a.pw) normalise<VE, V, TEAM>(v, red, t, threads, nvec, inv_d, a.center, a.eps, mu, ru);
        const uint32_t grow = a.gate ? a.gate_div.div((uint32_t)row) : 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = t + threads * i;
            if (c >= nvec) continue;
            float pw[VE], pb[VE], g[VE];
            weights<T, VE>(a.pw, model, a.d, c, 1.f, pw);
            weights<T, VE>(a.pb, model, a.d, c, 0.f, pb);
            weights<T, VE>(a.gate, grow, a.d, c, 1.f, g);
            Pack<T, VE> out;
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                v[i][j] = fmaf(a.scale * g[j], fmaf(v[i][j], pw[j], pb[j]), rx.get(i, j));
                out.v[j] = from_f<T>(v[i][j]);
            }
            *reinterpret_cast<Pack<T, VE>*>(static_cast<T*>(a.h) + row * a.d + (int64_t)c * VE) = out;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int j = 0; j < VE; ++j) v[i][j] = t + threads * i < nvec ? rx.get(i, j) : 0.f;
    }
    normalise<VE, V, TEAM>(v, red, t, threads, nvec, inv_d, a.center, a.eps, mh, rh);
    if (a.stats && t == 0) *reinterpret_cast<float4*>(a.stats + 4 * row) = make_float4(mu, ru, mh, rh);
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = t + threads * i;
        if (c >= nvec) continue;
        float w[VE], b[VE];
        weights<T, VE>(a.w, model, a.d, c, 1.f, w);
        weights<T, VE>(a.wb, model, a.d, c, 0.f, b);
#pragma unroll
        for (int j = 0; j < VE; ++j) v[i][j] = fmaf(v[i][j], w[j], b[j]);
        if constexpr (CODES) {
#pragma unroll
            for (int j = 0; j < VE; ++j) top = amax2(top, v[i][j]);
        } else {
            Pack<T, VE> out;
#pragma unroll
            for (int j = 0; j < VE; ++j) out.v[j] = from_f<T>(v[i][j]);
            *reinterpret_cast<Pack<T, VE>*>(static_cast<T*>(a.z) + row * a.d + (int64_t)c * VE) = out;
        }
    }
    if constexpr (CODES) {
        const float scale = code_scale(red.amax(top), true);
        if (t == 0) a.cscale[row] = scale;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = t + threads * i;
            if (c >= nvec) continue;
            Pack<uint8_t, VE> out;
            codes_i8<VE>(v[i], scale, out.v);
            *reinterpret_cast<Pack<uint8_t, VE>*>(static_cast<uint8_t*>(a.z) + row * a.ld + c * VE) = out;
        }
    }
}

struct ForwardLaunch {
    Args a;
    bool codes;
    cudaStream_t st;

    template <typename T, int VE, int V>
    int go(int threads) {
        const int64_t blocks = threads == 32 ? (a.rows + 3) / 4 : a.rows;
        if (threads == 32) {
            if (codes) forward_kernel<T, VE, V, WARP, true><<<blocks, 128, 0, st>>>(a);
            else forward_kernel<T, VE, V, WARP, false><<<blocks, 128, 0, st>>>(a);
        } else {
            if (codes) forward_kernel<T, VE, V, BLOCK, true><<<blocks, threads, 0, st>>>(a);
            else forward_kernel<T, VE, V, BLOCK, false><<<blocks, threads, 0, st>>>(a);
        }
        return check_launch("widek_residual_norm_fwd");
    }
    // 32 values a thread keep a row of 1024 in one warp; few rows are spread
    // over more threads instead.
    template <typename T, int VE>
    int pick() {
        const int sms = sm_count(current_device());
        int vt = a.d <= 256 ? 8 : a.d <= 512 ? 16 : 32;
        while (vt > 8 && a.rows * ((a.d + vt - 1) / vt) < (int64_t)sms * 512 && (a.d + vt / 2 - 1) / (vt / 2) <= 256)
            vt /= 2;
        int threads = 32;
        while (threads * vt < a.d) threads *= 2;
        if (vt == 8) return go<T, VE, 8 / VE>(threads);
        if (vt == 16) return go<T, VE, 16 / VE>(threads);
        return go<T, VE, 32 / VE>(threads);
    }
    template <typename T>
    int run() {
        int ve = vec_elems<T>(a.d, {a.x, a.y, a.w, a.wb, a.pw, a.pb, a.gate, a.h, codes ? nullptr : a.z});
        if constexpr (sizeof(T) == 2)
            if (ve == 8) return pick<T, 8>();
        return ve >= 4 ? pick<T, 4>() : pick<T, 1>();
    }
};

// Codes of rows of any length. Rows of up to VT values a thread stay in
// registers; longer ones are read twice (the second time from L2).
template <typename T, int VE, int V, int TEAM>
__global__ void __launch_bounds__(TEAM == TEAM == WARP ? 128 : 1024)
    quantize_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes, float* __restrict__ scales, int64_t rows, int d,
                    int64_t ld, int64_t x_ld) {
    __shared__ float slots[2][32];
    const int threads = TEAM == WARP ? 32 : blockDim.x;
    const int t = TEAM == WARP ? threadIdx.x & 31 : threadIdx.x;
    const int64_t row = TEAM == WARP ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= rows) return;
    Reduce<TEAM, 1> red{slots, 0};
    const int nvec = d / VE;
    const T* xr = x + row * x_ld;
    uint8_t* out = codes + row * ld;
    Raw<T, VE, V> raw;
    raw.load(xr, t, threads, nvec);
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (t + threads * i < nvec) {
#pragma unroll
            for (int j = 0; j < VE; ++j) top = amax2(top, raw.get(i, j));
        }
    for (int c = t + threads * V; c < nvec; c += threads) {
        const Pack<T, VE> p = *reinterpret_cast<const Pack<T, VE>*>(xr + (int64_t)c * VE);
#pragma unroll
        for (int j = 0; j < VE; ++j) top = amax2(top, to_f<T>(p.v[j]));
    }
    const float scale = code_scale(red.amax(top), true);
    if (t == 0) scales[row] = scale;
    auto put = [&](const Pack<T, VE>& p, int c) {
        float v[VE];
        Pack<uint8_t, VE> o;
#pragma unroll
        for (int j = 0; j < VE; ++j) v[j] = to_f<T>(p.v[j]);
        codes_i8<VE>(v, scale, o.v);
        *reinterpret_cast<Pack<uint8_t, VE>*>(out + (int64_t)c * VE) = o;
    };
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (t + threads * i < nvec) put(raw.p[i], t + threads * i);
    for (int c = t + threads * V; c < nvec; c += threads)
        put(*reinterpret_cast<const Pack<T, VE>*>(xr + (int64_t)c * VE), c);
}

struct QuantizeLaunch {
    const void* x;
    void* codes;
    float* scales;
    int64_t rows;
    int d;
    int64_t ld, x_ld;
    cudaStream_t st;

    template <typename T, int VE, int V>
    int go(int threads) {
        const T* p = static_cast<const T*>(x);
        uint8_t* c = static_cast<uint8_t*>(codes);
        if (threads == 32)
            quantize_kernel<T, VE, V, WARP><<<(rows + 3) / 4, 128, 0, st>>>(p, c, scales, rows, d, ld, x_ld);
        else
            quantize_kernel<T, VE, V, BLOCK><<<rows, threads, 0, st>>>(p, c, scales, rows, d, ld, x_ld);
        return check_launch("widek_quantize_rows_fwd");
    }
    template <typename T, int VE>
    int pick() {
        const int sms = sm_count(current_device());
        int vt = d <= 256 ? 8 : d <= 512 ? 16 : 32;
        while (vt > 8 && rows * ((d + vt - 1) / vt) < (int64_t)sms * 512 && (d + vt / 2 - 1) / (vt / 2) <= 512)
            vt /= 2;
        int threads = 32;
        while (threads * vt < d && threads < 1024) threads *= 2;
        if (vt == 8) return go<T, VE, 8 / VE>(threads);
        if (vt == 16) return go<T, VE, 16 / VE>(threads);
        return go<T, VE, 32 / VE>(threads);
    }
    template <typename T>
    int run() {
        int ve = vec_elems<T>(d, {x});
        while (ve > 1 && x_ld % ve != 0) ve = ve == 8 ? 4 : 1;
        if constexpr (sizeof(T) == 2)
            if (ve == 8) return pick<T, 8>();
        return ve >= 4 ? pick<T, 4>() : pick<T, 1>();
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
