// Attention of one new token of every sequence over a paged key-value cache.
//
//   z_p = scale q . k_p,  out = sum_p exp(z_p - m) v_p / sum_p exp(z_p - m),
//   m = max z, over the tokens max(0, len - window) <= p < len; zeros where
//   there is none.
//
// One block per query head, one token per warp at a time, the running maximum
// and sum of each warp joined at the end.
#include "paged_cache.cuh"

namespace widek {
namespace {

struct DecodeArgs {
    const void* q;
    const void* lengths;
    void* out;
    int64_t q_n, q_b, q_h, len_n, len_b;
    int n, b, hq, hk, d, group, len64, window;
    float scale_log2;            // scale * log2(e)
    PagedCache c;
    int* err;
};

constexpr int kWarps = 4;

enum CacheIn : int { IN_SAME = 1, IN_I8 = 2, IN_E4M3 = 3 };

template <typename T, int IN>
__device__ __forceinline__ float cache_value(const void* base, int64_t at) {
    if constexpr (IN == IN_I8) return (float)static_cast<const int8_t*>(base)[at];
    if constexpr (IN == IN_E4M3) return value_e4m3(static_cast<const uint8_t*>(base)[at]);
    return to_f<T>(static_cast<const T*>(base)[at]);
}

template <typename T, int IN>
__global__ void __launch_bounds__(32 * kWarps) decode_kernel(const __grid_constant__ DecodeArgs a) {
    constexpr int CH = 8;        // channels of a lane: lane + 32 j, up to 256
    __shared__ float sm[kWarps], sl[kWarps], so[kWarps][256];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int h = blockIdx.x % a.hq;
    const int b = (blockIdx.x / a.hq) % a.b;
    const int64_t i = blockIdx.x / a.hq / a.b;
    const int kh = h / a.group;
    int len = load_index(a.lengths, i * a.len_n + b * a.len_b, a.len64);
    if ((int64_t)len > (int64_t)a.c.cols * a.c.page) {
        len = a.c.cols * a.c.page;
        if (threadIdx.x == 0) raise_device_error(a.err, DEV_ERR_INDEX);
    }
    const int start = a.window > 0 && len > a.window ? len - a.window : 0;
    const T* q = static_cast<const T*>(a.q) + i * a.q_n + b * a.q_b + h * a.q_h;
    float qv[CH], acc[CH];
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        qv[j] = lane + 32 * j < a.d ? to_f<T>(q[lane + 32 * j]) * a.scale_log2 : 0.f;
        acc[j] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int p = start + warp; p < len; p += kWarps) {
        const int slot = a.c.row(i, b, a.hk, kh, p);
        if (slot < 0) {
            if (lane == 0) raise_device_error(a.err, DEV_ERR_INDEX);
            continue;
        }
        const int64_t at = i * a.c.pages * a.hk * a.c.page + slot;
        float z = 0.f;
#pragma unroll
        for (int j = 0; j < CH; ++j)
            if (lane + 32 * j < a.d) z += qv[j] * cache_value<T, IN>(a.c.k, at * a.d + lane + 32 * j);
        z = warp_sum(z);
        float vs = 1.f;
        if constexpr (IN != IN_SAME) {
            z *= a.c.ks[at];
            vs = a.c.vs[at];
        }
        const float top = fmaxf(m, z);
        const float ref = top == -INFINITY ? 0.f : top;
        const float keep = exp2f(m - ref), w = exp2f(z - ref);
        m = top;
        l = l * keep + w;
#pragma unroll
        for (int j = 0; j < CH; ++j)
            if (lane + 32 * j < a.d)
                acc[j] = acc[j] * keep + w * vs * cache_value<T, IN>(a.c.v, at * a.d + lane + 32 * j);
    }
    if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
    for (int j = 0; j < CH; ++j) so[warp][lane + 32 * j] = acc[j];
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w]);
    const float ref = top == -INFINITY ? 0.f : top;
    float total = 0.f, f[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        f[w] = exp2f(sm[w] - ref);
        total += f[w] * sl[w];
    }
    T* out = static_cast<T*>(a.out) + (int64_t)blockIdx.x * a.d;
    for (int c = threadIdx.x; c < a.d; c += 32 * kWarps) {
        float o = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) o += f[w] * so[w][c];
        out[c] = from_f<T>(total == 0.f ? 0.f : o / total);
    }
}

struct DecodeLaunch {
    DecodeArgs a;
    int fmt;
    cudaStream_t st;
    template <typename T>
    int run() {
        const unsigned blocks = (unsigned)a.n * a.b * a.hq;
        if (fmt == WIDEK_I8) decode_kernel<T, IN_I8><<<blocks, 32 * kWarps, 0, st>>>(a);
        else if (fmt == WIDEK_E4M3) decode_kernel<T, IN_E4M3><<<blocks, 32 * kWarps, 0, st>>>(a);
        else decode_kernel<T, IN_SAME><<<blocks, 32 * kWarps, 0, st>>>(a);
        return check_launch("widek_decode_attention_fwd");
    }
};

int decode_args(DecodeArgs& a, const char* what, const int64_t* g, int64_t window) {
    if (!g) return set_error(WIDEK_ERR_INVALID, "%s: null geometry", what);
    for (int i = 0; i < 5; ++i)
        if (g[i] < 0 || g[i] > 0x7fffffff)
            return set_error(WIDEK_ERR_INVALID, "%s: size %d out of range (%lld)", what, i, (long long)g[i]);
    if (g[4] > 256) return set_error(WIDEK_ERR_UNSUPPORTED, "%s: head size %lld above 256", what, (long long)g[4]);
    if (g[3] < 1 || g[2] < 1 || g[2] % g[3] != 0)
        return set_error(WIDEK_ERR_INVALID, "%s: %lld query heads over %lld key heads", what, (long long)g[2],
                         (long long)g[3]);
    if (window < 0) return set_error(WIDEK_ERR_INVALID, "%s: negative window", what);
    if ((double)g[0] * g[1] * g[2] > 2147483647.0)
        return set_error(WIDEK_ERR_INVALID, "%s: over 2^31 query heads", what);
    a = DecodeArgs{};
    a.n = (int)g[0], a.b = (int)g[1], a.hq = (int)g[2], a.hk = (int)g[3], a.d = (int)g[4];
    a.q_n = g[5], a.q_b = g[6], a.q_h = g[7], a.len_n = g[8], a.len_b = g[9];
    a.group = a.hq / a.hk;
    a.window = window > 0x7fffffff ? 0x7fffffff : (int)window;
    a.err = device_error_ptr();
    return WIDEK_OK;
}

}  // namespace
}  // namespace widek

using namespace widek;

extern "C" int64_t widek_decode_attention_workspace(const int64_t* geom, const int64_t* cgeom, int64_t window) {
    DecodeArgs a;
    if (!cgeom || decode_args(a, "widek_decode_attention_workspace", geom, window) != WIDEK_OK) return -1;
    return 0;
}

extern "C" int widek_decode_attention_fwd(const void* q, const void* kc, const void* vc, const float* ks,
                                          const float* vs, const void* table, const void* lengths, void* out,
                                          const int64_t* geom, const int64_t* cgeom, double scale, int64_t window,
                                          int len64, int fmt, int dtype, void* workspace, int64_t workspace_bytes,
                                          void* stream) {
    const char* what = "widek_decode_attention_fwd";
    DecodeArgs a;
    int rc = decode_args(a, what, geom, window);
    if (rc != WIDEK_OK) return rc;
    rc = cache_args(a.c, what, const_cast<void*>(kc), const_cast<void*>(vc), const_cast<float*>(ks),
                    const_cast<float*>(vs), table, cgeom, (int64_t)a.n * a.b, a.hk, a.d, fmt, dtype);
    if (rc != WIDEK_OK) return rc;
    if (a.n == 0 || a.b == 0 || a.d == 0) return WIDEK_OK;
    if (!q || !lengths || !out) return set_error(WIDEK_ERR_INVALID, "%s: null pointer", what);
    a.q = q, a.lengths = lengths, a.out = out, a.len64 = len64;
    a.scale_log2 = (float)(scale * 1.4426950408889634);
    DecodeLaunch L{a, fmt, (cudaStream_t)stream};
    return dispatch_dtype(dtype, L);
}
