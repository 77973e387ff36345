// Attention of one new token of every sequence over a paged key-value cache:
// the argument checks, the choice of how often a sequence is split, and the
// join of its ranges. The kernel is in decode_attention.cuh.
#include "decode_attention.cuh"

#include <algorithm>

namespace widek {
namespace {

constexpr int kJoinWarps = 4;
constexpr int kMostSplits = 512;

// out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s over the groups of a
// sequence's ranges, in their order; one warp per query head. Sequences of one
// group were finished by the attention itself.
__global__ void __launch_bounds__(32 * kJoinWarps) decode_join_kernel(const __grid_constant__ DecodeArgs a) {
    sm100::grid_dep_wait();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * kJoinWarps + (threadIdx.x >> 5), nb = row / a.hq;
    if (row >= (int64_t)a.n * a.b * a.hq) return;
    const DecodeRange rg(a, nb / a.b, nb % a.b);
    if (rg.active <= a.cluster) return;
    const int groups = (rg.active + a.cluster - 1) / a.cluster;
    const float2* ml = a.part_ml + row * a.groups;
    float top = -INFINITY;
    for (int s = lane; s < groups; s += 32) top = fmaxf(top, ml[s].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float ref = top == -INFINITY ? 0.f : top;
    float total = 0.f, acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = 0.f;
    const float* po = a.part_o + row * a.groups * a.d;
#pragma unroll 8
    for (int s = 0; s < groups; ++s) {
        const float2 x = ml[s];
        const float f = ex2(x.x - ref);
        total += f * x.y;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (lane + 32 * j < a.d) acc[j] += f * po[(int64_t)s * a.d + lane + 32 * j];
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (lane + 32 * j < a.d) store_out(a.out, row * a.d + lane + 32 * j, acc[j] * inv, a.dtype);
}

int decode_args(DecodeArgs& a, const char* what, const int64_t* g, const int64_t* cgeom, int64_t window, int fmt) {
    if (!g || !cgeom) return set_error(WIDEK_ERR_INVALID, "%s: null geometry", what);
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
    a.fmt = fmt;
    a.err = device_error_ptr();
    const int nt = decode_nt(a.group, a.d, fmt);
    a.tiles = (a.group + 8 * nt - 1) / (8 * nt);
    // Ranges of a sequence. The host does not know the lengths, only the most
    // tokens that a table row holds. Fewer blocks than the GPU has places: as many ranges as fill them once, of one tile for each warp or
    // more. More blocks: ranges for six rounds, which evens out ragged lengths
    // and the last round, as long as they keep 1024 tokens to start up for.
    const int64_t blocks = (int64_t)a.n * a.b * a.hk * a.tiles;
    const int64_t places = decode_places(a.d, fmt, nt) * (int64_t)sm_count(current_device());
    const double span = (double)cgeom[1] * (double)cgeom[2];
    int64_t tokens = span > 2147418112.0 ? 2147418112 : (int64_t)span;      // the cache's own check refuses such a span
    if (a.window > 0 && a.window < tokens) tokens = a.window;
    a.unit = decode_unit(a.d, fmt);
    int64_t splits = 1;
    if (blocks > 0 && blocks < places) splits = std::min(places / blocks, (tokens + a.unit - 1) / a.unit);
    else if (blocks > 0) splits = std::min((6 * places + blocks - 1) / blocks, tokens / 1024);
    splits = std::max<int64_t>(1, std::min<int64_t>(splits, kMostSplits));
    a.cluster = (int)std::min<int64_t>(splits, kMostCluster);
    a.groups = (int)(splits / a.cluster);
    a.splits = a.groups * a.cluster;
    return WIDEK_OK;
}

int64_t part_rows(const DecodeArgs& a) {
    return a.groups > 1 ? (int64_t)a.n * a.b * a.hq * a.groups : 0;
}

}  // namespace
}  // namespace widek

using namespace widek;

extern "C" int64_t widek_decode_attention_workspace(const int64_t* geom, const int64_t* cgeom, int64_t window,
                                                    int fmt) {
    DecodeArgs a;
    if (decode_args(a, "widek_decode_attention_workspace", geom, cgeom, window, fmt) != WIDEK_OK) return -1;
    return part_rows(a) * (int64_t)(sizeof(float2) + a.d * sizeof(float));
}

extern "C" int widek_decode_attention_fwd(const void* q, const void* kc, const void* vc, const float* ks,
                                          const float* vs, const void* table, const void* lengths, void* out,
                                          const int64_t* geom, const int64_t* cgeom, double scale, int64_t window,
                                          int len64, int fmt, int dtype, void* workspace, int64_t workspace_bytes,
                                          void* stream) {
    const char* what = "widek_decode_attention_fwd";
    DecodeArgs a;
    int rc = decode_args(a, what, geom, cgeom, window, fmt);
    if (rc != WIDEK_OK) return rc;
    if (dtype_size(dtype) == 0) return set_error(WIDEK_ERR_INVALID, "%s: unknown dtype code %d", what, dtype);
    rc = cache_args(a.c, what, const_cast<void*>(kc), const_cast<void*>(vc), const_cast<float*>(ks),
                    const_cast<float*>(vs), table, cgeom, (int64_t)a.n * a.b, a.hk, a.d, fmt, dtype);
    if (rc != WIDEK_OK) return rc;
    if (a.n == 0 || a.b == 0 || a.d == 0) return WIDEK_OK;
    if (!q || !lengths || !out) return set_error(WIDEK_ERR_INVALID, "%s: null pointer", what);
    const int64_t rows = part_rows(a), need = rows * (int64_t)(sizeof(float2) + a.d * sizeof(float));
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 7)))
        return set_error(WIDEK_ERR_INVALID, "%s: workspace of %lld bytes, %lld needed", what,
                         (long long)workspace_bytes, (long long)need);
    a.part_ml = static_cast<float2*>(workspace);
    a.part_o = reinterpret_cast<float*>(a.part_ml + rows);
    a.q = q, a.lengths = lengths, a.out = out, a.len64 = len64, a.dtype = dtype;
    a.scale_log2 = (float)(scale * 1.4426950408889634);
    const int64_t in16 = 16 / (int64_t)dtype_size(dtype);
    a.q_vec = aligned16(q) && a.q_n % in16 == 0 && a.q_b % in16 == 0 && a.q_h % in16 == 0;
    cudaStream_t st = (cudaStream_t)stream;
    if (fmt == WIDEK_I8)
        rc = dtype == WIDEK_F32 ? launch_decode<DK_I8, true>(a, st) : launch_decode<DK_I8, false>(a, st);
    else if (fmt == WIDEK_E4M3)
        rc = dtype == WIDEK_F32 ? launch_decode<DK_E4M3, true>(a, st) : launch_decode<DK_E4M3, false>(a, st);
    else if (fmt == WIDEK_BF16)
        rc = launch_decode<DK_BF16, false>(a, st);
    else if (fmt == WIDEK_F16)
        rc = launch_decode<DK_F16, false>(a, st);
    else
        rc = launch_decode<DK_F32, false>(a, st);
    if (rc != WIDEK_OK || a.groups == 1) return rc;
    // the join's blocks are set up while the attention's last ones run
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(((int64_t)a.n * a.b * a.hq + kJoinWarps - 1) / kJoinWarps));
    cfg.blockDim = dim3(32 * kJoinWarps);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, decode_join_kernel, a);
    return check_launch("widek_decode_attention_fwd (join)");
}
