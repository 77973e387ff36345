// Attention of one new token of every sequence over a paged key-value cache:
// the argument checks, the choice of how often a sequence is split, and the
// join of its ranges. The kernel is in decode_attention.cuh.
#include "decode_attention.cuh"

#include <algorithm>

namespace widek {
namespace {

constexpr int kJoinThreads = 256;
constexpr int kMostBlocks = 1024;
constexpr int kWideThreads = kMostBlocks;       // one for each block's maximum and sum
// Sequences whose steps every block adds up to find its place in line (32 for
// each thread).
constexpr int kMostInLine = 4096;

// out = sum_c 2^(m_c - m) o_c / sum_c 2^(m_c - m) l_c over the blocks c that a
// segment lies in, in a fixed order. WIDE: a block for 32 channels of a query
// head, its 32 warps taking every 32nd c, with the first outputs on their way
// while the factors are found; else a warp for each head. Segments that lie in
// one block were finished by the attention itself.
template <bool WIDE>
__global__ void __launch_bounds__(WIDE ? kWideThreads : kJoinThreads)
    decode_join_kernel(const __grid_constant__ DecodeArgs a) {
    constexpr int kWarps = (WIDE ? kWideThreads : kJoinThreads) / 32;
    __shared__ float factor[WIDE ? kMostBlocks : 1];
    __shared__ float red[WIDE ? kWarps : 1][33];
    __shared__ float2 red_ml[WIDE ? kWarps : 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t last = (int64_t)a.n * a.b * a.hq - 1;
    const int64_t row = WIDE ? blockIdx.x : min((int64_t)blockIdx.x * kWarps + warp, last);
    // the segment's place in line, while the attention still runs
    const int nb = (int)(row / a.hq), h = (int)(row - (int64_t)nb * a.hq), in_group = h % a.group;
    const int sequences = a.n * a.b, per_seq = a.hk * a.tiles;
    const int hp = h / a.group * a.tiles + in_group / (8 * a.nt);
    long long before = 0, all = 0;
    for (int s = lane; s < sequences; s += 32) {
        const int n = DecodeRange(a, s).steps(a.step);
        all += n;
        if (s < nb) before += n;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        all += __shfl_xor_sync(0xffffffffu, all, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    const long long per = (all * per_seq + a.blocks - 1) / a.blocks;
    const int n = DecodeRange(a, nb).steps(a.step);
    const long long f0 = before * per_seq + (long long)hp * n;
    const int c0 = (int)(f0 / per), c1 = (int)((f0 + n - 1) / per);
    sm100::grid_dep_wait();
    if (c0 == c1 || (!WIDE && (int64_t)blockIdx.x * kWarps + warp > last)) return;
    // a block's part 0 is the segment it starts in
    const int late = f0 > c0 * per ? 1 : 0;
    auto place = [&](int c) {
        return ((int64_t)c * 2 + (c == c0 ? late : 0)) * 8 * a.nt + in_group % (8 * a.nt);
    };
    float top = -INFINITY, total = 0.f;
    if constexpr (WIDE) {
        constexpr int kAhead = 8;
        const int ch = blockIdx.y * 32 + lane, count = c1 - c0 + 1;
        const bool mine = (int)threadIdx.x < count;
        const float2 x = mine ? a.part_ml[place(c0 + threadIdx.x)] : make_float2(-INFINITY, 0.f);
        float ahead[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int c = warp + kWarps * i;
            ahead[i] = c < count && ch < a.d ? a.part_o[place(c0 + c) * a.d + ch] : 0.f;
        }
        top = x.x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (lane == 0) red_ml[warp].x = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, red_ml[w].x);
        const float f = mine ? ex2(x.x - (top == -INFINITY ? 0.f : top)) : 0.f;
        factor[threadIdx.x] = f;
        total = warp_sum(f * x.y);
        if (lane == 0) red_ml[warp].y = total;
        __syncthreads();
        float o = 0.f;
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (warp + kWarps * i < count) o += factor[warp + kWarps * i] * ahead[i];
        if (ch < a.d) {
#pragma unroll 8
            for (int c = warp + kWarps * kAhead; c < count; c += kWarps) o += factor[c] * a.part_o[place(c0 + c) * a.d + ch];
        }
        red[warp][lane] = o;
        __syncthreads();
        if (warp == 0 && ch < a.d) {
            o = total = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) o += red[w][lane], total += red_ml[w].y;
            store_out(a.out, row * a.d + ch, total == 0.f ? 0.f : o / total, a.dtype);
        }
    } else {
        for (int c = c0 + lane; c <= c1; c += 32) top = fmaxf(top, a.part_ml[place(c)].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float ref = top == -INFINITY ? 0.f : top;
        float acc[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = 0.f;
#pragma unroll 4
        for (int c = c0; c <= c1; ++c) {
            const int64_t at = place(c);
            const float2 x = a.part_ml[at];
            const float f = ex2(x.x - ref);
            total += f * x.y;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (lane + 32 * j < a.d) acc[j] += f * a.part_o[at * a.d + lane + 32 * j];
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (lane + 32 * j < a.d) store_out(a.out, row * a.d + lane + 32 * j, acc[j] * inv, a.dtype);
    }
}

int decode_args(DecodeArgs& a, const char* what, const int64_t* g, const int64_t* cgeom, int64_t window, int fmt) {
    if (!g || !cgeom) return set_error(WIDEK_ERR_INVALID, "%s: null geometry", what);
    if (cache_fmt_size(fmt) == 0) return set_error(WIDEK_ERR_INVALID, "%s: unknown cache format %d", what, fmt);
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
    a.nt = decode_nt(a.group, a.d, fmt);
    a.tiles = (a.group + 8 * a.nt - 1) / (8 * a.nt);
    a.step = decode_step(a.d, fmt);
    // As many blocks as the GPU holds, or as there can be steps: the host does
    // not know the lengths, only the most tokens that a table row holds.
    const double span = (double)cgeom[1] * (double)cgeom[2];
    int64_t tokens = span > 2130706432.0 ? 2130706432 : (int64_t)span;      // the cache's check refuses larger ones
    if (a.window > 0 && a.window < tokens) tokens = a.window;
    const int64_t segments = (int64_t)a.n * a.b * a.hk * a.tiles;
    const int64_t steps = std::max<int64_t>(1, (tokens + a.step - 1) / a.step);
    const int64_t places =
        std::min<int64_t>(decode_places(a.d, fmt, a.nt) * sm_count(current_device()), kMostBlocks);
    a.blocks = (int)(segments < places && segments * steps < places ? std::max<int64_t>(segments * steps, 1) : places);
    // nothing to divide when every segment is one step, or too much to add up
    a.in_turn = steps == 1 || (int64_t)a.n * a.b > kMostInLine;
    return WIDEK_OK;
}

int64_t part_rows(const DecodeArgs& a) { return a.in_turn ? 0 : (int64_t)a.blocks * 2 * 8 * a.nt; }

// Totals of chains, where the table has room for segments of more than one.
int64_t done_floats(const DecodeArgs& a, const int64_t* cgeom) {
    const int dp = a.d <= 64 ? 64 : (a.d <= 128 ? 128 : 256);
    const bool more = (double)cgeom[1] * (double)cgeom[2] > (double)kChainTokens * kDecodeWarps;
    return a.fmt != WIDEK_F32 && more ? (int64_t)a.blocks * a.nt * (dp / 4 + 2) * 32 * kDecodeWarps : 0;
}

int64_t workspace_bytes_of(const DecodeArgs& a, const int64_t* cgeom) {
    return part_rows(a) * (int64_t)(sizeof(float2) + a.d * sizeof(float)) +
           done_floats(a, cgeom) * (int64_t)sizeof(float);
}

}  // namespace
}  // namespace widek

using namespace widek;

extern "C" int64_t widek_decode_attention_workspace(const int64_t* geom, const int64_t* cgeom, int64_t window,
                                                    int fmt) {
    DecodeArgs a;
    if (decode_args(a, "widek_decode_attention_workspace", geom, cgeom, window, fmt) != WIDEK_OK) return -1;
    return workspace_bytes_of(a, cgeom);
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
    // their kernels hold more and leave room for two blocks, not three (a third
    // of the line would come in a second wave)
    if (dtype == WIDEK_F32 && cache_fmt_8bit(fmt)) a.blocks = std::min(a.blocks, 2 * sm_count(current_device()));
    rc = cache_args(a.c, what, const_cast<void*>(kc), const_cast<void*>(vc), const_cast<float*>(ks),
                    const_cast<float*>(vs), table, cgeom, (int64_t)a.n * a.b, a.hk, a.d, fmt, dtype);
    if (rc != WIDEK_OK) return rc;
    if (a.n == 0 || a.b == 0 || a.d == 0) return WIDEK_OK;
    if (!q || !lengths || !out) return set_error(WIDEK_ERR_INVALID, "%s: null pointer", what);
    const int64_t rows = part_rows(a), need = workspace_bytes_of(a, cgeom);
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 7)))
        return set_error(WIDEK_ERR_INVALID, "%s: workspace of %lld bytes, %lld needed", what,
                         (long long)workspace_bytes, (long long)need);
    a.part_ml = static_cast<float2*>(workspace);
    a.part_o = reinterpret_cast<float*>(a.part_ml + rows);
    a.done = a.part_o + rows * a.d;
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
    if (rc != WIDEK_OK || a.in_turn) return rc;
    // The join is set up while the attention runs. A segment lies in about
    // blocks / segments of them: with more than 8 its heads are spread out.
    const int64_t heads = (int64_t)a.n * a.b * a.hq;
    const bool wide = a.blocks > 8 * (int64_t)a.n * a.b * a.hk * a.tiles;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = wide ? dim3((unsigned)heads, (unsigned)((a.d + 31) / 32))
                       : dim3((unsigned)((heads + kJoinThreads / 32 - 1) / (kJoinThreads / 32)));
    cfg.blockDim = dim3(wide ? kWideThreads : kJoinThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (wide) cudaLaunchKernelEx(&cfg, decode_join_kernel<true>, a);
    else cudaLaunchKernelEx(&cfg, decode_join_kernel<false>, a);
    return check_launch("widek_decode_attention_fwd (join)");
}
