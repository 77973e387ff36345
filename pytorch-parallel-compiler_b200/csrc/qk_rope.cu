// Row kernels of decoder attention: RMS norm of every query and key head with
// the position rotation, the paged cache's write and read, and the gradients
// of the norm + rotation.
//
// A row is one head of one token: D channels, D <= 256.
//   norm      u = x r w, r = 1 / sqrt(mean(x^2) + eps), w per (model, channel)
//   rotation  each pair (a, b) of the first R channels, turned by the angle of
//             its position: y_a = u_a cos - u_b sin, y_b = u_b cos + u_a sin.
//             Pairs are (i, i + R/2), or (2i, 2i + 1) when interleaved.
//   gradient  du = dy turned back, dw = sum over rows of du x r, g = du w,
//             dx = r (g - x r^2 mean(g x))
// A row whose position is negative is padding: zeros out, nothing written,
// zero gradient. A position outside the table records an index error and does
// the same; one outside the cache records it and writes nothing.
//
// Mapping: a power of two of lanes share a row and each lane holds both
// members of its pairs (vector A at u VEC and vector B at u VEC + R/2; one
// after the other for the interleaved order, the channels past R and rows
// without a rotation), so that the rotation needs no exchange between lanes
// and the norm one reduction. Every channel is read once and written once,
// in 16-byte vectors where sizes and strides allow it.
//
// Bound by memory (2 D bytes in and out per row of a 16-bit type), not far from
// the instructions' bound: at the copy rate there is time for about 22 of them
// a channel, and norm + rotation takes 15. So four heads of a token share its
// angles, weights and addresses, the weights are folded into the angles'
// coefficients, fp32 arithmetic runs two to an instruction, and codes and values
// change form by byte permutes.
// Measured (B200, floor at the measured copy rate): norm + rotation of 168 M
// bf16 values 137 us (103), its backward over 84 M 113 us (77), int8 write of
// 268 M 183 us (124), read 127 us (125).
#include "paged_cache.cuh"

#include <initializer_list>
#include <type_traits>

namespace widek {

int cache_args(PagedCache& c, const char* what, void* k, void* v, float* ks, float* vs, const void* table,
               const int64_t* cgeom, int64_t calls, int64_t hk, int64_t d, int fmt, int dtype) {
    if (!cgeom) return set_error(WIDEK_ERR_INVALID, "%s: null cache geometry", what);
    const int64_t pages = cgeom[0], page = cgeom[1], cols = cgeom[2];
    if (pages < 0 || page < 1 || cols < 0)
        return set_error(WIDEK_ERR_INVALID, "%s: bad cache sizes pages=%lld page=%lld columns=%lld", what,
                         (long long)pages, (long long)page, (long long)cols);
    if (!cache_fmt_8bit(fmt) && fmt != dtype)
        return set_error(WIDEK_ERR_INVALID, "%s: the cache's type %d is neither 8-bit nor the tensors' type %d", what,
                         fmt, dtype);
    if (page > 0x7fffffff || cols > 0x7fffffff || (hk > 0 && pages > 0x7fffffff / hk / page))
        return set_error(WIDEK_ERR_INVALID, "%s: one model's pool holds over 2^31 rows (pages=%lld, heads=%lld, "
                         "page=%lld)", what, (long long)pages, (long long)hk, (long long)page);
    if (cols * page > 0x7f000000)       // positions and the tiles past them stay 32-bit numbers
        return set_error(WIDEK_ERR_INVALID, "%s: a sequence spans about 2^31 tokens or more", what);
    if (calls > 0 && hk > 0 && d > 0 && pages > 0 && cols > 0 && (!k || !v || !table || (cache_fmt_8bit(fmt) && (!ks || !vs))))
        return set_error(WIDEK_ERR_INVALID, "%s: null cache pointer", what);
    c = PagedCache{k, v, ks, vs, static_cast<const int*>(table), cgeom[3], cgeom[4], (int)pages, (int)page, (int)cols,
                   FastDiv::make((uint32_t)page)};
    return WIDEK_OK;
}

namespace {

constexpr int kThreads = 128;

struct Strides {
    int64_t n, b, t, h;
};

struct RowArgs {
    const void *q, *k, *v, *qw, *kw;
    const float *cs, *sn;
    const void* pos;
    void *yq, *yk, *yv;
    Strides sq, sk, sv;
    int64_t pos_n, pos_b, pos_t;
    int pos64, n, b, t, hq, hk, d, rot, table_rows, inter, lanes_log2;
    uint32_t units;               // a unit: HPT heads of one kind of a token, one group of lanes
    int parts_q, parts_k;         // units of a token's q heads and k heads (and as many of v)
    float eps;
    FastDiv parts, tdiv, bdiv;
    PagedCache c;
    int* err;
};

// VEC consecutive elements of T as one load / store.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Pack<T, VEC>& r, float* out) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = to_f<T>(r.v[i]);
}

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float* out) {
    const Pack<T, VEC> r = *reinterpret_cast<const Pack<T, VEC>*>(p);
    unpack<T, VEC>(r, out);
}

// Loads that belong together are issued without branches around them (places
// outside a row read its first vector and are zeroed later): a branch around
// each kept them from being in flight at the same time.
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) {
    return *reinterpret_cast<const Pack<T, VEC>*>(p);
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* in) {
    Pack<T, VEC> r;
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.v[i] = from_f<T>(in[i]);
    *reinterpret_cast<Pack<T, VEC>*>(p) = r;
}

// VEC floats of a cos / sin row (16-byte loads at most).
template <int VEC>
__device__ __forceinline__ void load_table(const float* p, float* out) {
    constexpr int W = VEC < 4 ? VEC : 4;
#pragma unroll
    for (int i = 0; i < VEC; i += W) load_vec<float, W>(p + i, out + i);
}

// The lanes of this thread's row. A warp's rows may be of different kinds, so
// each row reduces among its own lanes, which always arrive together.
__device__ __forceinline__ unsigned group_mask(int lanes) {
    return lanes == 32 ? 0xffffffffu : ((1u << lanes) - 1u) << (threadIdx.x & 31 & ~(lanes - 1));
}

// Channels of unit u (first elements of its vectors A and B). Units below
// `turned` hold pairs of the rotation.
template <int VEC, bool INTER>
__device__ __forceinline__ void unit_channels(int u, int turned, int rot, int& a, int& b) {
    if (!INTER && u < turned) {
        a = u * VEC;
        b = a + rot / 2;
    } else {
        a = 2 * u * VEC;
        b = a + VEC;
    }
}

// The rotation of one unit as y_a = x_a ca + p_a sa, y_b = x_b cb + p_b sb with
// each channel's partner p: the coefficients, the norm's weights folded in
// (w_p belongs to the partner), from the angles' cosines and sines. SIGN -1
// turns back; then the weights apply after the turn and are left out.
template <int VEC, bool INTER>
struct Turn {
    float ca[VEC], sa[VEC], cb[VEC], sb[VEC];
    __device__ __forceinline__ void set(const float* co, const float* si, const float* wa, const float* wb) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if constexpr (!INTER || VEC == 1) {
                ca[j] = co[j] * wa[j];
                sa[j] = -si[j] * wb[j];
                cb[j] = co[j] * wb[j];
                sb[j] = si[j] * wa[j];
            } else {
                const int p = j / 2, q = VEC / 2 + j / 2;
                ca[j] = co[p] * wa[j];
                sa[j] = (j & 1 ? si[p] : -si[p]) * wa[j ^ 1];
                cb[j] = co[q] * wb[j];
                sb[j] = (j & 1 ? si[q] : -si[q]) * wb[j ^ 1];
            }
        }
    }
    // Channels that do not turn.
    __device__ __forceinline__ void keep(const float* wa, const float* wb) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) ca[j] = wa[j], cb[j] = wb[j], sa[j] = sb[j] = 0.f;
    }
    __device__ __forceinline__ void apply(float* a, float* b) const {
        float pa[VEC], pb[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            pa[j] = !INTER || VEC == 1 ? b[j] : a[VEC == 1 ? 0 : j ^ 1];
            pb[j] = !INTER || VEC == 1 ? a[j] : b[VEC == 1 ? 0 : j ^ 1];
        }
        mul_vec<VEC>(a, a, ca);
        mul_vec<VEC>(b, b, cb);
        fma_vec<VEC>(a, pa, sa, a);
        fma_vec<VEC>(b, pb, sb, b);
    }
};

enum RowOut : int { OUT_DENSE = 0, OUT_SAME = 1, OUT_I8 = 2, OUT_E4M3 = 3 };

// One vector of a cache row in the cache's format.
template <typename T, int VEC, int OUT>
__device__ __forceinline__ void store_code(void* base, int64_t at, const float* x, float scale, bool live) {
    if constexpr (OUT == OUT_I8 || OUT == OUT_E4M3) {
        Pack<uint8_t, VEC> p;
        if constexpr (OUT == OUT_I8) codes_i8<VEC>(x, scale, p.v);
        else codes_e4m3<VEC>(x, scale, p.v);
        if (live) *reinterpret_cast<Pack<uint8_t, VEC>*>(static_cast<uint8_t*>(base) + at) = p;
    } else {
        if (live) store_vec<T, VEC>(static_cast<T*>(base) + at, x);
    }
}

// Rows in: q heads (normed, rotated, dense out), k heads (the same, dense out
// or into the cache), v heads (into the cache). ROPE false: k and v heads go
// to the cache as they are. A group of lanes takes HPT heads of one token and
// kind at once: its loads are in flight together, and the angles and weights
// are read once (one row at a time reached 3.8 of 6.5 TB/s).
template <typename T, int VEC, int UPL, int HPT, int OUT, bool ROPE, bool INTER>
__global__ void __launch_bounds__(kThreads) rows_kernel(const __grid_constant__ RowArgs a) {
    const int lanes = 1 << a.lanes_log2;
    const int lane = threadIdx.x & (lanes - 1);
    const unsigned mask = group_mask(lanes);
    uint32_t unit = blockIdx.x * (kThreads >> a.lanes_log2) + (threadIdx.x >> a.lanes_log2);
    if (unit >= a.units) return;
    uint32_t part, t, b;
    const uint32_t tok = a.parts.divmod(unit, part);
    const uint32_t nb = a.tdiv.divmod(tok, t);
    const uint32_t i = a.bdiv.divmod(nb, b);
    const bool is_q = (int)part < a.parts_q;
    const bool is_v = (int)part >= a.parts_q + a.parts_k;
    const int h0 = HPT * (is_q ? (int)part : (is_v ? (int)part - a.parts_q - a.parts_k : (int)part - a.parts_q));
    const int nh = min(HPT, (is_q ? a.hq : a.hk) - h0);
    const Strides st = is_q ? a.sq : (is_v ? a.sv : a.sk);
    const T* src = static_cast<const T*>(is_q ? a.q : (is_v ? a.v : a.k)) + i * st.n + b * st.b + t * st.t + h0 * st.h;
    const int pos = load_index(a.pos, i * a.pos_n + b * a.pos_b + t * a.pos_t, a.pos64);

    const int turned = ROPE ? a.rot / 2 / VEC : 0;
    int ca[UPL], cb[UPL];
    Pack<T, VEC> ra[HPT][UPL], rb[HPT][UPL];
#pragma unroll
    for (int s = 0; s < UPL; ++s) unit_channels<VEC, INTER>(lane + s * lanes, turned, a.rot, ca[s], cb[s]);
#pragma unroll
    for (int r = 0; r < HPT; ++r)
#pragma unroll
        for (int s = 0; s < UPL; ++s) {
            const T* row = src + (r < nh ? r : 0) * (int64_t)(int)st.h;
            ra[r][s] = load_pack<T, VEC>(row + (ca[s] < a.d ? ca[s] : 0));
            rb[r][s] = load_pack<T, VEC>(row + (cb[s] < a.d ? cb[s] : 0));
        }

    bool keep = pos >= 0;
    const bool rope = ROPE && !is_v;
    if (ROPE && pos >= a.table_rows) {            // for the values as well: a slot gets both sides or neither
        keep = false;
        if (lane == 0) raise_device_error(a.err, DEV_ERR_INDEX);
    }
    Turn<VEC, INTER> turn[UPL];
    float norm[HPT];
    if (ROPE && rope) {
        const T* w = static_cast<const T*>(is_q ? a.qw : a.kw) + (int64_t)i * a.d;
        const int64_t trow = (int64_t)(keep ? pos : 0) * (a.rot / 2);
#pragma unroll
        for (int s = 0; s < UPL; ++s) {
            const int u = lane + s * lanes;
            float wa[VEC], wb[VEC];
            load_vec<T, VEC>(w + (ca[s] < a.d ? ca[s] : 0), wa);
            load_vec<T, VEC>(w + (cb[s] < a.d ? cb[s] : 0), wb);
            if (u < turned && a.table_rows > 0) {
                float co[VEC], si[VEC];
                load_table<VEC>(a.cs + trow + u * VEC, co);
                load_table<VEC>(a.sn + trow + u * VEC, si);
                turn[s].set(co, si, wa, wb);
            } else {
                turn[s].keep(wa, wb);
            }
        }
#pragma unroll
        for (int r = 0; r < HPT; ++r) {
            norm[r] = 0.f;
#pragma unroll
            for (int s = 0; s < UPL; ++s) {
                float x[VEC];
                unpack<T, VEC>(ra[r][s], x);
                norm[r] += ca[s] < a.d ? dot_vec<VEC>(x, x) : 0.f;
                unpack<T, VEC>(rb[r][s], x);
                norm[r] += cb[s] < a.d ? dot_vec<VEC>(x, x) : 0.f;
            }
        }
        for (int o = lanes >> 1; o > 0; o >>= 1)
#pragma unroll
            for (int r = 0; r < HPT; ++r) norm[r] += __shfl_xor_sync(mask, norm[r], o);
        const float inv_d = 1.f / (float)a.d;
#pragma unroll
        for (int r = 0; r < HPT; ++r) norm[r] = rsqrtf(norm[r] * inv_d + a.eps);
    }

    if ((is_q || OUT == OUT_DENSE) && !keep) {       // a padding row: zeros
        for (int r = 0; r < nh; ++r) {
            T* y = static_cast<T*>(is_q ? a.yq : a.yk) + ((int64_t)tok * (is_q ? a.hq : a.hk) + h0 + r) * a.d;
#pragma unroll
            for (int s = 0; s < UPL; ++s) {
                if (ca[s] < a.d) *reinterpret_cast<Pack<T, VEC>*>(y + ca[s]) = Pack<T, VEC>{};
                if (cb[s] < a.d) *reinterpret_cast<Pack<T, VEC>*>(y + cb[s]) = Pack<T, VEC>{};
            }
        }
        return;
    }
    int slot = -1;
    if (OUT != OUT_DENSE && !is_q && keep) {
        slot = a.c.row(i, b, a.hk, h0, pos);
        if (slot < 0 && lane == 0) raise_device_error(a.err, DEV_ERR_INDEX);
    }
#pragma unroll
    for (int r = 0; r < HPT; ++r) {
        float xa[UPL][VEC], xb[UPL][VEC];
#pragma unroll
        for (int s = 0; s < UPL; ++s) {
            unpack<T, VEC>(ra[r][s], xa[s]);
            unpack<T, VEC>(rb[r][s], xb[s]);
            if (ROPE && rope) {
                scale_vec<VEC>(xa[s], xa[s], norm[r]);
                scale_vec<VEC>(xb[s], xb[s], norm[r]);
                turn[s].apply(xa[s], xb[s]);
            }
        }
        if (is_q || OUT == OUT_DENSE) {
            T* y = static_cast<T*>(is_q ? a.yq : a.yk) + ((int64_t)tok * (is_q ? a.hq : a.hk) + h0 + r) * a.d;
#pragma unroll
            for (int s = 0; s < UPL; ++s) {
                if (r < nh && ca[s] < a.d) store_vec<T, VEC>(y + ca[s], xa[s]);
                if (r < nh && cb[s] < a.d) store_vec<T, VEC>(y + cb[s], xb[s]);
            }
        } else if constexpr (OUT != OUT_DENSE) {
            float scale = 1.f;
            if constexpr (OUT == OUT_I8 || OUT == OUT_E4M3) {
                float m = 0.f;
#pragma unroll
                for (int s = 0; s < UPL; ++s) {
                    float ma = 0.f, mb = 0.f;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) ma = amax2(ma, xa[s][j]), mb = amax2(mb, xb[s][j]);
                    m = amax2(m, amax2(ca[s] < a.d ? ma : 0.f, cb[s] < a.d ? mb : 0.f));
                }
                for (int o = lanes >> 1; o > 0; o >>= 1) m = amax2(m, __shfl_xor_sync(mask, m, o));
                scale = code_scale(m, OUT == OUT_I8);
            }
            const bool live = r < nh && slot >= 0;
            const int64_t at = (int64_t)i * a.c.pages * a.hk * a.c.page + slot + (int64_t)r * a.c.page;
            void* base = is_v ? a.c.v : a.c.k;
            if constexpr (OUT == OUT_I8 || OUT == OUT_E4M3) {
                if (live && lane == 0) (is_v ? a.c.vs : a.c.ks)[at] = scale;
            }
#pragma unroll
            for (int s = 0; s < UPL; ++s) {
                store_code<T, VEC, OUT>(base, at * a.d + ca[s], xa[s], scale, live && ca[s] < a.d);
                store_code<T, VEC, OUT>(base, at * a.d + cb[s], xb[s], scale, live && cb[s] < a.d);
            }
        }
    }
}

// Cache rows out: value = code * scale, rounded once to T; k and v heads of
// the tokens at `pos`, zeros for padding. HPT heads of a token at once.
template <typename T, int VEC, int UPL, int HPT, int IN>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const __grid_constant__ RowArgs a) {
    constexpr bool CODE = IN == OUT_I8 || IN == OUT_E4M3;
    using C = typename std::conditional<CODE, uint8_t, T>::type;
    const int lanes = 1 << a.lanes_log2;
    const int lane = threadIdx.x & (lanes - 1);
    const uint32_t unit = blockIdx.x * (kThreads >> a.lanes_log2) + (threadIdx.x >> a.lanes_log2);
    if (unit >= a.units) return;
    uint32_t part, t, b;
    const uint32_t tok = a.parts.divmod(unit, part);
    const uint32_t nb = a.tdiv.divmod(tok, t);
    const uint32_t i = a.bdiv.divmod(nb, b);
    const bool is_v = (int)part >= a.parts_k;
    const int h0 = HPT * (is_v ? (int)part - a.parts_k : (int)part);
    const int nh = min(HPT, a.hk - h0);
    const int pos = load_index(a.pos, i * a.pos_n + b * a.pos_b + t * a.pos_t, a.pos64);
    const int slot = pos < 0 ? -1 : a.c.row(i, b, a.hk, h0, pos);
    if (pos >= 0 && slot < 0 && lane == 0) raise_device_error(a.err, DEV_ERR_INDEX);
    Pack<C, VEC> raw[HPT][2 * UPL];
    float scale[HPT];
    if (slot >= 0) {
        const int64_t at = (int64_t)i * a.c.pages * a.hk * a.c.page + slot;
        const C* base = static_cast<const C*>(is_v ? a.c.v : a.c.k);
#pragma unroll
        for (int r = 0; r < HPT; ++r) {
            const int64_t row = at + (int64_t)min(r, nh - 1) * a.c.page;
            scale[r] = CODE ? __ldg((is_v ? a.c.vs : a.c.ks) + row) : 1.f;
#pragma unroll
            for (int s = 0; s < 2 * UPL; ++s) {
                const int c = (lane + s * lanes) * VEC;
                raw[r][s] = load_pack<C, VEC>(base + row * a.d + (c < a.d ? c : 0));
            }
        }
    } else {
#pragma unroll
        for (int r = 0; r < HPT; ++r) {
            scale[r] = 0.f;
#pragma unroll
            for (int s = 0; s < 2 * UPL; ++s) raw[r][s] = Pack<C, VEC>{};
        }
    }
#pragma unroll
    for (int r = 0; r < HPT; ++r) {
        T* y = static_cast<T*>(is_v ? a.yv : a.yk) + ((int64_t)tok * a.hk + h0 + r) * a.d;
#pragma unroll
        for (int s = 0; s < 2 * UPL; ++s) {
            const int c = (lane + s * lanes) * VEC;
            const bool live = r < nh && c < a.d;
            if constexpr (CODE) {
                float x[VEC];
                if constexpr (IN == OUT_I8) values_i8<VEC>(raw[r][s].v, x);
                else values_e4m3<VEC>(raw[r][s].v, x);
                scale_vec<VEC>(x, x, scale[r]);
                if (live) store_vec<T, VEC>(y + c, x);
            } else if (live) {
                *reinterpret_cast<Pack<T, VEC>*>(y + c) = raw[r][s];
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Gradients of the norm + rotation
// ---------------------------------------------------------------------------
struct GradArgs {
    RowArgs r;                  // q, k, weights, tables, positions as in the forward; yq / yk = dq / dk
    const void *dyq, *dyk;      // dense
    float* part;                // [n, chunks, d] fp32: one row of partial weight gradients per block
    void *dqw, *dkw;            // [n, d], nullable
    int cq, ck;                 // blocks per model for the q rows and the k rows
    uint32_t per_q, per_k;      // units of one block
    FastDiv q_parts, k_parts;
};

// A block takes consecutive units (HPT heads of a token) of one model's q (or
// k) side, and each of its groups of lanes every (threads / lanes)-th of them, keeping
// the weight gradient of its channels in registers; groups, warps and blocks
// are joined in a fixed order, so the sums do not depend on timing.
template <typename T, int VEC, int UPL, int HPT, bool INTER>
__global__ void __launch_bounds__(kThreads) rope_bwd_kernel(const __grid_constant__ GradArgs g) {
    const RowArgs& a = g.r;
    __shared__ float red[kThreads / 32][256];
    const int lanes = 1 << a.lanes_log2;
    const int lane = threadIdx.x & (lanes - 1);
    const unsigned mask = group_mask(lanes);
    const int groups = kThreads >> a.lanes_log2;
    const int chunks = g.cq + g.ck;
    const int i = blockIdx.x / chunks;
    const int chunk = blockIdx.x - i * chunks;
    const bool is_q = chunk < g.cq;
    const int heads = is_q ? a.hq : a.hk;
    const uint32_t all = (uint32_t)a.b * a.t * (is_q ? a.parts_q : a.parts_k);
    const uint32_t per = is_q ? g.per_q : g.per_k;
    const uint32_t first = (is_q ? chunk : chunk - g.cq) * per;
    const uint32_t last = min(all, first + per);
    const FastDiv parts = is_q ? g.q_parts : g.k_parts;
    const Strides st = is_q ? a.sq : a.sk;
    const T* x0 = static_cast<const T*>(is_q ? a.q : a.k) + (int64_t)i * st.n;
    const int64_t dense0 = (int64_t)i * a.b * a.t * heads;
    const T* dy0 = static_cast<const T*>(is_q ? g.dyq : g.dyk);
    T* dx0 = static_cast<T*>(is_q ? a.yq : a.yk);
    const T* w = static_cast<const T*>(is_q ? a.qw : a.kw) + (int64_t)i * a.d;
    const int turned = a.rot / 2 / VEC;

    int ca[UPL], cb[UPL];
    float wa[UPL][VEC], wb[UPL][VEC], da[UPL][VEC], db[UPL][VEC];
#pragma unroll
    for (int s = 0; s < UPL; ++s) {
        unit_channels<VEC, INTER>(lane + s * lanes, turned, a.rot, ca[s], cb[s]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) wa[s][j] = wb[s][j] = da[s][j] = db[s][j] = 0.f;
        if (ca[s] < a.d) load_vec<T, VEC>(w + ca[s], wa[s]);
        if (cb[s] < a.d) load_vec<T, VEC>(w + cb[s], wb[s]);
    }
    const float inv_d = 1.f / (float)a.d;
    // Where a unit lies, and its position, asked for a round ahead, as the
    // table's rows wait for it (118 -> 113 us over 84 M bf16 values; x and dy a
    // round ahead through shared memory as well: 124 us).
    struct Place {
        uint32_t part, bt, b, t;
        int pos;
    };
    auto find = [&](uint32_t unit) {
        Place p;
        p.bt = parts.divmod(min(unit, last - 1), p.part);
        p.b = a.tdiv.divmod(p.bt, p.t);
        p.pos = load_index(a.pos, i * a.pos_n + p.b * a.pos_b + p.t * a.pos_t, a.pos64);
        return p;
    };
    const uint32_t begin = first + (threadIdx.x >> a.lanes_log2);
    Place next = {};
    if (begin < last) next = find(begin);
    for (uint32_t unit = begin; unit < last; unit += groups) {
        const uint32_t part = next.part, bt = next.bt, b = next.b, t = next.t;
        const int pos = next.pos;
        const int h0 = (int)part * HPT, nh = min(HPT, heads - h0);
        const bool keep = pos >= 0 && pos < a.table_rows;
        const T* x = x0 + b * st.b + t * st.t + h0 * st.h;
        const int64_t dense = (dense0 + (int64_t)bt * heads + h0) * a.d;
        const T* dy = dy0 + dense;
        T* dx = dx0 + dense;
        Pack<T, VEC> ra[HPT][UPL], rb[HPT][UPL], sa[HPT][UPL], sb[HPT][UPL];
#pragma unroll
        for (int r = 0; r < HPT; ++r)
#pragma unroll
            for (int s = 0; s < UPL; ++s) {
                // places outside the row are read from its first vector and left out of the sums
                const int at = r < nh ? r : 0, pa = ca[s] < a.d ? ca[s] : 0, pb = cb[s] < a.d ? cb[s] : 0;
                const T* row = x + at * (int64_t)(int)st.h;
                ra[r][s] = load_pack<T, VEC>(row + pa);
                sa[r][s] = load_pack<T, VEC>(dy + at * a.d + pa);
                rb[r][s] = load_pack<T, VEC>(row + pb);
                sb[r][s] = load_pack<T, VEC>(dy + at * a.d + pb);
            }
        next = find(unit + groups);
        const int64_t trow = (int64_t)(keep ? pos : 0) * (a.rot / 2);
        Turn<VEC, INTER> turn[UPL];                 // back: the sines negated, no weights
#pragma unroll
        for (int s = 0; s < UPL; ++s) {
            const int u = lane + s * lanes;
            if (u < turned && a.table_rows > 0) {
                float co[VEC], si[VEC], one[VEC];
                load_table<VEC>(a.cs + trow + u * VEC, co);
                load_table<VEC>(a.sn + trow + u * VEC, si);
#pragma unroll
                for (int j = 0; j < VEC; ++j) si[j] = -si[j], one[j] = 1.f;
                turn[s].set(co, si, one, one);
            } else {
                float one[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) one[j] = 1.f;
                turn[s].keep(one, one);
            }
        }
        // du, and the sums over the row of x^2 and of g x with g = w du
        float ss[HPT], gx[HPT], ua[HPT][UPL][VEC], ub[HPT][UPL][VEC];
#pragma unroll
        for (int r = 0; r < HPT; ++r) {
            ss[r] = gx[r] = 0.f;
#pragma unroll
            for (int s = 0; s < UPL; ++s) {
                float x[VEC], g[VEC];
                unpack<T, VEC>(sa[r][s], ua[r][s]);
                unpack<T, VEC>(sb[r][s], ub[r][s]);
                turn[s].apply(ua[r][s], ub[r][s]);
                unpack<T, VEC>(ra[r][s], x);
                mul_vec<VEC>(g, ua[r][s], wa[s]);
                ss[r] += ca[s] < a.d ? dot_vec<VEC>(x, x) : 0.f;
                gx[r] += ca[s] < a.d ? dot_vec<VEC>(g, x) : 0.f;
                unpack<T, VEC>(rb[r][s], x);
                mul_vec<VEC>(g, ub[r][s], wb[s]);
                ss[r] += cb[s] < a.d ? dot_vec<VEC>(x, x) : 0.f;
                gx[r] += cb[s] < a.d ? dot_vec<VEC>(g, x) : 0.f;
            }
        }
        for (int o = lanes >> 1; o > 0; o >>= 1)
#pragma unroll
            for (int r = 0; r < HPT; ++r) {
                ss[r] += __shfl_xor_sync(mask, ss[r], o);
                gx[r] += __shfl_xor_sync(mask, gx[r], o);
            }
        if (!keep) {                         // padding adds nothing, not even a NaN that it holds
            for (int r = 0; r < nh; ++r)
#pragma unroll
                for (int s = 0; s < UPL; ++s) {
                    if (ca[s] < a.d) *reinterpret_cast<Pack<T, VEC>*>(dx + r * a.d + ca[s]) = Pack<T, VEC>{};
                    if (cb[s] < a.d) *reinterpret_cast<Pack<T, VEC>*>(dx + r * a.d + cb[s]) = Pack<T, VEC>{};
                }
            continue;
        }
#pragma unroll
        for (int r = 0; r < HPT; ++r) {
            const bool live = r < nh;
            const float rs = rsqrtf(ss[r] * inv_d + a.eps);
            const float m = -gx[r] * inv_d * rs * rs;
#pragma unroll
            for (int s = 0; s < UPL; ++s) {
                // t = x r; dw += du t; dx = r (w du) - t m
                auto one = [&](const Pack<T, VEC>& raw, float* u, const float* w, float* dw, int ch) {
                    float t[VEC], mt[VEC], td[VEC];
                    unpack<T, VEC>(raw, t);
                    scale_vec<VEC>(t, t, rs);
                    scale_vec<VEC>(td, t, live ? 1.f : 0.f);      // a head read twice counts once
                    fma_vec<VEC>(dw, u, td, dw);
                    scale_vec<VEC>(mt, t, m);
                    mul_vec<VEC>(u, u, w);
                    float rr[VEC];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) rr[j] = rs;
                    fma_vec<VEC>(u, u, rr, mt);
                    if (live && ch < a.d) store_vec<T, VEC>(dx + r * a.d + ch, u);
                };
                one(ra[r][s], ua[r][s], wa[s], da[s], ca[s]);
                one(rb[r][s], ub[r][s], wb[s], db[s], cb[s]);
            }
        }
    }
    __syncwarp();
    // groups of a warp, then the warps
#pragma unroll
    for (int s = 0; s < UPL; ++s)
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            for (int o = lanes; o < 32; o <<= 1) {
                da[s][j] += __shfl_xor_sync(0xffffffffu, da[s][j], o);
                db[s][j] += __shfl_xor_sync(0xffffffffu, db[s][j], o);
            }
    if ((threadIdx.x & 31) < lanes) {
#pragma unroll
        for (int s = 0; s < UPL; ++s)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (ca[s] < a.d) red[threadIdx.x >> 5][ca[s] + j] = da[s][j];
                if (cb[s] < a.d) red[threadIdx.x >> 5][cb[s] + j] = db[s][j];
            }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.d; c += kThreads) {
        float sum = 0.f;
#pragma unroll
        for (int wp = 0; wp < kThreads / 32; ++wp) sum += red[wp][c];
        g.part[(int64_t)blockIdx.x * a.d + c] = sum;
    }
}

// Weight gradients: the blocks' partial rows of one model and side, in order.
template <typename T>
__global__ void __launch_bounds__(kThreads) rope_bwd_join_kernel(const float* part, T* dqw, T* dkw, int cq, int ck,
                                                                 int d) {
    __shared__ float red[kThreads / 32][33];
    const int i = blockIdx.x >> 1;
    const bool is_q = (blockIdx.x & 1) == 0;
    T* out = is_q ? dqw : dkw;
    const int c = blockIdx.y * 32 + (threadIdx.x & 31);
    const float* p = part + ((int64_t)i * (cq + ck) + (is_q ? 0 : cq)) * d;
    float sum = 0.f;
    if (c < d)
        for (int r = threadIdx.x >> 5; r < (is_q ? cq : ck); r += kThreads / 32) sum += p[(int64_t)r * d + c];
    red[threadIdx.x >> 5][threadIdx.x & 31] = sum;
    __syncthreads();
    if (threadIdx.x < 32 && c < d && out) {
        sum = 0.f;
#pragma unroll
        for (int wp = 0; wp < kThreads / 32; ++wp) sum += red[wp][threadIdx.x];
        out[(int64_t)i * d + c] = from_f<T>(sum);
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
inline bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

inline bool strides_fit(const Strides& s, int vec) {
    return s.n % vec == 0 && s.b % vec == 0 && s.t % vec == 0 && s.h % vec == 0;
}

// Widest vector (elements) that every row address allows: 16 bytes, else 4 or 2
// elements, else 1. The halves of a rotation have to start on one too (bf16
// heads of 96 with 24 channels turned, 40 M values: 69 us with 4, 192 with 2).
int row_vec(const RowArgs& a, size_t esz, std::initializer_list<const void*> dense, bool cache_same) {
    for (int vec : {(int)(16 / esz), 4, 2}) {
        bool ok = a.d % vec == 0 && (a.rot / 2) % vec == 0;
        ok = ok && (!a.q || (aligned_to(a.q, vec * esz) && strides_fit(a.sq, vec)));
        ok = ok && (!a.k || (aligned_to(a.k, vec * esz) && strides_fit(a.sk, vec)));
        ok = ok && (!a.v || (aligned_to(a.v, vec * esz) && strides_fit(a.sv, vec)));
        for (const void* p : dense) ok = ok && (!p || aligned_to(p, vec * esz));
        for (const void* p : {(const void*)a.cs, (const void*)a.sn}) ok = ok && (!p || aligned_to(p, vec < 4 ? 4 * vec : 16));
        for (const void* p : {(const void*)a.c.k, (const void*)a.c.v})
            ok = ok && (!p || aligned_to(p, cache_same ? vec * esz : vec));
        if (ok) return vec;
    }
    return 1;
}

int lanes_log2(int d, int vec) {
    const int units = ((d + vec - 1) / vec + 1) / 2;
    int l = 0;
    while ((1 << l) < units && l < 5) ++l;
    return l;
}

// geom: n, b, t, hq, hk, d, rot, table rows, strides (n, b, t, head) of q, k
// and v, strides (n, b, t) of the positions.
int row_args(RowArgs& a, const char* what, const int64_t* g, int pos64) {
    if (!g) return set_error(WIDEK_ERR_INVALID, "%s: null geometry", what);
    for (int i = 0; i < 8; ++i)
        if (g[i] < 0 || g[i] > 0x7fffffff)
            return set_error(WIDEK_ERR_INVALID, "%s: size %d out of range (%lld)", what, i, (long long)g[i]);
    if (g[5] > 256) return set_error(WIDEK_ERR_UNSUPPORTED, "%s: head size %lld above 256", what, (long long)g[5]);
    if (g[6] > g[5] || g[6] % 2 != 0)
        return set_error(WIDEK_ERR_INVALID, "%s: %lld rotated channels of %lld (an even number of at most the head)",
                         what, (long long)g[6], (long long)g[5]);
    a = RowArgs{};
    a.n = (int)g[0], a.b = (int)g[1], a.t = (int)g[2], a.hq = (int)g[3], a.hk = (int)g[4], a.d = (int)g[5];
    a.rot = (int)g[6], a.table_rows = (int)g[7];
    a.sq = Strides{g[8], g[9], g[10], g[11]};
    a.sk = Strides{g[12], g[13], g[14], g[15]};
    a.sv = Strides{g[16], g[17], g[18], g[19]};
    a.pos_n = g[20], a.pos_b = g[21], a.pos_t = g[22];
    for (int64_t h : {a.sq.h, a.sk.h, a.sv.h})
        if (h > 0x7fffffff || h < -0x7fffffff)
            return set_error(WIDEK_ERR_UNSUPPORTED, "%s: heads %lld elements apart", what, (long long)h);
    a.pos64 = pos64;
    a.err = device_error_ptr();
    return WIDEK_OK;
}

// Heads that a group of lanes takes at once. 4 with 16-byte vectors (1, 2 and 8
// took 228, 194 and 193 us where 4 took 145, at 168 M values), one in the
// narrow paths, whose rows take more registers, and where there are so few
// rows that one each does not fill the GPU (a decoder step of 6144 rows: 4.8
// us, not 7.2). 2 with vectors of 4 16-bit channels, which rotations of 8 r + 4
// pairs take.
constexpr int kHeadsAtOnce = 4;

int heads_at_once(const RowArgs& a, int vec, size_t esz, int sides) {
    if (vec == 4 && esz == 2) return 2;
    if (vec != (int)(16 / esz)) return 1;
    const double lanes = (double)a.n * a.b * a.t * ((double)a.hq + (double)sides * a.hk) * (1 << lanes_log2(a.d, vec));
    return lanes > 2048.0 * sm_count(current_device()) ? kHeadsAtOnce : 1;
}

// Units of a call with `vec`-wide accesses, hpt heads at once; sides: 1 (k) or
// 2 (k and v).
int row_units(RowArgs& a, const char* what, int vec, int hpt, int sides) {
    a.parts_q = (a.hq + hpt - 1) / hpt;
    a.parts_k = (a.hk + hpt - 1) / hpt;
    const int64_t parts = (int64_t)a.parts_q + (int64_t)sides * a.parts_k;
    const double units = (double)a.n * a.b * a.t * (double)parts;
    if (units > 2147483647.0) return set_error(WIDEK_ERR_INVALID, "%s: over 2^31 rows (%.0f)", what, units);
    a.units = (uint32_t)units;
    if (a.units == 0) return WIDEK_OK;
    a.parts = FastDiv::make((uint32_t)parts);
    a.tdiv = FastDiv::make((uint32_t)a.t);
    a.bdiv = FastDiv::make((uint32_t)a.b);
    a.lanes_log2 = lanes_log2(a.d, vec);
    return WIDEK_OK;
}

// Whether the call has no rows at all.
bool no_rows(const RowArgs& a, int heads) { return a.n == 0 || a.b == 0 || a.t == 0 || heads == 0 || a.d == 0; }

template <int OUT, bool ROPE>
struct RowLaunch {
    RowArgs a;
    int vec, hpt;
    const char* what;
    cudaStream_t st;
    template <typename T, bool INTER>
    void go() {
        constexpr int W = 16 / sizeof(T), H = kHeadsAtOnce;
        const uint32_t per = kThreads >> a.lanes_log2;
        const unsigned blocks = (a.units + per - 1) / per;
        if (vec == W && hpt == H) rows_kernel<T, W, 1, H, OUT, ROPE, INTER><<<blocks, kThreads, 0, st>>>(a);
        else if (vec == W) rows_kernel<T, W, 1, 1, OUT, ROPE, INTER><<<blocks, kThreads, 0, st>>>(a);
        else if (W > 4 && vec == 4) rows_kernel<T, 4, 1, (W > 4 ? 2 : 1), OUT, ROPE, INTER><<<blocks, kThreads, 0, st>>>(a);
        else if (vec == 2) rows_kernel<T, 2, 2, 1, OUT, ROPE, INTER><<<blocks, kThreads, 0, st>>>(a);
        else rows_kernel<T, 1, 4, 1, OUT, ROPE, INTER><<<blocks, kThreads, 0, st>>>(a);
    }
    template <typename T>
    int run() {
        if constexpr (ROPE) {
            if (a.inter) go<T, true>();
            else go<T, false>();
        } else {
            go<T, false>();
        }
        return check_launch(what);
    }
};

template <int IN>
struct ReadLaunch {
    RowArgs a;
    int vec, hpt;
    cudaStream_t st;
    template <typename T>
    int run() {
        constexpr int W = 16 / sizeof(T);
        const uint32_t per = kThreads >> a.lanes_log2;
        const unsigned blocks = (a.units + per - 1) / per;
        if (vec == W && hpt > 1) cache_read_kernel<T, W, 1, kHeadsAtOnce, IN><<<blocks, kThreads, 0, st>>>(a);
        else if (vec == W) cache_read_kernel<T, W, 1, 1, IN><<<blocks, kThreads, 0, st>>>(a);
        else if (W > 4 && vec == 4) cache_read_kernel<T, 4, 1, (W > 4 ? 2 : 1), IN><<<blocks, kThreads, 0, st>>>(a);
        else if (vec == 2) cache_read_kernel<T, 2, 2, 1, IN><<<blocks, kThreads, 0, st>>>(a);
        else cache_read_kernel<T, 1, 4, 1, IN><<<blocks, kThreads, 0, st>>>(a);
        return check_launch("widek_cache_read_fwd");
    }
};

template <int OUT, bool ROPE>
int launch_rows(const RowArgs& a, int vec, int hpt, const char* what, int dtype, cudaStream_t st) {
    RowLaunch<OUT, ROPE> L{a, vec, hpt, what, st};
    return dispatch_dtype(dtype, L);
}

template <bool ROPE>
int launch_rows_fmt(const RowArgs& a, int vec, int hpt, const char* what, int fmt, int dtype, cudaStream_t st) {
    if (fmt == WIDEK_I8) return launch_rows<OUT_I8, ROPE>(a, vec, hpt, what, dtype, st);
    if (fmt == WIDEK_E4M3) return launch_rows<OUT_E4M3, ROPE>(a, vec, hpt, what, dtype, st);
    return launch_rows<OUT_SAME, ROPE>(a, vec, hpt, what, dtype, st);
}

// Blocks of the backward over all models, 3 for each SM of a B200: twice as many
// cost the join what they gave.
constexpr int kGradBlocks = 3 * 148;
constexpr int kGradHeads = 2;     // heads at once in the backward, whose rows take twice the registers
constexpr int grad_heads(int vec, size_t) { return vec >= 4 ? kGradHeads : 1; }

// Blocks per model of the backward: about three blocks for each SM over all
// models and both sides, none with fewer units than its groups of lanes.
void grad_chunks(const RowArgs& a, int vec, int hpt, int& cq, int& ck, uint32_t& per_q, uint32_t& per_k) {
    const int groups = kThreads >> lanes_log2(a.d, vec);
    const int64_t tokens = (int64_t)a.b * a.t;
    auto split = [&](int64_t heads, int& c, uint32_t& per) {
        const int64_t units = tokens * ((heads + hpt - 1) / hpt);
        int64_t want = (int64_t)kGradBlocks * heads / ((int64_t)a.n * ((int64_t)a.hq + a.hk));
        const int64_t most = (units + groups - 1) / groups;
        want = want < 1 ? 1 : (want > most ? most : want);
        per = (uint32_t)(((units + want - 1) / want + groups - 1) / groups * groups);
        c = (int)((units + per - 1) / per);
    };
    split(a.hq, cq, per_q);
    split(a.hk, ck, per_k);
}

struct GradLaunch {
    GradArgs g;
    int vec;
    cudaStream_t st;
    template <typename T, bool INTER>
    void go(unsigned blocks) {
        constexpr int W = 16 / sizeof(T);
        if (vec == W) rope_bwd_kernel<T, W, 1, grad_heads(W, sizeof(T)), INTER><<<blocks, kThreads, 0, st>>>(g);
        else if (W > 4 && vec == 4) rope_bwd_kernel<T, 4, 1, kGradHeads, INTER><<<blocks, kThreads, 0, st>>>(g);
        else if (vec == 2) rope_bwd_kernel<T, 2, 2, 1, INTER><<<blocks, kThreads, 0, st>>>(g);
        else rope_bwd_kernel<T, 1, 4, 1, INTER><<<blocks, kThreads, 0, st>>>(g);
    }
    template <typename T>
    int run() {
        const unsigned blocks = (unsigned)g.r.n * (g.cq + g.ck);
        if (g.r.inter) go<T, true>(blocks);
        else go<T, false>(blocks);
        int rc = check_launch("widek_qk_norm_rope_bwd");
        if (rc != WIDEK_OK || (!g.dqw && !g.dkw)) return rc;
        const dim3 grid(2 * g.r.n, (g.r.d + 31) / 32);
        rope_bwd_join_kernel<T><<<grid, kThreads, 0, st>>>(g.part, static_cast<T*>(g.dqw), static_cast<T*>(g.dkw), g.cq,
                                                           g.ck, g.r.d);
        return check_launch("widek_qk_norm_rope_bwd (join)");
    }
};

int rope_pointers(const RowArgs& a, const char* what) {
    if (a.hq < 1 || a.hk < 1) return set_error(WIDEK_ERR_INVALID, "%s: no heads (hq=%d, hk=%d)", what, a.hq, a.hk);
    if (!no_rows(a, a.hq) &&
        (!a.q || !a.k || !a.qw || !a.kw || !a.pos || !a.yq || (a.rot > 0 && a.table_rows > 0 && (!a.cs || !a.sn))))
        return set_error(WIDEK_ERR_INVALID, "%s: null pointer", what);
    return WIDEK_OK;
}

}  // namespace
}  // namespace widek

using namespace widek;

extern "C" int widek_qk_norm_rope_fwd(const void* q, const void* k, const void* qw, const void* kw, const float* cos,
                                      const float* sin, const void* positions, void* yq, void* yk,
                                      const int64_t* geom, double eps, int interleaved, int pos64, int dtype,
                                      void* stream) {
    const char* what = "widek_qk_norm_rope_fwd";
    RowArgs a;
    int rc = row_args(a, what, geom, pos64);
    if (rc != WIDEK_OK) return rc;
    a.q = q, a.k = k, a.qw = qw, a.kw = kw, a.cs = cos, a.sn = sin, a.pos = positions, a.yq = yq, a.yk = yk;
    a.eps = (float)eps, a.inter = interleaved;
    rc = rope_pointers(a, what);
    if (rc != WIDEK_OK) return rc;
    if (no_rows(a, a.hq)) return WIDEK_OK;
    if (!yk) return set_error(WIDEK_ERR_INVALID, "%s: null pointer", what);
    const size_t esz = dtype_size(dtype);
    if (esz == 0) return set_error(WIDEK_ERR_INVALID, "%s: unknown dtype code %d", what, dtype);
    const int vec = row_vec(a, esz, {qw, kw, yq, yk}, false);
    const int hpt = heads_at_once(a, vec, esz, 1);
    rc = row_units(a, what, vec, hpt, 1);
    if (rc != WIDEK_OK) return rc;
    return launch_rows<OUT_DENSE, true>(a, vec, hpt, what, dtype, (cudaStream_t)stream);
}

extern "C" int widek_qk_norm_rope_write_fwd(const void* q, const void* k, const void* v, const void* qw,
                                            const void* kw, const float* cos, const float* sin, const void* positions,
                                            void* yq, void* kc, void* vc, float* ks, float* vs, const void* table,
                                            const int64_t* geom, const int64_t* cgeom, double eps, int interleaved,
                                            int pos64, int fmt, int dtype, void* stream) {
    const char* what = "widek_qk_norm_rope_write_fwd";
    RowArgs a;
    int rc = row_args(a, what, geom, pos64);
    if (rc != WIDEK_OK) return rc;
    rc = cache_args(a.c, what, kc, vc, ks, vs, table, cgeom, (int64_t)a.n * a.b * a.t, a.hk, a.d, fmt, dtype);
    if (rc != WIDEK_OK) return rc;
    a.q = q, a.k = k, a.v = v, a.qw = qw, a.kw = kw, a.cs = cos, a.sn = sin, a.pos = positions, a.yq = yq;
    a.eps = (float)eps, a.inter = interleaved;
    rc = rope_pointers(a, what);
    if (rc != WIDEK_OK) return rc;
    if (no_rows(a, a.hq)) return WIDEK_OK;
    if (!v) return set_error(WIDEK_ERR_INVALID, "%s: null pointer", what);
    const size_t esz = dtype_size(dtype);
    if (esz == 0) return set_error(WIDEK_ERR_INVALID, "%s: unknown dtype code %d", what, dtype);
    const int vec = row_vec(a, esz, {qw, kw, yq}, !cache_fmt_8bit(fmt));
    const int hpt = heads_at_once(a, vec, esz, 2);
    rc = row_units(a, what, vec, hpt, 2);
    if (rc != WIDEK_OK) return rc;
    return launch_rows_fmt<true>(a, vec, hpt, what, fmt, dtype, (cudaStream_t)stream);
}

extern "C" int widek_cache_write_fwd(const void* k, const void* v, const void* positions, void* kc, void* vc,
                                     float* ks, float* vs, const void* table, const int64_t* geom,
                                     const int64_t* cgeom, int pos64, int fmt, int dtype, void* stream) {
    const char* what = "widek_cache_write_fwd";
    RowArgs a;
    int rc = row_args(a, what, geom, pos64);
    if (rc != WIDEK_OK) return rc;
    a.hq = 0, a.rot = 0;
    rc = cache_args(a.c, what, kc, vc, ks, vs, table, cgeom, (int64_t)a.n * a.b * a.t, a.hk, a.d, fmt, dtype);
    if (rc != WIDEK_OK) return rc;
    if (no_rows(a, a.hk)) return WIDEK_OK;
    if (!k || !v || !positions) return set_error(WIDEK_ERR_INVALID, "%s: null pointer", what);
    a.k = k, a.v = v, a.pos = positions;
    const size_t esz = dtype_size(dtype);
    if (esz == 0) return set_error(WIDEK_ERR_INVALID, "%s: unknown dtype code %d", what, dtype);
    const int vec = row_vec(a, esz, {}, !cache_fmt_8bit(fmt));
    const int hpt = heads_at_once(a, vec, esz, 2);
    rc = row_units(a, what, vec, hpt, 2);
    if (rc != WIDEK_OK) return rc;
    return launch_rows_fmt<false>(a, vec, hpt, what, fmt, dtype, (cudaStream_t)stream);
}

extern "C" int widek_cache_read_fwd(const void* kc, const void* vc, const float* ks, const float* vs,
                                    const void* table, const void* positions, void* k, void* v, const int64_t* geom,
                                    const int64_t* cgeom, int pos64, int fmt, int dtype, void* stream) {
    const char* what = "widek_cache_read_fwd";
    RowArgs a;
    int rc = row_args(a, what, geom, pos64);
    if (rc != WIDEK_OK) return rc;
    a.hq = 0, a.rot = 0;
    rc = cache_args(a.c, what, const_cast<void*>(kc), const_cast<void*>(vc), const_cast<float*>(ks),
                    const_cast<float*>(vs), table, cgeom, (int64_t)a.n * a.b * a.t, a.hk, a.d, fmt, dtype);
    if (rc != WIDEK_OK) return rc;
    if (no_rows(a, a.hk)) return WIDEK_OK;
    if (!k || !v || !positions) return set_error(WIDEK_ERR_INVALID, "%s: null pointer", what);
    a.yk = k, a.yv = v, a.pos = positions;
    const size_t esz = dtype_size(dtype);
    if (esz == 0) return set_error(WIDEK_ERR_INVALID, "%s: unknown dtype code %d", what, dtype);
    const int vec = row_vec(a, esz, {k, v}, !cache_fmt_8bit(fmt));
    const int hpt = heads_at_once(a, vec, esz, 2);
    rc = row_units(a, what, vec, hpt, 2);
    if (rc != WIDEK_OK) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    if (fmt == WIDEK_I8) {
        ReadLaunch<OUT_I8> L{a, vec, hpt, st};
        return dispatch_dtype(dtype, L);
    }
    if (fmt == WIDEK_E4M3) {
        ReadLaunch<OUT_E4M3> L{a, vec, hpt, st};
        return dispatch_dtype(dtype, L);
    }
    ReadLaunch<OUT_SAME> L{a, vec, hpt, st};
    return dispatch_dtype(dtype, L);
}

extern "C" int64_t widek_qk_norm_rope_bwd_workspace(const int64_t* geom) {
    RowArgs a;
    if (row_args(a, "widek_qk_norm_rope_bwd_workspace", geom, 0) != WIDEK_OK || a.hq < 1 || a.hk < 1) return -1;
    if (no_rows(a, a.hq)) return 0;
    // the most blocks of any vector width
    int64_t blocks = 0;
    for (int vec : {8, 4, 2, 1})
        for (int hpt : {1, kGradHeads}) {
            int cq, ck;
            uint32_t pq, pk;
            grad_chunks(a, vec, hpt, cq, ck, pq, pk);
            if (cq + ck > blocks) blocks = cq + ck;
        }
    return blocks * a.n * a.d * (int64_t)sizeof(float);
}

extern "C" int widek_qk_norm_rope_bwd(const void* q, const void* k, const void* qw, const void* kw, const float* cos,
                                      const float* sin, const void* positions, const void* dyq, const void* dyk,
                                      void* dq, void* dk, void* dqw, void* dkw, const int64_t* geom, double eps,
                                      int interleaved, int pos64, int dtype, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
    const char* what = "widek_qk_norm_rope_bwd";
    GradArgs g{};
    RowArgs& a = g.r;
    int rc = row_args(a, what, geom, pos64);
    if (rc != WIDEK_OK) return rc;
    a.q = q, a.k = k, a.qw = qw, a.kw = kw, a.cs = cos, a.sn = sin, a.pos = positions, a.yq = dq, a.yk = dk;
    a.eps = (float)eps, a.inter = interleaved;
    rc = rope_pointers(a, what);
    if (rc != WIDEK_OK) return rc;
    const size_t esz = dtype_size(dtype);
    if (esz == 0) return set_error(WIDEK_ERR_INVALID, "%s: unknown dtype code %d", what, dtype);
    if (no_rows(a, a.hq)) {                      // sums over nothing
        for (void* dw : {dqw, dkw})
            if (dw && a.n > 0 && a.d > 0 &&
                cudaMemsetAsync(dw, 0, (size_t)a.n * a.d * esz, (cudaStream_t)stream) != cudaSuccess)
                return check_launch(what);
        return WIDEK_OK;
    }
    if (!dk || !dyq || !dyk) return set_error(WIDEK_ERR_INVALID, "%s: null pointer", what);
    const int64_t need = widek_qk_norm_rope_bwd_workspace(geom);
    if (!workspace || workspace_bytes < need || !aligned_to(workspace, sizeof(float)))
        return set_error(WIDEK_ERR_INVALID, "%s: workspace of %lld bytes, %lld needed", what,
                         (long long)workspace_bytes, (long long)need);
    g.dyq = dyq, g.dyk = dyk, g.dqw = dqw, g.dkw = dkw, g.part = static_cast<float*>(workspace);
    const int vec = row_vec(a, esz, {qw, kw, dyq, dyk, dq, dk}, false);
    const int hpt = grad_heads(vec, esz);
    rc = row_units(a, what, 1, 1, 1);            // the narrowest: units of one head, for the size check
    if (rc != WIDEK_OK) return rc;
    grad_chunks(a, vec, hpt, g.cq, g.ck, g.per_q, g.per_k);
    a.lanes_log2 = lanes_log2(a.d, vec);
    a.parts_q = (a.hq + hpt - 1) / hpt;
    a.parts_k = (a.hk + hpt - 1) / hpt;
    g.q_parts = FastDiv::make((uint32_t)a.parts_q);
    g.k_parts = FastDiv::make((uint32_t)a.parts_k);
    GradLaunch L{g, vec, (cudaStream_t)stream};
    return dispatch_dtype(dtype, L);
}
