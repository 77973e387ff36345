// Entry points of the residual norm's gradients (kernels: residual_norm_bwd.cuh).
#include "residual_norm_bwd.cuh"

namespace widek {
namespace rnorm {

int bwd_mode(const Args& a, int64_t rows) {
    if (!a.gate) return a.pw ? MODEL : PLAIN;
    return (int64_t)a.gate_rows == rows ? MODEL : GROUPS;
}

int bwd_teams(int64_t n, int64_t rows, int d, int sms, int threads) {
    if (n < 1 || rows < 1) return 1;
    const TeamShape shape = team_shape(d, kBwdChannels);
    const int64_t blocks = (int64_t)sms * (threads / shape.threads);
    const int64_t wave = shape.team == PAIR ? blocks / 2 : blocks * shape.rows();
    int64_t teams = wave / n;
    if (teams > (rows + 1) / 2) teams = (rows + 1) / 2;
    return teams < 1 ? 1 : (int)teams;
}

}  // namespace rnorm
}  // namespace widek

using namespace widek;

extern "C" int64_t widek_residual_norm_bwd_workspace(int64_t n, int64_t rows, int64_t d, int64_t gate_rows, int has_post,
                                                     int center) {
    if (n < 0 || rows < 0 || d < 1 || d > rnorm::kMaxChannels || (n > 0 && rows > 0x7fffffff / n)) {
        set_error(WIDEK_ERR_INVALID, "widek_residual_norm_bwd_workspace: bad sizes n=%lld rows=%lld d=%lld", (long long)n,
                  (long long)rows, (long long)d);
        return -1;
    }
    rnorm::Args a{};
    a.gate = gate_rows > 0 ? &a : nullptr;
    a.pw = has_post ? &a : nullptr;
    a.gate_rows = (uint32_t)(gate_rows > 0 ? gate_rows : 0);
    const int teams = rnorm::bwd_teams(n, rows, (int)d, sm_count(current_device()), 1024);
    return n * teams * rnorm::slot_count(rnorm::bwd_mode(a, rows), center != 0) * d * (int64_t)sizeof(float);
}

extern "C" int widek_residual_norm_bwd(const void* x, const void* y, const void* w, const void* wb, const void* pw,
                                       const void* pb, const void* gate, const float* stats, const void* dh,
                                       const void* dz, void* dx, void* dy, void* dw, void* dwb, void* dpw, void* dpb,
                                       void* dgate, int64_t n, int64_t rows, int64_t d, int64_t gate_rows, double scale,
                                       double eps, int center, int dtype, void* workspace, int64_t workspace_bytes,
                                       void* stream) {
    const char* what = "widek_residual_norm_bwd";
    rnorm::BwdArgs a{};
    int rc = rnorm::make_args(a.f, what, x, y, w, wb, pw, pb, gate, n, rows, d, gate_rows, scale, eps, center, dtype);
    if (rc != WIDEK_OK) return rc;
    if ((dy && !y) || ((dpw || dpb) && !pw) || (dgate && !gate) || ((dwb || dpb) && !center))
        return set_error(WIDEK_ERR_INVALID, "%s: a gradient of an input that is not there", what);
    if (a.f.rows == 0) return WIDEK_OK;
    const int64_t need = widek_residual_norm_bwd_workspace(n, rows, d, gate ? gate_rows : -1, pw != nullptr, center);
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3))
        return set_error(WIDEK_ERR_INVALID, "%s: a workspace of %lld bytes, %lld needed (on a 4-byte border)", what,
                         (long long)workspace_bytes, (long long)need);
    if (!stats || !aligned16(stats)) return set_error(WIDEK_ERR_INVALID, "%s: no statistics, or off a 16-byte border", what);
    a.f.stats = const_cast<float*>(stats);
    a.dh = dh; a.dz = dz; a.dx = dx; a.dy = dy; a.dw = dw; a.dwb = dwb; a.dpw = dpw; a.dpb = dpb; a.dgate = dgate;
    a.part = static_cast<float*>(workspace);
    return dispatch_dtype(dtype, rnorm::BwdLaunch{a, rnorm::bwd_mode(a.f, rows), static_cast<cudaStream_t>(stream)});
}
