// extern "C" entry points of the selective state space block: argument checks before anything is launched.
#include "fwp_elements.hpp"

using namespace fwp;

namespace {

bool type_ok(int type) { return type == FWP_F32 || type == FWP_F16 || type == FWP_BF16; }
// a whole number of elements, as every view of a tensor is
bool element_aligned(const void *p, int type) { return reinterpret_cast<uintptr_t>(p) % (type == FWP_F32 ? 4 : 2) == 0; }
bool rows_ok(const fwp_rows &v, int type) { return v.ptr && element_aligned(v.ptr, type); }
bool rows_ok(const fwp_out_rows &v, int type) { return v.ptr && element_aligned(v.ptr, type); }

// Channels of 2^24 and steps of 2^30 are far beyond what fits the memory; below them every index within a row or sequence fits 32 bits.
bool dims_ok(int N, int H, int L) { return N >= 1 && H >= 1 && L >= 1 && L <= 1 << 30 && (int64_t)N * H < (int64_t(1) << 31); }
constexpr int kMaxChannels = 1 << 24, kMaxTaps = 8, kMaxKeys = 64, kMaxColumns = 8192;

int conv_check(const fwp_conv_args *a) {
    if (!a || !a->weight) return FWP_E_NULL;
    if (!type_ok(a->type) || !dims_ok(a->N, a->H, a->L) || a->D < 1 || a->D > kMaxChannels || a->K < 1 || a->K > kMaxTaps) return FWP_E_SHAPE;
    return rows_ok(a->x, a->type) ? 0 : FWP_E_NULL;
}

bool step_ok(int64_t sL) { return sL >= 0 && sL <= kScanMaxStep; }

int scan_dims(int N, int H, int L, int E, int M) {
    return dims_ok(N, H, L) && E >= 1 && E <= kMaxKeys && M >= 1 && M <= kMaxChannels ? 0 : FWP_E_SHAPE;
}

int norm_check(const fwp_norm_args *a) {
    if (!a || !a->y || !a->x || (a->after_bias && !a->after_weight) || (a->before_bias && !a->before_weight)) return FWP_E_NULL;
    if (!type_ok(a->type) || (a->stream_type != a->type && a->stream_type != FWP_F32) || a->rows < 1 || a->cols < 1 || a->cols > kMaxColumns ||
        (a->act != FWP_ACT_NONE && a->act != FWP_ACT_SIGMOID && a->act != FWP_ACT_SILU))
        return FWP_E_SHAPE;
    return 0;
}

}  // namespace

extern "C" {

int fwp_conv_fwd(const fwp_conv_args *a, void *state, fwp_out_rows y, void *stream) {
    if (int rc = conv_check(a)) return rc;
    if (!rows_ok(y, a->type)) return FWP_E_NULL;
    return conv_fwd(*a, a->K > 1 ? state : nullptr, y, (hipStream_t)stream);
}

long long fwp_conv_workspace(int N, int H, int L, int D, int K) {
    if (!dims_ok(N, H, L) || D < 1 || D > kMaxChannels || K < 1 || K > kMaxTaps) return FWP_E_SHAPE;
    return conv_workspace(N, H, L, D, K);
}

int fwp_conv_bwd(const fwp_conv_args *a, const void *state, fwp_rows grad_y, fwp_out_rows gx, float *gweight, float *gbias,
                 float *workspace, void *stream) {
    if (int rc = conv_check(a)) return rc;
    if (!rows_ok(grad_y, a->type) || !rows_ok(gx, a->type) || (gweight == nullptr) != (gbias == nullptr) || !workspace) return FWP_E_NULL;
    return conv_bwd(*a, a->K > 1 ? state : nullptr, grad_y, gx, gweight, gbias, workspace, (hipStream_t)stream);
}

long long fwp_scan_saved_floats(int N, int H, int L, int E, int M) {
    return scan_dims(N, H, L, E, M) ? FWP_E_SHAPE : scan_saved_floats(N, H, L, E, M);
}

long long fwp_scan_workspace(int N, int H, int L, int E, int M, int backward) {
    return scan_dims(N, H, L, E, M) ? FWP_E_SHAPE : scan_workspace(N, H, L, E, M, backward != 0);
}

int fwp_scan_fwd(const fwp_scan_args *a, float *W, fwp_out_rows out, float *saved, float *workspace, void *stream) {
    if (!a || !a->A) return FWP_E_NULL;
    if (!type_ok(a->type) || scan_dims(a->N, a->H, a->L, a->E, a->M)) return FWP_E_SHAPE;
    for (const fwp_rows *v : {&a->q, &a->k, &a->v, &a->delta})
        if (!rows_ok(*v, a->type)) return FWP_E_NULL;
    if (!element_aligned(a->z.ptr, a->type) || !rows_ok(out, a->type)) return FWP_E_NULL;
    for (const int64_t sL : {a->q.sL, a->k.sL, a->v.sL, a->delta.sL, a->z.ptr ? a->z.sL : 0, out.sL})
        if (!step_ok(sL)) return FWP_E_SHAPE;
    return scan_fwd(*a, W, out, saved, workspace, (hipStream_t)stream);
}

int fwp_scan_bwd(const fwp_scan_args *a, const float *saved, fwp_rows grad_out, fwp_out_rows gq, fwp_out_rows gk, fwp_out_rows gv,
                 fwp_out_rows gdelta, fwp_out_rows gz, float *gA, float *gD, float *gdelta_bias, float *workspace, void *stream) {
    if (!a || !a->A || !saved || !gA || !gD || !gdelta_bias || !workspace) return FWP_E_NULL;
    if (!type_ok(a->type) || scan_dims(a->N, a->H, a->L, a->E, a->M)) return FWP_E_SHAPE;
    for (const fwp_rows *v : {&a->q, &a->k, &a->v, &a->delta, (const fwp_rows *)&grad_out})
        if (!rows_ok(*v, a->type)) return FWP_E_NULL;
    for (const fwp_out_rows *v : {&gq, &gk, &gv, &gdelta})
        if (!rows_ok(*v, a->type)) return FWP_E_NULL;
    if (a->z.ptr && (!element_aligned(a->z.ptr, a->type) || !rows_ok(gz, a->type))) return FWP_E_NULL;
    for (const int64_t sL : {a->q.sL, a->k.sL, a->v.sL, a->delta.sL, grad_out.sL, gq.sL, gk.sL, gv.sL, gdelta.sL, a->z.ptr ? a->z.sL : 0, a->z.ptr ? gz.sL : 0})
        if (!step_ok(sL)) return FWP_E_SHAPE;
    return scan_bwd(*a, saved, grad_out, gq, gk, gv, gdelta, gz, gA, gD, gdelta_bias, workspace, (hipStream_t)stream);
}

int fwp_residual_norm_fwd(const fwp_norm_args *a, void *r, void *n, float *stats, void *stream) {
    if (int rc = norm_check(a)) return rc;
    if (!r || (a->before_weight != nullptr) != (n != nullptr) || reinterpret_cast<uintptr_t>(stats) % 16) return FWP_E_NULL;
    return residual_norm_fwd(*a, r, n, stats, (hipStream_t)stream);
}

long long fwp_residual_norm_workspace(int rows, int cols) {
    return rows < 1 || cols < 1 || cols > kMaxColumns ? FWP_E_SHAPE : residual_norm_workspace(rows, cols);
}

int fwp_residual_norm_bwd(const fwp_norm_args *a, const float *stats, const void *grad_r, const void *grad_n, const fwp_norm_grads *g,
                          float *workspace, void *stream) {
    if (int rc = norm_check(a)) return rc;
    if (!stats || reinterpret_cast<uintptr_t>(stats) % 16 || !g || !g->gy || !g->gx || (g->ggate && !a->gate) || !workspace) return FWP_E_NULL;
    return residual_norm_bwd(*a, stats, grad_r, grad_n, *g, workspace, (hipStream_t)stream);
}

}  // extern "C"
