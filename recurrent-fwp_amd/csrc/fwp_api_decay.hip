// extern "C" entry points of the decayed sum rule's block: argument checks before anything is launched.
#include "fwp_elements.hpp"

using namespace fwp;

namespace {

bool type_ok(int type) { return type == FWP_F32 || type == FWP_F16 || type == FWP_BF16; }
template <typename V>
bool rows_ok(const V &v, int type) {
    return v.ptr && reinterpret_cast<uintptr_t>(v.ptr) % (type == FWP_F32 ? 4 : 2) == 0;
}
// sixty-four steps and a row lie within 32 bits of bytes
template <typename V>
bool step_ok(const V &v) {
    return v.sL >= 0 && v.sL <= FWP_DSUM_MAX_STEP;
}
bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool divides(int part, int whole) { return part >= 1 && whole % part == 0; }

constexpr int kMaxKeys = 128, kMaxValues = 1 << 16, kMaxSteps = 1 << 30, kMaxWidth = 1 << 16, kMaxGroup = 1024, kMaxRows = 1 << 30;

bool dims_ok(int type, int N, int H, int L, int E, int M) {
    return type_ok(type) && N >= 1 && H >= 1 && L >= 1 && L <= kMaxSteps && (int64_t)N * H < (int64_t(1) << 31) && E >= 1 && E <= kMaxKeys && M >= 1 &&
           M <= kMaxValues;
}

int dsum_check(const fwp_dsum_args *a) {
    if (!a || !a->decay || reinterpret_cast<uintptr_t>(a->decay) % 4) return FWP_E_NULL;
    if (!dims_ok(a->type, a->N, a->H, a->L, a->E, a->M) || !divides(a->HQ, a->H) || !divides(a->HK, a->H) || !divides(a->HV, a->H) ||
        (a->per_head && (a->dN || a->dL)))
        return FWP_E_SHAPE;
    for (const fwp_rows *v : {&a->q, &a->k, &a->v}) {
        if (!rows_ok(*v, a->type)) return FWP_E_NULL;
        if (!step_ok(*v)) return FWP_E_SHAPE;
    }
    return 0;
}

int norm_check(const fwp_group_norm_args *a) {
    if (!a || !a->x) return FWP_E_NULL;
    if (!type_ok(a->type) || a->rows < 1 || a->rows > kMaxRows || a->groups < 1 || a->size < 1 || a->size > kMaxGroup || (int64_t)a->groups * a->size > kMaxWidth ||
        (a->act != FWP_ACT_NONE && a->act != FWP_ACT_SIGMOID && a->act != FWP_ACT_SILU))
        return FWP_E_SHAPE;
    return 0;
}

}  // namespace

extern "C" {

long long fwp_decayed_sum_saved_floats(int type, int N, int H, int L, int E, int M) {
    return dims_ok(type, N, H, L, E, M) ? dsum_saved_floats(type, N, H, L, E, M) : FWP_E_SHAPE;
}

long long fwp_decayed_sum_workspace(const fwp_dsum_args *a, int backward) {
    if (int rc = dsum_check(a)) return rc;
    return dsum_workspace(*a, backward != 0);
}

int fwp_decayed_sum_fwd(const fwp_dsum_args *a, float *W, fwp_out_rows out, float *saved, float *workspace, void *stream) {
    if (int rc = dsum_check(a)) return rc;
    if (!rows_ok(out, a->type) || !aligned16(saved) || !aligned16(workspace)) return FWP_E_NULL;
    if (!step_ok(out)) return FWP_E_SHAPE;
    return dsum_fwd(*a, W, out, saved, workspace, (hipStream_t)stream);
}

int fwp_decayed_sum_bwd(const fwp_dsum_args *a, const float *saved, fwp_rows grad_out, fwp_out_rows gq, fwp_out_rows gk, fwp_out_rows gv,
                        float *gdecay, float *workspace, void *stream) {
    if (int rc = dsum_check(a)) return rc;
    if (!saved || !aligned16(saved) || !gdecay || !aligned16(workspace) || (!workspace && dsum_workspace(*a, true)) || !rows_ok(grad_out, a->type))
        return FWP_E_NULL;
    if (!step_ok(grad_out)) return FWP_E_SHAPE;
    for (const fwp_out_rows *v : {&gq, &gk, &gv}) {
        if (!rows_ok(*v, a->type)) return FWP_E_NULL;
        if (!step_ok(*v)) return FWP_E_SHAPE;
    }
    return dsum_bwd(*a, saved, grad_out, gq, gk, gv, gdecay, workspace, (hipStream_t)stream);
}

int fwp_rotary(const fwp_rotary_args *a, fwp_out_rows oq, fwp_out_rows ok, void *stream) {
    if (!a || !a->frequencies || reinterpret_cast<uintptr_t>(a->frequencies) % 8) return FWP_E_NULL;
    if (!type_ok(a->type) || a->N < 1 || a->HQ < 1 || a->L < 1 || a->L > kMaxSteps || a->D < 1 || a->D > kMaxWidth || a->pairs < 1 ||
        2 * (int64_t)a->pairs > a->D || (a->k.ptr && a->HK < 1) || (int64_t)a->HQ + a->HK > (1 << 30))
        return FWP_E_SHAPE;
    if (!rows_ok(a->q, a->type) || !rows_ok(oq, a->type) || (a->k.ptr && (!rows_ok(a->k, a->type) || !rows_ok(ok, a->type)))) return FWP_E_NULL;
    return rotary(*a, oq, ok, (hipStream_t)stream);
}

int fwp_group_norm_fwd(const fwp_group_norm_args *a, void *y, void *stream) {
    if (int rc = norm_check(a)) return rc;
    return y ? group_norm_fwd(*a, y, (hipStream_t)stream) : FWP_E_NULL;
}

long long fwp_group_norm_workspace(int type, int rows, int groups, int size) {
    return !type_ok(type) || rows < 1 || rows > kMaxRows || groups < 1 || size < 1 || size > kMaxGroup || (int64_t)groups * size > kMaxWidth
               ? FWP_E_SHAPE
               : group_norm_workspace(type, rows, groups, size);
}

int fwp_group_norm_bwd(const fwp_group_norm_args *a, const void *grad_y, void *gx, void *ggate, float *gweight, float *gbias, float *workspace,
                       void *stream) {
    if (int rc = norm_check(a)) return rc;
    if (!grad_y || !gx || (a->gate != nullptr) != (ggate != nullptr) || ((gweight || gbias) && !workspace)) return FWP_E_NULL;
    return group_norm_bwd(*a, grad_y, gx, ggate, gweight, gbias, workspace, (hipStream_t)stream);
}

}  // extern "C"
