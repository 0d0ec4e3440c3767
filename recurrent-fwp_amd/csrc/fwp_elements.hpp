// Rows of fp32, fp16 or bf16 elements: loads to fp32, stores rounded to nearest even (half an ulp of the type, once per result).
#pragma once
#include "fwp_common.hpp"

namespace fwp {

using half_t = _Float16;
using bf16_t = __bf16;

template <typename T>
__device__ __forceinline__ float load(const T *p) {
    return (float)*p;
}
template <typename T>
__device__ __forceinline__ void store(T *p, float x) {
    *p = (T)x;
}

// The elements of row (n, h, t) of a view
template <typename T>
__device__ __forceinline__ const T *row(const fwp_rows &v, int n, int h, int64_t t) {
    return static_cast<const T *>(v.ptr) + n * v.sN + h * v.sH + t * v.sL;
}
template <typename T>
__device__ __forceinline__ T *row(const fwp_out_rows &v, int n, int h, int64_t t) {
    return static_cast<T *>(v.ptr) + n * v.sN + h * v.sH + t * v.sL;
}

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
// 1 / (1 + exp(-x)): 0 and 1 at the infinities, NaN stays
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + exp_of(-x)); }
// d/dx of x sigmoid(x) from s = sigmoid(x); at the infinities, where x (1 - s) would be inf 0, the limits 0 and 1
__device__ __forceinline__ float silu_slope(float x, float s) {
    const float t = 1.f - s;
    return t == 0.f ? s : s == 0.f ? 0.f : s * fmaf(x, t, 1.f);
}
// x sigmoid(x); 0 at -inf, where the product would be -inf 0
__device__ __forceinline__ float silu(float x, float s) { return s == 0.f ? 0.f : x * s; }

// log(1 + exp(x)) = max(x, 0) + log1p(u), u = exp(-|x|) in (0, 1], and log1p(u) = 2 atanh(s) with s = u / (2 + u) <= 1/3:
// s times a polynomial in s^2 (Chebyshev over [0, 1/9], 4e-9 off), so that small results keep their relative precision.
__device__ __forceinline__ float softplus(float x, float &u) {
    u = exp_of(-fabsf(x));
    const float s = u * __builtin_amdgcn_rcpf(2.f + u), y = s * s;
    float p = 0.1408732831478119f;
    p = fmaf(p, y, 0.1398070901632309f);
    p = fmaf(p, y, 0.20012426376342773f);
    p = fmaf(p, y, 0.3333315849304199f);
    p = fmaf(p, y, 1.f);
    return fmaf(2.f * s, p, x < 0.f ? 0.f : x);      // NaN stays
}
__device__ __forceinline__ float softplus(float x) {
    float u;
    return softplus(x, u);
}
// its slope, the sigmoid, from the same u
__device__ __forceinline__ float softplus_slope(float x, float u) { return (x < 0.f ? u : 1.f) * __builtin_amdgcn_rcpf(1.f + u); }

// An infinite decay as the largest finite one: exp(dt A) is 0 (or infinite) all the same for every dt from 1e-36 on, and 1, not NaN, for the dt of zero that rows
// behind a sequence have.
__device__ __forceinline__ float within_range(float x) {
    constexpr float most = 3.402823466e38f;
    return x < -most ? -most : x > most ? most : x;      // NaN stays
}

// The steps of sequence n that count
__device__ __forceinline__ int length_of(const int64_t *lengths, int n, int L) {
    if (!lengths) return L;
    const int64_t l = lengths[n];
    return l < 0 ? 0 : l < L ? (int)l : L;
}

// Calls f(T()) for the element type of a call; false for a type that is none.
template <typename F>
inline bool by_type(int type, F f) {
    if (type == FWP_F32) f(float());
    else if (type == FWP_F16) f(half_t());
    else if (type == FWP_BF16) f(bf16_t());
    else return false;
    return true;
}

int conv_fwd(const fwp_conv_args &a, void *state, fwp_out_rows y, hipStream_t s);
int64_t conv_workspace(int N, int H, int L, int D, int K);
int conv_bwd(const fwp_conv_args &a, const void *state, fwp_rows gy, fwp_out_rows gx, float *gweight, float *gbias, float *workspace,
             hipStream_t s);

// A launch has fewer than 2^32 threads.
inline bool fits_launch(int64_t blocks, int threads) { return blocks <= (int64_t(1) << 32) / threads - 1; }

// Elements between the steps of a view that the scan takes: sixteen steps and a row then lie within 32 bits of bytes.
constexpr int64_t kScanMaxStep = FWP_SCAN_MAX_STEP;
int64_t scan_saved_floats(int N, int H, int L, int E, int M);
int64_t scan_workspace(int N, int H, int L, int E, int M, bool backward);
int scan_fwd(const fwp_scan_args &a, float *W, fwp_out_rows out, float *saved, float *workspace, hipStream_t s);
int scan_bwd(const fwp_scan_args &a, const float *saved, fwp_rows gout, fwp_out_rows gq, fwp_out_rows gk, fwp_out_rows gv,
             fwp_out_rows gdelta, fwp_out_rows gz, float *gA, float *gD, float *gdelta_bias, float *workspace, hipStream_t s);

int64_t residual_norm_workspace(int rows, int cols);
int residual_norm_fwd(const fwp_norm_args &a, void *r, void *n, float *stats, hipStream_t s);
int residual_norm_bwd(const fwp_norm_args &a, const float *stats, const void *gr, const void *gn, const fwp_norm_grads &g,
                      float *workspace, hipStream_t s);

}  // namespace fwp
