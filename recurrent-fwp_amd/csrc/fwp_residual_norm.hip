// The norms around a block, fused with its gate, scale and residual addition, forward and backward.
//
//   u = norm(y) aw + ab    r = x + scale act(gate) u    n = norm(r) bw + bb
// and backwards, with hat for the normalised rows and s for 1 / spread:
//   dr = gr + s_r (h - mean(h) - rhat mean(h rhat)), h = gn bw    gx = dr    ggate = dr scale u act'(gate)    du = dr scale act(gate)
//   gy = s_y (h - mean(h) - yhat mean(h yhat)), h = du aw          (RMS norms: without the means that are subtracted)
// and the column sums for the five parameters.
//
// A row is read once and stays in registers: one wave to a row of up to 1024 columns, 4, 8 or 16 waves to wider ones, four neighbouring
// columns a lane and turn.  Means and variances (of the differences from the mean) are sums over the lanes by DPP and row exchanges, and over waves by way
// of LDS.  The backward pass forms r again from y, x and the gate; its workgroups go over many rows and keep the column sums in registers, and a
// second kernel adds the workgroups' sums in a fixed order.  Bound by memory.
#include "fwp_elements.hpp"
#include "fwp_wave.hpp"

#include <algorithm>

namespace fwp {
namespace {

constexpr int kBlocks = 512, kParams = 5;
constexpr int64_t kMaxBlocks = (int64_t(1) << 31) - 1;

// Elements c .. c + 3 of a row, as many as there are: at once where everything is aligned for that
template <typename T>
__device__ __forceinline__ void load4(float (&to)[4], const T *p, int c, int cols, bool whole) {
    struct alignas(4 * sizeof(T)) Four {
        T x[4];
    };
    if (whole) {
        if (c < cols) {
            const Four f = *reinterpret_cast<const Four *>(p + c);
#pragma unroll
            for (int i = 0; i < 4; i++) to[i] = (float)f.x[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) to[i] = 0.f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) to[i] = c + i < cols ? (float)p[c + i] : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store4(T *p, const float (&from)[4], int c, int cols, bool whole) {
    struct alignas(4 * sizeof(T)) Four {
        T x[4];
    };
    if (whole) {
        if (c >= cols) return;
        Four f;
#pragma unroll
        for (int i = 0; i < 4; i++) f.x[i] = (T)from[i];
        *reinterpret_cast<Four *>(p + c) = f;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (c + i < cols) p[c + i] = (T)from[i];
    }
}
// a parameter's columns, or `none` without it
__device__ __forceinline__ void param4(float (&to)[4], const float *p, float none, int c, int cols, bool whole) {
    if (p) load4(to, p, c, cols, whole);
    else {
#pragma unroll
        for (int i = 0; i < 4; i++) to[i] = none;
    }
}

// Sums over the lanes of a row, in all of them
template <int WAVES, int K>
__device__ __forceinline__ void row_sums(float (&x)[K], float (*sh)[16][3], int &turn) {
#pragma unroll
    for (int k = 0; k < K; k++) {
        float a = x[k], b = a;
        swap32(a, b);
        a += b, b = a;
        swap16(a, b);
        a += b;
        a += dpp<kRowRor8>(a);
        a += dpp<kRowRor4>(a);
        a += dpp<kQuadXor2>(a);
        a += dpp<kQuadXor1>(a);
        x[k] = a;
    }
    if constexpr (WAVES > 1) {
        const int wave = threadIdx.x / 64;
        float(*const s)[3] = sh[turn];
        turn ^= 1;      // the other half next time: one barrier a sum
        if (threadIdx.x % 64 == 0)
#pragma unroll
            for (int k = 0; k < K; k++) s[wave][k] = x[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; k++) {
            x[k] = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; w++) x[k] += s[w][k];
        }
    }
}

// act(g) and its slope
__device__ __forceinline__ float act_of(float g, int act) {
    if (act == FWP_ACT_NONE) return g;
    const float s = sigmoid(g);
    return act == FWP_ACT_SILU ? silu(g, s) : s;
}
__device__ __forceinline__ float act_slope(float g, int act) {
    if (act == FWP_ACT_NONE) return 1.f;
    const float s = sigmoid(g);
    return act == FWP_ACT_SILU ? silu_slope(g, s) : s * sigmoid(-g);
}

template <int NV>
struct Row {
    float x[NV][4];
};

// mean and 1 / spread of a row held in registers (columns beyond `cols` are left out)
template <int WAVES, int NV>
__device__ __forceinline__ float2 statistics(const Row<NV> &v, bool rms, int cols, float eps, int lane, float (*sh)[16][3], int &turn) {
    float mean = 0.f;
    if (!rms) {
        float s[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) s[0] += v.x[i][k];      // zeros beyond
        row_sums<WAVES, 1>(s, sh, turn);
        mean = s[0] / cols;
    }
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float d = v.x[i][k] - mean;
            s[0] += 4 * (lane + 64 * WAVES * i) + k < cols ? d * d : 0.f;
        }
    row_sums<WAVES, 1>(s, sh, turn);
    return make_float2(mean, 1.f / sqrtf(s[0] / cols + eps));
}

constexpr int rows_at_once(int waves) { return waves == 1 ? 4 : 1; }
constexpr int threads_of(int waves) { return waves == 1 ? 256 : 64 * waves; }

template <typename T, typename S, int WAVES, int NV>
__global__ __launch_bounds__(threads_of(WAVES)) void k_rnorm_fwd(fwp_norm_args a, S *__restrict__ r_out, T *__restrict__ n_out,
                                                                 float *__restrict__ stats, bool whole) {
    __shared__ float sh[2][16][3];
    int turn = 0;
    const int lane = threadIdx.x % (64 * WAVES);
    const int64_t row = (int64_t)blockIdx.x * rows_at_once(WAVES) + threadIdx.x / (64 * WAVES);
    if (row >= a.rows) return;      // all lanes of a row together, and the whole workgroup where it has one row
    const int64_t at = row * a.cols;
    Row<NV> y, r;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = 4 * (lane + 64 * WAVES * i);
        load4(y.x[i], static_cast<const T *>(a.y) + at, c, a.cols, whole);
        load4(r.x[i], static_cast<const S *>(a.x) + at, c, a.cols, whole);
    }
    float2 sy = make_float2(0.f, 1.f), sr = sy;
    if (a.after_weight) sy = statistics<WAVES, NV>(y, a.rms, a.cols, a.eps, lane, sh, turn);
    const float row_gate = a.gate && a.gate_rows ? act_of((float)static_cast<const T *>(a.gate)[row], a.act) : 1.f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = 4 * (lane + 64 * WAVES * i);
        float w[4], b[4], sc[4], g[4];
        param4(w, a.after_weight, 1.f, c, a.cols, whole);
        param4(b, a.after_bias, 0.f, c, a.cols, whole);
        param4(sc, a.scale, 1.f, c, a.cols, whole);
        if (a.gate && !a.gate_rows) load4(g, static_cast<const T *>(a.gate) + at, c, a.cols, whole);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float act = a.gate && !a.gate_rows ? act_of(g[k], a.act) : row_gate;
            const float u = fmaf((y.x[i][k] - sy.x) * sy.y, w[k], b[k]);
            r.x[i][k] = c + k < a.cols ? fmaf(sc[k] * act, u, r.x[i][k]) : 0.f;
        }
        store4(r_out + at, r.x[i], c, a.cols, whole);
    }
    if (a.before_weight) {
        sr = statistics<WAVES, NV>(r, a.rms, a.cols, a.eps, lane, sh, turn);
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = 4 * (lane + 64 * WAVES * i);
            float w[4], b[4], o[4];
            param4(w, a.before_weight, 1.f, c, a.cols, whole);
            param4(b, a.before_bias, 0.f, c, a.cols, whole);
#pragma unroll
            for (int k = 0; k < 4; k++) o[k] = fmaf((r.x[i][k] - sr.x) * sr.y, w[k], b[k]);
            store4(n_out + at, o, c, a.cols, whole);
        }
    }
    if (stats && lane == 0) *reinterpret_cast<float4 *>(stats + 4 * row) = make_float4(sy.x, sy.y, sr.x, sr.y);
}

// parts [blocks][scale, after weight, after bias, before weight, before bias][cols]
template <typename T, typename S, int WAVES, int NV>
__global__ __launch_bounds__(threads_of(WAVES)) void k_rnorm_bwd(fwp_norm_args a, const float *__restrict__ stats, const S *__restrict__ gr,
                                                                 const T *__restrict__ gn, T *__restrict__ gy, S *__restrict__ gx,
                                                                 T *__restrict__ gg, float *__restrict__ parts, bool whole) {
    __shared__ float sh[2][16][3];
    __shared__ float cs[4][64 * 4];
    int turn = 0;
    const int lane = threadIdx.x % (64 * WAVES);
    const bool element_gate = a.gate && !a.gate_rows, after = a.after_weight != nullptr;
    float col[kParams][NV][4] = {};
    const int64_t step = (int64_t)gridDim.x * rows_at_once(WAVES);
    for (int64_t row = (int64_t)blockIdx.x * rows_at_once(WAVES) + threadIdx.x / (64 * WAVES); row < a.rows; row += step) {
        const int64_t at = row * a.cols;
        const float4 st = *reinterpret_cast<const float4 *>(stats + 4 * row);
        Row<NV> y, x, g, dr, h;     // y: normalised (or itself); x: r normalised; h: gn times its weight, then du times its weight
        float sums[3] = {};
        const float row_gate = a.gate && a.gate_rows ? (float)static_cast<const T *>(a.gate)[row] : 0.f,
                    row_act = a.gate && a.gate_rows ? act_of(row_gate, a.act) : 1.f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = 4 * (lane + 64 * WAVES * i);
            load4(y.x[i], static_cast<const T *>(a.y) + at, c, a.cols, whole);
            load4(x.x[i], static_cast<const S *>(a.x) + at, c, a.cols, whole);
            if (element_gate) load4(g.x[i], static_cast<const T *>(a.gate) + at, c, a.cols, whole);
            if (gr) load4(dr.x[i], gr + at, c, a.cols, whole);
            else
#pragma unroll
                for (int k = 0; k < 4; k++) dr.x[i][k] = 0.f;
            if (gn && a.before_weight) load4(h.x[i], gn + at, c, a.cols, whole);
            else
#pragma unroll
                for (int k = 0; k < 4; k++) h.x[i][k] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = 4 * (lane + 64 * WAVES * i);
            float w[4], b[4], sc[4], bw[4];
            param4(w, a.after_weight, 1.f, c, a.cols, whole);
            param4(b, a.after_bias, 0.f, c, a.cols, whole);
            param4(sc, a.scale, 1.f, c, a.cols, whole);
            param4(bw, a.before_weight, 1.f, c, a.cols, whole);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                y.x[i][k] = c + k < a.cols ? (y.x[i][k] - st.x) * st.y : 0.f;
                const float act = element_gate ? act_of(g.x[i][k], a.act) : row_act, u = fmaf(y.x[i][k], w[k], b[k]);
                const float r = fmaf(sc[k] * act, u, x.x[i][k]);
                x.x[i][k] = c + k < a.cols ? (r - st.z) * st.w : 0.f;
                col[3][i][k] = fmaf(h.x[i][k], x.x[i][k], col[3][i][k]);
                col[4][i][k] += h.x[i][k];
                h.x[i][k] *= bw[k];
                sums[0] += h.x[i][k];
                sums[1] = fmaf(h.x[i][k], x.x[i][k], sums[1]);
            }
        }
        if (a.before_weight) row_sums<WAVES, 3>(sums, sh, turn);
        const float m0 = a.rms ? 0.f : sums[0] / a.cols, m1 = sums[1] / a.cols;
        sums[0] = sums[1] = sums[2] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = 4 * (lane + 64 * WAVES * i);
            float w[4], b[4], sc[4], o[4];
            param4(w, a.after_weight, 1.f, c, a.cols, whole);
            param4(b, a.after_bias, 0.f, c, a.cols, whole);
            param4(sc, a.scale, 1.f, c, a.cols, whole);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (a.before_weight) dr.x[i][k] = fmaf(st.w, fmaf(-x.x[i][k], m1, h.x[i][k] - m0), dr.x[i][k]);
                const float d = c + k < a.cols ? dr.x[i][k] : 0.f, act = element_gate ? act_of(g.x[i][k], a.act) : row_act;
                const float u = fmaf(y.x[i][k], w[k], b[k]), du = d * sc[k] * act;
                col[0][i][k] = fmaf(d * act, u, col[0][i][k]);
                col[1][i][k] = fmaf(du, y.x[i][k], col[1][i][k]);
                col[2][i][k] += du;
                const float slope = d * sc[k] * u;      // of act
                o[k] = element_gate ? slope * act_slope(g.x[i][k], a.act) : 0.f;
                h.x[i][k] = du * w[k];
                sums[0] += h.x[i][k];
                sums[1] = fmaf(h.x[i][k], y.x[i][k], sums[1]);
                sums[2] += slope;
            }
            store4(gx + at, dr.x[i], c, a.cols, whole);
            if (gg && element_gate) store4(gg + at, o, c, a.cols, whole);
        }
        if (after || (gg && a.gate_rows)) row_sums<WAVES, 3>(sums, sh, turn);
        const float n0 = a.rms || !after ? 0.f : sums[0] / a.cols, n1 = after ? sums[1] / a.cols : 0.f;
        if (gg && a.gate_rows && lane == 0) gg[row] = (T)(sums[2] * act_slope(row_gate, a.act));
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = 4 * (lane + 64 * WAVES * i);
            float o[4];
#pragma unroll
            for (int k = 0; k < 4; k++) o[k] = st.y * fmaf(-y.x[i][k], n1, h.x[i][k] - n0);
            store4(gy + at, o, c, a.cols, whole);
        }
    }
    // the column sums of this workgroup
#pragma unroll
    for (int q = 0; q < kParams; q++)
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = 4 * (lane + 64 * WAVES * i);
            float o[4];
#pragma unroll
            for (int k = 0; k < 4; k++) o[k] = col[q][i][k];
            if constexpr (WAVES == 1) {
                __syncthreads();
#pragma unroll
                for (int k = 0; k < 4; k++) cs[threadIdx.x / 64][4 * lane + k] = o[k];
                __syncthreads();
                if (threadIdx.x >= 64) continue;
#pragma unroll
                for (int k = 0; k < 4; k++) o[k] = (cs[0][4 * lane + k] + cs[1][4 * lane + k]) + (cs[2][4 * lane + k] + cs[3][4 * lane + k]);
            }
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (c + k < a.cols) parts[((int64_t)blockIdx.x * kParams + q) * a.cols + c + k] = o[k];
        }
}

// The workgroups' sums added up in a fixed order: 64 columns and four slices of the workgroups to a workgroup
__global__ __launch_bounds__(256) void k_rnorm_params(const float *__restrict__ parts, fwp_norm_grads g, int blocks, int cols) {
    __shared__ float sh[4][64];
    const int64_t per = (int64_t)kParams * cols, i = (int64_t)blockIdx.x * 64 + threadIdx.x % 64;
    const int slice = threadIdx.x / 64;
    float x = 0.f;
    if (i < per)
        for (int k = slice; k < blocks; k += 4) x += parts[k * per + i];
    sh[slice][threadIdx.x % 64] = x;
    __syncthreads();
    if (slice || i >= per) return;
    x = (sh[0][threadIdx.x] + sh[1][threadIdx.x]) + (sh[2][threadIdx.x] + sh[3][threadIdx.x]);
    const int q = (int)(i / cols);
    float *const to = q == 0 ? g.gscale : q == 1 ? g.gafter_weight : q == 2 ? g.gafter_bias : q == 3 ? g.gbefore_weight : g.gbefore_bias;
    if (to) to[i % cols] = x;
}

template <typename F>
void by_width(int cols, F f) {
    using std::integral_constant;
    if (cols <= 256) f(integral_constant<int, 1>(), integral_constant<int, 1>());
    else if (cols <= 512) f(integral_constant<int, 1>(), integral_constant<int, 2>());
    else if (cols <= 1024) f(integral_constant<int, 1>(), integral_constant<int, 4>());
    else if (cols <= 2048) f(integral_constant<int, 4>(), integral_constant<int, 2>());
    else if (cols <= 4096) f(integral_constant<int, 8>(), integral_constant<int, 2>());
    else f(integral_constant<int, 16>(), integral_constant<int, 2>());
}

// f(T(), S()): the block's type and the stream's
template <typename F>
void by_types(const fwp_norm_args &a, F f) {
    by_type(a.type, [&](auto t) {
        if (a.stream_type == FWP_F32) f(t, float());
        else f(t, t);
    });
}

bool aligned(const void *p, int to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Four columns at once for every tensor of a call?
bool whole_rows(const fwp_norm_args &a, std::initializer_list<const void *> blocks, std::initializer_list<const void *> streams,
                std::initializer_list<const void *> params) {
    if (a.cols % 4) return false;
    const int t = a.type == FWP_F32 ? 16 : 8, s = a.stream_type == FWP_F32 ? 16 : 8;
    for (const void *p : blocks)
        if (!aligned(p, t)) return false;
    for (const void *p : streams)
        if (!aligned(p, s)) return false;
    for (const void *p : params)
        if (!aligned(p, 16)) return false;
    return true;
}

int blocks_of(int rows, int cols) {
    const int at_once = cols <= 1024 ? 4 : 1;
    return (int)std::min<int64_t>(((int64_t)rows + at_once - 1) / at_once, kBlocks);
}

}  // namespace

int64_t residual_norm_workspace(int rows, int cols) { return (int64_t)blocks_of(rows, cols) * kParams * cols; }

int residual_norm_fwd(const fwp_norm_args &a, void *r, void *n, float *stats, hipStream_t s) {
    const bool whole = whole_rows(a, {a.y, a.gate_rows ? nullptr : a.gate, n}, {a.x, r},
                                  {a.scale, a.after_weight, a.after_bias, a.before_weight, a.before_bias});
    by_types(a, [&](auto t, auto st) {
        using T = decltype(t);
        using S = decltype(st);
        by_width(a.cols, [&](auto w, auto v) {
            constexpr int WAVES = decltype(w)::value, NV = decltype(v)::value;
            const unsigned grid = (unsigned)(((int64_t)a.rows + rows_at_once(WAVES) - 1) / rows_at_once(WAVES));
            hipLaunchKernelGGL((k_rnorm_fwd<T, S, WAVES, NV>), dim3(grid), dim3(threads_of(WAVES)), 0, s, a, (S *)r, (T *)n, stats, whole);
        });
    });
    return (int)hipGetLastError();
}

int residual_norm_bwd(const fwp_norm_args &a, const float *stats, const void *gr, const void *gn, const fwp_norm_grads &g, float *workspace,
                      hipStream_t s) {
    const bool whole = whole_rows(a, {a.y, a.gate_rows ? nullptr : a.gate, gn, g.gy, a.gate_rows ? nullptr : g.ggate}, {a.x, gr, g.gx},
                                  {a.scale, a.after_weight, a.after_bias, a.before_weight});
    const int blocks = blocks_of(a.rows, a.cols);
    by_types(a, [&](auto t, auto st) {
        using T = decltype(t);
        using S = decltype(st);
        by_width(a.cols, [&](auto w, auto v) {
            constexpr int WAVES = decltype(w)::value, NV = decltype(v)::value;
            hipLaunchKernelGGL((k_rnorm_bwd<T, S, WAVES, NV>), dim3(blocks), dim3(threads_of(WAVES)), 0, s, a, stats, (const S *)gr, (const T *)gn,
                               (T *)g.gy, (S *)g.gx, (T *)g.ggate, workspace, whole);
        });
    });
    if (g.gscale || g.gafter_weight || g.gafter_bias || g.gbefore_weight || g.gbefore_bias)
        hipLaunchKernelGGL(k_rnorm_params, dim3((kParams * a.cols + 63) / 64), dim3(256), 0, s, workspace, g, blocks, a.cols);
    return (int)hipGetLastError();
}

}  // namespace fwp
