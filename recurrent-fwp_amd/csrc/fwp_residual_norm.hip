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
// second kernel adds the workgroups' sums in a fixed order.  Bound by memory: 32768 x 256 fp32 with a gate, forward 33 us (168 MB, 5.1 TB/s), adjoint 51 (268 MB, 5.2 TB/s)
// and its sums 5; 16384 x 4096 bf16 on an fp32 stream, RMS, 144 us (0.81 GB, 5.6 TB/s), 225-249 (1.2 GB, 4.8-5.4 TB/s) and 8.
#include "fwp_elements.hpp"
#include "fwp_wave.hpp"

#include <algorithm>
#include <type_traits>

namespace fwp {
namespace {

constexpr int kParams = 5;

template <typename T>
struct alignas(4 * sizeof(T)) Four {
    T x[4];
};

// How rows lie: kWhole, all rows and parameters are aligned for reading four elements at once, and `cols` is a multiple of four; kRagged, anything else
// of four columns or more: the same loads without the alignment, and the lane that the row's end cuts reads its last four and moves them
// up; kTiny, fewer columns, one by one.  A lane has four neighbouring columns either way, so that a row's numbers do not depend on where it lies.
enum Lie { kWhole, kRagged, kTiny };

template <int WAVES>
__device__ __forceinline__ int column(int lane, int i, int k) {
    return 4 * (lane + 64 * WAVES * i) + k;
}
// Element c of a row: a 32-bit offset of bytes from an address that all lanes share, which costs no 64-bit sum
template <typename T>
__device__ __forceinline__ T *within(T *row, int c) {
    using Byte = std::conditional_t<std::is_const_v<T>, const char, char>;
    return reinterpret_cast<T *>(reinterpret_cast<Byte *>(row) + (unsigned)c * (unsigned)sizeof(T));
}
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Anywhere {
    T x[4];
};
// Four elements as they come.  Every lane loads, those beyond the row its last elements, which nobody uses: a branch around a load would wait for it at its end.
template <int LIE, int WAVES, typename T>
__device__ __forceinline__ Four<T> raw4(const T *p, int lane, int i, int cols) {
    const int c = column<WAVES>(lane, i, 0);
    if constexpr (LIE == kWhole) return *reinterpret_cast<const Four<T> *>(within(p, min(c, cols - 4)));
    Four<T> f;
    if constexpr (LIE == kRagged) {
        const Anywhere<T> u = *reinterpret_cast<const Anywhere<T> *>(within(p, min(c, cols - 4)));
#pragma unroll
        for (int k = 0; k < 4; k++) f.x[k] = u.x[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) f.x[k] = *within(p, min(c + k, cols - 1));
    }
    return f;
}
template <int LIE, int WAVES, typename T>
__device__ __forceinline__ void convert4(float (&to)[4], const Four<T> &f, int lane, int i, int cols) {
#pragma unroll
    for (int k = 0; k < 4; k++) to[k] = (float)f.x[k];
    if constexpr (LIE == kRagged) {
        const int s = column<WAVES>(lane, i, 0) - (cols - 4);       // how far the four that were read lie before the ones wanted
        to[0] = s == 1 ? to[1] : s == 2 ? to[2] : s == 3 ? to[3] : to[0];
        to[1] = s == 1 ? to[2] : s == 2 ? to[3] : to[1];
        to[2] = s == 1 ? to[3] : to[2];
    }
}
template <int LIE, int WAVES, typename T>
__device__ __forceinline__ void load4(float (&to)[4], const T *p, int lane, int i, int cols) {
    convert4<LIE, WAVES>(to, raw4<LIE, WAVES>(p, lane, i, cols), lane, i, cols);
}
template <int LIE, int WAVES, typename T>
__device__ __forceinline__ void store4(T *p, const float (&from)[4], int lane, int i, int cols) {
    const int c = column<WAVES>(lane, i, 0);
    if constexpr (LIE == kWhole) {
        Four<T> f;
#pragma unroll
        for (int k = 0; k < 4; k++) f.x[k] = (T)from[k];
        if (c < cols) *reinterpret_cast<Four<T> *>(within(p, c)) = f;
        return;
    }
    Anywhere<T> f;
#pragma unroll
    for (int k = 0; k < 4; k++) f.x[k] = (T)from[k];
    if (LIE == kRagged && c + 3 < cols) *reinterpret_cast<Anywhere<T> *>(within(p, c)) = f;
    else
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (c + k < cols) *within(p, c + k) = f.x[k];
}
// a parameter's columns, or `none` without it
template <int LIE, int WAVES>
__device__ __forceinline__ void param4(float (&to)[4], const float *p, float none, int lane, int i, int cols) {
    if (p) load4<LIE, WAVES>(to, p, lane, i, cols);
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
template <int LIE, int WAVES, int NV>
__device__ __forceinline__ float2 statistics(const Row<NV> &v, bool rms, int cols, float eps, int lane, float (*sh)[16][3], int &turn) {
    float mean = 0.f;
    if (!rms) {
        float s[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) s[0] += column<WAVES>(lane, i, k) < cols ? v.x[i][k] : 0.f;
        row_sums<WAVES, 1>(s, sh, turn);
        mean = s[0] / cols;
    }
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float d = v.x[i][k] - mean;
            s[0] += column<WAVES>(lane, i, k) < cols ? d * d : 0.f;
        }
    row_sums<WAVES, 1>(s, sh, turn);
    return make_float2(mean, 1.f / sqrtf(s[0] / cols + eps));
}

constexpr int rows_at_once(int waves) { return waves == 1 ? 4 : 1; }
constexpr int threads_of(int waves) { return waves == 1 ? 256 : 64 * waves; }
// which of a workgroup's rows this is: the same for the lanes of a wave, and known to be
template <int WAVES>
__device__ __forceinline__ int row_at_once() {
    return WAVES == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : 0;
}

template <typename T, typename S, int WAVES, int NV, int LIE>
__global__ __launch_bounds__(threads_of(WAVES)) void k_rnorm_fwd(fwp_norm_args a, S *__restrict__ r_out, T *__restrict__ n_out,
                                                                 float *__restrict__ stats) {
    __shared__ float sh[2][16][3];
    int turn = 0;
    const int lane = threadIdx.x % (64 * WAVES);
    const int64_t row = (int64_t)blockIdx.x * rows_at_once(WAVES) + row_at_once<WAVES>();
    if (row >= a.rows) return;      // all lanes of a row together, and the whole workgroup where it has one row
    const int64_t at = row * a.cols;
    const bool element_gate = a.gate && !a.gate_rows;
    Row<NV> y, r, gate;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        load4<LIE, WAVES>(y.x[i], static_cast<const T *>(a.y) + at, lane, i, a.cols);
        load4<LIE, WAVES>(r.x[i], static_cast<const S *>(a.x) + at, lane, i, a.cols);
        if (element_gate) load4<LIE, WAVES>(gate.x[i], static_cast<const T *>(a.gate) + at, lane, i, a.cols);
    }
    float2 sy = make_float2(0.f, 1.f), sr = sy;
    if (a.after_weight) sy = statistics<LIE, WAVES, NV>(y, a.rms, a.cols, a.eps, lane, sh, turn);
    const float row_gate = a.gate && a.gate_rows ? act_of((float)static_cast<const T *>(a.gate)[row], a.act) : 1.f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        float w[4], b[4], sc[4];
        param4<LIE, WAVES>(w, a.after_weight, 1.f, lane, i, a.cols);
        param4<LIE, WAVES>(b, a.after_bias, 0.f, lane, i, a.cols);
        param4<LIE, WAVES>(sc, a.scale, 1.f, lane, i, a.cols);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float act = element_gate ? act_of(gate.x[i][k], a.act) : row_gate;
            const float u = fmaf((y.x[i][k] - sy.x) * sy.y, w[k], b[k]);
            r.x[i][k] = fmaf(sc[k] * act, u, r.x[i][k]);
        }
        store4<LIE, WAVES>(r_out + at, r.x[i], lane, i, a.cols);
    }
    if (a.before_weight) {
        sr = statistics<LIE, WAVES, NV>(r, a.rms, a.cols, a.eps, lane, sh, turn);
#pragma unroll
        for (int i = 0; i < NV; i++) {
            float w[4], b[4], o[4];
            param4<LIE, WAVES>(w, a.before_weight, 1.f, lane, i, a.cols);
            param4<LIE, WAVES>(b, a.before_bias, 0.f, lane, i, a.cols);
#pragma unroll
            for (int k = 0; k < 4; k++) o[k] = fmaf((r.x[i][k] - sr.x) * sr.y, w[k], b[k]);
            store4<LIE, WAVES>(n_out + at, o, lane, i, a.cols);
        }
    }
    if (stats && lane == 0) *reinterpret_cast<float4 *>(stats + 4 * row) = make_float4(sy.x, sy.y, sr.x, sr.y);
}

// A row of the adjoint's inputs as they come from memory
template <typename T, typename S, int NV>
struct Inputs {
    Four<T> y[NV], gate[NV], gn[NV];
    Four<S> x[NV], gr[NV];
    float4 stats;
    float row_gate;
};

// parts [blocks][scale, after weight, after bias, before weight, before bias][cols]; BIAS: are there biases?  The next row is on its way while one is
// worked on, and the parameters' columns stay in registers where there is room for them.
template <typename T, typename S, int WAVES, int NV, bool BIAS, int LIE>
__global__ __launch_bounds__(threads_of(WAVES)) void k_rnorm_bwd(fwp_norm_args a, const float *__restrict__ stats, const S *__restrict__ gr,
                                                                 const T *__restrict__ gn, T *__restrict__ gy, S *__restrict__ gx,
                                                                 T *__restrict__ gg, float *__restrict__ parts) {
    constexpr bool HELD = NV <= 2, AHEAD = HELD;      // sixteen columns to a lane leave no registers for either
    constexpr int COLS = BIAS ? 5 : 3;      // scale, after weight, before weight, the biases
    __shared__ float sh[2][16][3];
    __shared__ float cs[4][64 * 4];
    __shared__ float4 kept[HELD ? 1 : 3][HELD ? 1 : NV][HELD ? 1 : threads_of(WAVES)];     // the columns' sums of sixteen columns a lane, which alone reads them
    int turn = 0;
    const int lane = threadIdx.x % (64 * WAVES);
    const bool element_gate = a.gate && !a.gate_rows, after = a.after_weight != nullptr, before = a.before_weight != nullptr,
               has_gn = gn && before;
    float col[COLS][HELD ? NV : 1][4] = {}, more[HELD || !BIAS ? 1 : 2][HELD ? 1 : NV][4] = {}, aw[HELD ? NV : 1][4], ab[HELD && BIAS ? NV : 1][4], sc[HELD ? NV : 1][4], bw[HELD ? NV : 1][4];
    const auto params = [&](int i, int to) {
        param4<LIE, WAVES>(aw[to], a.after_weight, 1.f, lane, i, a.cols);
        if constexpr (BIAS) param4<LIE, WAVES>(ab[to], a.after_bias, 0.f, lane, i, a.cols);
        param4<LIE, WAVES>(sc[to], a.scale, 1.f, lane, i, a.cols);
        param4<LIE, WAVES>(bw[to], a.before_weight, 1.f, lane, i, a.cols);
    };
    if constexpr (HELD) {
#pragma unroll
        for (int i = 0; i < NV; i++) params(i, i);
    } else {
#pragma unroll
        for (int q = 0; q < 3; q++)
#pragma unroll
            for (int i = 0; i < NV; i++) kept[q][i][threadIdx.x] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    // column sum q (scale, after weight, before weight, after bias, before bias) of turn i
    const auto add = [&](int q, int i, const float (&v)[4]) {
        if constexpr (HELD) {
#pragma unroll
            for (int k = 0; k < 4; k++) col[q][i][k] += v[k];
        } else if (q < 3) {
            float4 t = kept[q][i][threadIdx.x];
            t.x += v[0], t.y += v[1], t.z += v[2], t.w += v[3];
            kept[q][i][threadIdx.x] = t;
        } else if constexpr (BIAS) {
#pragma unroll
            for (int k = 0; k < 4; k++) more[q - 3][i][k] += v[k];
        }
    };
    // what is not there is read from y or x, and not used
    const T *const gate_at = static_cast<const T *>(element_gate ? a.gate : a.y), *const gn_at = has_gn ? gn : static_cast<const T *>(a.y);
    const S *const gr_at = gr ? gr : static_cast<const S *>(a.x);
    Inputs<T, S, NV> in;
    const auto fetch = [&](int64_t row) {
        const int64_t at = row * a.cols;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            in.y[i] = raw4<LIE, WAVES>(static_cast<const T *>(a.y) + at, lane, i, a.cols);
            in.x[i] = raw4<LIE, WAVES>(static_cast<const S *>(a.x) + at, lane, i, a.cols);
            in.gate[i] = raw4<LIE, WAVES>(gate_at + at, lane, i, a.cols);
            in.gr[i] = raw4<LIE, WAVES>(gr_at + at, lane, i, a.cols);
            in.gn[i] = raw4<LIE, WAVES>(gn_at + at, lane, i, a.cols);
        }
        in.stats = *reinterpret_cast<const float4 *>(stats + 4 * row);
        in.row_gate = (float)(a.gate && a.gate_rows ? static_cast<const T *>(a.gate)[row] : gate_at[at]);
    };
    const int64_t step = (int64_t)gridDim.x * rows_at_once(WAVES);
    int64_t row = (int64_t)blockIdx.x * rows_at_once(WAVES) + row_at_once<WAVES>();
    if (AHEAD && row < a.rows) fetch(row);
    for (; row < a.rows; row += step) {
        const int64_t at = row * a.cols;
        if constexpr (!AHEAD) {
            in.stats = *reinterpret_cast<const float4 *>(stats + 4 * row);
            in.row_gate = (float)(a.gate && a.gate_rows ? static_cast<const T *>(a.gate)[row] : gate_at[at]);
        }
        const float4 st = in.stats;
        Row<NV> y, x, g, dr, h;     // y: normalised (or itself); x: r normalised; h: gn times its weight, then du times its weight
        float sums[3] = {};
        const float row_gate = a.gate && a.gate_rows ? in.row_gate : 0.f, row_act = a.gate && a.gate_rows ? act_of(row_gate, a.act) : 1.f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            if constexpr (AHEAD) {
                convert4<LIE, WAVES>(y.x[i], in.y[i], lane, i, a.cols);
                convert4<LIE, WAVES>(x.x[i], in.x[i], lane, i, a.cols);
                convert4<LIE, WAVES>(g.x[i], in.gate[i], lane, i, a.cols);
                convert4<LIE, WAVES>(dr.x[i], in.gr[i], lane, i, a.cols);
                convert4<LIE, WAVES>(h.x[i], in.gn[i], lane, i, a.cols);
            } else {
                load4<LIE, WAVES>(y.x[i], static_cast<const T *>(a.y) + at, lane, i, a.cols);
                load4<LIE, WAVES>(x.x[i], static_cast<const S *>(a.x) + at, lane, i, a.cols);
                load4<LIE, WAVES>(g.x[i], gate_at + at, lane, i, a.cols);
                load4<LIE, WAVES>(dr.x[i], gr_at + at, lane, i, a.cols);
                load4<LIE, WAVES>(h.x[i], gn_at + at, lane, i, a.cols);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                g.x[i][k] = element_gate ? g.x[i][k] : 0.f;
                dr.x[i][k] = gr ? dr.x[i][k] : 0.f;
                h.x[i][k] = has_gn && column<WAVES>(lane, i, k) < a.cols ? h.x[i][k] : 0.f;
            }
        }
        if (AHEAD) fetch(row + step < a.rows ? row + step : row);
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int q = HELD ? i : 0;
            float v0[4], v1[4];
            if constexpr (!HELD) {
                __builtin_amdgcn_sched_barrier(0);      // one turn's parameters at a time
                params(i, 0);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                y.x[i][k] = column<WAVES>(lane, i, k) < a.cols ? (y.x[i][k] - st.x) * st.y : 0.f;
                const float act = element_gate ? act_of(g.x[i][k], a.act) : row_act, u = fmaf(y.x[i][k], aw[q][k], BIAS ? ab[q][k] : 0.f);
                const float r = fmaf(sc[q][k] * act, u, x.x[i][k]);
                x.x[i][k] = column<WAVES>(lane, i, k) < a.cols ? (r - st.z) * st.w : 0.f;
                v0[k] = h.x[i][k] * x.x[i][k], v1[k] = h.x[i][k];
                h.x[i][k] *= bw[q][k];
                sums[0] += h.x[i][k];
                sums[1] = fmaf(h.x[i][k], x.x[i][k], sums[1]);
            }
            add(2, i, v0);
            if constexpr (BIAS) add(4, i, v1);
        }
        if (before) row_sums<WAVES, 3>(sums, sh, turn);
        const float m0 = a.rms ? 0.f : sums[0] / a.cols, m1 = sums[1] / a.cols;
        sums[0] = sums[1] = sums[2] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int q = HELD ? i : 0;
            float o[4], v0[4], v1[4], v3[4];
            if constexpr (!HELD) {
                __builtin_amdgcn_sched_barrier(0);      // one turn's parameters at a time
                params(i, 0);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (before) dr.x[i][k] = fmaf(st.w, fmaf(-x.x[i][k], m1, h.x[i][k] - m0), dr.x[i][k]);
                const float d = column<WAVES>(lane, i, k) < a.cols ? dr.x[i][k] : 0.f, act = element_gate ? act_of(g.x[i][k], a.act) : row_act;
                const float u = fmaf(y.x[i][k], aw[q][k], BIAS ? ab[q][k] : 0.f), du = d * sc[q][k] * act;
                v0[k] = d * act * u, v1[k] = du * y.x[i][k], v3[k] = du;
                const float slope = d * sc[q][k] * u;      // of act
                o[k] = element_gate ? slope * act_slope(g.x[i][k], a.act) : 0.f;
                h.x[i][k] = du * aw[q][k];
                sums[0] += h.x[i][k];
                sums[1] = fmaf(h.x[i][k], y.x[i][k], sums[1]);
                sums[2] += slope;
            }
            add(0, i, v0), add(1, i, v1);
            if constexpr (BIAS) add(3, i, v3);
            store4<LIE, WAVES>(gx + at, dr.x[i], lane, i, a.cols);
            if (gg && element_gate) store4<LIE, WAVES>(gg + at, o, lane, i, a.cols);
        }
        if (after || (gg && a.gate_rows)) row_sums<WAVES, 3>(sums, sh, turn);
        const float n0 = a.rms || !after ? 0.f : sums[0] / a.cols, n1 = after ? sums[1] / a.cols : 0.f;
        if (gg && a.gate_rows && lane == 0) gg[row] = (T)(sums[2] * act_slope(row_gate, a.act));
#pragma unroll
        for (int i = 0; i < NV; i++) {
            float o[4];
#pragma unroll
            for (int k = 0; k < 4; k++) o[k] = after ? st.y * fmaf(-y.x[i][k], n1, h.x[i][k] - n0) : h.x[i][k];      // without a norm, not infinity times zero
            store4<LIE, WAVES>(gy + at, o, lane, i, a.cols);
        }
    }
    // the column sums of this workgroup, in the order scale, after weight, after bias, before weight, before bias
#pragma unroll
    for (int q = 0; q < COLS; q++)
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int to = q < 2 ? q : q == 2 ? 3 : q == 3 ? 2 : 4;
            float o[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if constexpr (HELD) o[k] = col[q][i][k];
                else if (q < 3) o[k] = reinterpret_cast<const float *>(&kept[q][i][threadIdx.x])[k];
                else o[k] = more[BIAS ? q - 3 : 0][i][k];
            }
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
                if (column<WAVES>(lane, i, k) < a.cols) parts[((int64_t)blockIdx.x * kParams + to) * a.cols + column<WAVES>(lane, i, k)] = o[k];
        }
}

// The workgroups' sums added up in a fixed order: 16 columns and 64 slices of the workgroups to a workgroup (four slices took 34 us for 512
// workgroups' 256 columns: too few loads at once)
__global__ __launch_bounds__(1024) void k_rnorm_params(const float *__restrict__ parts, fwp_norm_grads g, int blocks, int cols) {
    __shared__ float sh[64][17];
    const int64_t per = (int64_t)kParams * cols, i = (int64_t)blockIdx.x * 16 + threadIdx.x % 16;
    const int slice = threadIdx.x / 16, q = (int)(min(i, per - 1) / cols);
    float *const to = q == 0 ? g.gscale : q == 1 ? g.gafter_weight : q == 2 ? g.gafter_bias : q == 3 ? g.gbefore_weight : g.gbefore_bias;
    float x = 0.f;
    if (i < per && to)
#pragma unroll 8
        for (int k = slice; k < blocks; k += 64) x += parts[k * per + i];
    sh[slice][threadIdx.x % 16] = x;
    __syncthreads();
    if (threadIdx.x >= 256) return;
    const int c = threadIdx.x % 16, s = threadIdx.x / 16;
    x = (sh[4 * s][c] + sh[4 * s + 1][c]) + (sh[4 * s + 2][c] + sh[4 * s + 3][c]);
    __syncthreads();
    sh[s][c] = x;
    __syncthreads();
    if (s || i >= per || !to) return;
    x = 0.f;
#pragma unroll
    for (int k = 0; k < 16; k++) x += sh[k][c];
    to[i % cols] = x;
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

// The adjoint's, with the columns' sums in registers: 4096 columns took 230 us with eight columns a lane and 472 with four (16384 rows, bf16, RMS), since
// sixteen waves leave 128 registers to a lane, which then spills; 8192 columns 976 us that way.  Sixteen columns a lane (beyond 4096) need more than the 256
// registers there are all the same: with biases 2 to 18 of them go to scratch where rows are aligned, 23 to 25 where they are not; without biases none.
template <typename F>
void by_width_bwd(int cols, F f) {
    using std::integral_constant;
    if (cols <= 256) f(integral_constant<int, 1>(), integral_constant<int, 1>());
    else if (cols <= 512) f(integral_constant<int, 1>(), integral_constant<int, 2>());
    else if (cols <= 1024) f(integral_constant<int, 4>(), integral_constant<int, 1>());
    else if (cols <= 2048) f(integral_constant<int, 4>(), integral_constant<int, 2>());
    else if (cols <= 4096) f(integral_constant<int, 8>(), integral_constant<int, 2>());
    else f(integral_constant<int, 8>(), integral_constant<int, 4>());
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

// Workgroups of the adjoint: as many as the chip holds at once
int blocks_of(int rows, int cols) {
    const int at_once = cols <= 512 ? 4 : 1, most = cols <= 256 ? 1024 : cols <= 2048 ? 512 : 256;
    return (int)std::min<int64_t>(((int64_t)rows + at_once - 1) / at_once, most);
}

}  // namespace

int64_t residual_norm_workspace(int rows, int cols) { return (int64_t)blocks_of(rows, cols) * kParams * cols; }

int residual_norm_fwd(const fwp_norm_args &a, void *r, void *n, float *stats, hipStream_t s) {
    const bool whole = whole_rows(a, {a.y, a.gate_rows ? nullptr : a.gate, n}, {a.x, r},
                                  {a.scale, a.after_weight, a.after_bias, a.before_weight, a.before_bias});
    int rc = 0;
    by_types(a, [&](auto t, auto st) {
        using T = decltype(t);
        using S = decltype(st);
        by_width(a.cols, [&](auto w, auto v) {
            constexpr int WAVES = decltype(w)::value, NV = decltype(v)::value;
            const int64_t blocks = ((int64_t)a.rows + rows_at_once(WAVES) - 1) / rows_at_once(WAVES);
            if (!fits_launch(blocks, threads_of(WAVES))) {
                rc = FWP_E_SHAPE;
                return;
            }
            const dim3 grid((unsigned)blocks), block(threads_of(WAVES));
            if (whole) hipLaunchKernelGGL((k_rnorm_fwd<T, S, WAVES, NV, kWhole>), grid, block, 0, s, a, (S *)r, (T *)n, stats);
            else if (a.cols >= 4) hipLaunchKernelGGL((k_rnorm_fwd<T, S, WAVES, NV, kRagged>), grid, block, 0, s, a, (S *)r, (T *)n, stats);
            else hipLaunchKernelGGL((k_rnorm_fwd<T, S, 1, 1, kTiny>), grid, block, 0, s, a, (S *)r, (T *)n, stats);
        });
    });
    return rc ? rc : (int)hipGetLastError();
}

int residual_norm_bwd(const fwp_norm_args &a, const float *stats, const void *gr, const void *gn, const fwp_norm_grads &g, float *workspace,
                      hipStream_t s) {
    const bool whole = whole_rows(a, {a.y, a.gate_rows ? nullptr : a.gate, gn, g.gy, a.gate_rows ? nullptr : g.ggate}, {a.x, gr, g.gx},
                                  {a.scale, a.after_weight, a.after_bias, a.before_weight});
    const int blocks = blocks_of(a.rows, a.cols);
    by_types(a, [&](auto t, auto st) {
        using T = decltype(t);
        using S = decltype(st);
        by_width_bwd(a.cols, [&](auto w, auto v) {
            constexpr int WAVES = decltype(w)::value, NV = decltype(v)::value;
            const auto launch = [&](auto kernel, int threads) {
                hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), 0, s, a, stats, (const S *)gr, (const T *)gn, (T *)g.gy, (S *)g.gx,
                                   (T *)g.ggate, workspace);
            };
            const bool bias = a.after_bias || a.before_bias;
            if (a.cols < 4) launch(k_rnorm_bwd<T, S, 1, 1, true, kTiny>, threads_of(1));
            else if (!whole) launch(k_rnorm_bwd<T, S, WAVES, NV, true, kRagged>, threads_of(WAVES));
            else if (bias) launch(k_rnorm_bwd<T, S, WAVES, NV, true, kWhole>, threads_of(WAVES));
            else launch(k_rnorm_bwd<T, S, WAVES, NV, false, kWhole>, threads_of(WAVES));
        });
    });
    if (g.gscale || g.gafter_weight || g.gafter_bias || g.gbefore_weight || g.gbefore_bias)
        hipLaunchKernelGGL(k_rnorm_params, dim3((kParams * a.cols + 15) / 16), dim3(1024), 0, s, workspace, g, blocks, a.cols);
    return (int)hipGetLastError();
}

}  // namespace fwp
