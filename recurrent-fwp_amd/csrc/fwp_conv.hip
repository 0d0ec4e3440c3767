// Short causal convolution, a filter of K taps to each channel, forward and backward.
//
//   p[t] = bias + sum_j weight[j] x[t - K + 1 + j]    y = p, or p sigmoid(p)
//   d = gy act'(p)    gx[t] = sum_j weight[j] d[t + K - 1 - j]    gweight[j] = sum_t d[t] x[t - K + 1 + j]    gbias = sum_t d
//
// A thread takes V neighbouring channels over a run of steps and keeps the last K rows in registers, so a row is read once (and K - 1 rows
// again at the run's start; backward also K - 1 rows behind its end, whose d reaches back into the run); p is formed again from x in
// the backward pass rather than kept.  The loads of kAhead rows go out together.  Bound by memory: 32 x 1024 steps of 512 channels, four taps, fp32, forward
// 27 us (134 MB, 5.0 TB/s), adjoint 42 (201 MB, 4.8 TB/s) and its sums 4; a padded batch of 7 x 1531 steps of 1001 channels, three taps, fp16, 16 us (43 MB).
#include "fwp_elements.hpp"

#include <algorithm>

namespace fwp {
namespace {

constexpr int kThreads = 256, kAhead = 8;

// How rows lie: kWhole, four channels at a time, aligned for that everywhere; kRagged, any width from four on and any place: the same loads without the
// alignment, and the thread that the row's end cuts reads its last four and moves them up; kTiny, one channel to a thread.
enum Lie { kWhole, kRagged, kTiny };
constexpr int width_of(int lie) { return lie == kTiny ? 1 : 4; }

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T x[V];
};
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Anywhere {
    T x[V];
};

// Channels c .. c + V - 1 of a row, as they come: always a load, in the row (a branch around a load would wait for it at its end)
template <int LIE, typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T *row, int c, int D) {
    if constexpr (LIE == kWhole) return *reinterpret_cast<const Vec<T, V> *>(row + c);
    const Anywhere<T, V> u = *reinterpret_cast<const Anywhere<T, V> *>(row + min(c, D - V));
    Vec<T, V> v;
#pragma unroll
    for (int i = 0; i < V; i++) v.x[i] = u.x[i];
    return v;
}
// their values, zeros where the row does not count
template <int LIE, typename T, int V>
__device__ __forceinline__ void convert(float (&to)[V], const Vec<T, V> &v, bool in, int c, int D) {
#pragma unroll
    for (int i = 0; i < V; i++) to[i] = in ? (float)v.x[i] : 0.f;
    if constexpr (LIE == kRagged) {
        const int s = c - (D - V);      // how far the four that were read lie before the ones wanted
        to[0] = s == 1 ? to[1] : s == 2 ? to[2] : s == 3 ? to[3] : to[0];
        to[1] = s == 1 ? to[2] : s == 2 ? to[3] : to[1];
        to[2] = s == 1 ? to[3] : to[2];
    }
}
template <int LIE, typename T, int V>
__device__ __forceinline__ void store_vec(T *row, const float (&from)[V], int c, int D) {
    Anywhere<T, V> u;
#pragma unroll
    for (int i = 0; i < V; i++) u.x[i] = (T)from[i];
    if constexpr (LIE == kWhole) *reinterpret_cast<Vec<T, V> *>(row + c) = *reinterpret_cast<const Vec<T, V> *>(&u);
    else if (c + V <= D) *reinterpret_cast<Anywhere<T, V> *>(row + c) = u;
    else
#pragma unroll
        for (int i = 0; i < V; i++)
            if (c + i < D) row[c + i] = u.x[i];
}

// Steps to a run.  A longer one reads fewer rows twice and leaves fewer partial sums, a shorter one gives more threads.  16 / 32 steps, forward at 2.7 and 4.2 M
// rows of vectors 16.2 / 20.1 and 24 / 22 us, adjoint at 0.8 and 4.2 M 48 / 59 and 63 / 51 us; eight taps at 4.2 M, 32 / 64 steps: 75 / 60 us.
// 8 / 16 steps, forward at 0.5 and 1.05 M 4.6 / 6.0 and 8.0 / 8.0 us.
int run_of(int64_t vectors, int K, bool backward) {
    if (!backward && vectors < 1000000) return 8;
    if (vectors < (backward ? 2 : 4) * int64_t(1000000)) return 16;
    return backward && K > 4 && vectors >= 4000000 ? 64 : 32;
}

// How a workgroup's threads lie over channels and steps: `across` threads (a power of two) side by side over the channels, V each, the others
// over the runs.
struct Tiling {
    int across, blocks_d, run, runs, blocks_t;
    Tiling(int N, int H, int L, int D, int K, int V, bool backward) {
        const int vecs = (D + V - 1) / V;
        across = 64;
        while (across > 1 && across / 2 >= vecs) across /= 2;
        blocks_d = (vecs + across - 1) / across;
        run = run_of((int64_t)N * H * L * vecs, K, backward);
        runs = (L + run - 1) / run;
        const int at_once = kThreads / across;
        blocks_t = (runs + at_once - 1) / at_once;
    }
    int64_t grid(int N, int H) const { return (int64_t)N * H * blocks_d * blocks_t; }
};

// Which channels and steps a thread has
struct Spot {
    int n, h, c, t0, len;
    int64_t nh, bt;
    bool in;
    __device__ __forceinline__ Spot(const fwp_conv_args &a, const Tiling &g, int V) {
        int64_t b = blockIdx.x;
        const int bd = (int)(b % g.blocks_d);
        b /= g.blocks_d;
        bt = b % g.blocks_t, nh = b / g.blocks_t;
        n = (int)(nh / a.H), h = (int)(nh % a.H);
        c = (bd * g.across + threadIdx.x % g.across) * V;
        t0 = (int)(bt * (kThreads / g.across) + threadIdx.x / g.across) * g.run;
        len = length_of(a.lengths, n, a.L);
        in = c < a.D && t0 < a.L;
    }
};

template <int K, int V>
__device__ __forceinline__ void load_filter(float (&w)[K][V], float (&b)[V], const fwp_conv_args &a, const Spot &p) {
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int64_t at = (int64_t)p.h * a.D + min(p.c + i, a.D - 1);
#pragma unroll
        for (int j = 0; j < K; j++) w[j][i] = a.weight[at * K + j];
        b[i] = a.bias ? a.bias[at] : 0.f;
    }
}

// Row t of x, or the one nearest to it of those that count
template <typename T>
__device__ __forceinline__ const T *x_row(const fwp_rows &x, const Spot &p, int t) {
    return row<T>(x, p.n, p.h, max(0, min(t, p.len - 1)));
}
// x[t] as the filter sees it: the carried rows before the first, zeros without them and behind the last
template <int LIE, typename T, int K, int V>
__device__ __forceinline__ void load_x(float (&to)[V], const fwp_conv_args &a, const T *state, const Spot &p, int t) {
    const bool carried = t < 0 && state;
    const T *const r = carried ? state + (p.nh * (K - 1) + t + K - 1) * a.D : x_row<T>(a.x, p, t);
    convert<LIE, T, V>(to, load_vec<LIE, T, V>(r, p.c, a.D), carried || (t >= 0 && t < p.len), p.c, a.D);
}

template <typename T, int K, int LIE>
__global__ __launch_bounds__(kThreads) void k_conv_fwd(fwp_conv_args a, Tiling g, T *state, fwp_out_rows y) {
    constexpr int V = width_of(LIE);
    const Spot p(a, g, V);
    if (!p.in) return;
    float w[K][V], b[V], win[K][V];
    load_filter<K, V>(w, b, a, p);
    const int end = min(p.t0 + g.run, a.L);
    Vec<T, V> ahead[kAhead];
    const auto fetch = [&](int t) {
#pragma unroll
        for (int u = 0; u < kAhead; u++) ahead[u] = load_vec<LIE, T, V>(x_row<T>(a.x, p, t + u), p.c, a.D);
    };
    fetch(p.t0);
#pragma unroll
    for (int j = 0; j < K - 1; j++) load_x<LIE, T, K, V>(win[j + 1], a, state, p, p.t0 - (K - 1) + j);
    if (state && p.t0 == 0) {       // this thread alone reads and writes its channels' carried rows: the last K - 1 of (carried rows, x)
        float last[K > 1 ? K - 1 : 1][V];
#pragma unroll
        for (int i = 0; i < K - 1; i++) load_x<LIE, T, K, V>(last[i], a, state, p, p.len - (K - 1) + i);
#pragma unroll
        for (int i = 0; i < K - 1; i++) store_vec<LIE, T, V>(state + (p.nh * (K - 1) + i) * a.D, last[i], p.c, a.D);
    }
    for (int t = p.t0; t < end; t += kAhead) {
        float x[kAhead][V];
#pragma unroll
        for (int u = 0; u < kAhead; u++) convert<LIE, T, V>(x[u], ahead[u], t + u < p.len, p.c, a.D);
        if (t + kAhead < end) fetch(t + kAhead);
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            float o[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
#pragma unroll
                for (int j = 0; j < K - 1; j++) win[j][i] = win[j + 1][i];
                win[K - 1][i] = x[u][i];
                float s = b[i];
#pragma unroll
                for (int j = 0; j < K; j++) s = fmaf(w[j][i], win[j][i], s);
                if (a.silu) s = silu(s, sigmoid(s));
                o[i] = t + u < p.len ? s : 0.f;
            }
            if (t + u < end) store_vec<LIE, T, V>(row<T>(y, p.n, p.h, t + u), o, p.c, a.D);
        }
    }
}

// parts [N blocks_t][H][K + 1][D]: the sums of a workgroup's runs for gweight's taps and gbias
template <typename T, int K, int LIE>
__global__ __launch_bounds__(kThreads) void k_conv_bwd(fwp_conv_args a, Tiling g, const T *__restrict__ state, fwp_rows gy, fwp_out_rows gx,
                                                       float *__restrict__ parts) {
    constexpr int V = width_of(LIE), AHEAD = 4;      // eight rows' loads at once leave two waves a SIMD instead of three: 52 us against 45, 32 x 1024 x 512 fp32
    __shared__ float sh[kThreads * V];
    const Spot p(a, g, V);
    float gw[K + 1][V] = {};
    if (p.in) {
        float w[K][V], b[V], win[K][V], dwin[K][V] = {};
        load_filter<K, V>(w, b, a, p);
        const int end = min(p.t0 + g.run, a.L);
        Vec<T, V> x_ahead[AHEAD], d_ahead[AHEAD];
        const auto fetch = [&](int t) {
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                x_ahead[u] = load_vec<LIE, T, V>(x_row<T>(a.x, p, t + u), p.c, a.D);
                d_ahead[u] = load_vec<LIE, T, V>(x_row<T>(gy, p, t + u), p.c, a.D);
            }
        };
        fetch(p.t0);
#pragma unroll
        for (int j = 0; j < K - 1; j++) load_x<LIE, T, K, V>(win[j + 1], a, state, p, p.t0 - (K - 1) + j);
        for (int t = p.t0; t < end + K - 1; t += AHEAD) {
            float x[AHEAD][V], d[AHEAD][V];
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                convert<LIE, T, V>(x[u], x_ahead[u], t + u < p.len, p.c, a.D);
                convert<LIE, T, V>(d[u], d_ahead[u], t + u < p.len, p.c, a.D);
            }
            if (t + AHEAD < end + K - 1) fetch(t + AHEAD);
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                float o[V];
                const bool mine = t + u < end, in = t + u < p.len;
#pragma unroll
                for (int i = 0; i < V; i++) {
#pragma unroll
                    for (int j = 0; j < K - 1; j++) win[j][i] = win[j + 1][i], dwin[j][i] = dwin[j + 1][i];
                    win[K - 1][i] = x[u][i];
                    float e = d[u][i];
                    if (a.silu) {
                        float s = b[i];
#pragma unroll
                        for (int j = 0; j < K; j++) s = fmaf(w[j][i], win[j][i], s);
                        e *= silu_slope(s, sigmoid(s));
                    }
                    e = in ? e : 0.f;
                    dwin[K - 1][i] = e;
                    if (mine) {
#pragma unroll
                        for (int j = 0; j < K; j++) gw[j][i] = fmaf(e, win[j][i], gw[j][i]);
                        gw[K][i] += e;
                    }
                    float s = 0.f;
#pragma unroll
                    for (int j = 0; j < K; j++) s = fmaf(w[j][i], dwin[K - 1 - j][i], s);
                    o[i] = t + u - (K - 1) < p.len ? s : 0.f;
                }
                const int at = t + u - (K - 1);
                if (at >= p.t0 && at < end) store_vec<LIE, T, V>(row<T>(gx, p.n, p.h, at), o, p.c, a.D);
            }
        }
    }
    const int c = threadIdx.x % g.across, q = threadIdx.x / g.across, groups = kThreads / g.across;
    for (int j = 0; j <= K; j++) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; i++) sh[(q * g.across + c) * V + i] = gw[j][i];
        __syncthreads();
        for (int k = threadIdx.x; k < g.across * V; k += kThreads) {
            float s = 0.f;
            for (int r = 0; r < groups; r++) s += sh[r * g.across * V + k];
            const int col = (int)(blockIdx.x % g.blocks_d) * g.across * V + k;
            if (col < a.D) parts[(((p.n * (int64_t)g.blocks_t + p.bt) * a.H + p.h) * (K + 1) + j) * a.D + col] = s;
        }
    }
}

// gweight, gbias: the workgroups' sums added up in a fixed order, 16 columns and 64 slices of the terms to a workgroup
__global__ __launch_bounds__(1024) void k_conv_params(const float *__restrict__ parts, float *__restrict__ gweight, float *__restrict__ gbias,
                                                      int64_t terms, int H, int D, int K) {
    __shared__ float sh[64][17];
    const int64_t per = (int64_t)H * (K + 1) * D, i = (int64_t)blockIdx.x * 16 + threadIdx.x % 16;
    const int slice = threadIdx.x / 16;
    float x = 0.f;
    if (i < per)
#pragma unroll 8
        for (int64_t k = slice; k < terms; k += 64) x += parts[k * per + i];
    sh[slice][threadIdx.x % 16] = x;
    __syncthreads();
    const int c = threadIdx.x % 16, s = threadIdx.x / 16;
    if (s < 16) x = (sh[4 * s][c] + sh[4 * s + 1][c]) + (sh[4 * s + 2][c] + sh[4 * s + 3][c]);
    __syncthreads();
    if (s < 16) sh[s][c] = x;
    __syncthreads();
    if (s || i >= per) return;
    x = 0.f;
#pragma unroll
    for (int k = 0; k < 16; k++) x += sh[k][c];
    const int64_t h = i / ((int64_t)(K + 1) * D), j = i / D % (K + 1), ch = i % D;
    if (j < K) gweight[(h * D + ch) * K + j] = x;
    else gbias[h * D + ch] = x;
}

// How the rows of a call lie
int lie_of(const fwp_conv_args &a, std::initializer_list<fwp_rows> views, const void *state) {
    const int size = a.type == FWP_F32 ? 4 : 2;
    if (a.D < 4) return kTiny;
    if (a.D % 4 || reinterpret_cast<uintptr_t>(state) % (4 * size)) return kRagged;
    for (const fwp_rows &v : views)
        if (reinterpret_cast<uintptr_t>(v.ptr) % (4 * size) || v.sN % 4 || v.sH % 4 || v.sL % 4) return kRagged;
    return kWhole;
}

template <typename F>
void by_taps(int K, F f) {
    switch (K) {
        case 1: f(std::integral_constant<int, 1>()); break;
        case 2: f(std::integral_constant<int, 2>()); break;
        case 3: f(std::integral_constant<int, 3>()); break;
        case 4: f(std::integral_constant<int, 4>()); break;
        case 5: f(std::integral_constant<int, 5>()); break;
        case 6: f(std::integral_constant<int, 6>()); break;
        case 7: f(std::integral_constant<int, 7>()); break;
        default: f(std::integral_constant<int, 8>()); break;
    }
}

// f(T, K, Lie)
template <typename F>
void by_kind(const fwp_conv_args &a, int lie, F f) {
    using std::integral_constant;
    by_type(a.type, [&](auto t) {
        by_taps(a.K, [&](auto k) {
            if (lie == kWhole) f(t, k, integral_constant<int, kWhole>());
            else if (lie == kRagged) f(t, k, integral_constant<int, kRagged>());
            else f(t, k, integral_constant<int, kTiny>());
        });
    });
}

}  // namespace

int conv_fwd(const fwp_conv_args &a, void *state, fwp_out_rows y, hipStream_t s) {
    const int lie = lie_of(a, {a.x, {y.ptr, y.sN, y.sH, y.sL}}, state);
    const Tiling g(a.N, a.H, a.L, a.D, a.K, width_of(lie), false);
    if (!fits_launch(g.grid(a.N, a.H), kThreads)) return FWP_E_SHAPE;
    const dim3 grid((unsigned)g.grid(a.N, a.H));
    by_kind(a, lie, [&](auto t, auto k, auto l) {
        using T = decltype(t);
        hipLaunchKernelGGL((k_conv_fwd<T, decltype(k)::value, decltype(l)::value>), grid, dim3(kThreads), 0, s, a, g, (T *)state, y);
    });
    return (int)hipGetLastError();
}

int64_t conv_workspace(int N, int H, int L, int D, int K) {
    return (int64_t)N * Tiling(N, H, L, D, K, D < 4 ? 1 : 4, true).blocks_t * H * (K + 1) * D;
}

int conv_bwd(const fwp_conv_args &a, const void *state, fwp_rows gy, fwp_out_rows gx, float *gweight, float *gbias, float *workspace,
             hipStream_t s) {
    const int lie = lie_of(a, {a.x, gy, {gx.ptr, gx.sN, gx.sH, gx.sL}}, state);
    const Tiling g(a.N, a.H, a.L, a.D, a.K, width_of(lie), true);
    const int64_t param_blocks = ((int64_t)a.H * (a.K + 1) * a.D + 15) / 16;
    if (!fits_launch(g.grid(a.N, a.H), kThreads) || !fits_launch(param_blocks, 1024)) return FWP_E_SHAPE;
    const dim3 grid((unsigned)g.grid(a.N, a.H));
    by_kind(a, lie, [&](auto t, auto k, auto l) {
        using T = decltype(t);
        hipLaunchKernelGGL((k_conv_bwd<T, decltype(k)::value, decltype(l)::value>), grid, dim3(kThreads), 0, s, a, g, (const T *)state, gy, gx,
                           workspace);
    });
    if (gweight)
        hipLaunchKernelGGL(k_conv_params, dim3((unsigned)param_blocks), dim3(1024), 0, s, workspace, gweight, gbias, (int64_t)a.N * g.blocks_t, a.H,
                           a.D, a.K);
    return (int)hipGetLastError();
}

}  // namespace fwp
