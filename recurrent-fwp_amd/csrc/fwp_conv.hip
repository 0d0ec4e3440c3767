// Short causal convolution, a filter of K taps to each channel, forward and backward.
//
//   p[t] = bias + sum_j weight[j] x[t - K + 1 + j]    y = p, or p sigmoid(p)
//   d = gy act'(p)    gx[t] = sum_j weight[j] d[t + K - 1 - j]    gweight[j] = sum_t d[t] x[t - K + 1 + j]    gbias = sum_t d
//
// A thread takes V neighbouring channels over a run of kRun steps and keeps the last K rows in registers, so a row is read once (and K - 1 rows
// again at the run's start; backward also K - 1 rows behind its end, whose d reaches back into the run); p is formed again from x in
// the backward pass rather than kept.  The loads of kAhead rows go out together.  Bound by memory.
#include "fwp_elements.hpp"

#include <algorithm>

namespace fwp {
namespace {

constexpr int kThreads = 256, kAhead = 8, kRun = 32;
constexpr int64_t kMaxBlocks = (int64_t(1) << 31) - 1;

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T x[V];
};

template <typename T, int V>
__device__ __forceinline__ void load_vec(float (&to)[V], const T *p, bool in) {
    if (!in) {
#pragma unroll
        for (int i = 0; i < V; i++) to[i] = 0.f;
        return;
    }
    const Vec<T, V> v = *reinterpret_cast<const Vec<T, V> *>(p);
#pragma unroll
    for (int i = 0; i < V; i++) to[i] = (float)v.x[i];
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T *p, const float (&from)[V]) {
    Vec<T, V> v;
#pragma unroll
    for (int i = 0; i < V; i++) v.x[i] = (T)from[i];
    *reinterpret_cast<Vec<T, V> *>(p) = v;
}

// How a workgroup's threads lie over channels and steps: `across` threads (a power of two) side by side over the channels, V each, the others
// over the runs.
struct Tiling {
    int across, blocks_d, runs, blocks_t;
    Tiling(int L, int D, int V) {
        const int vecs = (D + V - 1) / V;
        across = 64;
        while (across > 1 && across / 2 >= vecs) across /= 2;
        blocks_d = (vecs + across - 1) / across;
        runs = (L + kRun - 1) / kRun;
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
        t0 = (int)(bt * (kThreads / g.across) + threadIdx.x / g.across) * kRun;
        len = length_of(a.lengths, n, a.L);
        in = c < a.D && t0 < a.L;
    }
};

template <int K, int V>
__device__ __forceinline__ void load_filter(float (&w)[K][V], float (&b)[V], const fwp_conv_args &a, const Spot &p) {
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int64_t at = (int64_t)p.h * a.D + p.c + i;
#pragma unroll
        for (int j = 0; j < K; j++) w[j][i] = a.weight[at * K + j];
        b[i] = a.bias ? a.bias[at] : 0.f;
    }
}

// x[t] as the filter sees it: the carried rows before the first, zeros without them and behind the last
template <typename T, int K, int V>
__device__ __forceinline__ void load_x(float (&to)[V], const fwp_conv_args &a, const T *state, const Spot &p, int t) {
    if (t >= 0) load_vec<T, V>(to, row<T>(a.x, p.n, p.h, t) + p.c, t < p.len);
    else load_vec<T, V>(to, state + (p.nh * (K - 1) + t + K - 1) * a.D + p.c, state != nullptr);
}

template <typename T, int K, int V>
__global__ __launch_bounds__(kThreads) void k_conv_fwd(fwp_conv_args a, Tiling g, T *state, fwp_out_rows y) {
    const Spot p(a, g, V);
    if (!p.in) return;
    float w[K][V], b[V], win[K][V];
    load_filter<K, V>(w, b, a, p);
#pragma unroll
    for (int j = 0; j < K - 1; j++) load_x<T, K, V>(win[j + 1], a, state, p, p.t0 - (K - 1) + j);
    if (state && p.t0 == 0) {       // this thread alone reads and writes its channels' carried rows: the last K - 1 of (carried rows, x)
        float last[K > 1 ? K - 1 : 1][V];
#pragma unroll
        for (int i = 0; i < K - 1; i++) load_x<T, K, V>(last[i], a, state, p, p.len - (K - 1) + i);
#pragma unroll
        for (int i = 0; i < K - 1; i++) store_vec<T, V>(state + (p.nh * (K - 1) + i) * a.D + p.c, last[i]);
    }
    const int end = min(p.t0 + kRun, a.L);
    for (int t = p.t0; t < end; t += kAhead) {
        float x[kAhead][V];
#pragma unroll
        for (int u = 0; u < kAhead; u++) load_vec<T, V>(x[u], row<T>(a.x, p.n, p.h, t + u) + p.c, t + u < p.len);
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
            if (t + u < end) store_vec<T, V>(row<T>(y, p.n, p.h, t + u) + p.c, o);
        }
    }
}

// parts [N blocks_t][H][K + 1][D]: the sums of a workgroup's runs for gweight's taps and gbias
template <typename T, int K, int V>
__global__ __launch_bounds__(kThreads) void k_conv_bwd(fwp_conv_args a, Tiling g, const T *__restrict__ state, fwp_rows gy, fwp_out_rows gx,
                                                       float *__restrict__ parts) {
    __shared__ float sh[kThreads * V];
    const Spot p(a, g, V);
    float gw[K + 1][V] = {};
    if (p.in) {
        float w[K][V], b[V], win[K][V], dwin[K][V] = {};
        load_filter<K, V>(w, b, a, p);
#pragma unroll
        for (int j = 0; j < K - 1; j++) load_x<T, K, V>(win[j + 1], a, state, p, p.t0 - (K - 1) + j);
        const int end = min(p.t0 + kRun, a.L);
        for (int t = p.t0; t < end + K - 1; t += kAhead) {
            float x[kAhead][V], d[kAhead][V];
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                const bool in = t + u < p.len && t + u < end + K - 1;
                load_vec<T, V>(x[u], row<T>(a.x, p.n, p.h, t + u) + p.c, in);
                load_vec<T, V>(d[u], row<T>(gy, p.n, p.h, t + u) + p.c, in);
            }
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
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
                if (at >= p.t0 && at < end) store_vec<T, V>(row<T>(gx, p.n, p.h, at) + p.c, o);
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

// gweight, gbias: the workgroups' sums added up in a fixed order, 64 columns and four slices of the terms to a workgroup
__global__ __launch_bounds__(kThreads) void k_conv_params(const float *__restrict__ parts, float *__restrict__ gweight,
                                                          float *__restrict__ gbias, int64_t terms, int H, int D, int K) {
    __shared__ float sh[4][64];
    const int64_t per = (int64_t)H * (K + 1) * D, i = (int64_t)blockIdx.x * 64 + threadIdx.x % 64;
    const int slice = threadIdx.x / 64;
    float x = 0.f;
    if (i < per)
        for (int64_t k = slice; k < terms; k += 4) x += parts[k * per + i];
    sh[slice][threadIdx.x % 64] = x;
    __syncthreads();
    if (slice || i >= per) return;
    x = (sh[0][threadIdx.x] + sh[1][threadIdx.x]) + (sh[2][threadIdx.x] + sh[3][threadIdx.x]);
    const int64_t h = i / ((int64_t)(K + 1) * D), j = i / D % (K + 1), c = i % D;
    if (j < K) gweight[(h * D + c) * K + j] = x;
    else gbias[h * D + c] = x;
}

// Four channels to a thread where every row can be read that way
bool by_four(const fwp_conv_args &a, std::initializer_list<fwp_rows> views, const void *state) {
    const int size = a.type == FWP_F32 ? 4 : 2;
    if (a.D % 4 || reinterpret_cast<uintptr_t>(state) % (4 * size)) return false;
    for (const fwp_rows &v : views)
        if (reinterpret_cast<uintptr_t>(v.ptr) % (4 * size) || v.sN % 4 || v.sH % 4 || v.sL % 4) return false;
    return true;
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

}  // namespace

int conv_fwd(const fwp_conv_args &a, void *state, fwp_out_rows y, hipStream_t s) {
    const bool four = by_four(a, {a.x, {y.ptr, y.sN, y.sH, y.sL}}, state);
    const Tiling g(a.L, a.D, four ? 4 : 1);
    if (g.grid(a.N, a.H) > kMaxBlocks) return FWP_E_SHAPE;
    const dim3 grid((unsigned)g.grid(a.N, a.H));
    by_type(a.type, [&](auto t) {
        using T = decltype(t);
        by_taps(a.K, [&](auto k) {
            constexpr int K = decltype(k)::value;
            if (four) hipLaunchKernelGGL((k_conv_fwd<T, K, 4>), grid, dim3(kThreads), 0, s, a, g, (T *)state, y);
            else hipLaunchKernelGGL((k_conv_fwd<T, K, 1>), grid, dim3(kThreads), 0, s, a, g, (T *)state, y);
        });
    });
    return (int)hipGetLastError();
}

int64_t conv_workspace(int N, int H, int L, int D, int K) {
    const int64_t blocks = std::max(Tiling(L, D, 1).blocks_t, Tiling(L, D, 4).blocks_t);
    return N * blocks * H * (K + 1) * D;
}

int conv_bwd(const fwp_conv_args &a, const void *state, fwp_rows gy, fwp_out_rows gx, float *gweight, float *gbias, float *workspace,
             hipStream_t s) {
    const bool four = by_four(a, {a.x, gy, {gx.ptr, gx.sN, gx.sH, gx.sL}}, state);
    const Tiling g(a.L, a.D, four ? 4 : 1);
    const int64_t param_blocks = ((int64_t)a.H * (a.K + 1) * a.D + 63) / 64;
    if (g.grid(a.N, a.H) > kMaxBlocks || param_blocks > kMaxBlocks) return FWP_E_SHAPE;
    const dim3 grid((unsigned)g.grid(a.N, a.H));
    by_type(a.type, [&](auto t) {
        using T = decltype(t);
        by_taps(a.K, [&](auto k) {
            constexpr int K = decltype(k)::value;
            if (four) hipLaunchKernelGGL((k_conv_bwd<T, K, 4>), grid, dim3(kThreads), 0, s, a, g, (const T *)state, gy, gx, workspace);
            else hipLaunchKernelGGL((k_conv_bwd<T, K, 1>), grid, dim3(kThreads), 0, s, a, g, (const T *)state, gy, gx, workspace);
        });
    });
    if (gweight)
        hipLaunchKernelGGL(k_conv_params, dim3((unsigned)param_blocks), dim3(kThreads), 0, s, workspace, gweight, gbias,
                           (int64_t)a.N * g.blocks_t, a.H, a.D, a.K);
    return (int)hipGetLastError();
}

}  // namespace fwp
