// Norm of groups of channels with an activation or a gate, channels last, forward and backward.
//
//   u = hat w + b,  hat = (x - mean) / sqrt(var + eps) (RMS: x / sqrt(mean(x^2) + eps));   y = act(gate) u, or act(u)
// and backwards
//   du = gy act(gate), or gy act'(u);  ggate = gy u act'(gate);  gw = sum du hat, gb = sum du over the rows
//   gx = (h - mean(h) - hat mean(h hat)) / spread,  h = du w          (RMS: without mean(h))
//
// A group is W lanes' worth of 16-byte runs, and a wave has as many neighbouring groups of a row as it has room for and goes from row to row with them: no
// sum ever leaves the wave, and parameters and their sums stay in registers.  The next row's loads are issued before a row is worked on.  Statistics are made again in
// the backward pass, which reads the rows anyway; the four waves of a workgroup add their sums in LDS, and a second kernel adds the workgroups' in a
// fixed order.  Bound by memory: 16384 rows of 32 groups of 128, bf16 with a gate, 79 us forward at 5.1 TB/s and 136 back at 4.9, the rate of copies, and 5 for the sums; 32768 rows of 8 groups of 32,
// fp32, 18 + 29 + 4.  The adjoint could take the statistics from memory, but then would read them, and has them at no time of its own.
#include <algorithm>

#include "fwp_elements.hpp"
#include "fwp_wave.hpp"

namespace fwp {
namespace {

struct NormWalk {
    const void *x, *gate, *gy;
    int64_t x_step, gate_step;
    void *y, *gx, *ggate;
    const float *weight, *bias;
    float *sums;      // [blocks][2][groups * size]
    float eps;
    int rms, act, rows, groups, size, blocks;      // blocks: workgroups for each run of groups
};

constexpr int kRowHalfMirror = 0x141, kRowMirror = 0x140;

// Sum over W neighbouring lanes, in all of them
template <int W>
__device__ __forceinline__ float lanes_sum(float x) {
    if constexpr (W >= 2) x += dpp<kQuadXor1>(x);
    if constexpr (W >= 4) x += dpp<kQuadXor2>(x);
    if constexpr (W >= 8) x += dpp<kRowHalfMirror>(x);
    if constexpr (W >= 16) x += dpp<kRowMirror>(x);
    if constexpr (W >= 32) {
        float y = x;
        swap16(x, y);
        x += y;
    }
    if constexpr (W >= 64) {
        float y = x;
        swap32(x, y);
        x += y;
    }
    return x;
}

// A lane's elements of a row: K runs of V, those of a group from `first` on.  Every lane loads, what lies beyond the group from the group's last elements: a branch
// around a load would wait for it at its end.  ODD: groups that are no multiple of a run, of which the last one is then shifted; groups shorter than one are
// read element by element.
template <typename T, int K, bool ODD>
struct Run {
    static constexpr int V = 16 / sizeof(T);
    typedef uint32_t Words __attribute__((ext_vector_type(4)));
    struct __attribute__((packed, aligned(sizeof(T)))) Anywhere { Words w; };
    struct Elements { T x[V]; };
    Words w[K];

    __device__ __forceinline__ void load(const T *at, int first, int step, int size) {
#pragma unroll
        for (int i = 0; i < K; i++) {
            const int c = first + i * step;
            if (!ODD || size >= V) {
                w[i] = reinterpret_cast<const Anywhere *>(at + min(c, size - V))->w;
            } else {
                Elements few;
#pragma unroll
                for (int e = 0; e < V; e++) few.x[e] = at[min(e, size - 1)];
                w[i] = __builtin_bit_cast(Words, few);
            }
        }
    }
    // as fp32, zero beyond the group
    __device__ __forceinline__ void get(float (&x)[K][V], int first, int step, int size) const {
#pragma unroll
        for (int i = 0; i < K; i++) {
            const Elements few = __builtin_bit_cast(Elements, w[i]);
            const int c = first + i * step;
#pragma unroll
            for (int e = 0; e < V; e++) x[i][e] = (float)few.x[e];
            if constexpr (ODD) {
                const int late = size >= V ? max(0, c - (size - V)) : 0;
#pragma unroll
                for (int b = 1; b < V; b *= 2)
#pragma unroll
                    for (int e = 0; e < V; e++) x[i][e] = late & b ? x[i][e + b < V ? e + b : e] : x[i][e];
#pragma unroll
                for (int e = 0; e < V; e++) x[i][e] = c + e < size ? x[i][e] : 0.f;
            } else {
#pragma unroll
                for (int e = 0; e < V; e++) x[i][e] = c < size ? x[i][e] : 0.f;
            }
        }
    }
    __device__ __forceinline__ static void store(const float (&x)[K][V], T *at, int first, int step, int size) {
#pragma unroll
        for (int i = 0; i < K; i++) {
            const int c = first + i * step;
            if (!ODD || c + V <= size) {
                Elements few;
#pragma unroll
                for (int e = 0; e < V; e++) few.x[e] = (T)x[i][e];
                if (c < size) reinterpret_cast<Anywhere *>(at + c)->w = __builtin_bit_cast(Words, few);
            } else {
#pragma unroll
                for (int e = 0; e < V; e++)
                    if (c + e < size) at[c + e] = (T)x[i][e];
            }
        }
    }
};

__device__ __forceinline__ float act_of(float x, int act) {
    if (act == FWP_ACT_NONE) return x;
    const float s = sigmoid(x);
    return act == FWP_ACT_SIGMOID ? s : silu(x, s);
}
__device__ __forceinline__ float slope_of(float x, int act) {
    if (act == FWP_ACT_NONE) return 1.f;
    const float s = sigmoid(x);
    return act == FWP_ACT_SIGMOID ? s * (1.f - s) : silu_slope(x, s);
}

// Where a lane of this wave works: W lanes a group, 64 / W groups a wave, K runs of V elements a lane.
template <typename T, int W, int K>
struct Lane {
    static constexpr int V = 16 / sizeof(T), kGroups = 64 / W, kStep = W * V;
    int group, first, wave, row0, rows_step;
    bool live;
    __device__ __forceinline__ explicit Lane(const NormWalk &w) {
        const int lane = threadIdx.x % 64;
        wave = threadIdx.x / 64;
        group = (int)(blockIdx.x / w.blocks) * kGroups + lane / W;
        first = lane % W * V;
        row0 = (int)(blockIdx.x % w.blocks) * 4 + wave;
        rows_step = w.blocks * 4;
        live = group < w.groups;
    }
};

// hat in place of x, and 1 / spread
template <int W, int K, int V>
__device__ __forceinline__ float normalise(float (&x)[K][V], int first, int step, int size, float eps, int rms) {
    const float inv = 1.f / (float)size;
    if (!rms) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < K; i++)
#pragma unroll
            for (int e = 0; e < V; e++) s += x[i][e];
        const float mean = lanes_sum<W>(s) * inv;
#pragma unroll
        for (int i = 0; i < K; i++)
#pragma unroll
            for (int e = 0; e < V; e++) x[i][e] = first + i * step + e < size ? x[i][e] - mean : 0.f;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < K; i++)
#pragma unroll
        for (int e = 0; e < V; e++) s = fmaf(x[i][e], x[i][e], s);
    const float rstd = 1.f / sqrtf(lanes_sum<W>(s) * inv + eps);
#pragma unroll
    for (int i = 0; i < K; i++)
#pragma unroll
        for (int e = 0; e < V; e++) x[i][e] *= rstd;
    return rstd;
}

template <int K, int V>
__device__ __forceinline__ void parameters(float (&to)[K][V], const float *p, float none, int first, int step, int size) {
#pragma unroll
    for (int i = 0; i < K; i++)
#pragma unroll
        for (int e = 0; e < V; e++) {
            const int c = first + i * step + e;
            to[i][e] = p && c < size ? p[c] : none;
        }
}

template <typename T, int W, int K, bool ODD>
__global__ __launch_bounds__(256) void k_group_norm_fwd(const NormWalk w) {
    using L = Lane<T, W, K>;
    constexpr int V = L::V, step = L::kStep;
    const L l(w);
    if (!l.live) return;
    const int64_t width = (int64_t)w.groups * w.size, off = (int64_t)l.group * w.size;
    const T *xs = static_cast<const T *>(w.x) + off, *gs = static_cast<const T *>(w.gate);
    if (gs) gs += off;
    T *ys = static_cast<T *>(w.y) + off;
    float weight[K][V], bias[K][V];
    parameters(weight, w.weight ? w.weight + off : nullptr, 1.f, l.first, step, w.size);
    parameters(bias, w.bias ? w.bias + off : nullptr, 0.f, l.first, step, w.size);
    Run<T, K, ODD> x, gate;
#pragma unroll
    for (int i = 0; i < K; i++) gate.w[i] = 0;
    if (l.row0 < w.rows) {
        x.load(xs + l.row0 * w.x_step, l.first, step, w.size);
        if (gs) gate.load(gs + l.row0 * w.gate_step, l.first, step, w.size);
    }
    for (int r = l.row0; r < w.rows; r += l.rows_step) {
        float h[K][V], g[K][V];
        x.get(h, l.first, step, w.size);
        gate.get(g, l.first, step, w.size);
        if (r + l.rows_step < w.rows) {
            x.load(xs + (r + l.rows_step) * w.x_step, l.first, step, w.size);
            if (gs) gate.load(gs + (r + l.rows_step) * w.gate_step, l.first, step, w.size);
        }
        normalise<W>(h, l.first, step, w.size, w.eps, w.rms);
#pragma unroll
        for (int i = 0; i < K; i++)
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float u = fmaf(h[i][e], weight[i][e], bias[i][e]);
                h[i][e] = gs ? u * act_of(g[i][e], w.act) : act_of(u, w.act);
            }
        Run<T, K, ODD>::store(h, ys + r * width, l.first, step, w.size);
    }
}

template <typename T, int W, int K, bool ODD>
__global__ __launch_bounds__(256) void k_group_norm_bwd(const NormWalk w) {
    using L = Lane<T, W, K>;
    constexpr int V = L::V, step = L::kStep;
    __shared__ float sums[3][2][64 * K * V];
    const L l(w);
    const int64_t width = (int64_t)w.groups * w.size, off = (int64_t)(l.live ? l.group : 0) * w.size;
    const T *xs = static_cast<const T *>(w.x) + off, *gs = static_cast<const T *>(w.gate), *ds = static_cast<const T *>(w.gy) + off;
    if (gs) gs += off;
    float weight[K][V], bias[K][V], gw[K][V], gb[K][V];
    parameters(weight, w.weight ? w.weight + off : nullptr, 1.f, l.first, step, w.size);
    parameters(bias, w.bias ? w.bias + off : nullptr, 0.f, l.first, step, w.size);
#pragma unroll
    for (int i = 0; i < K; i++)
#pragma unroll
        for (int e = 0; e < V; e++) gw[i][e] = gb[i][e] = 0.f;
    Run<T, K, ODD> x, gate, gy;
    const auto fetch = [&](int r) {
        x.load(xs + r * w.x_step, l.first, step, w.size);
        gy.load(ds + r * width, l.first, step, w.size);
        if (gs) gate.load(gs + r * w.gate_step, l.first, step, w.size);
    };
#pragma unroll
    for (int i = 0; i < K; i++) gate.w[i] = 0;
    if (l.live && l.row0 < w.rows) fetch(l.row0);
    for (int r = l.row0; l.live && r < w.rows; r += l.rows_step) {
        float h[K][V], g[K][V], d[K][V];
        x.get(h, l.first, step, w.size);
        gy.get(d, l.first, step, w.size);
        gate.get(g, l.first, step, w.size);
        if (r + l.rows_step < w.rows) fetch(r + l.rows_step);
        const float rstd = normalise<W>(h, l.first, step, w.size, w.eps, w.rms);
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int i = 0; i < K; i++)
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float u = fmaf(h[i][e], weight[i][e], bias[i][e]);
                float du;
                if (gs) {
                    du = d[i][e] * act_of(g[i][e], w.act);
                    g[i][e] = d[i][e] * u * slope_of(g[i][e], w.act);
                } else {
                    du = d[i][e] * slope_of(u, w.act);
                }
                gw[i][e] = fmaf(du, h[i][e], gw[i][e]), gb[i][e] += du;
                d[i][e] = du * weight[i][e];
                s0 += d[i][e], s1 = fmaf(d[i][e], h[i][e], s1);
            }
        const float inv = 1.f / (float)w.size, m0 = w.rms ? 0.f : lanes_sum<W>(s0) * inv, m1 = lanes_sum<W>(s1) * inv;
#pragma unroll
        for (int i = 0; i < K; i++)
#pragma unroll
            for (int e = 0; e < V; e++) d[i][e] = rstd * (d[i][e] - fmaf(h[i][e], m1, m0));
        Run<T, K, ODD>::store(d, static_cast<T *>(w.gx) + off + r * width, l.first, step, w.size);
        if (gs) Run<T, K, ODD>::store(g, static_cast<T *>(w.ggate) + off + r * width, l.first, step, w.size);
    }
    if (!w.sums) return;
    const int lane = threadIdx.x % 64;
    if (l.wave > 0) {
#pragma unroll
        for (int i = 0; i < K; i++)
#pragma unroll
            for (int e = 0; e < V; e++) sums[l.wave - 1][0][(i * V + e) * 64 + lane] = gw[i][e], sums[l.wave - 1][1][(i * V + e) * 64 + lane] = gb[i][e];
    }
    __syncthreads();
    if (l.wave > 0 || !l.live) return;
    float *to = w.sums + (blockIdx.x % w.blocks) * 2 * width + off;
#pragma unroll
    for (int i = 0; i < K; i++)
#pragma unroll
        for (int e = 0; e < V; e++) {
            const int at = (i * V + e) * 64 + lane, c = l.first + i * step + e;
            if (c >= w.size) continue;
            to[c] = (gw[i][e] + sums[0][0][at]) + (sums[1][0][at] + sums[2][0][at]);
            to[width + c] = (gb[i][e] + sums[0][1][at]) + (sums[1][1][at] + sums[2][1][at]);
        }
}

// The workgroups' sums added: 8 columns and 32 parts of the workgroups to a workgroup here
__global__ __launch_bounds__(256) void k_group_norm_sums(const float *sums, float *gweight, float *gbias, int blocks, int64_t width) {
    __shared__ float part[32][9];
    const int c = threadIdx.x % 8, y = threadIdx.x / 8;
    const int64_t col = (int64_t)blockIdx.x * 8 + c;
    float s = 0.f;
    if (col < 2 * width) {
#pragma unroll 8
        for (int b = y; b < blocks; b += 32) s += sums[b * 2 * width + col];
    }
    part[y][c] = s;
    __syncthreads();
    if (y || col >= 2 * width) return;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; i++) s += part[i][c];
    float *to = col < width ? gweight : gbias;
    if (to) to[col < width ? col : col - width] = s;
}

// The workgroups of a run of groups: four to a CU over all runs, and no more than have rows
int row_blocks(int rows, int runs) { return std::max(1, std::min((rows + 3) / 4, 256 * 4 / runs)); }
int lanes_of(int type, int size) {
    const int V = type == FWP_F32 ? 4 : 8;
    int W = 1;
    while (W * V < size && W < 64) W *= 2;
    return W;
}

template <typename T, int W, int K, bool BACKWARD>
void launch(NormWalk w, hipStream_t s) {
    const int runs = (w.groups + 64 / W - 1) / (64 / W);
    w.blocks = row_blocks(w.rows, runs);
    const unsigned grid = (unsigned)(runs * w.blocks);
    const bool odd = w.size % (16 / (int)sizeof(T)) != 0;
    if constexpr (BACKWARD) {
        if (odd) k_group_norm_bwd<T, W, K, true><<<grid, 256, 0, s>>>(w);
        else k_group_norm_bwd<T, W, K, false><<<grid, 256, 0, s>>>(w);
    } else {
        if (odd) k_group_norm_fwd<T, W, K, true><<<grid, 256, 0, s>>>(w);
        else k_group_norm_fwd<T, W, K, false><<<grid, 256, 0, s>>>(w);
    }
}
template <typename T, bool BACKWARD>
void by_size(const NormWalk &w, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int vecs = (w.size + V - 1) / V;
    if (vecs <= 1) launch<T, 1, 1, BACKWARD>(w, s);
    else if (vecs <= 2) launch<T, 2, 1, BACKWARD>(w, s);
    else if (vecs <= 4) launch<T, 4, 1, BACKWARD>(w, s);
    else if (vecs <= 8) launch<T, 8, 1, BACKWARD>(w, s);
    else if (vecs <= 16) launch<T, 16, 1, BACKWARD>(w, s);
    else if (vecs <= 32) launch<T, 32, 1, BACKWARD>(w, s);
    else if (vecs <= 64) launch<T, 64, 1, BACKWARD>(w, s);
    else if (vecs <= 128) launch<T, 64, 2, BACKWARD>(w, s);
    else if constexpr (sizeof(T) == 4) launch<T, 64, 4, BACKWARD>(w, s);
}

NormWalk walk_of(const fwp_group_norm_args &a) {
    NormWalk w{};
    w.x = a.x, w.gate = a.gate, w.x_step = a.x_step, w.gate_step = a.gate_step, w.weight = a.weight, w.bias = a.bias;
    w.eps = a.eps, w.rms = a.rms, w.act = a.act, w.rows = a.rows, w.groups = a.groups, w.size = a.size;
    return w;
}
int blocks_of(int type, int rows, int groups, int size) {
    const int per = 64 / lanes_of(type, size);
    return row_blocks(rows, (groups + per - 1) / per);
}

}  // namespace

int64_t group_norm_workspace(int type, int rows, int groups, int size) { return 2 * (int64_t)blocks_of(type, rows, groups, size) * groups * size; }

int group_norm_fwd(const fwp_group_norm_args &a, void *y, hipStream_t s) {
    NormWalk w = walk_of(a);
    w.y = y;
    by_type(a.type, [&](auto t) { by_size<decltype(t), false>(w, s); });
    return (int)hipGetLastError();
}

int group_norm_bwd(const fwp_group_norm_args &a, const void *gy, void *gx, void *ggate, float *gweight, float *gbias, float *workspace,
                   hipStream_t s) {
    NormWalk w = walk_of(a);
    w.gy = gy, w.gx = gx, w.ggate = ggate;
    w.sums = gweight || gbias ? workspace : nullptr;
    by_type(a.type, [&](auto t) { by_size<decltype(t), true>(w, s); });
    if (w.sums) {
        const int64_t width = (int64_t)a.groups * a.size;
        k_group_norm_sums<<<(unsigned)((2 * width + 7) / 8), 256, 0, s>>>(workspace, gweight, gbias, blocks_of(a.type, a.rows, a.groups, a.size), width);
    }
    return (int)hipGetLastError();
}

}  // namespace fwp
