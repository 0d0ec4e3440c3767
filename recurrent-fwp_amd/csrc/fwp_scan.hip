// Selective scan: the sum rule with a decay that depends on the token, forward and backward.
//
//   dt = softplus(delta + bias)    W[e][m] = exp(dt[m] A[e][m]) W[e][m] + dt[m] v[m] k[e]    o[m] = sum_e q[e] W[e][m] + D[m] v[m]
//   out = o z sigmoid(z)
// and backwards, with dy = gout z sigmoid(z) and g the gradient of the state after a step:
//   g = dy q + c,  c (of the state before the step) = a g,  a = exp(dt A),  w = a W_before g
//   gq = sum_m dy W    gk = sum_m g dt v    gv = dt sum_e g k + D dy    gdt = v sum_e g k + sum_e A w    gA = sum dt w    gD = sum dy v
//
// A workgroup takes 64 channels of one sequence and head: a lane is a channel, a wave four entries of the state (key rows), so
// that k and q of a step are scalars for the wave (packed as fp32 beforehand, read through the scalar cache), a state and its
// history stay in registers, and a sum over the channels is a sum over the lanes.  Steps go in tiles of kTile rows: each thread loads its
// rows of v, delta, z once, works out dt and dt v, and puts them into LDS for all waves; the waves' parts of a sum over e meet in LDS
// and the thread that loaded a row finishes it.
//
// Few sequences and channels leave most of the chip idle, so a long sequence is cut into segments that run at the same time:
// a first pass gives each segment's state from zeros and its sum of dt, a small kernel turns these into the state that each segment
// starts from (the decay over a segment is exp(A sum dt), whatever its length), and the second pass is the scan itself.  That doubles the
// exponentials, which is what bounds these kernels, so a call that fills the chip is not cut.
#include "fwp_elements.hpp"
#include "fwp_wave.hpp"

#include <algorithm>

namespace fwp {
namespace {

constexpr int kRowMirror8 = 0x141;      // lane i of 8 gets lane 7 - i

// For 1, 2, 4, 8 or 16 waves of four state rows each.  The widest states have half the tile: 16 waves leave 128 registers to a lane.
constexpr int tile_of(int waves) { return waves == 16 ? 8 : 16; }
int waves_of(int E) { return E <= 4 ? 1 : E <= 8 ? 2 : E <= 16 ? 4 : E <= 32 ? 8 : 16; }

using scalar_float = const float __attribute__((address_space(4)));

struct Dims {
    int N, H, L, E, M;
    int blocks_m;       // 64 channels each
    int segments, steps;      // per sequence, and steps of a segment (a multiple of the tile)
    int padded;         // L rounded up to whole tiles: rows of the packed k and q
    int tiles;
};

struct Plan : Dims {
    int waves, tile;
    int64_t heads, packed, states;      // N H; floats of packed k and q; floats of one set of states
    Plan(int N_, int H_, int L_, int E_, int M_, bool backward) {
        N = N_, H = H_, L = L_, E = E_, M = M_;
        waves = waves_of(E), tile = tile_of(waves);
        blocks_m = (M + 63) / 64;
        tiles = (L + tile - 1) / tile;
        padded = tiles * tile;
        heads = (int64_t)N * H;
        packed = heads * waves * padded * 8;
        states = heads * E * M;
        const int64_t blocks = heads * blocks_m;
        int64_t want = blocks >= 256 ? 1 : (512 + blocks - 1) / blocks;
        want = std::max<int64_t>(1, std::min<int64_t>(want, tiles / 4));
        const int per = (int)((tiles + want - 1) / want);      // tiles to a segment
        segments = (tiles + per - 1) / per;
        steps = per * tile;
        (void)backward;
    }
    int64_t grid() const { return heads * blocks_m * segments; }
    int64_t seg_states() const { return segments > 1 ? states * segments + heads * segments * M : 0; }      // the states and the sums of dt
};

// ------------------------------------------------------------------ k and q, packed

// kq [heads][waves][padded][k0..k3 | q0..q3], zero where there is no such row, step or entry (so that whatever a padded row holds stays out)
template <typename T>
__global__ __launch_bounds__(256) void k_pack(fwp_rows q, fwp_rows k, const int64_t *__restrict__ lengths, float *__restrict__ kq,
                                              int H, int L, int E, int padded, int chunks) {
    const int64_t nh = blockIdx.x / chunks;
    const int i = (blockIdx.x % chunks) * 256 + threadIdx.x, t = i / 8, j = i % 8, w = blockIdx.y, e = 4 * w + j % 4;
    if (t >= padded) return;
    const int n = (int)(nh / H), h = (int)(nh % H);
    float x = 0.f;
    if (e < E && t < length_of(lengths, n, L)) x = load(row<T>(j < 4 ? k : q, n, h, t) + e);
    kq[(nh * gridDim.y + w) * padded * 8 + i] = x;
}

// ------------------------------------------------------------------ what the passes share

struct Place {
    int n, h, m, seg, wave, lane;
    int64_t nh;
    bool live;      // a channel that exists
    __device__ __forceinline__ Place(const Dims &d) {
        int64_t b = blockIdx.x;
        const int mb = (int)(b % d.blocks_m);
        b /= d.blocks_m;
        seg = (int)(b % d.segments);
        nh = b / d.segments;
        n = (int)(nh / d.H), h = (int)(nh % d.H);
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
        m = mb * 64 + lane;
        live = m < d.M;
    }
    // state row e of this channel in a [.., E, M] array's block `at`
    __device__ __forceinline__ int64_t state(const Dims &d, int64_t at, int e) const { return (at * d.E + e) * d.M + m; }
};

// A log2(e) of the wave's four rows
__device__ __forceinline__ void load_decays(float (&a)[4], const float *A, const Dims &d, const Place &p) {
#pragma unroll
    for (int s = 0; s < 4; s++) {
        const int e = 4 * p.wave + s;
        a[s] = p.live && e < d.E ? A[p.state(d, p.h, e)] * kLog2e : 0.f;
    }
}
__device__ __forceinline__ void load_states(float (&x)[4], const float *from, int64_t at, const Dims &d, const Place &p) {
#pragma unroll
    for (int s = 0; s < 4; s++) {
        const int e = 4 * p.wave + s;
        x[s] = from && p.live && e < d.E ? from[p.state(d, at, e)] : 0.f;
    }
}
__device__ __forceinline__ void store_states(const float (&x)[4], float *to, int64_t at, const Dims &d, const Place &p) {
#pragma unroll
    for (int s = 0; s < 4; s++) {
        const int e = 4 * p.wave + s;
        if (p.live && e < d.E) to[p.state(d, at, e)] = x[s];
    }
}

// The parameters of a channel that the threads which load its rows need
struct Channel {
    float D, bias;
    __device__ __forceinline__ Channel(const fwp_scan_args &a, const Place &p) {
        const int64_t at = (int64_t)p.h * a.M + p.m;
        D = p.live && a.D ? a.D[at] : 0.f;
        bias = p.live && a.delta_bias ? a.delta_bias[at] : 0.f;
    }
};

// ------------------------------------------------------------------ forward

// LOCAL: only the state after the segment, from zeros, and the segment's sum of dt; otherwise the scan
template <typename T, int WAVES, bool LOCAL>
__global__ __launch_bounds__(64 * WAVES) void k_scan_fwd(fwp_scan_args a, Dims d, const float *__restrict__ kq, const float *init, float *W,
                                                         float *__restrict__ saved, float *__restrict__ sums, fwp_out_rows out) {
    constexpr int TILE = tile_of(WAVES), ROWS = (TILE + WAVES - 1) / WAVES;
    __shared__ float2 sx[TILE][64];                          // dt, dt v
    __shared__ float sy[LOCAL ? 1 : WAVES][TILE][64];        // the waves' parts of sum_e q W
    const Place p(d);
    const Channel ch(a, p);
    const int len = length_of(a.lengths, p.n, d.L), first = p.seg * d.steps, end = min(first + d.steps, d.L);
    float decay[4], state[4];
    load_decays(decay, a.A, d, p);
    load_states(state, LOCAL ? nullptr : init, p.nh * d.segments + p.seg, d, p);
    float sum = 0.f;
    for (int t0 = first; t0 < end; t0 += TILE) {
        if (t0 >= len) {        // behind the sequence
            if constexpr (!LOCAL)
#pragma unroll
                for (int j = 0; j < ROWS; j++) {
                    const int t = t0 + p.wave + WAVES * j;
                    if (p.wave + WAVES * j < TILE && t < end && p.live) store(row<T>(out, p.n, p.h, t) + p.m, 0.f);
                }
            continue;
        }
        if constexpr (!LOCAL)
            if (saved) store_states(state, saved, p.nh * d.tiles + t0 / TILE, d, p);
        float v[ROWS];
#pragma unroll
        for (int j = 0; j < ROWS; j++) {
            const int r = p.wave + WAVES * j, t = t0 + r;
            float dt = 0.f;
            v[j] = 0.f;
            if (r < TILE && t < len && p.live) {
                v[j] = load(row<T>(a.v, p.n, p.h, t) + p.m);
                dt = load(row<T>(a.delta, p.n, p.h, t) + p.m) + ch.bias;
                if (a.softplus) dt = softplus(dt);
            }
            if (r < TILE) sx[r][p.lane] = make_float2(dt, dt * v[j]);
        }
        __syncthreads();
        scalar_float *const ks = (scalar_float *)(kq + ((p.nh * WAVES + p.wave) * d.padded + t0) * 8);
#pragma unroll
        for (int r = 0; r < TILE; r++) {
            const float2 x = sx[r][p.lane];
            float y = 0.f;
#pragma unroll
            for (int s = 0; s < 4; s++) {
                state[s] = fmaf(__builtin_amdgcn_exp2f(x.x * decay[s]), state[s], x.y * ks[8 * r + s]);
                if constexpr (!LOCAL) y = fmaf(ks[8 * r + 4 + s], state[s], y);
            }
            if constexpr (LOCAL) sum += x.x;
            else sy[p.wave][r][p.lane] = y;
        }
        __syncthreads();
        if constexpr (!LOCAL)
#pragma unroll
            for (int j = 0; j < ROWS; j++) {
                const int r = p.wave + WAVES * j, t = t0 + r;
                if (r >= TILE || t >= end || !p.live) continue;
                float o = ch.D * v[j];
#pragma unroll
                for (int w = 0; w < WAVES; w++) o += sy[w][r][p.lane];
                if (a.z.ptr && t < len) {
                    const float z = load(row<T>(a.z, p.n, p.h, t) + p.m);
                    o *= silu(z, sigmoid(z));
                }
                store(row<T>(out, p.n, p.h, t) + p.m, t < len ? o : 0.f);
            }
    }
    if constexpr (LOCAL) {
        store_states(state, W, p.nh * d.segments + p.seg, d, p);
        if (p.wave == 0 && p.live) sums[(p.nh * d.segments + p.seg) * d.M + p.m] = sum;
    } else if (W) {
        store_states(state, W, p.nh, d, p);     // one segment: the state that the call keeps
    }
}

// From each segment's own state (or gradient) to the one it starts from: after a segment x becomes exp(A sum dt) x + own.  The
// exponential is applied as two halves, which reach twice as far before one of them is infinite.
template <bool REVERSE>
__global__ __launch_bounds__(256) void k_chain(const float *__restrict__ A, const float *__restrict__ sums, float *__restrict__ own,
                                               const float *W_in, float *W_out, Dims d) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = (int64_t)d.E * d.M;
    if (i >= (int64_t)d.N * d.H * per) return;
    const int64_t nh = i / per, em = i % per;
    const int m = (int)(em % d.M);
    const float half = 0.5f * kLog2e * A[(nh % d.H) * per + em];
    float x = W_in ? W_in[i] : 0.f;
    constexpr int AHEAD = 8;
    for (int s0 = 0; s0 < d.segments; s0 += AHEAD) {
        float o[AHEAD], dt[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            const int k = min(s0 + j, d.segments - 1), seg = REVERSE ? d.segments - 1 - k : k;
            const int64_t at = nh * d.segments + seg;
            o[j] = own[at * per + em];
            dt[j] = sums[at * d.M + m];
        }
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            if (s0 + j >= d.segments) continue;
            const int seg = REVERSE ? d.segments - 1 - (s0 + j) : s0 + j;
            own[(nh * d.segments + seg) * per + em] = x;
            const float e = __builtin_amdgcn_exp2f(half * dt[j]);
            x = fmaf(e, e * x, o[j]);
        }
    }
    if (W_out) W_out[i] = x;
}

// ------------------------------------------------------------------ backward

// The gradient of the state before the segment, from zeros behind it
template <typename T, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_scan_bwd_local(fwp_scan_args a, Dims d, const float *__restrict__ kq, fwp_rows gout,
                                                               float *__restrict__ own, float *__restrict__ sums) {
    constexpr int TILE = tile_of(WAVES), ROWS = (TILE + WAVES - 1) / WAVES;
    __shared__ float2 sx[TILE][64];     // dt, dy
    const Place p(d);
    const Channel ch(a, p);
    const int len = length_of(a.lengths, p.n, d.L), first = p.seg * d.steps, end = min(first + d.steps, d.L);
    float decay[4], c[4] = {}, sum = 0.f;
    load_decays(decay, a.A, d, p);
    for (int t0 = first + (end - first - 1) / TILE * TILE; t0 >= first; t0 -= TILE) {
        if (t0 >= len) continue;
#pragma unroll
        for (int j = 0; j < ROWS; j++) {
            const int r = p.wave + WAVES * j, t = t0 + r;
            float dt = 0.f, dy = 0.f;
            if (r < TILE && t < len && p.live) {
                dy = load(row<T>(gout, p.n, p.h, t) + p.m);
                dt = load(row<T>(a.delta, p.n, p.h, t) + p.m) + ch.bias;
                if (a.softplus) dt = softplus(dt);
                if (a.z.ptr) {
                    const float z = load(row<T>(a.z, p.n, p.h, t) + p.m);
                    dy *= silu(z, sigmoid(z));
                }
            }
            if (r < TILE) sx[r][p.lane] = make_float2(dt, dy);
        }
        __syncthreads();
        scalar_float *const ks = (scalar_float *)(kq + ((p.nh * WAVES + p.wave) * d.padded + t0) * 8);
#pragma unroll
        for (int r = TILE - 1; r >= 0; r--) {
            const float2 x = sx[r][p.lane];
#pragma unroll
            for (int s = 0; s < 4; s++) c[s] = fmaf(x.y, ks[8 * r + 4 + s], c[s]) * __builtin_amdgcn_exp2f(x.x * decay[s]);
            sum += x.x;
        }
        __syncthreads();
    }
    store_states(c, own, p.nh * d.segments + p.seg, d, p);
    if (p.wave == 0 && p.live) sums[(p.nh * d.segments + p.seg) * d.M + p.m] = sum;
}

// parts: [blocks_m][heads][padded][waves][gk0..gk3 | gq0..gq3], the sums over 64 channels
// params: [N segments][H][E + 2][M]: gA, gD, gdelta_bias of one segment
template <typename T, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_scan_bwd(fwp_scan_args a, Dims d, const float *__restrict__ kq, const float *__restrict__ saved,
                                                         const float *__restrict__ init, fwp_rows gout, fwp_out_rows gv, fwp_out_rows gdelta,
                                                         fwp_out_rows gz, float *__restrict__ parts, float *__restrict__ params) {
    constexpr int TILE = tile_of(WAVES), ROWS = (TILE + WAVES - 1) / WAVES;
    __shared__ float2 sx[TILE][64];                      // dt, dt v
    __shared__ float sg[TILE][64];                       // dy
    __shared__ float part[3][WAVES][TILE][64];           // the waves' parts of sum_e g k, sum_e A w (times log2 e), sum_e q W
    const Place p(d);
    const Channel ch(a, p);
    const int len = length_of(a.lengths, p.n, d.L), first = p.seg * d.steps, end = min(first + d.steps, d.L);
    float decay[4], c[4], gA[4] = {}, gD = 0.f, gbias = 0.f;
    load_decays(decay, a.A, d, p);
    load_states(c, init, p.nh * d.segments + p.seg, d, p);
    for (int t0 = first + (end - first - 1) / TILE * TILE; t0 >= first; t0 -= TILE) {
        if (t0 >= len) {
#pragma unroll
            for (int j = 0; j < ROWS; j++) {
                const int t = t0 + p.wave + WAVES * j;
                if (p.wave + WAVES * j >= TILE || t >= end || !p.live) continue;
                store(row<T>(gv, p.n, p.h, t) + p.m, 0.f);
                store(row<T>(gdelta, p.n, p.h, t) + p.m, 0.f);
                if (a.z.ptr) store(row<T>(gz, p.n, p.h, t) + p.m, 0.f);
            }
            continue;
        }
        float v[ROWS], pre[ROWS], go[ROWS], z[ROWS];
#pragma unroll
        for (int j = 0; j < ROWS; j++) {
            const int r = p.wave + WAVES * j, t = t0 + r;
            float dt = 0.f, dy = 0.f;
            v[j] = pre[j] = go[j] = z[j] = 0.f;
            if (r < TILE && t < len && p.live) {
                v[j] = load(row<T>(a.v, p.n, p.h, t) + p.m);
                pre[j] = load(row<T>(a.delta, p.n, p.h, t) + p.m) + ch.bias;
                dt = a.softplus ? softplus(pre[j]) : pre[j];
                dy = go[j] = load(row<T>(gout, p.n, p.h, t) + p.m);
                if (a.z.ptr) {
                    z[j] = load(row<T>(a.z, p.n, p.h, t) + p.m);
                    dy *= silu(z[j], sigmoid(z[j]));
                }
            }
            if (r < TILE) sx[r][p.lane] = make_float2(dt, dt * v[j]), sg[r][p.lane] = dy;
        }
        __syncthreads();
        scalar_float *const ks = (scalar_float *)(kq + ((p.nh * WAVES + p.wave) * d.padded + t0) * 8);
        float before[TILE + 1][4], al[TILE][4];      // the states before each step, and its decays
        load_states(before[0], saved, p.nh * d.tiles + t0 / TILE, d, p);
#pragma unroll
        for (int r = 0; r < TILE; r++) {
            const float2 x = sx[r][p.lane];
            float y = 0.f;
#pragma unroll
            for (int s = 0; s < 4; s++) {
                al[r][s] = __builtin_amdgcn_exp2f(x.x * decay[s]);
                before[r + 1][s] = fmaf(al[r][s], before[r][s], x.y * ks[8 * r + s]);
                y = fmaf(ks[8 * r + 4 + s], before[r + 1][s], y);
            }
            part[2][p.wave][r][p.lane] = y;
        }
        // One step back; what is summed over the channels comes out in `sums`: gk of the four rows, then gq
        const auto back = [&](int r, float (&sums)[8]) {
            const float2 x = sx[r][p.lane];
            const float dy = sg[r][p.lane];
            float read = 0.f, slope = 0.f;
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const float g = fmaf(dy, ks[8 * r + 4 + s], c[s]);
                sums[s] = g * x.y;
                sums[4 + s] = dy * before[r + 1][s];
                read = fmaf(g, ks[8 * r + s], read);
                c[s] = g * al[r][s];
                const float w = c[s] * before[r][s];
                slope = fmaf(w, decay[s], slope);
                gA[s] = fmaf(w, x.x, gA[s]);
            }
            part[0][p.wave][r][p.lane] = read;
            part[1][p.wave][r][p.lane] = slope;
        };
        // The sums over the lanes, halving what a lane holds as it goes: after eight steps lane l has the sum number l % 8 of the step whose bits
        // 0, 1, 2 are l's bits 5, 4, 3.
#pragma unroll
        for (int r0 = TILE - 8; r0 >= 0; r0 -= 8) {
            float eight[2][8];
#pragma unroll
            for (int q2 = 1; q2 >= 0; q2--) {
                float four[2][8];
#pragma unroll
                for (int q1 = 1; q1 >= 0; q1--) {
                    float odd[8], even[8];
                    back(r0 + 4 * q2 + 2 * q1 + 1, odd);
                    back(r0 + 4 * q2 + 2 * q1, even);
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        swap32(even[i], odd[i]);
                        four[q1][i] = even[i] + odd[i];
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    swap16(four[0][i], four[1][i]);
                    eight[q2][i] = pinned(four[0][i] + four[1][i]);
                }
            }
            const bool b3 = p.lane & 8, b2 = p.lane & 4, b1 = p.lane & 2, b0 = p.lane & 1;
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = pinned((b3 ? eight[1][i] : eight[0][i]) + dpp<kRowRor8>(b3 ? eight[0][i] : eight[1][i]));
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = pinned((b2 ? x[i + 4] : x[i]) + dpp<kRowMirror8>(b2 ? x[i] : x[i + 4]));
#pragma unroll
            for (int i = 0; i < 2; i++) x[i] = pinned((b1 ? x[i + 2] : x[i]) + dpp<kQuadXor2>(b1 ? x[i] : x[i + 2]));
            x[0] = pinned((b0 ? x[1] : x[0]) + dpp<kQuadXor1>(b0 ? x[0] : x[1]));
            const int t = t0 + r0 + (p.lane >> 5 & 1) + 2 * (p.lane >> 4 & 1) + 4 * (p.lane >> 3 & 1);
            const int64_t mb = blockIdx.x % d.blocks_m;
            parts[(((mb * d.N * d.H + p.nh) * d.padded + t) * WAVES + p.wave) * 8 + p.lane % 8] = x[0];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ROWS; j++) {
            const int r = p.wave + WAVES * j, t = t0 + r;
            if (r >= TILE || t >= end || !p.live) continue;
            float read = 0.f, slope = 0.f, o = ch.D * v[j];
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                read += part[0][w][r][p.lane];
                slope += part[1][w][r][p.lane];
                o += part[2][w][r][p.lane];
            }
            const float dt = sx[r][p.lane].x, dy = sg[r][p.lane];
            float gdt = fmaf(v[j], read, kLn2 * slope);
            if (a.softplus) gdt *= sigmoid(pre[j]);
            const bool in = t < len;
            store(row<T>(gv, p.n, p.h, t) + p.m, in ? fmaf(dt, read, ch.D * dy) : 0.f);
            store(row<T>(gdelta, p.n, p.h, t) + p.m, in ? gdt : 0.f);
            if (a.z.ptr) store(row<T>(gz, p.n, p.h, t) + p.m, in ? go[j] * o * silu_slope(z[j], sigmoid(z[j])) : 0.f);
            if (in) gD = fmaf(dy, v[j], gD), gbias += gdt;
        }
        __syncthreads();        // the next tile overwrites what this one's last rows are read from
    }
    float *const to = params + ((int64_t)(p.n * d.segments + p.seg) * d.H + p.h) * (d.E + 2) * d.M + p.m;
#pragma unroll
    for (int s = 0; s < 4; s++)
        if (p.live && 4 * p.wave + s < d.E) to[(int64_t)(4 * p.wave + s) * d.M] = gA[s];
    // the waves' rows of a channel
    part[0][p.wave][0][p.lane] = gD;
    part[1][p.wave][0][p.lane] = gbias;
    __syncthreads();
    if (p.wave == 0 && p.live) {
        for (int w = 1; w < WAVES; w++) gD += part[0][w][0][p.lane], gbias += part[1][w][0][p.lane];
        to[(int64_t)d.E * d.M] = gD;
        to[(int64_t)(d.E + 1) * d.M] = gbias;
    }
}

// The sums over the channels' blocks to gq and gk, and those over sequences and segments to the parameters' gradients, each in a fixed order
template <typename T>
__global__ __launch_bounds__(256) void k_scan_finish(const float *__restrict__ parts, const float *__restrict__ params, fwp_out_rows gq,
                                                     fwp_out_rows gk, float *__restrict__ gA, float *__restrict__ gD,
                                                     float *__restrict__ gbias, const int64_t *__restrict__ lengths, Dims d, int waves,
                                                     int64_t row_blocks) {
    if (blockIdx.x < row_blocks) {
        const int width = waves * 8;
        const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, heads = (int64_t)d.N * d.H;
        const int64_t nh = i / ((int64_t)d.L * width), rest = i % ((int64_t)d.L * width);
        const int t = (int)(rest / width), j = (int)(rest % width), e = j / 8 * 4 + j % 4;
        if (nh >= heads || e >= d.E) return;
        const int n = (int)(nh / d.H), h = (int)(nh % d.H);
        float x = 0.f;
        if (t < length_of(lengths, n, d.L))
            for (int mb = 0; mb < d.blocks_m; mb++) x += parts[((mb * heads + nh) * d.padded + t) * width + j];
        store(row<T>(j % 8 < 4 ? gk : gq, n, h, t) + e, x);
        return;
    }
    // 64 columns and four slices of the sequences and segments to a workgroup
    __shared__ float sh[4][64];
    const int64_t per = (int64_t)d.H * (d.E + 2) * d.M, i = (blockIdx.x - row_blocks) * 64 + threadIdx.x % 64;
    const int slice = threadIdx.x / 64, terms = d.N * d.segments;
    float x = 0.f;
    if (i < per)
        for (int k = slice; k < terms; k += 4) x += params[k * per + i];
    sh[slice][threadIdx.x % 64] = x;
    __syncthreads();
    if (slice || i >= per) return;
    x = (sh[0][threadIdx.x] + sh[1][threadIdx.x]) + (sh[2][threadIdx.x] + sh[3][threadIdx.x]);
    const int64_t h = i / ((int64_t)(d.E + 2) * d.M), em = i % ((int64_t)(d.E + 2) * d.M), rows = (int64_t)d.E * d.M;
    if (em < rows) gA[h * rows + em] = x;
    else if (em < rows + d.M) gD[h * d.M + em - rows] = x;
    else gbias[h * d.M + em - rows - d.M] = x;
}

// ------------------------------------------------------------------ one step

// Four waves share the state rows of 64 channels
template <typename T>
__global__ __launch_bounds__(256) void k_scan_step(fwp_scan_args a, float *__restrict__ W, fwp_out_rows out) {
    __shared__ float sy[4][64];
    const int blocks_m = (a.M + 63) / 64;
    const int64_t nh = blockIdx.x / blocks_m;
    const int n = (int)(nh / a.H), h = (int)(nh % a.H), lane = threadIdx.x % 64, m = (int)(blockIdx.x % blocks_m) * 64 + lane,
              wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const bool live = m < a.M;
    if (length_of(a.lengths, n, 1) == 0) {      // the whole workgroup
        if (wave == 0 && live) store(row<T>(out, n, h, 0) + m, 0.f);
        return;
    }
    const int64_t at = (int64_t)h * a.M + m;
    float y = 0.f, v = 0.f;
    if (live) {
        v = load(row<T>(a.v, n, h, 0) + m);
        float dt = load(row<T>(a.delta, n, h, 0) + m) + (a.delta_bias ? a.delta_bias[at] : 0.f);
        if (a.softplus) dt = softplus(dt);
        const T *const q = row<T>(a.q, n, h, 0), *const k = row<T>(a.k, n, h, 0);
        const float *const A = a.A + (int64_t)h * a.E * a.M + m;
        float *const w = W ? W + nh * a.E * a.M + m : nullptr;
#pragma unroll 4
        for (int e = wave; e < a.E; e += 4) {
            float x = dt * v * load(k + e);
            if (w) {
                x = fmaf(exp_of(dt * A[(int64_t)e * a.M]), w[(int64_t)e * a.M], x);
                w[(int64_t)e * a.M] = x;
            }
            y = fmaf(load(q + e), x, y);
        }
    }
    sy[wave][lane] = y;
    __syncthreads();
    if (wave || !live) return;
    float o = (sy[0][lane] + sy[1][lane]) + (sy[2][lane] + sy[3][lane]) + (a.D ? a.D[at] * v : 0.f);
    if (a.z.ptr) {
        const float z = load(row<T>(a.z, n, h, 0) + m);
        o *= silu(z, sigmoid(z));
    }
    store(row<T>(out, n, h, 0) + m, o);
}

// ------------------------------------------------------------------ launches

template <typename F>
void by_waves(int waves, F f) {
    switch (waves) {
        case 1: f(std::integral_constant<int, 1>()); break;
        case 2: f(std::integral_constant<int, 2>()); break;
        case 4: f(std::integral_constant<int, 4>()); break;
        case 8: f(std::integral_constant<int, 8>()); break;
        default: f(std::integral_constant<int, 16>()); break;
    }
}

constexpr int64_t kMaxBlocks = (int64_t(1) << 31) - 1;

}  // namespace

int64_t scan_saved_floats(int N, int H, int L, int E, int M) {
    const Plan p(N, H, L, E, M, false);
    return p.packed + p.states * p.tiles;
}

int64_t scan_workspace(int N, int H, int L, int E, int M, bool backward) {
    const Plan p(N, H, L, E, M, backward);
    if (!backward) return p.packed + p.seg_states();
    return p.blocks_m * p.heads * p.padded * p.waves * 8 + (int64_t)N * p.segments * H * (E + 2) * M + p.seg_states();
}

int scan_fwd(const fwp_scan_args &a, float *W, fwp_out_rows out, float *saved, float *workspace, hipStream_t s) {
    if (a.L == 1 && !saved) {
        const int64_t grid = (int64_t)a.N * a.H * ((a.M + 63) / 64);
        if (grid > kMaxBlocks) return FWP_E_SHAPE;
        by_type(a.type, [&](auto t) { hipLaunchKernelGGL((k_scan_step<decltype(t)>), dim3((unsigned)grid), dim3(256), 0, s, a, W, out); });
        return (int)hipGetLastError();
    }
    const Plan p(a.N, a.H, a.L, a.E, a.M, false);
    const int chunks = (int)(((int64_t)p.padded * 8 + 255) / 256);
    if (p.grid() > kMaxBlocks || p.heads * chunks > kMaxBlocks || (p.states + 255) / 256 > kMaxBlocks) return FWP_E_SHAPE;
    float *const kq = saved ? saved : workspace, *const ckpt = saved ? saved + p.packed : nullptr, *const seg = workspace + (saved ? 0 : p.packed),
                *const sums = seg + p.states * p.segments;
    const Dims d = p;
    by_type(a.type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((k_pack<T>), dim3((unsigned)(p.heads * chunks), p.waves), dim3(256), 0, s, a.q, a.k, a.lengths, kq, a.H, a.L, a.E,
                           p.padded, chunks);
        by_waves(p.waves, [&](auto w) {
            constexpr int WAVES = decltype(w)::value;
            const dim3 grid((unsigned)p.grid()), block(64 * WAVES);
            if (p.segments > 1) {
                hipLaunchKernelGGL((k_scan_fwd<T, WAVES, true>), grid, block, 0, s, a, d, kq, nullptr, seg, nullptr, sums, out);
                hipLaunchKernelGGL((k_chain<false>), dim3((unsigned)((p.states + 255) / 256)), dim3(256), 0, s, a.A, sums, seg, W, W, d);
            }
            hipLaunchKernelGGL((k_scan_fwd<T, WAVES, false>), grid, block, 0, s, a, d, kq, p.segments > 1 ? seg : W,
                               p.segments > 1 ? nullptr : W, ckpt, nullptr, out);
        });
    });
    return (int)hipGetLastError();
}

int scan_bwd(const fwp_scan_args &a, const float *saved, fwp_rows gout, fwp_out_rows gq, fwp_out_rows gk, fwp_out_rows gv,
             fwp_out_rows gdelta, fwp_out_rows gz, float *gA, float *gD, float *gdelta_bias, float *workspace, hipStream_t s) {
    const Plan p(a.N, a.H, a.L, a.E, a.M, true);
    const int64_t row_blocks = (p.heads * a.L * p.waves * 8 + 255) / 256,
                  param_blocks = ((int64_t)a.H * (a.E + 2) * a.M + 63) / 64;
    if (p.grid() > kMaxBlocks || row_blocks + param_blocks > kMaxBlocks || (p.states + 255) / 256 > kMaxBlocks ||
        (int64_t)a.N * p.segments > kMaxBlocks)
        return FWP_E_SHAPE;
    const float *const kq = saved, *const ckpt = saved + p.packed;
    float *const parts = workspace, *const params = parts + p.blocks_m * p.heads * p.padded * p.waves * 8,
                *const seg = params + (int64_t)a.N * p.segments * a.H * (a.E + 2) * a.M, *const sums = seg + p.states * p.segments;
    const Dims d = p;
    by_type(a.type, [&](auto t) {
        using T = decltype(t);
        by_waves(p.waves, [&](auto w) {
            constexpr int WAVES = decltype(w)::value;
            const dim3 grid((unsigned)p.grid()), block(64 * WAVES);
            if (p.segments > 1) {
                hipLaunchKernelGGL((k_scan_bwd_local<T, WAVES>), grid, block, 0, s, a, d, kq, gout, seg, sums);
                hipLaunchKernelGGL((k_chain<true>), dim3((unsigned)((p.states + 255) / 256)), dim3(256), 0, s, a.A, sums, seg, nullptr, nullptr, d);
            }
            hipLaunchKernelGGL((k_scan_bwd<T, WAVES>), grid, block, 0, s, a, d, kq, ckpt, p.segments > 1 ? seg : nullptr, gout, gv, gdelta, gz,
                               parts, params);
        });
        hipLaunchKernelGGL((k_scan_finish<T>), dim3((unsigned)(row_blocks + param_blocks)), dim3(256), 0, s, parts, params, gq, gk, gA, gD,
                           gdelta_bias, a.lengths, d, p.waves, row_blocks);
    });
    return (int)hipGetLastError();
}

}  // namespace fwp
