// Selective scan: the sum rule with a decay that depends on the token, forward and backward.
//
//   dt = softplus(delta + bias)    W[e][m] = exp(dt[m] A[e][m]) W[e][m] + dt[m] v[m] k[e]    o[m] = sum_e q[e] W[e][m] + D[m] v[m]
//   out = o z sigmoid(z)
// and backwards, with dy = gout z sigmoid(z) and g the gradient of the state after a step:
//   g = dy q + c,  c (of the state before the step) = a g,  a = exp(dt A),  w = a W_before g
//   gq = sum_m dy W    gk = sum_m g dt v    gv = dt sum_e g k + D dy    gdt = v sum_e g k + sum_e A w    gA = sum dt w    gD = sum dy v
//
// A workgroup takes 64 channels of one sequence and head: a lane is a channel, a wave two, four or eight entries of the state (key rows), so that a
// state and its history stay in registers, and a sum over the channels is a sum over the lanes.  Steps go in tiles of 16 (8 for 16 waves) rows: each thread
// loads its rows of v, delta, z once, works out dt and dt v, and puts them into LDS for all waves, as k and q are; the waves' parts of a sum
// over e meet in LDS and the thread that loaded a row finishes it.  The next tile's rows are on their way meanwhile.
//
// Few sequences and channels leave most of the chip idle, so a long sequence is cut into segments that run at the same time:
// a first pass gives each segment's state from zeros and its sum of dt, a small kernel turns these into the state that each segment
// starts from (the decay over a segment is exp(A sum dt), whatever its length), and the second pass is the scan itself.  That doubles the
// exponentials, and instructions are what bounds these kernels, so a call that fills the chip is not cut.
//
// Measured, 32 sequences x 1024 steps of 512 channels, 16 rows, fp32: forward 128 us, adjoint 300-320, its sums 10; their bytes would take 51 and 84 at 5 TB/s.  8 x 2048 steps of
// 2048 channels, bf16: 236-244, 551-568, 17 us.  An entry and step costs 8 vector instructions forward, 24 backward: 5 and 13 are the recurrences (the exponential takes
// the slots of four), a quarter of the rest the sums over the lanes, the other half the softplus, the gate and their slopes.  The vector pipes are at work 56 % of the
// forward and 71 % of the adjoint's time, with two waves a SIMD (the adjoint's LDS leaves no room for more), LDS another 12-13 %.  Without the sums over the lanes the
// adjoint's 603 us of an earlier stage were 543, without softplus and gate 509, with one wave's part instead of eight's 568, without exponentials 583, without k and q from LDS 555.
// Not kept: k and q by scalar loads (297 us forward, 186 from LDS at that stage), tiles of 8 steps with one barrier (149 us against 125) or of 32 (128), one barrier
// and all of a tile's LDS twice (158 against 140 us), steps and values held in registers between the adjoint's two sweeps as k and q are (no change).
//
// One long prompt, 8192 steps of 1024 channels, bf16, 32 segments: 33 + 7 + 47 us.
#include "fwp_elements.hpp"
#include "fwp_wave.hpp"

#include <algorithm>
#include <type_traits>

namespace fwp {
namespace {

constexpr int kRowMirror8 = 0x141;      // lane i of 8 gets lane 7 - i

// Waves of a workgroup and state rows of a wave (S).  Two rows a wave need half the registers of four, so that twice the waves are there to fill one another's
// gaps: 32 x 1024 steps of 512 channels, 16 rows, forward + backward 125 + 344 us against 158 + 526 us with four.  At 32 rows sixteen waves of two
// would not fit the LDS of the adjoint; forward they take 139 us against 151 with 256 workgroups and 275 against 229 with 512.  Fewer than four waves would load a tile's rows too slowly.
// Beyond 32 rows sixteen waves of four go forward, and eight of eight back, since sixteen leave 128 registers to a lane and a tile's history does not fit them
// (32 x 1024 steps of 512 channels, 64 rows: 2441 us, and 913 with eight).
// Sixteen waves of one row forward at 16 rows: 147 us against 127 with 256 workgroups, 256 against 157 with 512 (twice the parts of sum_e q W through LDS).
int rows_of(int E, bool backward) { return E <= 16 ? 2 : E <= 32 || !backward ? 4 : 8; }
int waves_of(int E, bool backward) { return E <= 8 ? 4 : E <= 32 || backward ? 8 : 16; }
// Steps from one saved state to the next, and of the adjoint's tiles, whose states a wave holds in registers
constexpr int tile_of(int rows, int waves) { return rows * waves > 32 ? 8 : 16; }

struct Dims {
    int N, H, L, E, M;
    int blocks_m;       // 64 channels each
    int segments, steps;      // per sequence, and steps of a segment (a multiple of the tile)
    int tiles, padded;  // whole tiles of a sequence, and their steps
};

struct Plan : Dims {
    int waves, rows, tile;
    int64_t heads, states;      // N H; floats of one set of states
    Plan(int N_, int H_, int L_, int E_, int M_, bool backward) {
        N = N_, H = H_, L = L_, E = E_, M = M_;
        rows = rows_of(E, backward), waves = waves_of(E, backward), tile = tile_of(rows, waves);
        blocks_m = (M + 63) / 64;
        tiles = (L + tile - 1) / tile;
        padded = tiles * tile;
        heads = (int64_t)N * H;
        states = heads * E * M;
        // Segments: with w of them the CUs have ceil(blocks w / 256) workgroups each, of 1 / w of the steps, and the pass before adds 0.7 (forward) and
        // 0.2 (backward) of the work.  Workgroups that share a CU fill one another's gaps in the forward pass, where three fit: two take
        // 1.36 times as long as one.  Measured, 256 workgroups cut into 1, 2, 4: 231, 282, 261 us and 587, 718, 718 us; 16 into
        // 8, 16, 32, 64: 186, 116, 84, 85 us forward.  A segment has eight tiles at least, or the two launches more cost what it saves.
        // Workgroups of four waves (up to 8 rows) leave more of a CU idle, forward and backward: two take 1.2 times as long as one, eight 3.5 times, and the pass before 0.4 of the
        // adjoint.  128 workgroups (1024 steps) cut into 1, 2, 4, 8: 118, 103, 68, 55 and 268, 190, 125, 126 us; 256: 124, 127, 103, 96 and 288, 245, 243, 254;
        // 512: 152, 188, 176, 171 and 350, 434, 435, 465.
        const int64_t blocks = heads * blocks_m;
        double best = 0;
        segments = 1, steps = padded;
        for (int w = 1; w <= 64 && (w == 1 || w <= tiles / 8); w++) {
            const double turns = (double)((blocks * w + 255) / 256);
            const double side_by_side = waves == 4 ? (backward ? 0.6 * turns : 0.35 + 0.42 * turns) : backward ? turns : 0.68 * turns;
            const double cost = (turns > 1 ? side_by_side : 1) / w * (w == 1 ? 1 : !backward ? 1.7 : waves == 4 ? 1.4 : 1.2);
            if (w > 1 && cost >= best) continue;
            best = cost;
            const int per = (tiles + w - 1) / w;
            segments = (tiles + per - 1) / per, steps = per * tile;
        }
    }
    int64_t grid() const { return heads * blocks_m * segments; }
    int64_t seg_states() const { return segments > 1 ? states * segments + heads * segments * M : 0; }      // the states and the sums of dt
};

// ------------------------------------------------------------------ what the passes share

struct Place {
    int n, h, m, mb, seg, wave, lane, nh;
    bool live;      // a channel that exists
    __device__ __forceinline__ Place(const Dims &d) {
        unsigned b = blockIdx.x;        // 32-bit divisions: those of 64 bits take a microsecond
        mb = b % d.blocks_m;
        b /= d.blocks_m;
        seg = b % d.segments;
        nh = b / d.segments;
        n = nh / d.H, h = nh % d.H;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
        m = mb * 64 + lane;
        live = m < d.M;
    }
    // state row e of this channel in a [.., E, M] array's block `at`
    __device__ __forceinline__ int64_t state(const Dims &d, int64_t at, int e) const { return (at * d.E + e) * d.M + m; }
};

// A log2(e) of the wave's S rows
template <int S>
__device__ __forceinline__ void load_decays(float (&a)[S], const float *A, const Dims &d, const Place &p) {
#pragma unroll
    for (int s = 0; s < S; s++) {
        const int e = S * p.wave + s;
        a[s] = p.live && e < d.E ? within_range(A[p.state(d, p.h, e)] * kLog2e) : 0.f;
    }
}
template <int S>
__device__ __forceinline__ void load_states(float (&x)[S], const float *from, int64_t at, const Dims &d, const Place &p) {
#pragma unroll
    for (int s = 0; s < S; s++) {
        const int e = S * p.wave + s;
        x[s] = from && p.live && e < d.E ? from[p.state(d, at, e)] : 0.f;
    }
}
template <int S>
__device__ __forceinline__ void store_states(const float (&x)[S], float *to, int64_t at, const Dims &d, const Place &p) {
#pragma unroll
    for (int s = 0; s < S; s++) {
        const int e = S * p.wave + s;
        if (p.live && e < d.E) to[p.state(d, at, e)] = x[s];
    }
}

// The rows of a tile in an [N,H,L,M] view, by the channel of the lane.  Addresses are a 64-bit base, the same for all lanes, that goes from tile to
// tile, and 32-bit offsets in the tile (steps of up to kScanMaxStep elements).  Every lane loads: channels that do not exist read the last one, rows
// behind the sequence its last row, and what they read is not used.  So no load waits behind a branch, and those of the next tile are on
// their way while this one is worked on.
template <typename T>
struct Column {
    char *base;
    unsigned step, col;     // in bytes
    template <typename V>
    __device__ __forceinline__ Column(const V &v, const Place &at, const Dims &d, int t0)
        : base((char *)v.ptr + (at.n * v.sN + at.h * v.sH + t0 * v.sL) * (int64_t)sizeof(T)), step((unsigned)v.sL * sizeof(T)),
          col(min(at.m, d.M - 1) * (unsigned)sizeof(T)) {}
    __device__ __forceinline__ T &operator[](int r) const { return *(T *)(base + (r * step + col)); }
    __device__ __forceinline__ void go(int rows) { base += (int64_t)rows * step; }
    // rows wave, wave + waves, .. as far as the last one that there is
    template <typename U, int ROWS>
    __device__ __forceinline__ void load(U (&to)[ROWS], int most, int wave, int waves) const {
#pragma unroll
        for (int j = 0; j < ROWS; j++) to[j] = (*this)[min(wave + waves * j, most)];
    }
};

// A tile of k and q in LDS, [TILE][WAVES][S of k | S of q], or (PARTS 1) one of them, loaded the same way; zero where there is no
// such entry or step (so that whatever a padded row holds stays out).
template <typename T, int WAVES, int S, int TILE, int PARTS>
struct Keys {
    static constexpr int WIDTH = S * PARTS, ROW = WAVES * WIDTH, EACH = TILE * WIDTH > 64 ? TILE * WIDTH / 64 : 1, APART = 64 / WIDTH;
    const char *p;
    unsigned step;
    int row, at;
    bool in;
    __device__ __forceinline__ Keys(const fwp_rows &k, const fwp_rows &q, const Place &w, const Dims &d, int t0) {
        at = threadIdx.x % ROW, row = threadIdx.x / ROW;
        const int e = at / WIDTH * S + at % S;
        const bool is_k = at % WIDTH < S;
        in = e < d.E;
        const int64_t sL = is_k ? k.sL : q.sL;
        p = (is_k ? (const char *)k.ptr + (w.n * k.sN + w.h * k.sH) * (int64_t)sizeof(T) : (const char *)q.ptr + (w.n * q.sN + w.h * q.sH) * (int64_t)sizeof(T)) +
            (t0 * sL + min(e, d.E - 1)) * (int64_t)sizeof(T);
        step = (unsigned)sL * sizeof(T);
    }
    __device__ __forceinline__ void go(int rows) { p += (int64_t)rows * step; }
    __device__ __forceinline__ void load(T (&to)[EACH], int most) const {
#pragma unroll
        for (int j = 0; j < EACH; j++) to[j] = *(const T *)(p + min(row + APART * j, most) * step);
    }
    __device__ __forceinline__ void put(float (*to)[ROW], const T (&from)[EACH], int steps) const {
#pragma unroll
        for (int j = 0; j < EACH; j++)
            if (row + APART * j < TILE) to[row + APART * j][at] = in && row + APART * j < steps ? (float)from[j] : 0.f;
    }
};

// Where a state has fewer rows than the waves (not FULL), the others hold zeros, whatever values meet their k and q of zero: an infinite value then
// gives infinity, not infinity times zero.  2 us of 47 (30 x 8 heads of 391 steps, 11 x 49); the adjoint, where it would be 12 of 120, goes without: gradients that meet
// an infinity may be NaN.
template <int S, bool FULL>
struct Existing {
    int mask[S];
    __device__ __forceinline__ Existing(const Dims &d, const Place &p) {
#pragma unroll
        for (int s = 0; s < S; s++) mask[s] = __builtin_amdgcn_readfirstlane(S * p.wave + s < d.E ? -1 : 0);
    }
    __device__ __forceinline__ float operator()(float x, int s) const { return FULL ? x : __int_as_float(__float_as_int(x) & mask[s]); }
};

// The parameters of a channel that the threads which load its rows need
struct Channel {
    float D, bias;
    int has_D;
    __device__ __forceinline__ Channel(const fwp_scan_args &a, const Place &p) {
        const int64_t at = (int64_t)p.h * a.M + p.m;
        D = p.live && a.D ? a.D[at] : 0.f;
        bias = p.live && a.delta_bias ? a.delta_bias[at] : 0.f;
        has_D = __builtin_amdgcn_readfirstlane(a.D ? -1 : 0);
    }
    // D x, or 0 for any x without D
    __device__ __forceinline__ float skip(float x) const { return D * __int_as_float(__float_as_int(x) & has_D); }
};

// ------------------------------------------------------------------ forward

// LOCAL: only the state after the segment, from zeros, and the segment's sum of dt; otherwise the scan.  FULL: every row of every wave is one of the state's.
template <typename T, int WAVES, int S, bool LOCAL, bool FULL>
__global__ __launch_bounds__(64 * WAVES) void k_scan_fwd(fwp_scan_args a, Dims d, const float *init, float *W, float *__restrict__ saved,
                                                         float *__restrict__ sums, fwp_out_rows out) {
    constexpr int TILE = 16, ROWS = (TILE + WAVES - 1) / WAVES, KEEP = tile_of(S, WAVES);
    using K = Keys<T, WAVES, S, TILE, LOCAL ? 1 : 2>;
    __shared__ alignas(16) float kq[TILE][K::ROW];
    __shared__ float2 sx[TILE][64];                          // dt, dt v
    __shared__ float sy[LOCAL ? 1 : WAVES][TILE][64];        // the waves' parts of sum_e q W
    const Place p(d);
    const Channel ch(a, p);
    const int len = length_of(a.lengths, p.n, d.L), first = p.seg * d.steps, end = min(first + d.steps, d.L), last = min(end, len);
    const bool gated = !LOCAL && a.z.ptr;
    Column<const T> V(a.v, p, d, first), DT(a.delta, p, d, first), Z(gated ? a.z : a.v, p, d, first);
    Column<T> O(LOCAL ? fwp_out_rows{(void *)a.v.ptr, 0, 0, 0} : out, p, d, first);
    K keys(a.k, a.q, p, d, first);
    const Existing<S, FULL> keep(d, p);
    float decay[S], state[S], sum = 0.f;
    load_decays(decay, a.A, d, p);
    load_states(state, LOCAL ? nullptr : init, (int64_t)p.nh * d.segments + p.seg, d, p);
    T v[ROWS], dt[ROWS], z[ROWS], key[K::EACH];
    // the rows of the tile that the columns are at, which starts at step t0
    const auto fetch = [&](int t0) {
        const int most = min(last - 1 - t0, TILE - 1);
        V.load(v, most, p.wave, WAVES);
        DT.load(dt, most, p.wave, WAVES);
        if (gated) Z.load(z, most, p.wave, WAVES);
        keys.load(key, most);
        V.go(TILE), DT.go(TILE), Z.go(TILE), keys.go(TILE);
    };
    if (first < last) fetch(first);
    for (int t0 = first; t0 < last; t0 += TILE) {
        float dv[ROWS], gate[ROWS];       // D v and the gate of this thread's rows
#pragma unroll
        for (int j = 0; j < ROWS; j++) {
            const int r = p.wave + WAVES * j;
            const bool in = t0 + r < last && p.live;
            float x = (float)dt[j] + ch.bias;
            if (a.softplus) x = softplus(x);
            x = in ? x : 0.f;
            const float vs = in ? (float)v[j] : 0.f;
            dv[j] = ch.skip(vs);
            gate[j] = gated ? silu((float)z[j], sigmoid((float)z[j])) : 1.f;
            if (r < TILE) sx[r][p.lane] = make_float2(x, x * vs);
        }
        keys.put(kq, key, last - t0);
        __syncthreads();
        if (t0 + TILE < last) fetch(t0 + TILE);
#pragma unroll
        for (int r = 0; r < TILE; r++) {
            if constexpr (!LOCAL)
                if (r % KEEP == 0)
                    if (saved && t0 + r < last) store_states(state, saved, (int64_t)p.nh * d.tiles + (t0 + r) / KEEP, d, p);
            const float2 x = sx[r][p.lane];
            const float *const k = kq[r] + K::WIDTH * p.wave, *const q = k + S;
            float y = 0.f;
#pragma unroll
            for (int s = 0; s < S; s++) {
                state[s] = keep(fmaf(__builtin_amdgcn_exp2f(x.x * decay[s]), state[s], x.y * k[s]), s);
                if constexpr (!LOCAL) y = fmaf(q[s], state[s], y);
            }
            if constexpr (LOCAL) sum += x.x;
            else sy[p.wave][r][p.lane] = y;
        }
        __syncthreads();
        if constexpr (!LOCAL) {
#pragma unroll
            for (int j = 0; j < ROWS; j++) {
                const int r = p.wave + WAVES * j, t = t0 + r;
                if (r >= TILE) continue;
                float o = dv[j];
#pragma unroll
                for (int w = 0; w < WAVES; w++) o += sy[w][r][p.lane];
                if (gated) o *= gate[j];
                if (t < end && p.live) O[r] = (T)(t < len ? o : 0.f);
            }
            O.go(TILE);
        }
    }
    if constexpr (LOCAL) {
        store_states(state, W, (int64_t)p.nh * d.segments + p.seg, d, p);
        if (p.wave == 0 && p.live) sums[((int64_t)p.nh * d.segments + p.seg) * d.M + p.m] = sum;
    } else {
        if (W) store_states(state, W, p.nh, d, p);      // one segment: the state that the call keeps
        for (int t = first + (max(last - first, 0) + TILE - 1) / TILE * TILE + p.wave; t < end; t += WAVES)      // tiles behind the sequence
            if (p.live) *(row<T>(out, p.n, p.h, t) + p.m) = (T)0.f;
    }
}

// From each segment's own state (or gradient) to the one it starts from: after a segment x becomes exp(A sum dt) x + own.  The
// exponential is applied as two halves, which reach twice as far before one of them is infinite.  An infinite x stays infinite as step by step,
// also where exp(A sum dt) is zero: unless the steps' decays cannot all be above zero (2^-126 each).
template <bool REVERSE>
__global__ __launch_bounds__(256) void k_chain(const float *__restrict__ A, const float *__restrict__ sums, float *__restrict__ own,
                                               const float *W_in, float *W_out, Dims d) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = (int64_t)d.E * d.M;
    if (i >= (int64_t)d.N * d.H * per) return;
    const int64_t nh = i / per, em = i % per;
    const int m = (int)(em % d.M);
    const float half = within_range(0.5f * kLog2e * A[(nh % d.H) * per + em]);
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
            const float exponent = half * dt[j];
            float e = __builtin_amdgcn_exp2f(exponent);
            if (fabsf(x) == __builtin_inff() && exponent >= -63.f * d.steps) e = fmaxf(e, 1.17549435e-38f);
            x = x == 0.f ? o[j] : fmaf(e, e * x, o[j]);       // nothing grows out of nothing, however large exp(A sum dt)
        }
    }
    if (W_out) W_out[i] = x;
}

// ------------------------------------------------------------------ backward

// The gradient of the state before the segment, from zeros behind it
template <typename T, int WAVES, int S>
__global__ __launch_bounds__(64 * WAVES) void k_scan_bwd_local(fwp_scan_args a, Dims d, fwp_rows gout, float *__restrict__ own,
                                                               float *__restrict__ sums) {
    constexpr int TILE = 16, ROWS = (TILE + WAVES - 1) / WAVES;
    using K = Keys<T, WAVES, S, TILE, 1>;
    __shared__ alignas(16) float sq[TILE][K::ROW];
    __shared__ float2 sx[TILE][64];     // dt, dy
    const Place p(d);
    const Channel ch(a, p);
    const int len = length_of(a.lengths, p.n, d.L), first = p.seg * d.steps, end = min(first + d.steps, d.L), last = min(end, len);
    const int top = first < last ? first + (last - first - 1) / TILE * TILE : first;
    const bool gated = a.z.ptr != nullptr;
    Column<const T> DT(a.delta, p, d, top), GO(gout, p, d, top), Z(gated ? a.z : a.v, p, d, top);
    K keys(a.q, a.q, p, d, top);
    float decay[S], c[S] = {}, sum = 0.f;
    load_decays(decay, a.A, d, p);
    T dt[ROWS], go[ROWS], z[ROWS], key[K::EACH];
    const auto fetch = [&](int t0) {
        const int most = min(last - 1 - t0, TILE - 1);
        DT.load(dt, most, p.wave, WAVES);
        GO.load(go, most, p.wave, WAVES);
        if (gated) Z.load(z, most, p.wave, WAVES);
        keys.load(key, most);
        DT.go(-TILE), GO.go(-TILE), Z.go(-TILE), keys.go(-TILE);
    };
    if (first < last) fetch(top);
    for (int t0 = top; t0 >= first && first < last; t0 -= TILE) {
#pragma unroll
        for (int j = 0; j < ROWS; j++) {
            const int r = p.wave + WAVES * j;
            const bool in = t0 + r < last && p.live;
            float x = (float)dt[j] + ch.bias, dy = (float)go[j];
            if (a.softplus) x = softplus(x);
            if (gated) dy *= silu((float)z[j], sigmoid((float)z[j]));
            if (r < TILE) sx[r][p.lane] = in ? make_float2(x, dy) : make_float2(0.f, 0.f);
        }
        keys.put(sq, key, last - t0);
        __syncthreads();
        if (t0 > first) fetch(t0 - TILE);
#pragma unroll
        for (int r = TILE - 1; r >= 0; r--) {
            const float2 x = sx[r][p.lane];
#pragma unroll
            for (int s = 0; s < S; s++) c[s] = fmaf(x.y, sq[r][S * p.wave + s], c[s]) * __builtin_amdgcn_exp2f(x.x * decay[s]);
            sum += x.x;
        }
        __syncthreads();
    }
    store_states(c, own, (int64_t)p.nh * d.segments + p.seg, d, p);
    if (p.wave == 0 && p.live) sums[((int64_t)p.nh * d.segments + p.seg) * d.M + p.m] = sum;
}

// parts: [blocks_m][heads][padded][WAVES][S of gk | S of gq], the sums over 64 channels
// params: [N segments][H][E + 2][M]: gA, gD, gdelta_bias of one segment
template <typename T, int WAVES, int S>
__global__ __launch_bounds__(64 * WAVES, 2) void k_scan_bwd(fwp_scan_args a, Dims d, const float *__restrict__ saved, const float *__restrict__ init,
                                                         fwp_rows gout, fwp_out_rows gv, fwp_out_rows gdelta, fwp_out_rows gz,
                                                         float *__restrict__ parts, float *__restrict__ params) {
    constexpr int TILE = tile_of(S, WAVES), ROWS = (TILE + WAVES - 1) / WAVES;
    using K = Keys<T, WAVES, S, TILE, 2>;
    __shared__ alignas(16) float kqs[2][TILE][K::ROW];
    __shared__ float2 sxs[2][TILE][64];                  // dt, dt v
    __shared__ float sgs[2][TILE][64];                   // dy
    __shared__ float part[3][WAVES][TILE][64];           // the waves' parts of sum_e g k, sum_e A w (times log2 e), sum_e q W
    const Place p(d);
    const Channel ch(a, p);
    const int len = length_of(a.lengths, p.n, d.L), first = p.seg * d.steps, end = min(first + d.steps, d.L), last = min(end, len);
    const int top = first < last ? first + (last - first - 1) / TILE * TILE : first - TILE;
    const bool gated = a.z.ptr != nullptr;
    Column<T> GV(gv, p, d, top), GD(gdelta, p, d, top), GZ(gated ? gz : gv, p, d, top);
    // whole tiles behind the sequence
    for (int t = top + TILE + p.wave; t < end; t += WAVES)
        if (p.live) {
            Column<T> gv0(gv, p, d, t), gd0(gdelta, p, d, t), gz0(gated ? gz : gv, p, d, t);
            gv0[0] = gd0[0] = (T)0.f;
            if (gated) gz0[0] = (T)0.f;
        }
    Column<const T> V(a.v, p, d, max(top, 0)), DT(a.delta, p, d, max(top, 0)), GO(gout, p, d, max(top, 0)), Z(gated ? a.z : a.v, p, d, max(top, 0));
    K keys(a.k, a.q, p, d, max(top, 0));
    float decay[S], c[S], gA[S] = {}, gD = 0.f, gbias = 0.f;
    load_decays(decay, a.A, d, p);
    load_states(c, init, (int64_t)p.nh * d.segments + p.seg, d, p);
    T v[ROWS], dt[ROWS], go[ROWS], z[ROWS], key[K::EACH];
    float next[S];
    const auto fetch = [&](int t0) {
        const int most = min(last - 1 - t0, TILE - 1);
        V.load(v, most, p.wave, WAVES);
        DT.load(dt, most, p.wave, WAVES);
        GO.load(go, most, p.wave, WAVES);
        if (gated) Z.load(z, most, p.wave, WAVES);
        keys.load(key, most);
        load_states(next, saved, (int64_t)p.nh * d.tiles + t0 / TILE, d, p);
        V.go(-TILE), DT.go(-TILE), GO.go(-TILE), Z.go(-TILE), keys.go(-TILE);
    };
    // What the last lines of a tile need of its rows: v, the slope of dt, gout times the slope of the gate.  Set [0] is the tile's at work, [1] the next one's.
    float vs[2][ROWS], slope_dt[2][ROWS], slope_z[2][ROWS], before0[S];
    const auto stage = [&](int t0, int half) {
#pragma unroll
        for (int j = 0; j < ROWS; j++) {
            const int r = p.wave + WAVES * j;
            const bool in = t0 + r < last && p.live;
            const float pre = (float)dt[j] + ch.bias, g = in ? (float)go[j] : 0.f;
            vs[1][j] = in ? (float)v[j] : 0.f;
            float x = pre, dy = g;
            slope_dt[1][j] = 1.f;
            if (a.softplus) {
                float u;
                x = softplus(pre, u);
                slope_dt[1][j] = softplus_slope(pre, u);
            }
            x = in ? x : 0.f;
            if (gated) {
                const float z_ = in ? (float)z[j] : 0.f, s = sigmoid(z_);
                dy = g * silu(z_, s);
                slope_z[1][j] = g * silu_slope(z_, s);
            }
            if (r < TILE) sxs[half][r][p.lane] = make_float2(x, x * vs[1][j]), sgs[half][r][p.lane] = dy;
        }
        keys.put(kqs[half], key, last - t0);
    };
    const auto turn = [&] {
#pragma unroll
        for (int j = 0; j < ROWS; j++) vs[0][j] = vs[1][j], slope_dt[0][j] = slope_dt[1][j], slope_z[0][j] = slope_z[1][j];
#pragma unroll
        for (int s = 0; s < S; s++) before0[s] = next[s];
    };
    if (first < last) {
        fetch(top);
        stage(top, 0);
    }
    int half = 0;
    for (int t0 = top; t0 >= first; t0 -= TILE, half ^= 1) {
        __syncthreads();        // this tile's rows are in LDS, and nobody reads `part` any more
        const auto sx = sxs[half];
        const auto sg = sgs[half];
        const auto kq = kqs[half];
        turn();
        if (t0 > first) fetch(t0 - TILE);
        constexpr bool AGAIN = S == 8;               // no registers for them: formed again on the way back
        float before[TILE + 1][S], al[AGAIN ? 1 : TILE][S];      // the states before each step, and its decays
        // k and q of the tile for the way back as well, where the registers are there for it (two rows a wave: 551 us against 568, 8 x 2048 steps of 2048
        // channels; four rows spill 115 registers)
        constexpr bool HELD = S == 2;
        float kq_held[HELD ? TILE : 1][2 * S];
#pragma unroll
        for (int s = 0; s < S; s++) before[0][s] = before0[s];
#pragma unroll
        for (int r = 0; r < TILE; r++) {
            const float2 x = sx[r][p.lane];
            if constexpr (HELD)
#pragma unroll
                for (int i = 0; i < 2 * S; i++) kq_held[r][i] = kq[r][K::WIDTH * p.wave + i];
            const float *const k = HELD ? kq_held[HELD ? r : 0] : kq[r] + K::WIDTH * p.wave, *const q = k + S;
            float y = 0.f;
#pragma unroll
            for (int s = 0; s < S; s++) {
                const float e = __builtin_amdgcn_exp2f(x.x * decay[s]);
                if constexpr (!AGAIN) al[r][s] = e;
                before[r + 1][s] = fmaf(e, before[r][s], x.y * k[s]);
                y = fmaf(q[s], before[r + 1][s], y);
            }
            part[2][p.wave][r][p.lane] = y;
        }
        float tile_gA[S] = {};      // a tile's share first: the sum over a sequence then has a sixteenth of the terms
        // One step back; what is summed over the channels comes out in `sums`: gk of the wave's rows, then gq
        constexpr int SUMS = 2 * S;
        const auto back = [&](int r, float (&sums)[SUMS]) {
            const float2 x = sx[r][p.lane];
            const float dy = sg[r][p.lane], *const k = HELD ? kq_held[HELD ? r : 0] : kq[r] + K::WIDTH * p.wave, *const q = k + S;
            float read = 0.f, slope = 0.f;
#pragma unroll
            for (int s = 0; s < S; s++) {
                const float g = fmaf(dy, q[s], c[s]);
                sums[s] = g * x.y;
                sums[S + s] = dy * before[r + 1][s];
                read = fmaf(g, k[s], read);
                c[s] = g * (AGAIN ? __builtin_amdgcn_exp2f(x.x * decay[s]) : al[AGAIN ? 0 : r][s]);
                const float w = c[s] * before[r][s];
                slope = fmaf(w, decay[s], slope);
                tile_gA[s] = fmaf(w, x.x, tile_gA[s]);
            }
            part[0][p.wave][r][p.lane] = read;
            part[1][p.wave][r][p.lane] = slope;
        };
        // The sums over the lanes, halving what a lane holds as it goes, over 64 / SUMS steps (4, 8 or 16): lane l then has the sum
        // number l % SUMS of the step whose bits 0, 1 (2, and 3) are l's bits 5, 4 (3, and 2).
        const bool b3 = p.lane & 8, b2 = p.lane & 4, b1 = p.lane & 2, b0 = p.lane & 1;
        float *const to = parts + (((int64_t)p.mb * d.N * d.H + p.nh) * d.padded + t0) * WAVES * SUMS +
                          ((p.lane >> 5 & 1) + 2 * (p.lane >> 4 & 1) + (S <= 4 ? 4 * (p.lane >> 3 & 1) : 0) + (S == 2 ? 8 * (p.lane >> 2 & 1) : 0)) * WAVES * SUMS +
                          p.wave * SUMS + p.lane % SUMS;
        const auto four_back = [&](int r0, float (&x)[SUMS]) {
            float two[2][SUMS];
#pragma unroll
            for (int q1 = 1; q1 >= 0; q1--) {
                float odd[SUMS], even[SUMS];
                back(r0 + 2 * q1 + 1, odd);
                back(r0 + 2 * q1, even);
#pragma unroll
                for (int i = 0; i < SUMS; i++) {
                    swap32(even[i], odd[i]);
                    two[q1][i] = even[i] + odd[i];
                }
            }
#pragma unroll
            for (int i = 0; i < SUMS; i++) {
                swap16(two[0][i], two[1][i]);
                x[i] = pinned(two[0][i] + two[1][i]);
            }
        };
        const auto eight_back = [&](int r0, float (&x)[SUMS]) {
            float eight[2][SUMS];
            four_back(r0 + 4, eight[1]);
            four_back(r0, eight[0]);
#pragma unroll
            for (int i = 0; i < SUMS; i++) x[i] = pinned((b3 ? eight[1][i] : eight[0][i]) + dpp<kRowRor8>(b3 ? eight[0][i] : eight[1][i]));
        };
        const auto four_lanes = [&](float (&x)[4]) {
#pragma unroll
            for (int i = 0; i < 2; i++) x[i] = pinned((b1 ? x[i + 2] : x[i]) + dpp<kQuadXor2>(b1 ? x[i] : x[i + 2]));
            return pinned((b0 ? x[1] : x[0]) + dpp<kQuadXor1>(b0 ? x[0] : x[1]));
        };
        if constexpr (S == 8) {
#pragma unroll
            for (int r0 = TILE - 4; r0 >= 0; r0 -= 4) {
                float x[SUMS], y[8], u[4];
                four_back(r0, x);
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] = pinned((b3 ? x[i + 8] : x[i]) + dpp<kRowRor8>(b3 ? x[i] : x[i + 8]));
#pragma unroll
                for (int i = 0; i < 4; i++) u[i] = pinned((b2 ? y[i + 4] : y[i]) + dpp<kRowMirror8>(b2 ? y[i] : y[i + 4]));
                to[r0 * WAVES * SUMS] = four_lanes(u);
            }
        } else if constexpr (S == 4) {
#pragma unroll
            for (int r0 = TILE - 8; r0 >= 0; r0 -= 8) {
                float x[8], y[4];
                eight_back(r0, x);
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] = pinned((b2 ? x[i + 4] : x[i]) + dpp<kRowMirror8>(b2 ? x[i] : x[i + 4]));
                to[r0 * WAVES * SUMS] = four_lanes(y);
            }
        } else {
            float hi[4], lo[4], y[4];
            eight_back(8, hi);
            eight_back(0, lo);
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = pinned((b2 ? hi[i] : lo[i]) + dpp<kRowMirror8>(b2 ? lo[i] : hi[i]));
            *to = four_lanes(y);
        }
#pragma unroll
        for (int s = 0; s < S; s++) gA[s] += tile_gA[s];
        if (t0 > first) stage(t0 - TILE, half ^ 1);
        __syncthreads();
        float tile_gD = 0.f, tile_gbias = 0.f;
#pragma unroll
        for (int j = 0; j < ROWS; j++) {
            const int r = p.wave + WAVES * j, t = t0 + r;
            if (r >= TILE) continue;
            float read = 0.f, slope = 0.f, o = ch.D * vs[0][j];
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                read += part[0][w][r][p.lane];
                slope += part[1][w][r][p.lane];
                o += part[2][w][r][p.lane];
            }
            const float x = sx[r][p.lane].x, dy = sg[r][p.lane];
            float gdt = fmaf(vs[0][j], read, kLn2 * slope) * slope_dt[0][j];
            const bool in = t < len;
            gdt = in ? gdt : 0.f;
            if (t < end && p.live) {
                GV[r] = (T)(in ? fmaf(x, read, ch.D * dy) : 0.f);
                GD[r] = (T)gdt;
                if (gated) GZ[r] = (T)(in ? slope_z[0][j] * o : 0.f);
            }
            if (in) tile_gD = fmaf(dy, vs[0][j], tile_gD), tile_gbias += gdt;
        }
        GV.go(-TILE), GD.go(-TILE), GZ.go(-TILE);
        gD += tile_gD, gbias += tile_gbias;
    }
    __syncthreads();
    float *const to = params + ((int64_t)(p.n * d.segments + p.seg) * d.H + p.h) * (d.E + 2) * d.M + p.m;
#pragma unroll
    for (int s = 0; s < S; s++)
        if (p.live && S * p.wave + s < d.E) to[(int64_t)(S * p.wave + s) * d.M] = gA[s];
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
                                                     int S, unsigned param_blocks) {
    if (blockIdx.x >= param_blocks) {       // the parameters' first: they take longer
        const unsigned width = waves * 2 * S, heads = (unsigned)d.N * d.H, i = (blockIdx.x - param_blocks) * 256 + threadIdx.x;      // a launch's threads fit 32 bits
        const unsigned row_of = i / width, j = i % width, nh = row_of / d.L, t = row_of % d.L;
        const int e = (int)(j / (2 * S) * S + j % S);
        if (nh >= heads || e >= d.E) return;
        const int n = (int)(nh / d.H), h = (int)(nh % d.H);
        float x = 0.f;
        if ((int)t < length_of(lengths, n, d.L)) {
            const float *from = parts + ((int64_t)nh * d.padded + t) * width + j;
            const int64_t step = (int64_t)heads * d.padded * width;
#pragma unroll 8
            for (int mb = 0; mb < d.blocks_m; mb++) x += from[mb * step];
        }
        store(row<T>(j % (2 * S) < S ? gk : gq, n, h, t) + e, x);
        return;
    }
    // 64 columns and four slices of the sequences and segments to a workgroup
    __shared__ float sh[4][64];
    const int64_t per = (int64_t)d.H * (d.E + 2) * d.M, i = (int64_t)blockIdx.x * 64 + threadIdx.x % 64;
    const int slice = threadIdx.x / 64, terms = d.N * d.segments;
    float x = 0.f;
    if (i < per)
#pragma unroll 8
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

template <int V>
struct alignas(4 * V) Floats {
    float x[V];
};

// Four waves share the state rows of 64 V channels, V neighbours to a lane.  Bound by the state's bytes: 256 sequences x 2048 channels x 16 rows, read and
// written, in 17.3 us with V = 4 and 20.8 with V = 1 (14.3 at 5 TB/s); 131072 channels in all 7.3 and 7.5, 16384 4.8 and 3.1 us.
template <typename T, int V>
__global__ __launch_bounds__(256) void k_scan_step(fwp_scan_args a, float *__restrict__ W, fwp_out_rows out) {
    __shared__ Floats<V> sy[4][64];
    const unsigned blocks_m = (a.M + 64 * V - 1) / (64 * V);
    const int nh = blockIdx.x / blocks_m, n = nh / a.H, h = nh % a.H, lane = threadIdx.x % 64,
              m = ((int)(blockIdx.x % blocks_m) * 64 + lane) * V, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const bool live = m < a.M;      // V divides M
    if (length_of(a.lengths, n, 1) == 0) {      // the whole workgroup
        if (wave == 0 && live)
#pragma unroll
            for (int i = 0; i < V; i++) store(row<T>(out, n, h, 0) + m + i, 0.f);
        return;
    }
    const int64_t at = (int64_t)h * a.M + min(m, a.M - V), rows = (int64_t)a.M;
    Floats<V> y = {};
    float v[V], dt[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int c = min(m, a.M - V) + i;
        v[i] = load(row<T>(a.v, n, h, 0) + c);
        dt[i] = load(row<T>(a.delta, n, h, 0) + c) + (a.delta_bias ? a.delta_bias[at + i] : 0.f);
        if (a.softplus) dt[i] = softplus(dt[i]);
    }
    const T *const q = row<T>(a.q, n, h, 0), *const k = row<T>(a.k, n, h, 0);
    const float *const A = a.A + (int64_t)h * a.E * a.M + min(m, a.M - V);
    float *const w = W ? W + (int64_t)nh * a.E * a.M + min(m, a.M - V) : nullptr;
    // four rows' loads at once; rows that do not exist read the last one
    for (int e0 = wave; e0 < a.E; e0 += 16) {
        Floats<V> al[4], st[4] = {};
        float ks[4], qs[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int e = min(e0 + 4 * j, a.E - 1);
            al[j] = *reinterpret_cast<const Floats<V> *>(A + e * rows);
            if (w) st[j] = *reinterpret_cast<const Floats<V> *>(w + e * rows);
            ks[j] = load(k + e), qs[j] = load(q + e);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int e = e0 + 4 * j;
            if (e >= a.E) continue;
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float x = dt[i] * v[i] * ks[j];
                st[j].x[i] = w ? fmaf(exp_of(dt[i] * within_range(al[j].x[i])), st[j].x[i], x) : x;
                y.x[i] = fmaf(qs[j], st[j].x[i], y.x[i]);
            }
            if (w && live) *reinterpret_cast<Floats<V> *>(w + e * rows) = st[j];
        }
    }
    sy[wave][lane] = y;
    __syncthreads();
    if (wave || !live) return;
#pragma unroll
    for (int i = 0; i < V; i++) {
        float o = (sy[0][lane].x[i] + sy[1][lane].x[i]) + (sy[2][lane].x[i] + sy[3][lane].x[i]) + (a.D ? a.D[at + i] * v[i] : 0.f);
        if (a.z.ptr) {
            const float z = load(row<T>(a.z, n, h, 0) + m + i);
            o *= silu(z, sigmoid(z));
        }
        store(row<T>(out, n, h, 0) + m + i, o);
    }
}

// ------------------------------------------------------------------ launches

// f(WAVES, S)
template <bool BACKWARD, typename F>
void by_waves(const Plan &p, F f) {
    using std::integral_constant;
    if (p.waves == 4) f(integral_constant<int, 4>(), integral_constant<int, 2>());
    else if (p.E > 32) f(integral_constant<int, BACKWARD ? 8 : 16>(), integral_constant<int, BACKWARD ? 8 : 4>());
    else if (p.rows == 2) f(integral_constant<int, 8>(), integral_constant<int, 2>());
    else f(integral_constant<int, 8>(), integral_constant<int, 4>());
}

}  // namespace

int64_t scan_saved_floats(int N, int H, int L, int E, int M) {
    const Plan p(N, H, L, E, M, false);
    return p.states * p.tiles;
}

int64_t scan_workspace(int N, int H, int L, int E, int M, bool backward) {
    const Plan p(N, H, L, E, M, backward);
    if (!backward) return p.seg_states();
    return p.blocks_m * p.heads * p.padded * p.waves * 2 * p.rows + (int64_t)N * p.segments * H * (E + 2) * M + p.seg_states();
}

int scan_fwd(const fwp_scan_args &a, float *W, fwp_out_rows out, float *saved, float *workspace, hipStream_t s) {
    if (a.L == 1 && !saved) {
        const bool four = a.M % 4 == 0 && a.M >= 256 && reinterpret_cast<uintptr_t>(W) % 16 == 0 && reinterpret_cast<uintptr_t>(a.A) % 16 == 0 &&
                          (int64_t)a.N * a.H * a.M >= 1 << 18;
        const int across = four ? 256 : 64;
        const int64_t grid = (int64_t)a.N * a.H * ((a.M + across - 1) / across);
        if (!fits_launch(grid, 256)) return FWP_E_SHAPE;
        by_type(a.type, [&](auto t) {
            using T = decltype(t);
            if (four) hipLaunchKernelGGL((k_scan_step<T, 4>), dim3((unsigned)grid), dim3(256), 0, s, a, W, out);
            else hipLaunchKernelGGL((k_scan_step<T, 1>), dim3((unsigned)grid), dim3(256), 0, s, a, W, out);
        });
        return (int)hipGetLastError();
    }
    const Plan p(a.N, a.H, a.L, a.E, a.M, false);
    if (!fits_launch(p.grid(), 64 * p.waves) || (p.segments > 1 && !fits_launch((p.states + 255) / 256, 256))) return FWP_E_SHAPE;
    if (p.segments > 1 && !workspace) return FWP_E_NULL;
    float *const seg = workspace, *const sums = seg + p.states * p.segments;
    const Dims d = p;
    by_type(a.type, [&](auto t) {
        using T = decltype(t);
        by_waves<false>(p, [&](auto w, auto r) {
            constexpr int WAVES = decltype(w)::value, S = decltype(r)::value;
            const dim3 grid((unsigned)p.grid()), block(64 * WAVES);
            if (p.segments > 1) {
                hipLaunchKernelGGL((k_scan_fwd<T, WAVES, S, true, true>), grid, block, 0, s, a, d, nullptr, seg, nullptr, sums, out);
                hipLaunchKernelGGL((k_chain<false>), dim3((unsigned)((p.states + 255) / 256)), dim3(256), 0, s, a.A, sums, seg, W, W, d);
            }
            const auto scan = [&](auto full) {
                hipLaunchKernelGGL((k_scan_fwd<T, WAVES, S, false, decltype(full)::value>), grid, block, 0, s, a, d, p.segments > 1 ? seg : W,
                                   p.segments > 1 ? nullptr : W, saved, nullptr, out);
            };
            if (p.E == WAVES * S) scan(std::true_type());
            else scan(std::false_type());
        });
    });
    return (int)hipGetLastError();
}

int scan_bwd(const fwp_scan_args &a, const float *saved, fwp_rows gout, fwp_out_rows gq, fwp_out_rows gk, fwp_out_rows gv,
             fwp_out_rows gdelta, fwp_out_rows gz, float *gA, float *gD, float *gdelta_bias, float *workspace, hipStream_t s) {
    const Plan p(a.N, a.H, a.L, a.E, a.M, true);
    const int64_t row_blocks = (p.heads * a.L * p.waves * 2 * p.rows + 255) / 256,
                  param_blocks = ((int64_t)a.H * (a.E + 2) * a.M + 63) / 64;
    if (!fits_launch(p.grid(), 64 * p.waves) || !fits_launch(row_blocks + param_blocks, 256) ||
        (p.segments > 1 && !fits_launch((p.states + 255) / 256, 256)))
        return FWP_E_SHAPE;
    float *const parts = workspace, *const params = parts + p.blocks_m * p.heads * p.padded * p.waves * 2 * p.rows,
                *const seg = params + (int64_t)a.N * p.segments * a.H * (a.E + 2) * a.M, *const sums = seg + p.states * p.segments;
    const Dims d = p;
    by_type(a.type, [&](auto t) {
        using T = decltype(t);
        by_waves<true>(p, [&](auto w, auto r) {
            constexpr int WAVES = decltype(w)::value, S = decltype(r)::value;
            const dim3 grid((unsigned)p.grid()), block(64 * WAVES);
            if (p.segments > 1) {
                hipLaunchKernelGGL((k_scan_bwd_local<T, WAVES, S>), grid, block, 0, s, a, d, gout, seg, sums);
                hipLaunchKernelGGL((k_chain<true>), dim3((unsigned)((p.states + 255) / 256)), dim3(256), 0, s, a.A, sums, seg, nullptr, nullptr, d);
            }
            hipLaunchKernelGGL((k_scan_bwd<T, WAVES, S>), grid, block, 0, s, a, d, saved, p.segments > 1 ? seg : nullptr, gout, gv, gdelta, gz, parts,
                               params);
        });
        hipLaunchKernelGGL((k_scan_finish<T>), dim3((unsigned)(row_blocks + param_blocks)), dim3(256), 0, s, parts, params, gq, gk, gA, gD,
                           gdelta_bias, a.lengths, d, p.waves, p.rows, (unsigned)param_blocks);
    });
    return (int)hipGetLastError();
}

}  // namespace fwp
