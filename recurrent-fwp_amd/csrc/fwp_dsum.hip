// The decayed sum rule: how a call is cut into workgroups, what joins its parts, and single steps.
#include <algorithm>
#include <type_traits>

#include "fwp_dsum.hpp"

namespace fwp {
namespace {

// What the segments leave, joined in order: every segment's first state from the one before it.  Slot s of `ends` holds what segment s - 1 leaves when it
// starts from zero, and then the state that segment s starts from; BACKWARD: of segment s + 1, from the last to the first.  A lane has one number of the state, and
// the slots of WAVES * K segments are loaded at once: the time is that of the loads' round trips (8 heads of 64 x 64, 86 segments: 6.3 us; one wave with 16 loads ahead 8.2).  Each of the WAVES waves folds the K slots that are its own from
// zero, takes what the waves before it have come to, and folds again from there.
constexpr int kJoinWaves = 8;
template <bool BACKWARD, int K>
__global__ __launch_bounds__(64 * kJoinWaves) void k_dsum_join(float *ends, const float *factors, const float *from, int E, int M, int Ep, int Mp, int segments) {
    constexpr int WAVES = kJoinWaves;
    __shared__ float left[WAVES][64], through[WAVES];
    const int cells = Ep * Mp, blocks = cells / 64, lane = threadIdx.x % 64, wave = threadIdx.x / 64, cell = blockIdx.x % blocks * 64 + lane;      // at least 32 x 32
    const int64_t head = blockIdx.x / blocks;
    float *at = ends + head * segments * cells + cell;
    const float *f = factors + head * segments;
    const auto slot_of = [&](int s) { return BACKWARD ? segments - 1 - s : s; };
    float cur = 0.f;
    if (!BACKWARD && from) {
        const int e = cell / Mp, m = cell % Mp;
        if (e < E && m < M) cur = from[(head * E + e) * M + m];
    }
    if (wave == 0) at[(int64_t)slot_of(0) * cells] = cur;
    for (int s0 = 1; s0 < segments; s0 += WAVES * K) {
        const int mine = s0 + wave * K;
        float x[K], y[K];
#pragma unroll
        for (int i = 0; i < K; i++) {
            const int slot = slot_of(min(mine + i, segments - 1));
            x[i] = at[(int64_t)slot * cells];
            y[i] = f[BACKWARD ? slot + 1 : slot - 1];
        }
        float start = cur, z = 0.f, by = 1.f;
#pragma unroll
        for (int i = 0; i < K; i++) z = fmaf(y[i], z, x[i]), by *= y[i];
        left[wave][lane] = z;
        if (lane == 0) through[wave] = by;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            cur = fmaf(through[w], cur, left[w][lane]);
            if (w + 1 == wave) start = cur;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < K; i++) {
            start = fmaf(y[i], start, x[i]);
            if (mine + i < segments) at[(int64_t)slot_of(mine + i) * cells] = start;
        }
    }
}

// rows [N,G,L,D] of type T as the sum of `parts` fp32 tensors of that shape, in their order; K elements a thread, of one row, and the loads of eight parts at once.  Bound by memory:
// 32 parts of 4 x 4096 x 128 in 63 us, 4.2 TB/s (one element a thread: 127).
template <typename T, int K>
__global__ __launch_bounds__(256) void k_sum_parts(const float *x, fwp_out_rows out, int parts, int64_t total, int G, int L, int D) {
    struct __attribute__((aligned(4 * K))) Run { float x[K]; };
    struct __attribute__((packed, aligned(sizeof(T)))) Anywhere { T x[K]; };
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * K; i < total; i += (int64_t)gridDim.x * 256 * K) {
        float s[K] = {};
#pragma unroll 8
        for (int p = 0; p < parts; p++) {
            const Run r = *reinterpret_cast<const Run *>(x + p * total + i);
#pragma unroll
            for (int k = 0; k < K; k++) s[k] += r.x[k];
        }
        const int d = i % D;
        int64_t r = i / D;
        const int64_t t = r % L;
        r /= L;
        Anywhere a;
#pragma unroll
        for (int k = 0; k < K; k++) a.x[k] = (T)s[k];
        *reinterpret_cast<Anywhere *>(row<T>(out, r / G, r % G, t) + d) = a;
    }
}
template <typename T>
void sum_parts(const float *x, fwp_out_rows out, int parts, int N, int G, int L, int D, hipStream_t s) {
    const int64_t total = (int64_t)N * G * L * D;
    const auto blocks = [](int64_t n) { return (unsigned)std::min<int64_t>((n + 255) / 256, 8192); };
    if (D % 4 == 0) k_sum_parts<T, 4><<<blocks(total / 4), 256, 0, s>>>(x, out, parts, total, G, L, D);
    else k_sum_parts<T, 1><<<blocks(total), 256, 0, s>>>(x, out, parts, total, G, L, D);
}

// [H] = sums over n and the parts of each head of x [N,H,parts], one workgroup a head: a launch, 4.3 us
__global__ __launch_bounds__(256) void k_sum_heads(const float *x, float *out, int N, int H, int parts) {
    __shared__ float part[4];
    const int h = blockIdx.x;
    float s = 0.f;
    for (int64_t i = threadIdx.x; i < (int64_t)N * parts; i += 256) s += x[(i / parts * H + h) * parts + i % parts];
#pragma unroll
    for (int off = 1; off < 64; off *= 2) s += __shfl_xor(s, off);
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = s;
    __syncthreads();
    if (threadIdx.x == 0) out[h] = (part[0] + part[1]) + (part[2] + part[3]);
}

// One step: S = exp(g) S + k (x) v, o = scale S^T q.  Bound by the state, which is read and written once: a lane holds four columns of R rows, all loaded before
// any is used; X lanes lie side by side on a row.  No cache line of it is used again within a step: 256 x 16 states of 128 x 128 (0.54 GB) 127 us at 4.2 TB/s, 138 without saying so.
// 32 x 8 states of 32 x 32: 4.4 us, a launch and two round trips.
template <typename T, int R>
__global__ __launch_bounds__(256) void k_dsum_step(const DsumWalk a, int X, int blocks) {
    __shared__ float part[4][128 + 4];
    const int tid = threadIdx.x, x = tid % X, y = tid / X, Y = 256 / X;
    const int head = blockIdx.x / blocks, block = blockIdx.x % blocks, h = head % a.H, n = head / a.H, m = (block * X + x) * 4;
    const T *q = row<T>(a.q, n, h / (a.H / a.HQ), 0), *k = row<T>(a.k, n, h / (a.H / a.HK), 0), *v = row<T>(a.v, n, h / (a.H / a.HV), 0);
    T *out = row<T>(a.out, n, h, 0);
    const bool counts = length_of(a.lengths, n, 1) > 0;
    if (!counts) {
        if (y == 0)
            for (int i = 0; i < 4; i++)
                if (m + i < a.M) out[m + i] = (T)0.f;
        return;
    }
    typedef float Quad __attribute__((ext_vector_type(4), aligned(4)));
    const float *from = a.from ? a.from + ((int64_t)n * a.H + h) * a.E * a.M : nullptr;
    const bool whole = m + 4 <= a.M;
    float S[R][4], kv[R], qv[R], vv[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int e = y + r * Y;
        kv[r] = e < a.E ? (float)k[e] : 0.f, qv[r] = e < a.E ? (float)q[e] : 0.f;
        if (from && e < a.E && whole) {
            const Quad s = __builtin_nontemporal_load(reinterpret_cast<const Quad *>(from + (int64_t)e * a.M + m));
#pragma unroll
            for (int i = 0; i < 4; i++) S[r][i] = s[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) S[r][i] = from && e < a.E && m + i < a.M ? from[(int64_t)e * a.M + m + i] : 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) vv[i] = m + i < a.M ? (float)v[m + i] : 0.f;
    const float decay = exp_of(a.decay[n * a.dN + h * a.dH]);
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int e = y + r * Y;
        Quad s;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            s[i] = fmaf(kv[r], vv[i], decay * S[r][i]);
            if (e < a.E) o[i] = fmaf(qv[r], s[i], o[i]);
        }
        if (!a.to || e >= a.E) continue;
        float *to = a.to + (((int64_t)n * a.H + h) * a.E + e) * a.M + m;
        if (whole) __builtin_nontemporal_store(s, reinterpret_cast<Quad *>(to));
        else
            for (int i = 0; i < 4; i++)
                if (m + i < a.M) to[i] = s[i];
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        for (int off = X; off < 64; off *= 2) o[i] += __shfl_xor(o[i], off);
    const int wave = tid / 64, lane = tid % 64;
    if (lane < X) {
#pragma unroll
        for (int i = 0; i < 4; i++) part[wave][4 * lane + i] = o[i];
    }
    __syncthreads();
    if (tid < 4 * X && block * X * 4 + tid < a.M)
        store(out + block * X * 4 + tid, a.scale * ((part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid])));
}

// Up to so many segments, every workgroup of the walk joins what it starts from itself: 8 x 16 sequences of 4096 steps, 64 x 64 bf16, six segments forward and four back, 357 us for both with
// their walks, 370 with a kernel of its own for each; eight segments of 32 x 8 x 1024, 32 x 32 fp32, 170 and 174.  Many segments would read most of `ends` again and again.
constexpr int kFewSegments = 9;

// A plan has more than kFewSegments segments only where heads times slices are fewer than half of what the GPU holds: its workgroups always fit a launch.
template <bool BACKWARD>
void join(const DsumWalk &w, const float *from, int64_t heads, int Ep, hipStream_t s) {
    const unsigned blocks = (unsigned)(heads * (Ep * w.Mp / 64));
    const auto launch = [&](auto slots) { k_dsum_join<BACKWARD, slots><<<blocks, 64 * kJoinWaves, 0, s>>>(w.ends, w.factors, from, w.E, w.M, Ep, w.Mp, w.segments); };
    if (w.segments <= 33) launch(std::integral_constant<int, 4>{});
    else launch(std::integral_constant<int, 16>{});
}

struct Plan {
    int Ep, MS, Mp, slices, chunk, chunks, segments, per;
    int64_t heads, cells, ends;      // ends: floats of the segments' states and factors
};

int resident_of(int type, int which, int Ep, int MS) {
    int n = 1;
    by_type(type, [&](auto t) { n = dsum_launch<decltype(t)>(which, nullptr, Ep, MS, 0, nullptr); });
    return std::max(n, 1);
}

// How a pass is cut.  Segments by a model of its time in chunks of the walk: workgroups go in rounds of as many as the GPU holds, each as long as its chunks and 2.5 for the way into them and out; a
// last round of fewer to a CU is shorter, but not below half.  Cutting sequences adds the walk that finds the segments' states (a chunk of it is 0.45 of a chunk forward and 0.3 backward where it fills the
// GPU, and half of that at least) and joining them.  Measured at 1 to 640 heads of 1024 to 16384 steps in up to 256 segments: the choice is within 7 % of the best one there is.  64 x 64 bf16: 8 x 16 sequences
// of 64 chunks forward 203 us in one piece, 138, 99, 96 and 113 in 2, 4, 6 and 8 segments, backward 410, 264, 217, 254 and 265; 32 x 16 of 32 chunks forward 146 in one, 182 in two, 193 in four.
Plan plan_of(int type, int N, int H, int L, int E, int M, bool backward) {
    Plan p{};
    p.Ep = E <= 32 ? 32 : E <= 64 ? 64 : 128;
    // Slices of 128 columns make P once for twice as many (32 x 16 sequences of 1024 steps, 64 keys, 128 columns, fp16: 591 us for training, 869 in two of 64; 128 keys 1404 and 1430), but three of 64
    // beat two of 128 (150 columns, training: 64 keys fp16 1274 for 1357, bf16 1137 for 1055, fp32 1552 for 1645; 128 keys 2255 for 3257, 2188 for 2882, 2740 for 4324).
    p.MS = M <= 32 ? 32 : M <= 64 || (M > 128 && M <= 192) ? 64 : 128;
    p.slices = (M + p.MS - 1) / p.MS;
    p.Mp = p.slices * p.MS;
    by_type(type, [&](auto t) { p.chunk = kChunkOf<decltype(t)>; });
    p.chunks = (L + p.chunk - 1) / p.chunk;
    p.heads = (int64_t)N * H;
    p.cells = (int64_t)p.Ep * p.Mp;
    const int64_t units = p.heads * p.slices, walks = 256 * resident_of(type, backward ? kDsumBackward : kDsumForward, p.Ep, p.MS),
                  ends = 256 * resident_of(type, backward ? kDsumBackwardEnds : kDsumForwardEnds, p.Ep, p.MS);
    const auto rounds = [](int64_t blocks, int64_t held) { return (double)((blocks + held - 1) / held); };
    // rounds of workgroups of which a CU holds `held / 256`
    const auto share = [](int64_t blocks, int64_t held) {
        const int64_t rest = blocks % held;
        return (double)(blocks / held) + (rest ? std::max(0.5, 0.2 + 0.8 * (double)((rest + 255) / 256 * 256) / held) : 0.0);
    };
    double best = 0;
    // every length of a segment once, and the fewest segments that have it
    for (int64_t s = 1, per; s <= std::max(1, p.chunks / 2) && (s == 1 || units * (s - 1) < 4 * walks); s = (p.chunks + per - 2) / (per - 1)) {
        per = (p.chunks + s - 1) / s;
        const int64_t segments = (p.chunks + per - 1) / per;
        double time = share(units * segments, walks) * (per + 2.5);
        if (segments > 1) {
            const double blocks = (double)units * (segments - 1);
            time += (per + 1) * (backward ? 0.3 : 0.45) * std::max(0.5 * rounds(units * (segments - 1), ends), blocks / ends);
            time += segments > kFewSegments ? 0.6 + 0.004 * segments : 0.3;
        }
        if (s == 1 || time < best) best = time, p.per = (int)per, p.segments = (int)segments;
        if (per == 1) break;
    }
    p.ends = p.segments > 1 ? p.heads * p.segments * (p.cells + 1) : 0;
    return p;
}

int64_t padded(int64_t n) { return (n + 3) & ~int64_t(3); }

struct BackwardRoom {
    int64_t q, k, v, decay, total;
};
BackwardRoom backward_room(const fwp_dsum_args &a, const Plan &p) {
    BackwardRoom r{};
    const int64_t rows = p.heads * a.L;
    r.q = a.HQ < a.H || p.slices > 1 ? rows * p.slices * a.E : 0;
    r.k = a.HK < a.H || p.slices > 1 ? rows * p.slices * a.E : 0;
    r.v = a.HV < a.H ? rows * a.M : 0;
    r.decay = a.per_head ? p.heads * p.slices * p.segments : p.slices > 1 ? rows * p.slices : 0;
    r.total = padded(p.ends) + padded(r.q) + padded(r.k) + padded(r.v) + padded(r.decay);
    return r;
}

DsumWalk walk_of(const fwp_dsum_args &a, const Plan &p) {
    DsumWalk w{};
    w.q = a.q, w.k = a.k, w.v = a.v;
    w.decay = a.decay, w.dN = a.dN, w.dH = a.dH, w.dL = a.dL;
    w.lengths = a.lengths;
    w.scale = a.scale;
    w.N = a.N, w.H = a.H, w.L = a.L, w.E = a.E, w.M = a.M, w.HQ = a.HQ, w.HK = a.HK, w.HV = a.HV;
    w.Mp = p.Mp, w.slices = p.slices, w.segments = p.segments, w.per = p.per;
    w.sum_decay = a.per_head;
    return w;
}

int launch(int which, const fwp_dsum_args &a, const Plan &p, const DsumWalk &w, int segments, hipStream_t s) {
    const int64_t blocks = p.heads * p.slices * segments;
    if (!fits_launch(blocks, 512)) return FWP_E_SHAPE;
    bool done = false;
    by_type(a.type, [&](auto t) { done = dsum_launch<decltype(t)>(which, &w, p.Ep, p.MS, (unsigned)blocks, s) > 0; });
    return done ? 0 : FWP_E_SHAPE;
}

template <typename T>
int launch_step(const DsumWalk &w, hipStream_t s) {
    const int columns = (w.M + 3) / 4;
    int X = 1;
    while (X < columns && X < 32) X *= 2;
    const int rows = (w.E + 256 / X - 1) / (256 / X);
    const int blocks = (columns + X - 1) / X;
    const int64_t grid = (int64_t)blocks * w.N * w.H;
    if (!fits_launch(grid, 256)) return FWP_E_SHAPE;
    if (rows <= 1) k_dsum_step<T, 1><<<(unsigned)grid, 256, 0, s>>>(w, X, blocks);
    else if (rows <= 2) k_dsum_step<T, 2><<<(unsigned)grid, 256, 0, s>>>(w, X, blocks);
    else if (rows <= 4) k_dsum_step<T, 4><<<(unsigned)grid, 256, 0, s>>>(w, X, blocks);
    else if (rows <= 8) k_dsum_step<T, 8><<<(unsigned)grid, 256, 0, s>>>(w, X, blocks);
    else k_dsum_step<T, 16><<<(unsigned)grid, 256, 0, s>>>(w, X, blocks);
    return (int)hipGetLastError();
}

}  // namespace

int64_t dsum_saved_floats(int type, int N, int H, int L, int E, int M) {
    const Plan p = plan_of(type, N, H, L, E, M, false);
    return p.heads * p.chunks * p.cells;
}

int64_t dsum_workspace(const fwp_dsum_args &a, bool backward) {
    const Plan p = plan_of(a.type, a.N, a.H, a.L, a.E, a.M, backward);
    return backward ? backward_room(a, p).total : p.ends;
}

int dsum_fwd(const fwp_dsum_args &a, float *W, fwp_out_rows out, float *saved, float *workspace, hipStream_t s) {
    const Plan p = plan_of(a.type, a.N, a.H, a.L, a.E, a.M, false);
    DsumWalk w = walk_of(a, p);
    w.out = out;
    w.from = w.to = W;
    w.saved = saved;
    if (a.L == 1 && !saved) {
        int rc = FWP_E_SHAPE;
        by_type(a.type, [&](auto t) { rc = launch_step<decltype(t)>(w, s); });
        return rc;
    }
    if (p.segments > 1) {
        if (!workspace) return FWP_E_NULL;
        w.ends = workspace;
        w.factors = workspace + p.heads * p.segments * p.cells;
        w.joined = p.segments > kFewSegments;
        if (int rc = launch(kDsumForwardEnds, a, p, w, p.segments - 1, s)) return rc;
        if (w.joined) join<false>(w, W, p.heads, p.Ep, s);
    }
    if (int rc = launch(kDsumForward, a, p, w, p.segments, s)) return rc;
    return (int)hipGetLastError();
}

int dsum_bwd(const fwp_dsum_args &a, const float *saved, fwp_rows gout, fwp_out_rows gq, fwp_out_rows gk, fwp_out_rows gv, float *gdecay,
             float *workspace, hipStream_t s) {
    const Plan p = plan_of(a.type, a.N, a.H, a.L, a.E, a.M, true);
    const BackwardRoom room = backward_room(a, p);
    DsumWalk w = walk_of(a, p);
    w.go = gout;
    w.gq = gq, w.gk = gk, w.gv = gv;
    w.saved = const_cast<float *>(saved);
    float *at = workspace;
    const auto take = [&](int64_t n) {
        float *r = n ? at : nullptr;
        at += padded(n);
        return r;
    };
    w.ends = take(p.ends);
    w.factors = w.ends ? w.ends + p.heads * p.segments * p.cells : nullptr;
    w.pq = take(room.q), w.pk = take(room.k), w.pv = take(room.v);
    float *parts = take(room.decay);
    w.gdecay = parts ? parts : gdecay;
    if (p.segments > 1) {
        if (int rc = launch(kDsumBackwardEnds, a, p, w, p.segments - 1, s)) return rc;
        w.joined = p.segments > kFewSegments;
        if (w.joined) join<true>(w, nullptr, p.heads, p.Ep, s);
    }
    if (int rc = launch(kDsumBackward, a, p, w, p.segments, s)) return rc;
    by_type(a.type, [&](auto t) {
        using T = decltype(t);
        if (w.pq) sum_parts<T>(w.pq, gq, a.H / a.HQ * p.slices, a.N, a.HQ, a.L, a.E, s);
        if (w.pk) sum_parts<T>(w.pk, gk, a.H / a.HK * p.slices, a.N, a.HK, a.L, a.E, s);
        if (w.pv) sum_parts<T>(w.pv, gv, a.H / a.HV, a.N, a.HV, a.L, a.M, s);
    });
    if (a.per_head) {
        k_sum_heads<<<a.H, 256, 0, s>>>(parts, gdecay, a.N, a.H, p.slices * p.segments);
    } else if (parts) {
        // its rows are those of the heads, L numbers each
        sum_parts<float>(parts, fwp_out_rows{gdecay, (int64_t)a.H * a.L, a.L, 0}, p.slices, a.N, a.H, 1, a.L, s);
    }
    return (int)hipGetLastError();
}

}  // namespace fwp
