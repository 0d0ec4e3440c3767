// The sum rule with a decay for each head, in chunks on the matrix cores.
//
//   S_t = a_t S_{t-1} + k_t (x) v_t,  o_t = scale S_t^T q_t,  a_t = exp(g_t), g_t of a head or of a step of a head
//
// Over a chunk of C steps with b_t = g_1 + .. + g_t, S the state before it and G the adjoint of the state behind it (both without `scale`):
//
//   P_ts = exp(b_t - b_s) q_t . k_s (s <= t)       o  = scale (P V + exp(b) Q S)         S' = exp(b_C) S + K^T (exp(b_C - b) V)
//   R_ts = exp(b_t - b_s) do_t . v_s (s <= t)      dq = scale (R K + exp(b) dO S^T)      dk = scale (R^T Q + exp(b_C - b) V G^T)
//   G'   = exp(b_C) G + Q^T (exp(b) dO)            dv = scale (P^T dO + exp(b_C - b) K G)
//   dg_t = sum_{s >= t in the chunk} (q_s . dq_s - k_s . dk_s) + scale <G, S'>
//
// Every factor is exp of a difference that is itself a sum of decays, at most 1 where they are not positive.  The sums b are made in 64 bits and kept as a
// pair of floats: behind a step of strong decay, differences of small ones would otherwise have lost their digits.  The inner product <G, S'> at every
// chunk's end keeps the decays' gradients from being differences of sums over the whole sequence.
//
// A workgroup owns a sequence's head and a slice of its value columns, and walks over the chunks of a segment with the state in registers:
// a wave holds all key rows of MW x 16 columns.  A sequence is cut into segments where there are too few of them to fill the GPU: a first kernel walks over each
// but the last from zero, and the walk proper starts every segment from what those before it leave, joined by itself or, of many, by a kernel between the two.
//
// Why chunks: a step by itself has no matrix product in it and 4 E M vector operations; in chunks of 64 (bf16, 32 where a tile takes two or three times the LDS) nearly all is products
// of 16 x 16 x 32, at an eighth of the time of the rows' way through memory.  8 x 16 sequences of 4096 steps, 64 x 64 bf16 in chunks of 32: 128 us forward and 245 back, then
// 105 and 213 in chunks of 64.  Neither the products (20 % of the time) nor the bytes alone bound the walks: vector instructions, which scale, split and store (49 % forward, 58 % back), and what
// two or three waves a SIMD do not hide of loads and barriers (34 % and 28 % of a wave's time).
#pragma once
#include "fwp_parts.hpp"
#include "fwp_wave.hpp"

namespace fwp {

template <typename T>
constexpr int kChunkOf = std::is_same_v<T, bf16_t> ? 64 : 32;
// Parts of rows of type T and of what is made of them: numbers that end in results of fewer bits than fp32 keep 2^-16, far below their rounding,
// those that end in the state, its adjoint and the decays' gradients 2^-24.
// Rows of fp32 with up to 32 keys have products of fp32 itself: 256 sequences of 1024 steps, 32 x 32, 53 + 125 us against 57 + 144 with six products of parts.
// Wider ones have more products in every chunk and gain by the parts: 64 of 2048 steps, 64 x 64, 95 + 115 us with parts, 111 + 136 without.
template <typename T, int NE>
struct Parts {
    static constexpr bool kWhole = std::is_same_v<T, float> && NE <= 2;
    static constexpr int P = kWhole ? kPlain : kPartsOf<T>, O = kWhole ? kPlain : sizeof(T) == 2 ? 2 : 3, X = kWhole ? kPlain : 3;
};

struct DsumWalk {
    fwp_rows q, k, v, go;
    fwp_out_rows out, gq, gk, gv;      // gq, gk, gv: used where the partial buffers are NULL
    const float *decay;
    int64_t dN, dH, dL;
    const int64_t *lengths;
    const float *from;                 // the state a sequence starts from (NULL: zeros), [N,H,E,M]
    float *to;                         // the state after the last step (NULL: not kept)
    float *saved;                      // [N,H,chunks,Ep,Mp]: the states before each chunk
    float *ends, *factors;             // [N,H,segments,Ep,Mp], [N,H,segments]
    float *pq, *pk, *pv;               // partial gradients [parts][N,G,L,E|M]
    float *gdecay;                     // [slices][N,H,L], or [N,H,slices,segments] where a head has one decay
    float scale;
    int N, H, L, E, M, HQ, HK, HV, Mp, slices, segments, per;      // per: chunks of a segment
    int sum_decay;
    int joined;                        // the segments' first states are in `ends`; else each workgroup joins those that it needs, and slot 0 is `from`
};

// Workgroups b, b + 8, .. run on one XCD: neighbours in the order of the work get numbers that lie 8 apart.  Slices and heads come first in that order: they share
// rows, or read rows that lie side by side where steps are outermost, at about the same time.
__device__ __forceinline__ uint32_t by_xcd(uint32_t b, uint32_t n) {
    const uint32_t whole = n / 8 * 8;
    return b < whole ? b % 8 * (n / 8) + b / 8 : b;
}

template <int C>
struct alignas(16) Decays {
    float hi[C], lo[C], into[C], rest[C];
    float whole, pad[3];

    // One wave: the sums over a chunk of its steps' decays, lane t those up to step t.  A decay below -1e5 is 0 all the same.
    __device__ __forceinline__ double sum(float g, int lane) {
        constexpr float least = -1e5f;
        double x = (double)(g < least ? least : g) * 1.4426950408889634074;
        x += shifted<0x111, 0xf>(x);      // row_shr:1, 2, 4, 8
        x += shifted<0x112, 0xf>(x);
        x += shifted<0x114, 0xf>(x);
        x += shifted<0x118, 0xf>(x);
        x += shifted<kRowBcast15, 0xa>(x);
        x += shifted<kRowBcast31, 0xc>(x);
        const double total = __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)__builtin_bit_cast(uint64_t, x), 63) |
                                                            (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(__builtin_bit_cast(uint64_t, x) >> 32), 63) << 32);
        if (lane < C) {
            const float h = (float)x;
            hi[lane] = h;
            lo[lane] = (float)(x - (double)h);
            into[lane] = __builtin_amdgcn_exp2f(h);
            rest[lane] = __builtin_amdgcn_exp2f((float)(total - x));
        }
        if (lane == 0) whole = __builtin_amdgcn_exp2f((float)total);
        return total;
    }
    // x of another lane of the wave, 0 where there is none
    template <int CTRL, int ROWS>
    static __device__ __forceinline__ double shifted(double x) {
        const uint64_t u = __builtin_bit_cast(uint64_t, x);
        const uint32_t l = __builtin_amdgcn_update_dpp(0, (int)u, CTRL, ROWS, 0xf, true), h = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, 0xf, true);
        return __builtin_bit_cast(double, (uint64_t)h << 32 | l);
    }
    // exp(b_t - b_s) for the four steps s ..; 0 where s > t
    __device__ __forceinline__ v4f between(int t, int s) const {
        const v4f h = *reinterpret_cast<const v4f *>(&hi[s]), l = *reinterpret_cast<const v4f *>(&lo[s]);
        const float ht = hi[t], lt = lo[t];
        v4f f;
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = s + i <= t ? __builtin_amdgcn_exp2f((ht - h[i]) + (lt - l[i])) : 0.f;
        return f;
    }
};

// A fragment times the steps' factors, split again
template <int Q, int P>
__device__ __forceinline__ Frag<Q> scaled(const Frag<P> &f, const float *factors, int sb, int g) {
    const v4f r0 = *reinterpret_cast<const v4f *>(&factors[32 * sb + 8 * g]), r1 = *reinterpret_cast<const v4f *>(&factors[32 * sb + 8 * g + 4]);
    float x[8];
    join8(f, x);
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] *= r0[i], x[i + 4] *= r1[i];
    return split8<Q>(x);
}

// A state, or an adjoint, and the products of a block of 32 steps.  APART, where a chunk is one block: it goes over the chunk as well, whose sum is made by itself first.  Added to the state product by
// product, the sum is rounded to the state's digits up to eight times a chunk: 32 x 8 sequences of 1024 steps, 32 x 32 fp32, results off by 3.7e-7 of their norm and decays' gradients by 5.0e-7, apart 2.2e-7 and
// 3.4e-7; 155 us both.  Else the state has gone over the chunk before: two blocks would need twice the fragments at once.
template <bool APART, int ORDERS, int PA, int PB>
__device__ __forceinline__ v4f go_on(const v4f &S, float whole, const Frag<PA> &a, const Frag<PB> &b) {
    if constexpr (!APART) return product<ORDERS>(a, b, S);
    const v4f added = product<ORDERS>(a, b, v4f{0, 0, 0, 0});
    v4f r;
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = fmaf(S[i], whole, added[i]);
    return r;
}

// Sums over the four groups of 16 lanes, and over the lanes of a group, in every lane
__device__ __forceinline__ float over_groups(float x) {
    float y = x;
    swap16(x, y);
    x += y, y = x;
    swap32(x, y);
    return x + y;
}
__device__ __forceinline__ float over_sixteen(float x) {
    x += dpp<kQuadXor1>(x);
    x += dpp<kQuadXor2>(x);
    x += dpp<kRowRor4>(x);
    return x + dpp<kRowRor8>(x);
}

// A number as it is, but one the compiler knows nothing of: what follows from it is worked out where it is needed, instead of being kept in scalar registers that
// run out, or turned into addresses of their own for every row, which take vector registers and are advanced from chunk to chunk.
__device__ __forceinline__ int opaque(int x) {
    asm volatile("" : "+s"(x));
    return x;
}

// W consecutive numbers of a row from element `at` of `base` on, in stores of up to 16 bytes at an element's address
template <typename T, int W>
__device__ __forceinline__ void store_whole(T *base, uint32_t at, const float (&x)[W]) {
    constexpr int kWords = sizeof(T) * W / 4, kStep = kWords < 4 ? kWords : 4;
    typedef uint32_t Words __attribute__((ext_vector_type(kStep)));
    struct __attribute__((packed, aligned(sizeof(T)))) Anywhere { Words w; };
    struct Split { Words w[kWords / kStep]; };
    Split split;
    if constexpr (std::is_same_v<T, bf16_t>) {
        struct { uint32_t w[kWords]; } words;
#pragma unroll
        for (int i = 0; i < kWords; i++) {
            float a = x[2 * i], b = x[2 * i + 1];
            words.w[i] = next_parts(a, b, true);
        }
        split = __builtin_bit_cast(Split, words);
    } else {
        struct { T x[W]; } row;
#pragma unroll
        for (int i = 0; i < W; i++) row.x[i] = (T)x[i];
        split = __builtin_bit_cast(Split, row);
    }
    asm volatile("" : "+v"(at));      // made here, or the compiler keeps 64 bits of it for every row
    Anywhere *to = reinterpret_cast<Anywhere *>(from(base, at));
#pragma unroll
    for (int i = 0; i < kWords / kStep; i++) to[i].w = split.w[i];
}
// A chunk's results, columns col .. of rows 16 I + c.  base: its first row, the same for all lanes; C rows lie within 32 bits of bytes.  live: the chunk's rows that
// count, the others become zero; there: those that are there at all.  cols: this lane's columns that are there, of 4 J (all where WHOLE).
template <bool WHOLE, typename T, int C, int J>
__device__ __forceinline__ void store_rows(T *base, int stride, int col, const v4f (&acc)[C / 16][J], float scale, int live, int there, int cols, int c) {
    const auto result = [&](int I, float (&x)[4 * J]) {
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) x[4 * j + i] = acc[I][j][i] * scale;
        return (uint32_t)(16 * I + c) * (uint32_t)stride + (uint32_t)col;
    };
    if (WHOLE && live >= C) {
#pragma unroll
        for (int I = 0; I < C / 16; I++) {
            float x[4 * J];
            const uint32_t at = result(I, x);
            store_whole<T, 4 * J>(base, at, x);
        }
        return;
    }
#pragma unroll
    for (int I = 0; I < C / 16; I++) {
        float x[4 * J];
        const uint32_t at = result(I, x);
        if (16 * I + c >= there) continue;
#pragma unroll
        for (int i = 0; i < 4 * J; i++) x[i] = 16 * I + c < live ? x[i] : 0.f;
        if (WHOLE || cols >= 4 * J) {
            store_whole<T, 4 * J>(base, at, x);
        } else {
            T *to = from(base, at);
#pragma unroll
            for (int i = 0; i < 4 * J; i++)
                if (i < cols) to[i] = (T)x[i];
        }
    }
}

// The i-th of the pairs of a block of 32 steps s and a tile I of 16 steps t that meet on or below the diagonal: LOWER, t behind s (I >= 2 sb); else s in front of t (I < 2 sb + 2).
template <int TT, bool LOWER>
struct Pairs {
    static constexpr int SB = TT / 2, kCount = SB * (SB + 1);
    int sb, I;
    __device__ __forceinline__ constexpr explicit Pairs(int i) : sb(0), I(0) {
        int n = LOWER ? TT : 2;
        while (i >= n) i -= n, sb++, n += LOWER ? -2 : 2;
        I = LOWER ? 2 * sb + i : i;
    }
};

// A first state from those that the segments leave, slots lo .. hi of `ends` one after another (backwards from lo down to hi where STEP is -1): what slot lo holds, then S = factor S + what the
// slot holds.  each(use) has use(number, four of the state's numbers, their offsets in a slot) called for all that the lane has; the loads of K slots go out together, as many as there are registers for.
template <int STEP, int COUNT, typename Each>
__device__ __forceinline__ void fold_segments(const float *ends, int64_t cells, const float *factors, int lo, int hi, Each each) {
    constexpr int K = COUNT <= 8 ? 4 : 2;
#pragma unroll 1
    for (int s0 = lo; STEP * s0 <= STEP * hi; s0 += STEP * K) {
        v4f x[K][COUNT];
        float y[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int slot = STEP > 0 ? min(s0 + k, hi) : max(s0 - k, hi);
            const float *at = ends + slot * cells;
            y[k] = slot == lo ? 0.f : factors[slot - STEP];
            each([&](int n, v4f &, auto place) {
#pragma unroll
                for (int i = 0; i < 4; i++) x[k][n][i] = at[place(i)];
            });
        }
#pragma unroll
        for (int k = 0; k < K; k++)
            if (STEP * (s0 + STEP * k) <= STEP * hi) each([&](int n, v4f &S, auto) { S = y[k] * S + x[k][n]; });
    }
}
__device__ __forceinline__ void pin(v4f &x) {
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = pinned(x[i]);
}

// Workgroups of a kernel that a CU holds at once at the least: 160 KB of LDS, and registers for `waves` on each of four SIMDs, which the kernel's launch bounds ask for.  Where the compiler needs
// fewer registers there may be up to twice as many, which plans do not count on.
constexpr int resident(size_t lds, int waves, int NW) { return (int)(160 * 1024 / lds) < 4 * waves / NW ? (int)(160 * 1024 / lds) : 4 * waves / NW; }

// ------------------------------------------------------------------ forward

template <typename T, int NE, int NW, int MW>
struct DsumForward {
    static constexpr int C = kChunkOf<T>, P = Parts<T, NE>::P, O = Parts<T, NE>::O, X = Parts<T, NE>::X, E = 16 * NE, MS = 16 * MW * NW, kThreads = 64 * NW;
    static constexpr int NB = NE / 2, SB = C / 32, TT = C / 16;
    struct Shared {
        Tile<C, E, P> q, k;
        Tile<C, MS, P> v;
        Tile<C, C, O> p;
        Decays<C> d[2];
    };
    struct Ends {
        Tile<C, E, P> k;
        Tile<C, MS, P> v;
        Decays<C> d[2];
    };
    static constexpr int kWaves = P == kPlain ? 4 : NE <= 4 ? 3 : 2, kEndWaves = NE <= 4 ? 4 : 3;
};

// ENDS: the state that a segment leaves when it starts from zero (the first from `from`, where nothing joins), and the segment's whole decay; nothing else.
// 8 x 16 sequences of 4096 steps, 64 x 64 bf16, six segments: ENDS 29 us at 4.2 TB/s, the walk 105 at 3.8 with the states it saves, a third of its bytes (24.5 without them for an eighth of the
// sequences).  32 x 8 of 1024 steps, 32 x 32 fp32, four segments: 14 and 39, 3.4 and 4.3 TB/s.
template <typename T, int NE, int NW, int MW, bool WHOLE, bool ENDS>
__global__ __launch_bounds__(64 * NW, (ENDS ? DsumForward<T, NE, NW, MW>::kEndWaves : DsumForward<T, NE, NW, MW>::kWaves)) void k_dsum_fwd(const DsumWalk a) {
    using F = DsumForward<T, NE, NW, MW>;
    constexpr int C = F::C, P = F::P, O = F::O, X = F::X, E = F::E, MS = F::MS, NB = F::NB, SB = F::SB, TT = F::TT;
    constexpr bool APART = SB == 1;
    __shared__ std::conditional_t<ENDS, typename F::Ends, typename F::Shared> sh;
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, g = lane / 16, c = lane % 16;

    uint32_t w = by_xcd(blockIdx.x, gridDim.x);
    const int slice = w % (uint32_t)a.slices;
    w /= (uint32_t)a.slices;
    const int h = w % (uint32_t)a.H;
    w /= (uint32_t)a.H;
    const int n = w % (uint32_t)a.N, seg = w / (uint32_t)a.N;

    const int len = length_of(a.lengths, n, a.L), chunks = (a.L + C - 1) / C, live = (len + C - 1) / C;
    const int first = seg * a.per, last = min(first + a.per, chunks), stop = min(last, live);
    const int hq = h / (a.H / a.HQ), hk = h / (a.H / a.HK), hv = h / (a.H / a.HV), m0 = slice * MS, mcols = min(a.M - m0, MS), mw = wave * 16 * MW;
    const T *qb = row<T>(a.q, n, hq, 0), *kb = row<T>(a.k, n, hk, 0), *vb = row<T>(a.v, n, hv, 0) + m0;
    const float *gb = a.decay + n * a.dN + h * a.dH;
    T *ob = nullptr;
    if constexpr (!ENDS) ob = row<T>(a.out, n, h, 0) + m0;

    v4f S[NB][2][MW];
    const int64_t head = (int64_t)n * a.H + h;
    const auto each = [&](auto use) {
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int j = 0; j < MW; j++)
                    use((b * 2 + u) * MW + j, S[b][u][j], [&](int i) { return (32 * b + 8 * g + 4 * u + i) * a.Mp + m0 + mw + place(MW, c, j); });
    };
    each([](int, v4f &x, auto) { x = v4f{0, 0, 0, 0}; });
    // A walk in segments takes its first states from `ends` alone: the last segment's workgroup writes `to`, which is `from`, and may have done so before the other
    // segments' have started.  Where nothing joins, the kernel that runs before starts the first segment from `from` and puts that into slot 0.
    if (a.from && (ENDS ? seg == 0 && !a.joined : a.segments == 1)) {
        const float *from = a.from + head * a.E * a.M;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int j = 0; j < MW; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int e = 32 * b + 8 * g + 4 * u + i, m = m0 + mw + place(MW, c, j);
                        if (e < a.E && m < a.M) S[b][u][j][i] = from[(int64_t)e * a.M + m];
                    }
        if constexpr (ENDS) {
            float *at = a.ends + head * a.segments * E * a.Mp;
            each([&](int, v4f &x, auto place) {
#pragma unroll
                for (int i = 0; i < 4; i++) at[place(i)] = x[i];
            });
        }
    }
    if constexpr (!ENDS) {
        if (a.segments > 1 && (seg > 0 || a.from))
            fold_segments<1, NB * 2 * MW>(a.ends + head * a.segments * E * a.Mp, (int64_t)E * a.Mp, a.factors + head * a.segments, a.joined ? seg : min(seg, 1), seg, each);
        // arrived, as everything that is loaded ahead of the loop: a wait that its first round needs would be one of all rounds
        each([](int, v4f &x, auto) { pin(x); });
    }
    if constexpr (!ENDS) {      // tiles of P above the diagonal stay zero
        for (int i = tid; i < (int)(sizeof(sh.p) / 16); i += 64 * NW) reinterpret_cast<v4f *>(&sh.p)[i] = v4f{0, 0, 0, 0};
    }

    Stage<T, C, E, 64 * NW, WHOLE> sq, sk;
    Stage<T, C, MS, 64 * NW, WHOLE> sv;
    double total = 0;
    float gnext = 0;
    const auto fetch = [&](int chunk) {
        const int64_t t0 = (int64_t)opaque(chunk) * C;
        const int rows = len - (int)t0;
        if constexpr (!ENDS) sq.load(qb + t0 * a.q.sL, (int)a.q.sL, rows, a.E, tid);
        sk.load(kb + t0 * a.k.sL, (int)a.k.sL, rows, a.E, tid);
        sv.load(vb + t0 * a.v.sL, (int)a.v.sL, rows, mcols, tid);
    };
    // the last wave, which has the fewest tiles of P, sums up the next chunk's decays
    const auto fetch_decay = [&](int chunk) { gnext = gb[min((int64_t)chunk * C + lane, (int64_t)len - 1) * a.dL]; };
    const auto sum_decay = [&](int chunk) { total += sh.d[chunk & 1].sum(lane < C && chunk * C + lane < len ? gnext : 0.f, lane); };
    if (first < stop) {
        if (wave == NW - 1) fetch_decay(first);
        fetch(first);
        if (wave == NW - 1) {
            sum_decay(first);
            if (first + 1 < stop) fetch_decay(first + 1);
        }
        if constexpr (!ENDS) sq.arrive();
        sk.arrive(), sv.arrive();
    }
    for (int chunk = first; chunk < stop; chunk++) {
        const int rows = len - chunk * C, keys = opaque(a.E), values = opaque(mcols);
        if constexpr (!ENDS) sq.put(sh.q, rows, keys, tid);
        sk.put(sh.k, rows, keys, tid);
        sv.put(sh.v, rows, values, tid);
        lds_barrier();
        const Decays<C> &d = sh.d[chunk & 1];
        if (wave == NW - 1 && chunk + 1 < stop) {
            sum_decay(chunk + 1);
            if (chunk + 2 < stop) fetch_decay(chunk + 2);
        }
        if (chunk + 1 < stop) fetch(chunk + 1);

        v4f acc[TT][MW];
        if constexpr (!ENDS) {
            if (a.saved) {
                float *at = a.saved + (head * chunks + opaque(chunk)) * E * a.Mp + m0;
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int j = 0; j < MW; j++)
#pragma unroll
                            for (int i = 0; i < 4; i++) *from(at, (uint32_t)(32 * b + 8 * g + 4 * u + i) * (uint32_t)a.Mp + mw + place(MW, c, j)) = S[b][u][j][i];
            }
            // P, a 16 x 16 tile of it at a time
            for (int tile = wave; tile < TT * (TT + 1) / 2; tile += NW) {
                int I = 0, J = tile;
                while (J > I) J -= ++I;
                struct Frags {
                    Frag<P> a, b;
                };
                v4f p = {0, 0, 0, 0};
                ahead<NB, kAhead<P>>([&](int b) { return Frags{sh.k.rows(16 * J, 32 * b, g, c), sh.q.rows(16 * I, 32 * b, g, c)}; },
                                     [&](int, const Frags &f) { p = product<O>(f.a, f.b, p); });
                const int t = 16 * I + c, s = 16 * J + 4 * g;
                const v4f f = d.between(t, s);
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = s + i <= t ? p[i] * f[i] : 0.f;      // a product beyond the diagonal may be infinite
                sh.p.put4(t, s, x);
            }
            // what the queries read from the state
#pragma unroll
            for (int I = 0; I < TT; I++)
#pragma unroll
                for (int j = 0; j < MW; j++) acc[I][j] = v4f{0, 0, 0, 0};
            Frag<O> state[MW];
            ahead<NB * TT, kAhead<P>>([&](int i) { return sh.q.rows(16 * (i % TT), 32 * (i / TT), g, c); },
                                      [&](int i, const Frag<P> &q) {
                                          const int b = i / TT, I = i % TT;
#pragma unroll
                                          for (int j = 0; j < MW; j++) {
                                              if (I == 0) state[j] = split8<O>(S[b][0][j], S[b][1][j]);
                                              acc[I][j] = product<O>(state[j], q, acc[I][j]);
                                          }
                                      });
#pragma unroll
            for (int I = 0; I < TT; I++) {
                const float f = d.into[16 * I + c];
#pragma unroll
                for (int j = 0; j < MW; j++) acc[I][j] *= f;
            }
            lds_barrier();
        }
        if constexpr (!APART) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int j = 0; j < MW; j++) S[b][u][j] *= d.whole;
        }
        Frag<P> v[SB][MW];
#pragma unroll
        for (int sb = 0; sb < SB; sb++)
#pragma unroll
            for (int j = 0; j < MW; j++) v[sb][j] = sh.v.template columns<MW>(mw, j, 32 * sb, g, c);
        [[maybe_unused]] int bad[MW];      // the first step whose value in this lane's column is infinite or NaN; C: none
        [[maybe_unused]] bool any_bad = false;
        if constexpr (!ENDS) {
            // such a value must not reach the steps before it through the zeros of P: it is taken for zero, and results from its step on, and the state, are NaN
            float x = 0.f;
#pragma unroll
            for (int sb = 0; sb < SB; sb++)
#pragma unroll
                for (int j = 0; j < MW; j++) x = unless_finite(v[sb][j], x);
            any_bad = __any(x != 0.f);
            if (any_bad) {
#pragma unroll
                for (int j = 0; j < MW; j++) {
                    bad[j] = C;
#pragma unroll
                    for (int sb = 0; sb < SB; sb++)
                        take_out(v[sb][j], [&](int i) { bad[j] = min(bad[j], 32 * sb + 8 * g + i); });
                    bad[j] = min(bad[j], __shfl_xor(bad[j], 16));
                    bad[j] = min(bad[j], __shfl_xor(bad[j], 32));
                }
            }
            using Below = Pairs<TT, true>;
            ahead<Below::kCount, kAhead<O>>([&](int i) { return sh.p.rows(16 * Below(i).I, 32 * Below(i).sb, g, c); },
                                            [&](int i, const Frag<O> &p) {
#pragma unroll
                                                for (int j = 0; j < MW; j++) acc[Below(i).I][j] = product<O>(v[Below(i).sb][j], p, acc[Below(i).I][j]);
                                            });
        }
        Frag<X> vs[MW];
        ahead<SB * NB * 2, kAhead<P>>([&](int i) { return sh.k.template columns<2>(32 * (i / 2 % NB), i % 2, 32 * (i / 2 / NB), g, c); },
                                      [&](int i, const Frag<P> &k) {
                                          const int sb = i / 2 / NB, b = i / 2 % NB, u = i % 2;
#pragma unroll
                                          for (int j = 0; j < MW; j++) {
                                              if (b == 0 && u == 0) vs[j] = scaled<X>(v[sb][j], d.rest, sb, g);
                                              S[b][u][j] = go_on<APART, X>(S[b][u][j], d.whole, k, vs[j]);
                                          }
                                      });
        if constexpr (!ENDS) {
            if (any_bad) {
                const float nan = __builtin_nanf("");
#pragma unroll
                for (int j = 0; j < MW; j++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        // results lie with their columns along the groups of lanes, v with them along a group's lanes
                        const int from_step = __shfl(bad[j], 4 * g + i);
#pragma unroll
                        for (int I = 0; I < TT; I++) acc[I][j][i] = 16 * I + c >= from_step ? nan : acc[I][j][i];
                    }
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int u = 0; u < 2; u++) S[b][u][j] = bad[j] < C ? v4f{nan, nan, nan, nan} : S[b][u][j];
                }
            }
            sq.arrive(), sk.arrive(), sv.arrive();
            gnext = pinned(gnext);
            const int col = mw + 4 * MW * g;
            store_rows<WHOLE, T, C, MW>(ob + (int64_t)opaque(chunk) * C * a.out.sL, (int)a.out.sL, col, acc, a.scale, rows, a.L - chunk * C, values - col, c);
        }
        lds_barrier();
    }

    if constexpr (ENDS) {
        float *at = a.ends + (head * a.segments + seg + 1) * E * a.Mp + m0 + mw;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int j = 0; j < MW; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++) at[(32 * b + 8 * g + 4 * u + i) * a.Mp + place(MW, c, j)] = S[b][u][j][i];
        if (tid == 64 * (NW - 1) && slice == 0) a.factors[head * a.segments + seg] = __builtin_amdgcn_exp2f((float)total);
    } else {
        // rows behind the sequence
        for (int64_t i = (int64_t)max(stop, first) * C * MS + tid; i < (int64_t)min(last * C, a.L) * MS; i += 64 * NW) {
            const int64_t t = i / MS;
            const int m = i % MS;
            if (m < mcols) ob[t * a.out.sL + m] = (T)0.f;
        }
        if (a.to && last == chunks) {
            float *to = a.to + head * a.E * a.M;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int j = 0; j < MW; j++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int e = 32 * b + 8 * g + 4 * u + i, m = m0 + mw + place(MW, c, j);
                            if (e < a.E && m < a.M) to[(int64_t)e * a.M + m] = S[b][u][j][i];
                        }
        }
    }
}

// ------------------------------------------------------------------ backward

// A workgroup's waves share the walk back by what they own: KW key waves have EW tiles of 16 key rows each, the gradients of q and k there and the adjoint's
// rows (all value columns, transposed); VW value waves have MW tiles of 16 value columns each, the gradient of v and the adjoint's columns, and make P and R.
// The adjoint is held twice so that no product waits for another wave's share of it.  Up to 64 keys and columns a wave is of both kinds, which leaves room for two workgroups of four waves on a
// CU: 8 x 16 sequences of 4096 steps, 64 x 64 bf16, 213 us, 223 with eight waves of one kind each.  Wider ones have no registers for that: 4 x 32 heads, 128 x 64, queries and keys
// shared, 8 waves of one kind 736 us for the training step, 4 of both 864; 8 key waves of one tile each 60 us more.  With LDS reads and loads ahead of their use (ahead, Stage::arrive) the walk is at
// 180-190 us for the first of these (0.6 GB, 3.2 TB/s) and at 383 for the second (1 GB of which half are the heads' partial gradients).  Two kernels, one for the adjoints before every chunk and one that
// works on all chunks at once, take longer: 295 + 65 and 437 + 172 us.
// The walk back has fewer registers to spare
template <int P>
constexpr int kAheadBack = kAhead<P> < 2 ? kAhead<P> : 2;

template <typename T, int NE, int NW, int MW>
struct DsumBackward {
    static constexpr int C = kChunkOf<T>, P = Parts<T, NE>::P, O = Parts<T, NE>::O, X = Parts<T, NE>::X, E = 16 * NE, MS = 16 * MW * NW;
    static constexpr int NB = NE / 2, SB = C / 32, TT = C / 16, MB = MS / 32;
    static constexpr int KW = NE < 4 ? NE : 4, EW = NE / KW, VW = MS / 16 < 4 ? MS / 16 : 4, VM = MS / 16 / VW;
    static constexpr bool kBoth = NE <= 4 && MS <= 64;      // every wave is of both kinds
    static constexpr int kCount = kBoth ? (KW > VW ? KW : VW) : KW + VW, kThreads = 64 * kCount, kTileWaves = kBoth ? kCount : VW;
    struct Shared {
        Tile<C, E, P> q, k;
        Tile<C, MS, P> v, go;
        Tile<C, C, O> p, r;
        Decays<C> d[2];
        float sums[2][KW][C], within[2][TT + 1][C], inner[2][KW];
    };
    struct Ends {
        Tile<C, E, P> q;
        Tile<C, MS, P> go;
        Decays<C> d[2];
    };
    static constexpr int kWaves = 2, kEndWaves = NE <= 4 ? 4 : 3;
};

// The adjoint of a segment's first state when that of its last one is zero, and the segment's whole decay.  8 x 16 sequences of 4096 steps, 64 x 64 bf16, four segments: 29 us at 3.7 TB/s.
template <typename T, int NE, int NW, int MW, bool WHOLE>
__global__ __launch_bounds__(64 * NW, (DsumBackward<T, NE, NW, MW>::kEndWaves)) void k_dsum_bwd_ends(const DsumWalk a) {
    using F = DsumBackward<T, NE, NW, MW>;
    constexpr int C = F::C, P = F::P, X = F::X, E = F::E, MS = F::MS, NB = F::NB, SB = F::SB;
    constexpr bool APART = SB == 1;
    __shared__ typename F::Ends sh;
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, g = lane / 16, c = lane % 16;
    uint32_t w = by_xcd(blockIdx.x, gridDim.x);
    const int slice = w % (uint32_t)a.slices;
    w /= (uint32_t)a.slices;
    const int h = w % (uint32_t)a.H;
    w /= (uint32_t)a.H;
    const int n = w % (uint32_t)a.N, seg = w / (uint32_t)a.N + 1;
    const int len = length_of(a.lengths, n, a.L), chunks = (a.L + C - 1) / C, live = (len + C - 1) / C;
    const int first = seg * a.per, stop = min(min(first + a.per, chunks), live);
    const int hq = h / (a.H / a.HQ), m0 = slice * MS, mcols = min(a.M - m0, MS), mw = wave * 16 * MW;
    const T *qb = row<T>(a.q, n, hq, 0), *db = row<T>(a.go, n, h, 0) + m0;
    const float *gb = a.decay + n * a.dN + h * a.dH;
    const int64_t head = (int64_t)n * a.H + h;
    v4f G[NB][2][MW];
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int j = 0; j < MW; j++) G[b][u][j] = v4f{0, 0, 0, 0};
    Stage<T, C, E, 64 * NW, WHOLE> sq;
    Stage<T, C, MS, 64 * NW, WHOLE> sd;
    double total = 0;
    float gnext = 0;
    const auto fetch = [&](int chunk) {
        const int64_t t0 = (int64_t)opaque(chunk) * C;
        const int rows = len - (int)t0;
        sq.load(qb + t0 * a.q.sL, (int)a.q.sL, rows, a.E, tid);
        sd.load(db + t0 * a.go.sL, (int)a.go.sL, rows, mcols, tid);
    };
    const auto fetch_decay = [&](int chunk) { gnext = gb[min((int64_t)chunk * C + lane, (int64_t)len - 1) * a.dL]; };
    const auto sum_decay = [&](int chunk) { total += sh.d[chunk & 1].sum(lane < C && chunk * C + lane < len ? gnext : 0.f, lane); };
    if (first < stop) {
        if (wave == NW - 1) fetch_decay(stop - 1);
        fetch(stop - 1);
        if (wave == NW - 1) {
            sum_decay(stop - 1);
            if (stop - 1 > first) fetch_decay(stop - 2);
        }
    }
    for (int chunk = stop - 1; chunk >= first; chunk--) {
        const int rows = len - chunk * C;
        sq.put(sh.q, rows, opaque(a.E), tid);
        sd.put(sh.go, rows, opaque(mcols), tid);
        lds_barrier();
        const Decays<C> &d = sh.d[chunk & 1];
        if (wave == NW - 1 && chunk > first) {
            sum_decay(chunk - 1);
            if (chunk - 1 > first) fetch_decay(chunk - 2);
        }
        if (chunk > first) fetch(chunk - 1);
        if constexpr (!APART) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int j = 0; j < MW; j++) G[b][u][j] *= d.whole;
        }
        Frag<P> go[SB][MW];
#pragma unroll
        for (int sb = 0; sb < SB; sb++)
#pragma unroll
            for (int j = 0; j < MW; j++) go[sb][j] = sh.go.template columns<MW>(mw, j, 32 * sb, g, c);
        Frag<X> ds[MW];
        ahead<SB * NB * 2, kAhead<P>>([&](int i) { return sh.q.template columns<2>(32 * (i / 2 % NB), i % 2, 32 * (i / 2 / NB), g, c); },
                                      [&](int i, const Frag<P> &q) {
                                          const int sb = i / 2 / NB, b = i / 2 % NB, u = i % 2;
#pragma unroll
                                          for (int j = 0; j < MW; j++) {
                                              if (b == 0 && u == 0) ds[j] = scaled<X>(go[sb][j], d.into, sb, g);
                                              G[b][u][j] = go_on<APART, X>(G[b][u][j], d.whole, q, ds[j]);
                                          }
                                      });
        lds_barrier();
    }
    float *at = a.ends + (head * a.segments + seg - 1) * E * a.Mp + m0 + mw;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int j = 0; j < MW; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) at[(32 * b + 8 * g + 4 * u + i) * a.Mp + place(MW, c, j)] = G[b][u][j][i];
    if (tid == 64 * (NW - 1) && slice == 0) a.factors[head * a.segments + seg] = __builtin_amdgcn_exp2f((float)total);
}

// The walk of one kind of waves; `wave` counts them, `tid` all threads.
template <bool KEYS, bool VALUES, typename T, int NE, int NW, int MW, bool WHOLE>
__device__ __forceinline__ void dsum_walk_back(const DsumWalk &a, typename DsumBackward<T, NE, NW, MW>::Shared &sh, int wave, int tid) {
    using F = DsumBackward<T, NE, NW, MW>;
    constexpr int C = F::C, P = F::P, O = F::O, X = F::X, E = F::E, MS = F::MS, NB = F::NB, SB = F::SB, TT = F::TT, MB = F::MB, EW = F::EW, VM = F::VM,
                  kThreads = F::kThreads;
    // 128 x 128 has no registers for it: 8 x 8 sequences of 1024 steps, fp32, training 358 us and gradients of k and v off by 3.3e-7, 427 and 2.8e-7 with it; fp16 250 us and 323
    constexpr bool APART = SB == 1 && (E < 128 || MS < 128);
    const int lane = tid % 64, g = lane / 16, c = lane % 16;
    uint32_t w = by_xcd(blockIdx.x, gridDim.x);
    const int slice = w % (uint32_t)a.slices;
    w /= (uint32_t)a.slices;
    const int h = w % (uint32_t)a.H;
    w /= (uint32_t)a.H;
    const int n = w % (uint32_t)a.N, seg = w / (uint32_t)a.N;
    const int len = length_of(a.lengths, n, a.L), chunks = (a.L + C - 1) / C, live = (len + C - 1) / C;
    const int first = seg * a.per, last = min(first + a.per, chunks), stop = min(last, live);
    const int rq = a.H / a.HQ, rk = a.H / a.HK, rv = a.H / a.HV, m0 = slice * MS, mcols = min(a.M - m0, MS), mw = wave * 16 * VM, ew = wave * 16 * EW;
    const T *qb = row<T>(a.q, n, h / rq, 0), *kb = row<T>(a.k, n, h / rk, 0), *vb = row<T>(a.v, n, h / rv, 0) + m0, *db = row<T>(a.go, n, h, 0) + m0;
    const float *gb = a.decay + n * a.dN + h * a.dH;
    const int64_t head = (int64_t)n * a.H + h;
    const bool sums_decay = VALUES && wave == F::kTileWaves - 1, grades_decay = VALUES && wave == F::kTileWaves - 2;
    const bool keys = KEYS && wave < F::KW, values = VALUES && wave < F::VW;      // a wave of both kinds may be beyond the rows or columns there are

    // the adjoint: key waves H, all value columns of their key rows, transposed; value waves G, all key rows of their value columns
    v4f H[KEYS ? MB : 1][2][EW], G[VALUES ? NB : 1][2][VM];
    constexpr int kOfH = KEYS ? MB * 2 * EW : 0, kOfG = VALUES ? NB * 2 * VM : 0;
    const auto each = [&](auto use) {
        if constexpr (KEYS) {
#pragma unroll
            for (int b = 0; b < MB; b++)
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int j = 0; j < EW; j++)
                        use((b * 2 + u) * EW + j, H[b][u][j], [&](int i) { return ((keys ? ew : 0) + place(EW, c, j)) * a.Mp + m0 + 32 * b + 8 * g + 4 * u + i; });
        }
        if constexpr (VALUES) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int j = 0; j < VM; j++)
                        use(kOfH + (b * 2 + u) * VM + j, G[b][u][j], [&](int i) { return (32 * b + 8 * g + 4 * u + i) * a.Mp + m0 + (values ? mw : 0) + place(VM, c, j); });
        }
    };
    each([](int, v4f &x, auto) { x = v4f{0, 0, 0, 0}; });
    if (a.segments > 1)
        fold_segments<-1, kOfH + kOfG>(a.ends + head * a.segments * E * a.Mp, (int64_t)E * a.Mp, a.factors + head * a.segments, a.joined ? seg : a.segments - 2, seg, each);
    each([](int, v4f &x, auto) { pin(x); });
#pragma unroll 1
    for (int i = tid; i < (int)(sizeof(sh.p) / 16); i += kThreads) reinterpret_cast<v4f *>(&sh.p)[i] = v4f{0, 0, 0, 0};
#pragma unroll 1
    for (int i = tid; i < (int)(sizeof(sh.r) / 16); i += kThreads) reinterpret_cast<v4f *>(&sh.r)[i] = v4f{0, 0, 0, 0};

    // a chunk's first state, as this key wave reads it
    float S[KEYS ? MB : 1][EW][8];
    const auto load_state = [&](int chunk) {
        const float *base = a.saved + (head * chunks + opaque(chunk)) * E * a.Mp + m0;
#pragma unroll
        for (int b = 0; b < MB; b++)
#pragma unroll
            for (int j = 0; j < EW; j++) {
                const float *at = from(base, (uint32_t)((keys ? ew : 0) + place(EW, c, j)) * (uint32_t)a.Mp + 32 * b + 8 * g);
                const float4 lo = *reinterpret_cast<const float4 *>(at), hi = *reinterpret_cast<const float4 *>(at + 4);
                S[b][j][0] = lo.x, S[b][j][1] = lo.y, S[b][j][2] = lo.z, S[b][j][3] = lo.w, S[b][j][4] = hi.x, S[b][j][5] = hi.y, S[b][j][6] = hi.z, S[b][j][7] = hi.w;
            }
    };
    const auto state_arrives = [&] {
#pragma unroll
        for (int b = 0; b < MB; b++)
#pragma unroll
            for (int j = 0; j < EW; j++)
#pragma unroll
                for (int i = 0; i < 8; i++) S[b][j][i] = pinned(S[b][j][i]);
    };
    // <H, S>, this wave's part
    const auto inner = [&] {
        float s = 0.f;
#pragma unroll
        for (int b = 0; b < MB; b++)
#pragma unroll
            for (int j = 0; j < EW; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) s = fmaf(S[b][j][i], H[b][0][j][i], s), s = fmaf(S[b][j][i + 4], H[b][1][j][i], s);
        return over_groups(over_sixteen(s));
    };

    Stage<T, C, E, kThreads, WHOLE> sq, sk;
    Stage<T, C, MS, kThreads, WHOLE> sv, sd;
    float gnext = 0, all = 0, x_end = 0;
    const auto fetch = [&](int chunk) {
        const int64_t t0 = (int64_t)opaque(chunk) * C;
        const int rows = len - (int)t0, wide = opaque(a.E), cols = opaque(mcols);
        sq.load(qb + t0 * a.q.sL, (int)a.q.sL, rows, wide, tid);
        sk.load(kb + t0 * a.k.sL, (int)a.k.sL, rows, wide, tid);
        sv.load(vb + t0 * a.v.sL, (int)a.v.sL, rows, cols, tid);
        sd.load(db + t0 * a.go.sL, (int)a.go.sL, rows, cols, tid);
    };
    const auto fetch_decay = [&](int chunk) { gnext = gb[min((int64_t)chunk * C + lane, (int64_t)len - 1) * a.dL]; };
    const auto sum_decay = [&](int chunk) { sh.d[chunk & 1].sum(lane < C && chunk * C + lane < len ? gnext : 0.f, lane); };
    // the decays' gradients of a chunk, from what the waves have left in LDS
    const auto decay_gradients = [&](int chunk) {
        float s = 0.f, x = 0.f;
#pragma unroll
        for (int i = 0; i < F::KW; i++) s += sh.sums[chunk & 1][i][lane % C], x += sh.inner[chunk & 1][i];
#pragma unroll
        for (int i = 0; i <= TT; i++) s += sh.within[chunk & 1][i][lane % C];
        if (lane >= C) s = 0.f;
#pragma unroll
        for (int off = 1; off < C; off *= 2) {
            const float y = __shfl_down(s, off);
            if (lane + off < C) s += y;
        }
        const int t = chunk * C + lane;
        s = lane < C && t < len ? (s + x) * a.scale : 0.f;
        if (a.sum_decay) all += s;
        else if (lane < C && t < a.L) a.gdecay[(((int64_t)slice * a.N + n) * a.H + h) * a.L + t] = s;
    };
    if (first < stop) {
        if (sums_decay) fetch_decay(stop - 1);
        fetch(stop - 1);
        if (sums_decay) {
            sum_decay(stop - 1);
            if (stop - 1 > first) fetch_decay(stop - 2);
        }
        if constexpr (KEYS) {
            // the inner product at the segment's end, with the next segment's first state; behind the last chunk the adjoint is zero
            if (stop == last && stop < live) {
                load_state(stop);
                x_end = inner();
            }
            load_state(stop - 1);
            state_arrives();
        }
        sq.arrive(), sk.arrive(), sv.arrive(), sd.arrive();
    }

    for (int chunk = stop - 1; chunk >= first; chunk--) {
        const int rows = len - chunk * C, there = a.L - chunk * C;
        {
            const int wide = opaque(a.E), cols = opaque(mcols);
            sq.put(sh.q, rows, wide, tid);
            sk.put(sh.k, rows, wide, tid);
            sv.put(sh.v, rows, cols, tid);
            sd.put(sh.go, rows, cols, tid);
        }
        if (keys && lane == 0) sh.inner[chunk & 1][wave] = x_end;
        lds_barrier();
        const Decays<C> &d = sh.d[chunk & 1];
        if (sums_decay && chunk > first) {
            sum_decay(chunk - 1);
            if (chunk - 1 > first) fetch_decay(chunk - 2);
        }
        if (chunk > first) fetch(chunk - 1);
        if (grades_decay && chunk + 1 < stop) decay_gradients(chunk + 1);

        // P and R, a 16 x 16 tile of each at a time
        if (VALUES)
            for (int tile = wave; tile < TT * (TT + 1) / 2; tile += F::kTileWaves) {
                int I = 0, J = tile;
                while (J > I) J -= ++I;
                struct Frags {
                    Frag<P> a, b;
                };
                v4f p = {0, 0, 0, 0}, r = {0, 0, 0, 0};
                ahead<NB + MB, kAheadBack<P>>([&](int i) {
                                              return i < NB ? Frags{sh.k.rows(16 * J, 32 * i, g, c), sh.q.rows(16 * I, 32 * i, g, c)}
                                                            : Frags{sh.v.rows(16 * J, 32 * (i - NB), g, c), sh.go.rows(16 * I, 32 * (i - NB), g, c)};
                                          },
                                          [&](int i, const Frags &f) {
                                              if (i < NB) p = product<X>(f.a, f.b, p);
                                              else r = product<X>(f.a, f.b, r);
                                          });
                const int t = 16 * I + c, s = 16 * J + 4 * g;
                const v4f f = d.between(t, s);
                float x[4], y[4], u = 0.f, z[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x[i] = s + i <= t ? p[i] * f[i] : 0.f, y[i] = s + i <= t ? r[i] * f[i] : 0.f;
                    z[i] = s + i < t ? x[i] * r[i] : 0.f;
                    u += z[i];
                }
                // what step t reads of what step s wrote counts for the decays between them: sums over s for every t, and over t for every s
                u = over_groups(u);
#pragma unroll
                for (int i = 0; i < 4; i++) z[i] = over_sixteen(z[i]);
                if (g == 0) sh.within[chunk & 1][J][t] = u;
                if (c == 0) *reinterpret_cast<v4f *>(&sh.within[chunk & 1][I == J ? TT : I][s]) = v4f{-z[0], -z[1], -z[2], -z[3]};
                sh.p.put4(t, s, x);
                sh.r.put4(t, s, y);
            }

        v4f dq[TT][EW], dk[TT][EW], dv[TT][VM];
        if (keys) {
#pragma unroll
            for (int I = 0; I < TT; I++)
#pragma unroll
                for (int j = 0; j < EW; j++) dq[I][j] = dk[I][j] = v4f{0, 0, 0, 0};
            // through the states before and behind the chunk
            Frag<X> state[EW];
            ahead<MB * 2 * TT, kAheadBack<P>>(
                [&](int i) { return i / TT % 2 ? sh.v.rows(16 * (i % TT), 32 * (i / TT / 2), g, c) : sh.go.rows(16 * (i % TT), 32 * (i / TT / 2), g, c); },
                [&](int i, const Frag<P> &f) {
                    const int b = i / TT / 2, I = i % TT;
                    const bool adjoint = i / TT % 2;
#pragma unroll
                    for (int j = 0; j < EW; j++) {
                        if (I == 0) state[j] = adjoint ? split8<X>(H[b][0][j], H[b][1][j]) : split8<X>(S[b][j]);
                        if (adjoint) dk[I][j] = product<X>(state[j], f, dk[I][j]);
                        else dq[I][j] = product<X>(state[j], f, dq[I][j]);
                    }
                });
            // What the rows read of the state before the chunk, and wrote into what is read behind it, counts for the decays; and what was there before and is read by the
            // chunk or behind it, for those of the chunk before: <G', S> = exp(b_C) <G, S> + the sum of what the rows read.
            const float through = inner() * d.whole;
            if (chunk > first) load_state(chunk - 1);
            float read = 0.f;
#pragma unroll
            for (int I = 0; I < TT; I++) {
                const int r = 16 * I + c;
                const float into = d.into[r], rest = d.rest[r];
                float u = 0.f, w = 0.f;
#pragma unroll
                for (int j = 0; j < EW; j++) {
                    dq[I][j] *= into, dk[I][j] *= rest;
                    const v4f q = sh.q.four(r, ew + 4 * EW * g + 4 * j), k = sh.k.four(r, ew + 4 * EW * g + 4 * j);
#pragma unroll
                    for (int i = 0; i < 4; i++) u = fmaf(q[i], dq[I][j][i], u), w = fmaf(k[i], dk[I][j][i], w);
                }
                read += u;
                u = over_groups(u - w);
                if (g == 0) sh.sums[chunk & 1][wave][r] = u;
            }
            x_end = through + over_groups(over_sixteen(read));
        }
        if (values) {
#pragma unroll
            for (int I = 0; I < TT; I++)
#pragma unroll
                for (int j = 0; j < VM; j++) dv[I][j] = v4f{0, 0, 0, 0};
            Frag<O> state[VM];
            ahead<NB * TT, kAheadBack<P>>([&](int i) { return sh.k.rows(16 * (i % TT), 32 * (i / TT), g, c); },
                                      [&](int i, const Frag<P> &k) {
                                          const int b = i / TT, I = i % TT;
#pragma unroll
                                          for (int j = 0; j < VM; j++) {
                                              if (I == 0) state[j] = split8<O>(G[b][0][j], G[b][1][j]);
                                              dv[I][j] = product<O>(state[j], k, dv[I][j]);
                                          }
                                      });
#pragma unroll
            for (int I = 0; I < TT; I++) {
                const float rest = d.rest[16 * I + c];
#pragma unroll
                for (int j = 0; j < VM; j++) dv[I][j] *= rest;
            }
        }
        lds_barrier();
        gnext = pinned(gnext);

        if (keys) {
            // within the chunk, and the adjoint of the state before it
            if constexpr (!APART) {
#pragma unroll
                for (int b = 0; b < MB; b++)
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int j = 0; j < EW; j++) H[b][u][j] *= d.whole;
            }
            Frag<P> q[SB][EW], k[SB][EW];
#pragma unroll
            for (int sb = 0; sb < SB; sb++)
#pragma unroll
                for (int j = 0; j < EW; j++) k[sb][j] = sh.k.template columns<EW>(ew, j, 32 * sb, g, c), q[sb][j] = sh.q.template columns<EW>(ew, j, 32 * sb, g, c);
            using Below = Pairs<TT, true>;
            using Above = Pairs<TT, false>;
            ahead<Below::kCount, kAheadBack<O>>([&](int i) { return sh.r.rows(16 * Below(i).I, 32 * Below(i).sb, g, c); },
                                            [&](int i, const Frag<O> &r) {
#pragma unroll
                                                for (int j = 0; j < EW; j++) dq[Below(i).I][j] = product<O>(k[Below(i).sb][j], r, dq[Below(i).I][j]);
                                            });
            ahead<Above::kCount, kAheadBack<O>>([&](int i) { return sh.r.template columns<1>(16 * Above(i).I, 0, 32 * Above(i).sb, g, c); },
                                            [&](int i, const Frag<O> &r) {
#pragma unroll
                                                for (int j = 0; j < EW; j++) dk[Above(i).I][j] = product<O>(q[Above(i).sb][j], r, dk[Above(i).I][j]);
                                            });
            Frag<X> qs[EW];
            ahead<SB * MB * 2, kAheadBack<P>>([&](int i) { return sh.go.template columns<2>(32 * (i / 2 % MB), i % 2, 32 * (i / 2 / MB), g, c); },
                                          [&](int i, const Frag<P> &go) {
                                              const int sb = i / 2 / MB, b = i / 2 % MB, u = i % 2;
#pragma unroll
                                              for (int j = 0; j < EW; j++) {
                                                  if (b == 0 && u == 0) qs[j] = scaled<X>(q[sb][j], d.into, sb, g);
                                                  H[b][u][j] = go_on<APART, X>(H[b][u][j], d.whole, go, qs[j]);
                                              }
                                          });
            sq.arrive(), sk.arrive(), sv.arrive(), sd.arrive();
            state_arrives();
            {
                const int wide = opaque(a.E), col = ew + 4 * EW * g;
                if (a.pq) {
                    float *pq = a.pq + ((((int64_t)(h % rq) * a.slices + slice) * a.N + n) * a.HQ + h / rq) * a.L * wide;
                    store_rows<WHOLE, float, C, EW>(pq + (int64_t)opaque(chunk) * C * wide, wide, col, dq, a.scale, rows, there, wide - col, c);
                } else {
                    store_rows<WHOLE, T, C, EW>(row<T>(a.gq, n, h, (int64_t)opaque(chunk) * C), (int)a.gq.sL, col, dq, a.scale, rows, there, wide - col, c);
                }
                if (a.pk) {
                    float *pk = a.pk + ((((int64_t)(h % rk) * a.slices + slice) * a.N + n) * a.HK + h / rk) * a.L * wide;
                    store_rows<WHOLE, float, C, EW>(pk + (int64_t)opaque(chunk) * C * wide, wide, col, dk, a.scale, rows, there, wide - col, c);
                } else {
                    store_rows<WHOLE, T, C, EW>(row<T>(a.gk, n, h, (int64_t)opaque(chunk) * C), (int)a.gk.sL, col, dk, a.scale, rows, there, wide - col, c);
                }
            }
        }
        if (values) {
            if constexpr (!APART) {
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int j = 0; j < VM; j++) G[b][u][j] *= d.whole;
            }
            Frag<P> go[SB][VM];
#pragma unroll
            for (int sb = 0; sb < SB; sb++)
#pragma unroll
                for (int j = 0; j < VM; j++) go[sb][j] = sh.go.template columns<VM>(mw, j, 32 * sb, g, c);
            using Above = Pairs<TT, false>;
            ahead<Above::kCount, kAheadBack<O>>([&](int i) { return sh.p.template columns<1>(16 * Above(i).I, 0, 32 * Above(i).sb, g, c); },
                                            [&](int i, const Frag<O> &p) {
#pragma unroll
                                                for (int j = 0; j < VM; j++) dv[Above(i).I][j] = product<O>(go[Above(i).sb][j], p, dv[Above(i).I][j]);
                                            });
            // this side of the adjoint ends in the gradient of v alone
            Frag<O> ds[VM];
            ahead<SB * NB * 2, kAheadBack<P>>([&](int i) { return sh.q.template columns<2>(32 * (i / 2 % NB), i % 2, 32 * (i / 2 / NB), g, c); },
                                          [&](int i, const Frag<P> &q) {
                                              const int sb = i / 2 / NB, b = i / 2 % NB, u = i % 2;
#pragma unroll
                                              for (int j = 0; j < VM; j++) {
                                                  if (b == 0 && u == 0) ds[j] = scaled<O>(go[sb][j], d.into, sb, g);
                                                  G[b][u][j] = go_on<APART, O>(G[b][u][j], d.whole, q, ds[j]);
                                              }
                                          });
            if (!KEYS) sq.arrive(), sk.arrive(), sv.arrive(), sd.arrive();
            {
                const int cols = opaque(mcols), col = mw + 4 * VM * g;
                if (a.pv) {
                    float *pv = a.pv + (((int64_t)(h % rv) * a.N + n) * a.HV + h / rv) * a.L * a.M + m0;
                    store_rows<WHOLE, float, C, VM>(pv + (int64_t)opaque(chunk) * C * a.M, a.M, col, dv, a.scale, rows, there, cols - col, c);
                } else {
                    store_rows<WHOLE, T, C, VM>(row<T>(a.gv, n, h, (int64_t)opaque(chunk) * C) + m0, (int)a.gv.sL, col, dv, a.scale, rows, there, cols - col, c);
                }
            }
        }
        lds_barrier();
    }
    if (first < stop && grades_decay) decay_gradients(first);

    // rows behind the sequence
    const int64_t t0 = (int64_t)max(stop, first) * C, t1 = min((int64_t)last * C, (int64_t)a.L);
    if (t0 < t1) {
        float *const pq = a.pq + ((((int64_t)(h % rq) * a.slices + slice) * a.N + n) * a.HQ + h / rq) * a.L * a.E;
        float *const pk = a.pk + ((((int64_t)(h % rk) * a.slices + slice) * a.N + n) * a.HK + h / rk) * a.L * a.E;
        float *const pv = a.pv + (((int64_t)(h % rv) * a.N + n) * a.HV + h / rv) * a.L * a.M + m0;
#pragma unroll 1
        for (int64_t i = t0 * E + tid; i < t1 * E; i += kThreads) {
            const int64_t t = i / E;
            const int e = i % E;
            if (e >= a.E) continue;
            if (a.pq) pq[t * a.E + e] = 0.f;
            else row<T>(a.gq, n, h, t)[e] = (T)0.f;
            if (a.pk) pk[t * a.E + e] = 0.f;
            else row<T>(a.gk, n, h, t)[e] = (T)0.f;
        }
#pragma unroll 1
        for (int64_t i = t0 * MS + tid; i < t1 * MS; i += kThreads) {
            const int64_t t = i / MS;
            const int m = i % MS;
            if (m >= mcols) continue;
            if (a.pv) pv[t * a.M + m] = 0.f;
            else row<T>(a.gv, n, h, t)[m0 + m] = (T)0.f;
        }
        if (!a.sum_decay)
            for (int64_t t = t0 + tid; t < t1; t += kThreads) a.gdecay[(((int64_t)slice * a.N + n) * a.H + h) * a.L + t] = 0.f;
    }
    if (a.sum_decay && grades_decay) {
        all = over_groups(over_sixteen(all));
        if (lane == 0) a.gdecay[(head * a.slices + slice) * a.segments + seg] = all;
    }
}

template <typename T, int NE, int NW, int MW, bool WHOLE>
__global__ __launch_bounds__((DsumBackward<T, NE, NW, MW>::kThreads), (DsumBackward<T, NE, NW, MW>::kWaves)) void k_dsum_bwd(const DsumWalk a) {
    using F = DsumBackward<T, NE, NW, MW>;
    __shared__ typename F::Shared sh;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    if constexpr (F::kBoth) {
        dsum_walk_back<true, true, T, NE, NW, MW, WHOLE>(a, sh, wave, tid);
    } else {
        if (wave < F::KW) dsum_walk_back<true, false, T, NE, NW, MW, WHOLE>(a, sh, wave, tid);
        else dsum_walk_back<false, true, T, NE, NW, MW, WHOLE>(a, sh, wave - F::KW, tid);
    }
}

// ------------------------------------------------------------------ launches

enum { kDsumForward, kDsumForwardEnds, kDsumBackward, kDsumBackwardEnds };

// Launches one of the four for states of Ep keys and slices of MS value columns, or with `a` NULL only says how many of its workgroups a CU holds at once; 0: there
// is no such kernel.
template <typename T>
int dsum_launch(int which, const DsumWalk *a, int Ep, int MS, unsigned blocks, hipStream_t s);

template <typename T, int NE, int NW, int MW, bool WHOLE>
int dsum_launch_one(int which, const DsumWalk *a, unsigned blocks, hipStream_t s) {
    using F = DsumForward<T, NE, NW, MW>;
    using B = DsumBackward<T, NE, NW, MW>;
    const dim3 grid(blocks), block(64 * NW);
    switch (which) {
        case kDsumForward:
            if (a) k_dsum_fwd<T, NE, NW, MW, WHOLE, false><<<grid, block, 0, s>>>(*a);
            return resident(sizeof(typename F::Shared), F::kWaves, NW);
        case kDsumForwardEnds:
            if (a) k_dsum_fwd<T, NE, NW, MW, WHOLE, true><<<grid, block, 0, s>>>(*a);
            return resident(sizeof(typename F::Ends), F::kEndWaves, NW);
        case kDsumBackward:
            if (a) k_dsum_bwd<T, NE, NW, MW, WHOLE><<<grid, dim3(B::kThreads), 0, s>>>(*a);
            return resident(sizeof(typename B::Shared), B::kWaves, B::kCount);
        default:
            if (a) k_dsum_bwd_ends<T, NE, NW, MW, WHOLE><<<grid, block, 0, s>>>(*a);
            return resident(sizeof(typename B::Ends), B::kEndWaves, NW);
    }
}

template <typename T, int NE>
int dsum_launch_keys(int which, const DsumWalk *a, int MS, unsigned blocks, hipStream_t s) {
    // all rows as wide as their tiles: nothing to cut off, and half the code
    const bool whole = a && a->E == 16 * NE && a->M % MS == 0;
    if (MS == 32) return whole ? dsum_launch_one<T, NE, 2, 1, true>(which, a, blocks, s) : dsum_launch_one<T, NE, 2, 1, false>(which, a, blocks, s);
    if (MS == 64) return whole ? dsum_launch_one<T, NE, 4, 1, true>(which, a, blocks, s) : dsum_launch_one<T, NE, 4, 1, false>(which, a, blocks, s);
    if (MS == 128) return whole ? dsum_launch_one<T, NE, 8, 1, true>(which, a, blocks, s) : dsum_launch_one<T, NE, 8, 1, false>(which, a, blocks, s);
    return 0;
}

#define FWP_DSUM_INSTANCES(T)                                                                            \
    template <>                                                                                          \
    int dsum_launch<T>(int which, const DsumWalk *a, int Ep, int MS, unsigned blocks, hipStream_t s) {   \
        if (Ep == 32) return dsum_launch_keys<T, 2>(which, a, MS, blocks, s);                            \
        if (Ep == 64) return dsum_launch_keys<T, 4>(which, a, MS, blocks, s);                            \
        if (Ep == 128) return dsum_launch_keys<T, 8>(which, a, MS, blocks, s);                           \
        return 0;                                                                                        \
    }

}  // namespace fwp
