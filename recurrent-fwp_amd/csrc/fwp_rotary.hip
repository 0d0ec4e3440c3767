// Rotary positions: the first 2 `pairs` channels of every row turn by an angle of the row's position, pair by pair.
//
//   (a, b) -> scale (a cos - b sin, a sin + b cos),  angle = position * frequency
//
// The angle of a far position has lost its fraction of a turn in 32 bits, so position * frequency and its remainder to a quarter of a turn are made in 64;
// what is left, at most pi / 4, goes through the series of sine and cosine, which end below 2^-27 there.  That costs some 40 instructions a pair, so a thread
// makes the angles of its pairs once and turns those of several heads by them.  Bound by memory: every row is read and written once, 16 bytes a lane.
// 32 x 8 + 8 heads of 1024 steps of 32 channels, fp32: 23 us (134 MB, in part cached); 32 + 8 heads of 32768 steps of 128 channels, bf16, 64 of them turning: 153 us at 4.4 TB/s.
#include <algorithm>

#include "fwp_elements.hpp"

namespace fwp {
namespace {

struct RotaryWalk {
    fwp_rotary_args a;
    fwp_out_rows oq, ok;
    int units, turning, groups, per;      // units of a row, those of them that turn; groups of heads, heads of a group
};

template <typename T>
struct Run {
    static constexpr int V = 16 / sizeof(T);
    typedef uint32_t Words __attribute__((ext_vector_type(4)));
    struct __attribute__((packed, aligned(sizeof(T)))) Anywhere { Words w; };
    struct Elements { T x[V]; };
    Words w;
    // elements c .. of a row.  WHOLE: all V are there, and no branch makes a load wait for the one before it; else those from `end` on are zero.
    template <bool WHOLE>
    __device__ __forceinline__ void load(const T *at, int c, int end) {
        if (WHOLE || c + V <= end) {
            w = reinterpret_cast<const Anywhere *>(at + c)->w;
        } else {
            Elements few;
#pragma unroll
            for (int i = 0; i < V; i++) few.x[i] = c + i < end ? at[c + i] : (T)0.f;
            w = __builtin_bit_cast(Words, few);
        }
    }
    __device__ __forceinline__ void get(float (&x)[V]) const {
        const Elements few = __builtin_bit_cast(Elements, w);
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = (float)few.x[i];
    }
    template <bool WHOLE>
    static __device__ __forceinline__ void store(const float (&x)[V], T *at, int c, int end) {
        Elements few;
#pragma unroll
        for (int i = 0; i < V; i++) few.x[i] = (T)x[i];
        if (WHOLE || c + V <= end) {
            reinterpret_cast<Anywhere *>(at + c)->w = __builtin_bit_cast(Words, few);
        } else {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (c + i < end) at[c + i] = few.x[i];
        }
    }
};

__device__ __forceinline__ void sine_cosine(double angle, float &s, float &c) {
    const double quarters = angle * 0.63661977236758134308, whole = rint(quarters);
    const float y = (float)((quarters - whole) * 1.57079632679489661923), z = y * y;
    float p = fmaf(z, 1.f / 362880, -1.f / 5040);
    p = fmaf(p, z, 1.f / 120);
    p = fmaf(p, z, -1.f / 6);
    const float sn = fmaf(p * z, y, y);
    p = fmaf(z, -1.f / 3628800, 1.f / 40320);
    p = fmaf(p, z, -1.f / 720);
    p = fmaf(p, z, 1.f / 24);
    p = fmaf(p, z, -0.5f);
    const float cs = fmaf(p, z, 1.f);
    const int q = (int)(whole - 4.0 * floor(whole * 0.25));      // 0 .. 3
    s = q & 1 ? cs : sn;
    c = q & 1 ? sn : cs;
    if (q & 2) s = -s;
    if (q == 1 || q == 2) c = -c;
}

// A thread has one unit of 2 V channels (V pairs, or as many of the channels that stay) of one step, for the heads of its group: those of q, then those of k.
// WHOLE: all units have all of their channels.
template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void k_rotary(const RotaryWalk w) {
    constexpr int V = 16 / sizeof(T), kAhead = 4;
    const fwp_rotary_args &a = w.a;
    int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int u = i % w.units;
    i /= w.units;
    const int t = i % a.L;
    i /= a.L;
    const int n = i % a.N, group = i / a.N;
    if (group >= w.groups) return;
    const bool counts = t < length_of(a.lengths, n, a.L), turns = u < w.turning;
    // the unit's channels: two runs of V
    int c0, c1, e0, e1;
    if (!turns) c0 = 2 * a.pairs + (u - w.turning) * 2 * V, c1 = c0 + V, e0 = e1 = a.D;
    else if (a.interleaved) c0 = u * 2 * V, c1 = c0 + V, e0 = e1 = 2 * a.pairs;
    else c0 = u * V, c1 = a.pairs + c0, e0 = a.pairs, e1 = 2 * a.pairs;
    if (!counts) {      // rows behind a sequence are not read: 8 x (32 + 8) heads of 4096 x 128, bf16, an eighth of them counting, 84 us, 127 where all do
        const float none[V] = {};
#pragma unroll 1
        for (int h = group * w.per; h < min((group + 1) * w.per, a.HQ + a.HK); h++) {
            T *to = h >= a.HQ ? row<T>(w.ok, n, h - a.HQ, t) : row<T>(w.oq, n, h, t);
            Run<T>::template store<WHOLE>(none, to, c0, e0), Run<T>::template store<WHOLE>(none, to, c1, e1);
        }
        return;
    }
    float sn[V], cs[V];
#pragma unroll
    for (int p = 0; p < V; p++) sn[p] = 0.f, cs[p] = 1.f;
    if (turns) {
        int64_t at = t;
        if (a.positions) at = a.each_step ? a.positions[(int64_t)n * a.L + t] : a.positions[n] + t;
        const double position = (double)at;
#pragma unroll
        for (int p = 0; p < V; p++) {
            sine_cosine(position * a.frequencies[min(u * V + p, a.pairs - 1)], sn[p], cs[p]);
            sn[p] *= a.inverse ? -a.scale : a.scale, cs[p] *= a.scale;
        }
    }
    const int last = min((group + 1) * w.per, a.HQ + a.HK);
    const auto source = [&](int h) { return h >= a.HQ ? row<T>(a.k, n, h - a.HQ, t) : row<T>(a.q, n, h, t); };
    for (int h = group * w.per; h < last; h += kAhead) {
        Run<T> x[kAhead], y[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const T *from = source(min(h + j, last - 1));
            x[j].template load<WHOLE>(from, c0, e0), y[j].template load<WHOLE>(from, c1, e1);
        }
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            if (h + j >= last) break;
            T *to = h + j >= a.HQ ? row<T>(w.ok, n, h + j - a.HQ, t) : row<T>(w.oq, n, h + j, t);
            float p0[V], p1[V], r0[V], r1[V];
            x[j].get(p0), y[j].get(p1);
            if (!turns) {
#pragma unroll
                for (int p = 0; p < V; p++) r0[p] = p0[p], r1[p] = p1[p];
            } else if (a.interleaved) {
#pragma unroll
                for (int p = 0; p < V; p += 2) {
                    r0[p] = fmaf(p0[p], cs[p / 2], -(p0[p + 1] * sn[p / 2])), r0[p + 1] = fmaf(p0[p], sn[p / 2], p0[p + 1] * cs[p / 2]);
                    r1[p] = fmaf(p1[p], cs[(V + p) / 2], -(p1[p + 1] * sn[(V + p) / 2])), r1[p + 1] = fmaf(p1[p], sn[(V + p) / 2], p1[p + 1] * cs[(V + p) / 2]);
                }
            } else {
#pragma unroll
                for (int p = 0; p < V; p++) r0[p] = fmaf(p0[p], cs[p], -(p1[p] * sn[p])), r1[p] = fmaf(p0[p], sn[p], p1[p] * cs[p]);
            }
            Run<T>::template store<WHOLE>(r0, to, c0, e0), Run<T>::template store<WHOLE>(r1, to, c1, e1);
        }
    }
}

}  // namespace

int rotary(const fwp_rotary_args &a, fwp_out_rows oq, fwp_out_rows ok, hipStream_t s) {
    RotaryWalk w{a, oq, ok};
    const int V = a.type == FWP_F32 ? 4 : 8, heads = a.HQ + (a.k.ptr ? a.HK : 0);
    if (!a.k.ptr) w.a.HK = 0;
    w.turning = (a.pairs + V - 1) / V;
    w.units = w.turning + (a.D - 2 * a.pairs + 2 * V - 1) / (2 * V);
    const int64_t rows = (int64_t)a.N * a.L * w.units;
    // all heads to a thread where there are threads enough: 2048 of them on each of 256 CUs
    w.groups = (int)std::min<int64_t>(heads, std::max<int64_t>(1, ((int64_t)1 << 19) / rows));
    w.per = (heads + w.groups - 1) / w.groups;
    w.groups = (heads + w.per - 1) / w.per;
    const int64_t blocks = (rows * w.groups + 255) / 256;
    if (!fits_launch(blocks, 256)) return FWP_E_SHAPE;
    const bool whole = a.pairs % V == 0 && (a.D - 2 * a.pairs) % (2 * V) == 0;
    by_type(a.type, [&](auto t) {
        if (whole) k_rotary<decltype(t), true><<<(unsigned)blocks, 256, 0, s>>>(w);
        else k_rotary<decltype(t), false><<<(unsigned)blocks, 256, 0, s>>>(w);
    });
    return (int)hipGetLastError();
}

}  // namespace fwp
