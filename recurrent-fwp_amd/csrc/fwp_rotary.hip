// Rotary positions: the first 2 `pairs` channels of every row turn by an angle of the row's position, pair by pair.
//
//   (a, b) -> scale (a cos - b sin, a sin + b cos),  angle = position * frequency
//
// The angle of a far position has lost its fraction of a turn in 32 bits, so position * frequency and its remainder to a quarter of a turn are made in 64;
// what is left, at most pi / 4, goes through the series of sine and cosine, which end below 2^-27 there.  That costs some 40 instructions a pair, so a thread
// makes the angles of its pairs once and turns those of several heads by them.  Bound by memory: every row is read and written once, 16 bytes a lane.
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
struct __attribute__((packed, aligned(sizeof(T)))) Vec {
    T x[16 / sizeof(T)];
};

// elements [c, c + V) of a row, those below `end`
template <typename T, int V>
__device__ __forceinline__ void load_some(float (&x)[V], const T *at, int c, int end) {
    if (c + V <= end) {
        const Vec<T> v = *reinterpret_cast<const Vec<T> *>(at + c);
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = (float)v.x[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = c + i < end ? (float)at[c + i] : 0.f;
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_some(const float (&x)[V], T *at, int c, int end) {
    if (c + V <= end) {
        Vec<T> v;
#pragma unroll
        for (int i = 0; i < V; i++) v.x[i] = (T)x[i];
        *reinterpret_cast<Vec<T> *>(at + c) = v;
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (c + i < end) at[c + i] = (T)x[i];
    }
}

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
template <typename T>
__global__ __launch_bounds__(256) void k_rotary(const RotaryWalk w) {
    constexpr int V = 16 / sizeof(T);
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
    float sn[V], cs[V];
    if (turns && counts) {
        int64_t at = t;
        if (a.positions) at = a.each_step ? a.positions[(int64_t)n * a.L + t] : a.positions[n] + t;
        const double position = (double)at;
#pragma unroll
        for (int p = 0; p < V; p++) {
            const int pair = u * V + p;
            sine_cosine(pair < a.pairs ? position * a.frequencies[pair] : 0.0, sn[p], cs[p]);
            sn[p] *= a.inverse ? -a.scale : a.scale, cs[p] *= a.scale;
        }
    }
    const int last = min((group + 1) * w.per, a.HQ + a.HK);
#pragma unroll 4
    for (int h = group * w.per; h < last; h++) {
        const bool key = h >= a.HQ;
        const T *from = row<T>(key ? a.k : a.q, n, key ? h - a.HQ : h, t);
        T *to = row<T>(key ? w.ok : w.oq, n, key ? h - a.HQ : h, t);
        float x[V], y[V];
#pragma unroll
        for (int p = 0; p < V; p++) x[p] = y[p] = 0.f;
        if (counts) load_some<T, V>(x, from, c0, e0), load_some<T, V>(y, from, c1, e1);
        if (turns && counts) {
            if (a.interleaved) {
                float r[2 * V];
#pragma unroll
                for (int p = 0; p < V; p++) {
                    const float p0 = p < V / 2 ? x[2 * p % V] : y[2 * p % V], p1 = p < V / 2 ? x[2 * p % V + 1] : y[2 * p % V + 1];
                    r[2 * p] = fmaf(p0, cs[p], -(p1 * sn[p])), r[2 * p + 1] = fmaf(p0, sn[p], p1 * cs[p]);
                }
#pragma unroll
                for (int p = 0; p < V; p++) x[p] = r[p], y[p] = r[V + p];
            } else {
#pragma unroll
                for (int p = 0; p < V; p++) {
                    const float p0 = x[p], p1 = y[p];
                    x[p] = fmaf(p0, cs[p], -(p1 * sn[p])), y[p] = fmaf(p0, sn[p], p1 * cs[p]);
                }
            }
        }
        store_some<T, V>(x, to, c0, e0), store_some<T, V>(y, to, c1, e1);
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
    by_type(a.type, [&](auto t) { k_rotary<decltype(t)><<<(unsigned)blocks, 256, 0, s>>>(w); });
    return (int)hipGetLastError();
}

}  // namespace fwp
