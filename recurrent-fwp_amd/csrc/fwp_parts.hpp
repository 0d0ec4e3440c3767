// Tiles of rows in LDS as sums of bfloat16 parts, and products of such sums on the matrix cores.
//
// An fp32 number is the sum of three bfloat16 numbers (8 significant bits each), an fp16 number that of two, and a product of two sums
// keeps the pairs of parts whose orders add up to less than a stated number: three orders leave out 2^-24 of a product, two 2^-16.  The 16-bit
// products run at 16 times the rate of v_mfma_f32_16x16x4_f32, so six of them are 2.7 times as fast as one fp32 product, and every type takes
// the same path.
//
// Fragments of v_mfma_f32_16x16x32_bf16, lane l = 16 g + c: an operand holds, for its row (A) or column (B) c, the summation indexes 8 g .. 8 g + 7; a
// result holds rows 4 g .. 4 g + 3 of column c.  Two results whose rows stand for the indexes 8 g + i and 8 g + 4 + i are therefore an operand of the next
// product as they are: nothing moves between lanes.  place() gives such an order to the 16 rows of each of `tiles` results.
#pragma once
#include <type_traits>

#include "fwp_elements.hpp"
#include "fwp_mfma.hpp"

namespace fwp {

typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef __bf16 v4b __attribute__((ext_vector_type(4)));
typedef short v4h __attribute__((ext_vector_type(4)));

// bfloat16 parts that hold a row element of this type whole
template <typename T>
constexpr int kPartsOf = std::is_same_v<T, bf16_t> ? 1 : std::is_same_v<T, half_t> ? 2 : 3;
// In place of parts: fp32 numbers as they are, and v_mfma_f32_16x16x4_f32, eight for 32 summation indexes of the same fragments
constexpr int kPlain = 0;

template <int P>
struct Frag {
    v8b p[P];
};
template <>
struct Frag<kPlain> {
    float x[8];
};

// Two numbers' next parts, rounded to nearest even, in one register; what they leave goes on in a and b.
__device__ __forceinline__ uint32_t next_parts(float &a, float &b, bool last) {
    typedef float v2f __attribute__((ext_vector_type(2)));
    typedef __bf16 v2b __attribute__((ext_vector_type(2)));
    const uint32_t u = __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{a, b}), v2b));
    if (!last) a -= __uint_as_float(u << 16), b -= __uint_as_float(u & 0xffff0000u);
    return u;
}

// x[i] as the sum of P parts: each takes what the ones before it left, which is exact.
template <int P, int W, typename V>
__device__ __forceinline__ void split(const float (&x)[W], V (&out)[P]) {
    struct Words { uint32_t w[W / 2]; };
    Words words[P];
#pragma unroll
    for (int i = 0; i < W; i += 2) {
        float a = x[i], b = x[i + 1];
#pragma unroll
        for (int p = 0; p < P; p++) words[p].w[i / 2] = next_parts(a, b, p + 1 == P);
    }
#pragma unroll
    for (int p = 0; p < P; p++) out[p] = __builtin_bit_cast(V, words[p]);
}

template <int P>
__device__ __forceinline__ Frag<P> split8(const float (&x)[8]) {
    Frag<P> f;
    if constexpr (P == kPlain) {
#pragma unroll
        for (int i = 0; i < 8; i++) f.x[i] = x[i];
    } else {
        split<P, 8>(x, f.p);
    }
    return f;
}

template <int P>
__device__ __forceinline__ Frag<P> split8(const v4f &lo, const v4f &hi) {
    const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return split8<P>(x);
}

template <int P>
__device__ __forceinline__ void join8(const Frag<P> &f, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if constexpr (P == kPlain) {
            x[i] = f.x[i];
        } else {
            x[i] = (float)f.p[P - 1][i];
#pragma unroll
            for (int p = P - 2; p >= 0; p--) x[i] += (float)f.p[p][i];
        }
    }
}

// Zero if the eight numbers are finite, else NaN
template <int P>
__device__ __forceinline__ float unless_finite(const Frag<P> &f, float acc) {
    if constexpr (P == kPlain) {
#pragma unroll
        for (int i = 0; i < 8; i++) acc = fmaf(f.x[i], 0.f, acc);
    } else {
        typedef __bf16 v2b __attribute__((ext_vector_type(2)));
        struct { v2b p[4]; } pairs = __builtin_bit_cast(decltype(pairs), f.p[0]);
#pragma unroll
        for (int i = 0; i < 4; i++) acc = __builtin_amdgcn_fdot2_f32_bf16(pairs.p[i], v2b{0, 0}, acc, false);
    }
    return acc;
}

// Takes what is not finite for zero; found(i) for each
template <int P, typename Found>
__device__ __forceinline__ void take_out(Frag<P> &f, Found found) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if constexpr (P == kPlain) {
            if (!(fmaf(f.x[i], 0.f, 0.f) == 0.f)) found(i), f.x[i] = 0.f;
        } else {
            if (!((float)f.p[0][i] * 0.f == 0.f)) {
                found(i);
#pragma unroll
                for (int p = 0; p < P; p++) f.p[p][i] = (__bf16)0.f;
            }
        }
    }
}

// acc + A B over 32 summation indexes, pairs of parts of orders below ORDERS
template <int ORDERS, int PA, int PB>
__device__ __forceinline__ v4f product(const Frag<PA> &a, const Frag<PB> &b, v4f acc) {
    if constexpr (PA == kPlain) {
#pragma unroll
        for (int i = 0; i < 8; i++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x[i], b.x[i], acc, 0, 0, 0);
        return acc;
    } else
#pragma unroll
    for (int i = 0; i < PA; i++)
#pragma unroll
        for (int j = 0; j < PB; j++)
            if (i + j < ORDERS) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[j], acc, 0, 0, 0);
    return acc;
}

// N steps, each with what load(i) reads from LDS, whose reads are issued D steps ahead: left to itself the compiler puts a read right before its use and waits for it, some
// 130 cycles for three products of 16.  The steps' numbers are constants.
template <int N, int D, typename Load, typename Use>
__device__ __forceinline__ void ahead(Load load, Use use) {
    decltype(load(0)) f[D + 1];
#pragma unroll
    for (int i = 0; i < D && i < N; i++) f[i] = load(i);
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (i + D < N) f[(i + D) % (D + 1)] = load(i + D);
        __builtin_amdgcn_sched_barrier(0);
        use(i, f[i % (D + 1)]);
    }
}
// How far ahead: what P parts leave of the registers
template <int P>
constexpr int kAhead = P == 1 ? 3 : P == 2 ? 2 : P == kPlain ? 2 : 1;

// Row (or column) a of the j-th of `tiles` results that lie side by side: four consecutive numbers a lane, 4 * tiles in a row of them.
__device__ __forceinline__ constexpr int place(int tiles, int a, int j) { return 4 * tiles * (a / 4) + 4 * j + a % 4; }

// R rows of W elements as P parts.  The 16-byte runs of a row lie in an order of its own: run q of row r is at q ^ key(r), so that every access below meets all banks evenly:
// the same run of 16 rows, one run after another of a row, and four neighbouring runs of rows 4 i .. 4 i + 3.
template <int R, int W, int P>
struct alignas(16) Tile {
    static_assert(W == 32 || W == 64 || W == 128, "row lengths that key() spreads");
    static constexpr int kPart = R * W;
    __bf16 x[P * kPart];

    // rows that share their banks' place (W / 32 of four, two or one) differ here, rows 4 i .. 4 i + 3 by whole groups of four runs
    static __device__ __forceinline__ int key(int r) {
        if constexpr (W == 32) return r / 4 % 4;
        else if constexpr (W == 64) return r / 2 % 2 * 4 + r / 4 % 2 + r / 8 % 2 * 2;
        else return r % 4 * 4 + r / 4 % 4;
    }
    static __device__ __forceinline__ int place_of(int r, int col) { return r * W + (((col >> 3) ^ key(r)) << 3) + (col & 7); }

    __device__ __forceinline__ void put(int p, int r, int col, const v8b &v) { *reinterpret_cast<v8b *>(&x[p * kPart + place_of(r, col)]) = v; }
    __device__ __forceinline__ void put(int r, int col, const float (&f)[8]) {
        const Frag<P> s = split8<P>(f);
#pragma unroll
        for (int p = 0; p < P; p++) put(p, r, col, s.p[p]);
    }
    __device__ __forceinline__ void put4(int r, int col, const float (&f)[4]) {
        v4b s[P];
        split<P, 4>(f, s);
#pragma unroll
        for (int p = 0; p < P; p++) *reinterpret_cast<v4b *>(&x[p * kPart + place_of(r, col)]) = s[p];
    }

    // rows r0 .. r0 + 15 against columns k0 .. k0 + 31 as they lie; r0 is a multiple of 16, k0 of 32
    __device__ __forceinline__ Frag<P> rows(int r0, int k0, int g, int c) const {
        const int at = c * W + (((g ^ key(c)) << 3) ^ k0) + r0 * W;
        Frag<P> f;
#pragma unroll
        for (int p = 0; p < P; p++) f.p[p] = *reinterpret_cast<const v8b *>(&x[p * kPart + at]);
        return f;
    }
    // columns c0 + place(TILES, c, j) against rows k0 .. k0 + 31; c0 is a multiple of 16 TILES, k0 of 32.  ds_read_b64_tr_b16: each lane names four elements, the 16 lanes of
    // a group four rows of 16, and lane c of the group gets the four rows' c-th.
    template <int TILES>
    __device__ __forceinline__ Frag<P> columns(int c0, int j, int k0, int g, int c) const {
        typedef __attribute__((address_space(3))) v4h *lds4;
        const int r = 8 * g + c / 4, col = 4 * TILES * (c % 4) + 4 * j;
        const int lo = r * W + ((((col >> 3) ^ key(r)) << 3) ^ c0) + (col & 7) + k0 * W, hi = lo + 4 * W + ((((col >> 3) ^ key(r + 4)) << 3) ^ c0) - ((((col >> 3) ^ key(r)) << 3) ^ c0);
        Frag<P> f;
#pragma unroll
        for (int p = 0; p < P; p++) {
            const v4h a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)&x[p * kPart + lo]), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)&x[p * kPart + hi]);
            const v4b l = __builtin_bit_cast(v4b, a), h = __builtin_bit_cast(v4b, b);
            f.p[p] = v8b{l[0], l[1], l[2], l[3], h[0], h[1], h[2], h[3]};
        }
        return f;
    }
    // four elements of a row, summed up again
    __device__ __forceinline__ v4f four(int r, int col) const {
        v4f s = {0, 0, 0, 0};
#pragma unroll
        for (int p = P - 1; p >= 0; p--) {
            const v4b v = *reinterpret_cast<const v4b *>(&x[p * kPart + place_of(r, col)]);
#pragma unroll
            for (int i = 0; i < 4; i++) s[i] += (float)v[i];
        }
        return s;
    }
};

template <int R, int W>
struct alignas(16) Tile<R, W, kPlain> {
    static constexpr int kStride = W + 4;
    float x[R * kStride];

    __device__ __forceinline__ void put(int r, int col, const float (&f)[8]) {
        *reinterpret_cast<v4f *>(&x[r * kStride + col]) = v4f{f[0], f[1], f[2], f[3]};
        *reinterpret_cast<v4f *>(&x[r * kStride + col + 4]) = v4f{f[4], f[5], f[6], f[7]};
    }
    __device__ __forceinline__ void put4(int r, int col, const float (&f)[4]) { *reinterpret_cast<v4f *>(&x[r * kStride + col]) = v4f{f[0], f[1], f[2], f[3]}; }
    __device__ __forceinline__ Frag<kPlain> rows(int r0, int k0, int g, int c) const {
        const v4f a = four(r0 + c, k0 + 8 * g), b = four(r0 + c, k0 + 8 * g + 4);
        return {{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}};
    }
    template <int TILES>
    __device__ __forceinline__ Frag<kPlain> columns(int c0, int j, int k0, int g, int c) const {
        Frag<kPlain> f;
#pragma unroll
        for (int i = 0; i < 8; i++) f.x[i] = x[(k0 + 8 * g + i) * kStride + c0 + place(TILES, c, j)];
        return f;
    }
    __device__ __forceinline__ v4f four(int r, int col) const { return *reinterpret_cast<const v4f *>(&x[r * kStride + col]); }
};

// Element i of memory that starts at an address all lanes share: a 32-bit offset of bytes, which costs no 64-bit sum
template <typename T>
__device__ __forceinline__ T *from(T *base, uint32_t i) {
    using Byte = std::conditional_t<std::is_const_v<T>, const char, char>;
    return reinterpret_cast<T *>(reinterpret_cast<Byte *>(base) + (uint32_t)(i * (uint32_t)sizeof(T)));
}

// A block of R rows of up to W elements on its way from memory to a Tile: load() starts the loads, put() converts and writes what they brought.  Rows from
// `rows` on and columns from `cols` on are not read and become zero; at least one row is there.  Every lane loads 16 bytes at an element's address (the
// hardware takes any), those beyond the block's rows the last row, those beyond its columns the last eight: a branch around a load would wait for
// it at its end, and there would be no loads ahead.  put() zeroes and shifts what was read from elsewhere.
template <typename T, int R, int W, int THREADS, bool WHOLE>
struct Stage {
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
    static constexpr int kRow = W / 8, kVecs = R * kRow, kPer = (kVecs + THREADS - 1) / THREADS, kRegs = sizeof(T) / 2;
    struct Eight {
        v4u x[kRegs];
    };
    struct __attribute__((packed, aligned(sizeof(T)))) Anywhere {
        Eight e;
    };
    Eight x[kPer];

    // base: the block's first row, the same for all lanes; R rows lie within 32 bits of bytes
    __device__ __forceinline__ void load(const T *base, int stride, int rows, int cols, int tid) {
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int v = tid + i * THREADS, r = min(v / kRow, min(rows, R) - 1), col = v % kRow * 8;
            if (WHOLE) {
                x[i] = reinterpret_cast<const Anywhere *>(from(base, (uint32_t)r * (uint32_t)stride + (uint32_t)col))->e;
            } else if (cols >= 8) {
                x[i] = reinterpret_cast<const Anywhere *>(from(base, (uint32_t)r * (uint32_t)stride + (uint32_t)min(col, cols - 8)))->e;
            } else {
                struct { T e[8]; } few;
#pragma unroll
                for (int e = 0; e < 8; e++) few.e[e] = *from(base, (uint32_t)r * (uint32_t)stride + (uint32_t)min(e, cols - 1));
                x[i] = __builtin_bit_cast(Eight, few);
            }
        }
    }
    // Waits for the loads.  The counter of outstanding accesses runs in order over loads and stores, and the compiler does not count over branches: a load that is still
    // waited for behind a kernel's stores waits for them too, some 2 us.
    __device__ __forceinline__ void arrive() {
#pragma unroll
        for (int i = 0; i < kPer; i++)
#pragma unroll
            for (int r = 0; r < kRegs; r++) asm volatile("" : "+v"(x[i].x[r]));
    }
    template <int P>
    __device__ __forceinline__ void put(Tile<R, W, P> &t, int rows, int cols, int tid) const {
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int v = tid + i * THREADS, r = v / kRow, col = v % kRow * 8;
            if (kVecs % THREADS && v >= kVecs) continue;
            const bool some = r < rows && (WHOLE || col < cols);
            if constexpr (P == 1)
                if (WHOLE || cols % 8 == 0) {
                    t.put(0, r, col, __builtin_bit_cast(v8b, some ? x[i].x[0] : v4u{0, 0, 0, 0}));
                    continue;
                }
            struct Few { T e[8]; };
            const Few few = __builtin_bit_cast(Few, x[i]);
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] = some ? (float)few.e[e] : 0.f;
            if (!WHOLE && cols % 8) {
                if (cols >= 8) {      // the last run of a row holds its last eight elements
                    const int late = max(0, col - (cols - 8));
#pragma unroll
                    for (int b = 1; b < 8; b *= 2)
#pragma unroll
                        for (int e = 0; e < 8; e++) f[e] = late & b ? (e + b < 8 ? f[e + b] : 0.f) : f[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) f[e] = e < cols ? f[e] : 0.f;
                }
            }
            t.put(r, col, f);
        }
    }
};

}  // namespace fwp
