// Rotary positions on eight neighbouring columns of a row, shared by the rotary and the append kernels.
//
// Columns i < R of a row turn in pairs: (i, i + R / 2), or neighbours (2 i, 2 i + 1) where interleaved. A pair
// (x1, x2) at position p becomes (x1 c - x2 s, x2 c + x1 s) with c = cos[p][i], s = sin[p][i]; its gradient is the
// same with -s. Column by column that is y = x c + x' s', x' the other column of the pair and s' = -s or s: products
// and sum are rounded one by one in fp32 (as separate operators round them), the result once to the row's type.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace ktt {

// Tables and layout of a rotation, as the kernels read them.
struct Turn {
    const float* cos;   // null: nothing turns
    const float* sin;
    int64_t stride;     // fp32 values from a position's row to the next
    int64_t rows;
    int half;           // R / 2
    int interleaved;
    int inverse;
};

template <typename T>
__device__ __forceinline__ float to_f32(T x) { return static_cast<float>(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Two fp32 values that one instruction works on, each rounded as by itself; but a product and a sum behind it are joined into
// one rounding by the compiler, whatever the instructions say, so what rounds them one by one stays with __fmul_rn and __fadd_rn.
struct Pair {
    unsigned long long v;
    __device__ __forceinline__ Pair() {}
    __device__ __forceinline__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ explicit Pair(float a) : Pair(a, a) {}
    __device__ __forceinline__ float low() const { return __uint_as_float(static_cast<uint32_t>(v)); }
    __device__ __forceinline__ float high() const { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
};
__device__ __forceinline__ Pair operator*(const Pair& a, const Pair& b) {
    Pair c;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(c.v) : "l"(a.v), "l"(b.v));
    return c;
}
__device__ __forceinline__ Pair operator+(const Pair& a, const Pair& b) {
    Pair c;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(c.v) : "l"(a.v), "l"(b.v));
    return c;
}
__device__ __forceinline__ Pair sub(const Pair& a, const Pair& b) {
    Pair c;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(c.v) : "l"(a.v), "l"(b.v));
    return c;
}
__device__ __forceinline__ Pair fma(const Pair& a, const Pair& b, const Pair& c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}

// Eight values in 16-byte pieces (one of 16-bit types, two of fp32).
template <typename T>
struct Eight {
    static constexpr int kPieces = static_cast<int>(8 * sizeof(T) / 16);
    uint4 raw[kPieces];
    __device__ __forceinline__ T get(int e) const { return reinterpret_cast<const T*>(raw)[e]; }
    __device__ __forceinline__ void set(int e, T x) { reinterpret_cast<T*>(raw)[e] = x; }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) raw[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void store(T* p) const {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) reinterpret_cast<uint4*>(p)[i] = raw[i];
    }
    // The n first values one by one (any alignment).
    __device__ __forceinline__ void load_some(const T* p, int n) {
#pragma unroll
        for (int e = 0; e < 8; ++e) set(e, e < n ? p[e] : from_f32<T>(0.f));
    }
    __device__ __forceinline__ void store_some(T* p, int n) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e < n) p[e] = get(e);
        }
    }
};

// The turn of columns [col, col + 8) at one position: kept in registers over the heads of a token.
// kFast: the columns all turn or none does, their partners are eight neighbours too, and table rows are read in
// 16-byte pieces.
template <bool kFast>
struct Turned {
    float c[8], s[8];
    int partner;     // kFast: column of the first partner (half layout), or -1: in the same eight columns
    int count;       // columns of the eight that turn

    __device__ __forceinline__ void load(const Turn& t, int64_t position, int col) {
        const int part = t.cos ? 2 * t.half : 0;
        count = min(max(part - col, 0), 8);
        partner = -1;
        if (count == 0) return;
        position = position < 0 ? 0 : (position >= t.rows ? t.rows - 1 : position);
        const float* cr = t.cos + position * t.stride;
        const float* sr = t.sin + position * t.stride;
        const float flip = t.inverse ? -1.f : 1.f;
        if (kFast) {
            if (t.interleaved) {
                const float4 a = *reinterpret_cast<const float4*>(cr + col / 2), b = *reinterpret_cast<const float4*>(sr + col / 2);
                const float cs[4] = {a.x, a.y, a.z, a.w}, sn[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    c[e] = cs[e >> 1];
                    s[e] = (e & 1 ? flip : -flip) * sn[e >> 1];
                }
            } else {
                const bool low = col < t.half;
                const int at = low ? col : col - t.half;
                partner = low ? col + t.half : at;
                const float sign = low ? -flip : flip;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float4 a = *reinterpret_cast<const float4*>(cr + at + 4 * i), b = *reinterpret_cast<const float4*>(sr + at + 4 * i);
                    c[4 * i] = a.x; c[4 * i + 1] = a.y; c[4 * i + 2] = a.z; c[4 * i + 3] = a.w;
                    s[4 * i] = sign * b.x; s[4 * i + 1] = sign * b.y; s[4 * i + 2] = sign * b.z; s[4 * i + 3] = sign * b.w;
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int i = col + e;
                const bool low = t.interleaved ? !(i & 1) : i < t.half;
                const int at = t.interleaved ? i >> 1 : (low ? i : i - t.half);
                c[e] = e < count ? cr[at] : 1.f;
                s[e] = e < count ? (low ? -flip : flip) * sr[at] : 0.f;
            }
        }
    }

    // x: columns [col, col + 8) of a row of d columns that starts at `row`.
    template <typename T>
    __device__ __forceinline__ void apply(const Turn& t, Eight<T>& x, const Eight<T>& other, const T* row, int col) const {
        if (count == 0) return;
        const Eight<T> old = x;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float p;
            if (t.interleaved) p = to_f32(old.get(e ^ 1));
            else if (kFast) p = to_f32(other.get(e));
            else p = e < count ? to_f32(row[col + e < t.half ? col + e + t.half : col + e - t.half]) : 0.f;
            // A column that does not turn is copied, whatever its neighbours hold.
            if (kFast || e < count) x.set(e, from_f32<T>(__fadd_rn(__fmul_rn(to_f32(old.get(e)), c[e]), __fmul_rn(p, s[e]))));
        }
    }
};

// Whether Turned<true> may be used for columns of rows like these.
inline bool turn_is_fast(const Turn& t) {
    if (!t.cos) return true;
    if ((t.interleaved ? 2 * t.half : t.half) % 8) return false;
    return t.stride % 4 == 0 && ((reinterpret_cast<uintptr_t>(t.cos) | reinterpret_cast<uintptr_t>(t.sin)) & 15) == 0;
}

}  // namespace ktt
