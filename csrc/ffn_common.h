// Shared by the feed-forward operators (layernorm.hip, linear.hip): types of
// 16 and 32 bits behind one name, 16-byte chunks at any alignment, the
// activations with their slopes, and the 8-bit form of an activation.
#pragma once
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

enum Act { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

// values of a row that share one scale in the 8-bit form
#define ACT8_GROUP 128
// under this largest magnitude 127 / a overflows: such a group is kept as zeros
#define ACT8_LEAST 0x1p-119f

// ---- chunks of 8 values ----------------------------------------------------
// Rows of odd length start at any multiple of the type's size; the vector
// types below say so, and gfx950 takes such addresses in one instruction.
template <typename T> struct Chunk;
template <> struct Chunk<bf16_t> {
    typedef bf16_t V __attribute__((ext_vector_type(8), aligned(2)));
};
template <> struct Chunk<f16_t> {
    typedef f16_t V __attribute__((ext_vector_type(8), aligned(2)));
};
template <> struct Chunk<float> {
    typedef float V __attribute__((ext_vector_type(8), aligned(4)));
};
typedef signed char i8x8 __attribute__((ext_vector_type(8), aligned(1)));

// `left` values are there (1..8); the others read as 0 and are not written
template <typename T>
__device__ __forceinline__ void load8(const T* p, int left, float* v) {
    if (left >= 8) {
        const typename Chunk<T>::V c =
            *reinterpret_cast<const typename Chunk<T>::V*>(p);
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)c[i];
    } else {
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? (float)p[i] : 0.0f;
    }
}

// E values from column c of a row of `dim`, as they lie in memory, for rows that
// may end inside a chunk: nothing branches between the load and its use, so that
// many are on their way at once.  Where the chunk ends past the row, its last E
// values come instead, and settle() moves them; `c` may lie past the row.
template <typename V, int E, typename T>
__device__ __forceinline__ V fetch(const T* row, int c, int dim) {
    if (dim >= E)
        return *reinterpret_cast<const V*>(row + (c < dim - E ? c : dim - E));
    V v;
    #pragma unroll
    for (int i = 0; i < E; ++i) v[i] = i < dim ? row[i] : (T)0.0f;
    return v;
}
template <typename T>
__device__ __forceinline__ typename Chunk<T>::V fetch8(const T* row, int c,
                                                       int dim) {
    return fetch<typename Chunk<T>::V, 8>(row, c, dim);
}

// What fetch() brought, with the columns where they belong and zeros in those that
// are not there: shifted down as a whole, and only where a lane's chunk ends past
// the row (done on single values by all lanes, this took as long as the rest of
// the norm).
template <int E, typename V>
__device__ __forceinline__ V settle(V raw, int c, int dim) {
    constexpr int W = sizeof(V) / 4, SZ = sizeof(V) / E;
    const int over = dim >= E ? c - (dim - E) : c;
    if (!__any(over > 0)) return raw;
    const int by = over <= 0 ? 0 : over < E && dim >= E ? over * SZ : E * SZ;
    union { V v; unsigned d[W]; } u;
    u.v = raw;
    #pragma unroll
    for (int b = SZ; b < 4; b *= 2)
        #pragma unroll
        for (int i = 0; i < W; ++i)
            u.d[i] = by & b
                ? __builtin_amdgcn_alignbyte(i + 1 < W ? u.d[i + 1] : 0u,
                                             u.d[i], b)
                : u.d[i];
    #pragma unroll
    for (int b = SZ < 4 ? 4 : SZ; b < E * SZ; b *= 2)
        #pragma unroll
        for (int i = 0; i < W; ++i)
            u.d[i] = by & b ? (i + b / 4 < W ? u.d[i + b / 4] : 0u) : u.d[i];
    #pragma unroll
    for (int i = 0; i < W; ++i) u.d[i] = by == E * SZ ? 0u : u.d[i];
    return u.v;
}

// `whole`: no lane's chunk ends past the row (the same for all lanes)
template <typename V>
__device__ __forceinline__ void unpack8(V raw, int c, int dim, bool whole,
                                        float* v) {
    if (!whole) raw = settle<8>(raw, c, dim);
    #pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)raw[i];
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int left, const float* v) {
    if (left >= 8) {
        typename Chunk<T>::V c;
        #pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = (T)v[i];
        *reinterpret_cast<typename Chunk<T>::V*>(p) = c;
    } else {
        #pragma unroll
        for (int i = 0; i < 8; ++i) if (i < left) p[i] = (T)v[i];
    }
}

__device__ __forceinline__ void load8_codes(const signed char* p, int left,
                                            float* v) {
    if (left >= 8) {
        const i8x8 c = *reinterpret_cast<const i8x8*>(p);
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)c[i];
    } else {
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? (float)p[i] : 0.0f;
    }
}

// ---- 8-bit form ------------------------------------------------------------
// c = rint(x * fl(127 / a)), s = fl(a * fl(1 / 127)), a = max |x| of the
// group.  x * fl(127 / a) is at most 127 (1 + 2^-23), so rint never leaves
// [-127, 127].  A group with an infinity or a NaN gets s = NaN and codes 0:
// all of it reads as NaN, so a broken activation shows in the gradients.
struct Act8Scale { float by, scale; };

// the group's largest magnitude comes as the bits of |x|, which order as the
// values do, infinities and then NaN at the end
__device__ __forceinline__ Act8Scale act8_scale(unsigned bits) {
    Act8Scale s;
    const float a = __uint_as_float(bits);
    const bool finite = bits < 0x7f800000u;
    const bool some = finite && a >= ACT8_LEAST;
    s.by = some ? 127.0f / a : 0.0f;
    s.scale = !finite ? __builtin_nanf("")
                      : some ? a * (1.0f / 127.0f) : 0.0f;
    return s;
}

// largest magnitude of 8 values, as bits
__device__ __forceinline__ unsigned max8(const float* v) {
    unsigned a = 0;
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned m = __float_as_uint(v[i]) & 0x7fffffffu;
        a = a > m ? a : m;
    }
    return a;
}

// rint by adding 1.5 * 2^23, which leaves the integer in the low bits: the same
// for products up to 127 (1 + 2^-23); the bytes are then picked, four to a word
__device__ __forceinline__ void store8_codes(signed char* p, int left,
                                             const float* v, float by) {
    // the product rounds by itself, by definition: no fma
    #pragma clang fp contract(off)
    unsigned q[8], w[2];
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = v[i] * by;
        q[i] = __float_as_uint(x + 12582912.0f);
    }
    #pragma unroll
    for (int h = 0; h < 2; ++h) {
        const unsigned lo = __builtin_amdgcn_perm(q[4 * h + 1], q[4 * h],
                                                  0x0c0c0400u);
        const unsigned hi = __builtin_amdgcn_perm(q[4 * h + 3], q[4 * h + 2],
                                                  0x04000c0cu);
        // groups of zeros, and those that are not finite
        w[h] = by == 0.0f ? 0u : lo | hi;
    }
    if (left >= 8) {
        typedef unsigned V __attribute__((ext_vector_type(2), aligned(1)));
        V c;
        c[0] = w[0];
        c[1] = w[1];
        *reinterpret_cast<V*>(p) = c;
    } else {
        #pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) p[i] = (signed char)(w[i >> 2] >> (8 * (i & 3)));
    }
}

// lane values moved within the wave by the vector unit itself: a few cycles,
// where a shuffle by way of LDS takes about a hundred
template <int CTRL, int ROWS>
__device__ __forceinline__ float moved(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(
        0, __float_as_int(v), CTRL, ROWS, 0xf, true));
}

// max over 16 neighbouring lanes (one group of 128 values, 8 a lane): each lane
// takes in the one 8, 4, 2 and 1 lanes round
template <int CTRL>
__device__ __forceinline__ unsigned max_moved(unsigned a) {
    const unsigned b = __builtin_amdgcn_update_dpp(0, a, CTRL, 0xf, 0xf, true);
    return a > b ? a : b;
}
__device__ __forceinline__ unsigned max16(unsigned a) {
    a = max_moved<0x128>(a);
    a = max_moved<0x124>(a);
    a = max_moved<0x122>(a);
    return max_moved<0x121>(a);
}

// sum over the wave, the same in all lanes: over 16 lanes from the left, then
// row 0 onto 1 and 2 onto 3, then the lower half onto the upper
__device__ __forceinline__ float wave_sum(float v) {
    v += moved<0x111, 0xf>(v);
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);
    v += moved<0x143, 0xc>(v);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// ---- activations -----------------------------------------------------------
// q = Phi(-|u|), the normal distribution's tail, and e = exp(-u^2 / 2).  Below 0
// gelu is u q, and its slope q + u phi: q has to be right relative to itself,
// as far down as the types hold it.  FAST, for 16 bits: q = e t P(t), t = 1 / (1
// + p |u|), the form of Abramowitz & Stegun 7.1.26, with p and the 6 coefficients
// of P fitted over 0..14 for the least relative error of q, which may be min(1 /
// (2 q), 32) times as large as at 0: 2^-21 there, 2^-16 in the tail.  In fp32
// arithmetic under 2^-21 absolute, and 2^-15.7 of q down to u = -13; 16-bit types
// round by 2^-11 at best.  (Fitted for the absolute error, as published, it is off
// by 2^-11 of q at u = -4 and 2^-6 at -9.)  One exp and one reciprocal; the epilogues
// that use it are bound by the vector unit.  Otherwise erfcf.
template <bool FAST>
__device__ __forceinline__ float normal_tail(float u, float* e) {
    const float z = fabsf(u);
    if (FAST) {
        // exp2(-u^2 / 2 * log2(e))
        *e = __builtin_amdgcn_exp2f(u * (u * -0.72134752044f));
        const float t = __builtin_amdgcn_rcpf(
            __builtin_fmaf(z, 0.29928696f, 1.0f));
        float q = __builtin_fmaf(t, -0.08004875f, 0.22636297f);
        q = __builtin_fmaf(t, q, -0.027499145f);
        q = __builtin_fmaf(t, q, 0.14891709f);
        q = __builtin_fmaf(t, q, 0.11239303f);
        q = __builtin_fmaf(t, q, 0.11987457f);
        return q * t * *e;
    }
    *e = expf(-0.5f * u * u);
    return 0.5f * erfcf(z * 0.7071067811865476f);
}

template <bool FAST>
__device__ __forceinline__ float act_value(float u, int act) {
    if (act == ACT_RELU) return u > 0.0f || u != u ? u : 0.0f;
    if (act == ACT_GELU) {
        // u Phi(u): u - u q above 0, u q below; q = 0 from 16 on, and infinity
        // times 0 is not 0
        float e;
        const float q = normal_tail<FAST>(u, &e);
        return __builtin_fmaf(-fminf(fabsf(u), 16.0f), q,
                              u > 0.0f || u != u ? u : 0.0f);
    }
    if (act == ACT_SILU) {
        if (FAST) return u * __builtin_amdgcn_rcpf(
            1.0f + __builtin_amdgcn_exp2f(u * -1.44269504089f));
        return u / (1.0f + expf(-u));
    }
    return u;
}

template <bool FAST>
__device__ __forceinline__ float act_slope(float u, int act) {
    if (act == ACT_GELU) {
        // Phi(u) + u phi(u), phi(u) = e / sqrt(2 pi); a NaN is in cdf
        float e;
        const float q = normal_tail<FAST>(u, &e);
        const float cdf = u < 0.0f ? q : 1.0f - q;
        return __builtin_fmaf(__builtin_amdgcn_fmed3f(u, -16.0f, 16.0f) * e,
                              0.3989422804014327f, cdf);
    }
    if (act == ACT_SILU) {
        const float s = FAST
            ? __builtin_amdgcn_rcpf(
                  1.0f + __builtin_amdgcn_exp2f(u * -1.44269504089f))
            : 1.0f / (1.0f + expf(-u));
        return s * __builtin_fmaf(__builtin_amdgcn_fmed3f(u, -128.0f, 128.0f),
                                  1.0f - s, 1.0f);
    }
    return 1.0f;
}
