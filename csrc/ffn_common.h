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

// 8 values from column c of a row of `dim`, as they lie in memory, for rows that
// may end inside a chunk: nothing branches between the load and its use, so that
// many are on their way at once.  Where the chunk ends past the row, its last 8
// values come instead, and unpack8() moves them; `c` may lie past the row.
template <typename T>
__device__ __forceinline__ typename Chunk<T>::V fetch8(const T* row, int c,
                                                       int dim) {
    if (dim >= 8)
        return *reinterpret_cast<const typename Chunk<T>::V*>(
            row + (c < dim - 8 ? c : dim - 8));
    typename Chunk<T>::V v;
    #pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < dim ? row[i] : (T)0.0f;
    return v;
}

// columns that are not there become 0.  `whole`: no lane's chunk ends past the
// row (the same for all lanes).
__device__ __forceinline__ void settle8(int c, int dim, bool whole, float* v) {
    if (whole) return;
    const int by = dim >= 8 && c > dim - 8 ? c - (dim - 8) : 0;
    #pragma unroll
    for (int b = 1; b < 8; b *= 2)
        #pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = by & b ? (i + b < 8 ? v[i + b] : 0.0f) : v[i];
    #pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < dim ? v[i] : 0.0f;
}

template <typename V>
__device__ __forceinline__ void unpack8(V raw, int c, int dim, bool whole,
                                        float* v) {
    #pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)raw[i];
    settle8(c, dim, whole, v);
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
                                            float scale, float* v) {
    if (left >= 8) {
        const i8x8 c = *reinterpret_cast<const i8x8*>(p);
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)c[i] * scale;
    } else {
        #pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = i < left ? (float)p[i] * scale : 0.0f;
    }
}

// ---- 8-bit form ------------------------------------------------------------
// c = rint(x * fl(127 / a)), s = fl(a * fl(1 / 127)), a = max |x| of the
// group.  x * fl(127 / a) is at most 127 (1 + 2^-23), so rint never leaves
// [-127, 127].  A group with an infinity or a NaN gets s = NaN and codes 0:
// all of it reads as NaN, so a broken activation shows in the gradients.
struct Act8Scale { float by, scale; };

__device__ __forceinline__ Act8Scale act8_scale(float a, bool finite) {
    Act8Scale s;
    const bool some = a >= ACT8_LEAST;
    s.by = some && finite ? 127.0f / a : 0.0f;
    s.scale = !finite ? __builtin_nanf("")
                      : some ? a * (1.0f / 127.0f) : 0.0f;
    return s;
}

// max |x| over 8 values; `finite` falls where one is an infinity or NaN
__device__ __forceinline__ float max8(const float* v) {
    // fmax drops NaN, so NaN is carried as an infinity
    float a = 0.0f;
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float m = fabsf(v[i]);
        a = fmaxf(a, m == m ? m : __builtin_inff());
    }
    return a;
}

__device__ __forceinline__ void store8_codes(signed char* p, int left,
                                             const float* v, float by) {
    i8x8 c;
    #pragma unroll
    for (int i = 0; i < 8; ++i)
        // by is 0 in a group of zeros and in one that is not finite
        c[i] = by == 0.0f ? (signed char)0
                          : (signed char)(int)rintf(v[i] * by);
    if (left >= 8) {
        *reinterpret_cast<i8x8*>(p) = c;
    } else {
        #pragma unroll
        for (int i = 0; i < 8; ++i) if (i < left) p[i] = c[i];
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
__device__ __forceinline__ float max16(float a) {
    a = fmaxf(a, moved<0x128, 0xf>(a));
    a = fmaxf(a, moved<0x124, 0xf>(a));
    a = fmaxf(a, moved<0x122, 0xf>(a));
    return fmaxf(a, moved<0x121, 0xf>(a));
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
// q = Phi(-|u|), the normal distribution's tail, and e = exp(-u^2 / 2).  FAST:
// Abramowitz & Stegun 7.1.26, erf(z) = 1 - t P(t) exp(-z^2) with t = 1 / (1 + p z)
// and z = |u| / sqrt(2), |error| < 1.5e-7: under 2^-22, while the 16-bit types
// that it serves round to 2^-12 at best.  One exp and one reciprocal; the
// epilogues that use it are bound by the vector unit.  Otherwise erfcf.
template <bool FAST>
__device__ __forceinline__ float normal_tail(float u, float* e) {
    const float z = fabsf(u);
    if (FAST) {
        // exp2(-u^2 / 2 * log2(e))
        *e = __builtin_amdgcn_exp2f(u * (u * -0.72134752044f));
        // p / sqrt(2); the coefficients are halved
        const float t = __builtin_amdgcn_rcpf(
            __builtin_fmaf(z, 0.23164189f, 1.0f));
        float q = __builtin_fmaf(t, 0.5307027145f, -0.7265760135f);
        q = __builtin_fmaf(t, q, 0.7107068705f);
        q = __builtin_fmaf(t, q, -0.142248368f);
        q = __builtin_fmaf(t, q, 0.127414796f);
        return q * t * *e;
    }
    *e = expf(-0.5f * u * u);
    return 0.5f * erfcf(z * 0.7071067811865476f);
}

template <bool FAST>
__device__ __forceinline__ float act_value(float u, int act) {
    if (act == ACT_RELU) return u > 0.0f || u != u ? u : 0.0f;
    if (act == ACT_GELU) {
        // u Phi(u): u - u q above 0, u q below
        float e;
        const float q = normal_tail<FAST>(u, &e);
        return __builtin_fmaf(-fabsf(u), q, u > 0.0f || u != u ? u : 0.0f);
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
        // Phi(u) + u phi(u), phi(u) = e / sqrt(2 pi)
        float e;
        const float q = normal_tail<FAST>(u, &e);
        const float cdf = 0.5f + __builtin_copysignf(0.5f - q, u);
        return __builtin_fmaf(u * e, 0.3989422804014327f, cdf);
    }
    if (act == ACT_SILU) {
        const float s = FAST
            ? __builtin_amdgcn_rcpf(
                  1.0f + __builtin_amdgcn_exp2f(u * -1.44269504089f))
            : 1.0f / (1.0f + expf(-u));
        return s * __builtin_fmaf(u, 1.0f - s, 1.0f);
    }
    return 1.0f;
}
