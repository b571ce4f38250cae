// Kernels of the layer norm, of the 8-bit form of activations, and of sums
// over rows.
#pragma once
#include <hip/hip_runtime.h>
#include "ffn_common.h"

// ---- reductions --------------------------------------------------------------
// sums of two values over the NT threads of a team (a wave or a block).  slot:
// 2 * 16 floats that no thread still reads; blocks alternate between two.
template <int NT>
__device__ __forceinline__ void team_sum2(float& a, float& b, float* slot) {
    a = wave_sum(a);
    b = wave_sum(b);
    if (NT > 64) {
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) { slot[w] = a; slot[16 + w] = b; }
        __syncthreads();
        a = b = 0.0f;
        #pragma unroll
        for (int i = 0; i < NT / 64; ++i) { a += slot[i]; b += slot[16 + i]; }
    }
}

// ---- layer norm ---------------------------------------------------------------
struct NormArgs {
    const void* x;        // [rows, dim] of T, rows ld apart
    long long ld;
    const void* gamma;    // [dim] of T, or of float where p32; null: ones
    const void* beta;     // null: zeros
    void* y;              // [rows, dim], rows ld_y apart
    long long ld_y;
    float* mean;          // [rows], with rstd; null: not kept
    float* rstd;
    signed char* x8;      // 8-bit form of x, or null
    float* x8_scale;
    signed char* y8;      // 8-bit form of y, or null
    float* y8_scale;
    int rows, dim, p32;
    float eps;
};

__device__ __forceinline__ int groups_of(int dim) {
    return (dim + ACT8_GROUP - 1) / ACT8_GROUP;
}

template <typename T>
__device__ __forceinline__ void load_param(const void* p, int p32, int c,
                                           int left, float other, float* v) {
    if (!p) {
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = other;
    } else if (p32) {
        load8((const float*)p + c, left, v);
    } else {
        load8((const T*)p + c, left, v);
    }
}

// the 8-bit form of 8 columns from c on; 16 lanes hold a group
__device__ __forceinline__ void keep8(signed char* codes, float* scales,
                                      long long row, int c, int left, int dim,
                                      const float* v) {
    const Act8Scale s = act8_scale(max16(max8(v)));
    if (left > 0) {
        store8_codes(codes + row * dim + c, left, v, s.by);
        if (c % ACT8_GROUP == 0)
            scales[row * groups_of(dim) + c / ACT8_GROUP] = s.scale;
    }
}

// From q, the sum of d^2, and `more`, that of d = x - mean, which rounding of
// the mean leaves: the mean without it, and 1 / the deviation.  A row of one
// value far from 0 so keeps no trace of its size.
__device__ __forceinline__ float norm_rstd(float q, float more, float n,
                                           float eps, float* mean) {
    more /= n;
    *mean += more;
    const float var = q / n - more * more;
    return 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + eps);
}

// A team of NT threads takes a row at a time and holds it in registers, R
// chunks of 8 a thread: x is read once, the mean comes first and the variance
// from what is left of it.  Bound by memory: 32768 x 2048 in fp32 99 us (5.4
// TB/s), and nearly so by instructions in 16 bits with the 8-bit form: 17920 x
// 1500 32 us (4.2 TB/s).  Four chunks for each of 1024 threads, rows of 16385 to
// 32768 values, do not fit their 128 registers: 68 (16 bits) or 300 bytes a lane
// go to scratch memory, and 32768 values go at 2.8 and 2.1 TB/s where 8192 go at
// 5.3.
template <typename T, int NT, int R>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void norm_forward_kernel(
        NormArgs p) {
    constexpr int TEAMS = NT < 256 ? 256 / NT : 1;
    __shared__ float slots[2][32];
    const int t = threadIdx.x % NT;
    float g[R][8], b[R][8];
    #pragma unroll
    for (int i = 0; i < R; ++i) {
        const int c = (i * NT + t) * 8;
        load_param<T>(p.gamma, p.p32, c, p.dim - c, 1.0f, g[i]);
        load_param<T>(p.beta, p.p32, c, p.dim - c, 0.0f, b[i]);
    }
    const float n = p.dim;
    for (int row = blockIdx.x * TEAMS + threadIdx.x / NT; row < p.rows;
         row += gridDim.x * TEAMS) {
        const T* x = (const T*)p.x + row * p.ld;
        float v[R][8], s = 0.0f, q = 0.0f, none = 0.0f;
        typename Chunk<T>::V raw[R];
        #pragma unroll
        for (int i = 0; i < R; ++i)
            raw[i] = fetch8(x, (i * NT + t) * 8, p.dim);
        #pragma unroll
        for (int i = 0; i < R; ++i) {
            const int c = (i * NT + t) * 8;
            unpack8(raw[i], c, p.dim, (i + 1) * NT * 8 <= p.dim, v[i]);
            #pragma unroll
            for (int j = 0; j < 8; ++j) s += v[i][j];
            if (p.x8)
                keep8(p.x8, p.x8_scale, row, c, p.dim - c, p.dim, v[i]);
        }
        team_sum2<NT>(s, none, slots[0]);
        float mean = s / n, more = 0.0f;
        #pragma unroll
        for (int i = 0; i < R; ++i) {
            const int left = p.dim - (i * NT + t) * 8;
            if ((i + 1) * NT * 8 > p.dim) {
                // columns that are not there count nothing
                #pragma unroll
                for (int j = 0; j < 8; ++j)
                    v[i][j] = j < left ? v[i][j] : mean;
            }
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float d = v[i][j] - mean;
                q += d * d;
                more += d;
            }
        }
        team_sum2<NT>(q, more, slots[1]);
        const float rstd = norm_rstd(q, more, n, p.eps, &mean);
        if (t == 0 && p.mean) { p.mean[row] = mean; p.rstd[row] = rstd; }
        #pragma unroll
        for (int i = 0; i < R; ++i) {
            const int c = (i * NT + t) * 8, left = p.dim - c;
            #pragma unroll
            for (int j = 0; j < 8; ++j)
                v[i][j] = (v[i][j] - mean) * rstd * g[i][j] + b[i][j];
            if (left > 0)
                store8((T*)p.y + row * p.ld_y + c, left, v[i]);
            if (p.y8) {
                #pragma unroll
                for (int j = 0; j < 8; ++j)
                    v[i][j] = j < left ? (float)(T)v[i][j] : 0.0f;
                keep8(p.y8, p.y8_scale, row, c, left, p.dim, v[i]);
            }
        }
    }
}

struct NormGradArgs {
    const void* x;        // [rows, dim] of T, or its 8-bit form
    long long ld;
    const signed char* x8;
    const float* x8_scale;
    const void* dy;       // [rows, dim] of T, rows ld_dy apart
    long long ld_dy;
    const void* add;      // [rows, dim] of T that goes onto dx, or null
    long long ld_add;
    const void* gamma;
    const float* mean;
    const float* rstd;
    void* dx;             // [rows, dim], or null
    float* part;          // [blocks, 2, dim]: sums of dy xh, of dy; or null
    int rows, dim, p32;
};

// 8 columns of the kept x as they lie in memory: values, or codes with their
// group's scale
template <typename T, bool X8> struct KeptRaw {
    typename Chunk<T>::V raw;
    __device__ __forceinline__ void fetch(const NormGradArgs& p, int row,
                                          int c) {
        raw = fetch8((const T*)p.x + row * p.ld, c, p.dim);
    }
    __device__ __forceinline__ void unpack(int c, int dim, bool whole,
                                           float* v) const {
        unpack8(raw, c, dim, whole, v);
    }
    // x - mean, of what unpack() brought
    __device__ __forceinline__ float from(float v, float mean) const {
        return v - mean;
    }
};
template <typename T> struct KeptRaw<T, true> {
    u32x2 raw;
    float scale;
    __device__ __forceinline__ void fetch(const NormGradArgs& p, int row_,
                                          int c) {
        const long long row = row_;
        const signed char* q = p.x8 + row * p.dim;
        i8x8 r;
        if (p.dim >= 8) {
            r = *reinterpret_cast<const i8x8*>(
                q + (c < p.dim - 8 ? c : p.dim - 8));
        } else {
            #pragma unroll
            for (int i = 0; i < 8; ++i)
                r[i] = i < p.dim ? q[i] : (signed char)0;
        }
        raw = __builtin_bit_cast(u32x2, r);
        const int g = c < p.dim ? c / ACT8_GROUP : groups_of(p.dim) - 1;
        scale = p.x8_scale[row * groups_of(p.dim) + g];
    }
    __device__ __forceinline__ void unpack(int c, int dim, bool whole,
                                           float* v) const {
        unpack8(__builtin_bit_cast(i8x8, raw), c, dim, whole, v);
    }
    __device__ __forceinline__ float from(float v, float mean) const {
        return __builtin_fmaf(v, scale, -mean);
    }
};

// x - mean for 8 columns of the kept x, from c on
template <typename T>
__device__ __forceinline__ void load_kept(const NormGradArgs& p, long long row,
                                          int c, int left, float mean,
                                          float* v) {
    float scale = 1.0f;
    if (p.x8) {
        load8_codes(p.x8 + row * p.dim + c, left, v);
        scale = p.x8_scale[row * groups_of(p.dim) + c / ACT8_GROUP];
    } else {
        load8((const T*)p.x + row * p.ld + c, left, v);
    }
    #pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __builtin_fmaf(v[i], scale, -mean);
}

// dx = rstd (g dy - mean(g dy) - xh mean(g dy xh)).  x and dy are read once;
// each thread sums dy xh and dy for its own columns over the rows that it
// sees, the teams of a block add theirs in turn, and column_sum_kernel adds
// the blocks': no atomics, the same result each time.  32768 x 2048 in fp32 151
// us (5.3 TB/s).  Two and four chunks a thread, rows of 8193 to 32768 values, do
// not fit the 128 registers that 1024 threads leave each: 112 to 276 and 824 to
// 860 bytes a lane go to scratch memory.  Forward and backward, TB/s of x twice,
// dy, y and dx, in bf16 and fp32: 8192 values 4.9 and 5.2; 9216 2.2 and 2.6, a
// second chunk that is nearly empty; 16384 3.0 and 3.7; 32768 0.8 and 1.6; 40960,
// by the kernels for longer rows, 2.7 and 2.6.
template <typename T, int NT, int R, bool X8>
__global__ __launch_bounds__(NT < 128 ? 256 : NT) void norm_backward_kernel(
        NormGradArgs p) {
    constexpr int TEAMS = NT < 128 ? 256 / NT : 1;
    __shared__ float slots[2][32];
    __shared__ float all[TEAMS > 1 ? 2 * NT * R * 8 : 1];
    const int t = threadIdx.x % NT, team = threadIdx.x / NT;
    float g[R][8], sg[R][8], sb[R][8];
    #pragma unroll
    for (int i = 0; i < R; ++i) {
        const int c = (i * NT + t) * 8;
        load_param<T>(p.gamma, p.p32, c, p.dim - c, 1.0f, g[i]);
        #pragma unroll
        for (int j = 0; j < 8; ++j) sg[i][j] = sb[i][j] = 0.0f;
    }
    const float inv = 1.0f / p.dim;
    int turn = 0;
    for (int row = blockIdx.x * TEAMS + team; row < p.rows;
         row += gridDim.x * TEAMS, turn ^= 1) {
        const float mean = p.mean[row], rstd = p.rstd[row];
        float s1 = 0.0f, s2 = 0.0f;
        KeptRaw<T, X8> rh[R];
        typename Chunk<T>::V rd[R];
        #pragma unroll
        for (int i = 0; i < R; ++i) {
            const int c = (i * NT + t) * 8;
            rh[i].fetch(p, row, c);
            rd[i] = fetch8((const T*)p.dy + row * p.ld_dy, c, p.dim);
        }
        // xh = (x - mean) rstd, x a code times its scale: the difference first,
        // since products with rstd round by steps of x, and in a row far from 0
        // for its spread nothing else would be left of xh.  Columns that are not
        // there have dy = 0.
        float h[R][8], d[R][8];
        #pragma unroll
        for (int i = 0; i < R; ++i) {
            const int c = (i * NT + t) * 8;
            const bool whole = (i + 1) * NT * 8 <= p.dim;
            rh[i].unpack(c, p.dim, whole, h[i]);
            unpack8(rd[i], c, p.dim, whole, d[i]);
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                h[i][j] = rh[i].from(h[i][j], mean) * rstd;
                sg[i][j] = __builtin_fmaf(d[i][j], h[i][j], sg[i][j]);
                sb[i][j] += d[i][j];
                d[i][j] *= g[i][j];
                s1 += d[i][j];
                s2 = __builtin_fmaf(d[i][j], h[i][j], s2);
            }
        }
        if (!p.dx) continue;
        team_sum2<NT>(s1, s2, slots[turn]);
        s1 *= -inv * rstd;
        s2 *= -inv * rstd;
        #pragma unroll
        for (int i = 0; i < R; ++i) {
            const int c = (i * NT + t) * 8, left = p.dim - c;
            float a[8];
            if (p.add)
                unpack8(fetch8((const T*)p.add + row * p.ld_add, c, p.dim), c,
                        p.dim, (i + 1) * NT * 8 <= p.dim, a);
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float v = __builtin_fmaf(
                    h[i][j], s2, __builtin_fmaf(d[i][j], rstd, s1));
                d[i][j] = p.add ? v + a[j] : v;
            }
            if (left > 0)
                store8((T*)p.dx + (long long)row * p.dim + c, left, d[i]);
        }
    }
    if (!p.part) return;
    float* out = p.part + (long long)blockIdx.x * 2 * p.dim;
    if (TEAMS == 1) {
        #pragma unroll
        for (int i = 0; i < R; ++i) {
            const int c = (i * NT + t) * 8, left = p.dim - c;
            if (left <= 0) continue;
            store8(out + c, left, sg[i]);
            store8(out + p.dim + c, left, sb[i]);
        }
        return;
    }
    for (int w = 0; w < TEAMS; ++w) {
        if (team == w) {
            #pragma unroll
            for (int i = 0; i < R; ++i)
                #pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float* a = all + (i * 8 + j) * NT + t;
                    a[0] = (w ? a[0] : 0.0f) + sg[i][j];
                    a[R * 8 * NT] = (w ? a[R * 8 * NT] : 0.0f) + sb[i][j];
                }
        }
        __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * p.dim; c += blockDim.x) {
        const int col = c < p.dim ? c : c - p.dim;
        const int k = col >> 3, at = ((k / NT) * 8 + (col & 7)) * NT + k % NT;
        out[c] = all[(c < p.dim ? 0 : R * 8 * NT) + at];
    }
}

// rows too long for a block's registers: they are read again for each step
template <typename T>
__global__ __launch_bounds__(1024) void norm_forward_wide_kernel(NormArgs p) {
    __shared__ float slots[2][32];
    const int row = blockIdx.x, step = 1024 * 8;
    const T* x = (const T*)p.x + row * p.ld;
    float s = 0.0f, q = 0.0f, none = 0.0f, v[8], g[8], b[8];
    for (int c = threadIdx.x * 8; c < p.dim; c += step) {
        load8(x + c, p.dim - c, v);
        #pragma unroll
        for (int j = 0; j < 8; ++j) s += v[j];
    }
    team_sum2<1024>(s, none, slots[0]);
    const float n = p.dim;
    float mean = s / n, more = 0.0f;
    for (int c = threadIdx.x * 8; c < p.dim; c += step) {
        load8(x + c, p.dim - c, v);
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float d = j < p.dim - c ? v[j] - mean : 0.0f;
            q += d * d;
            more += d;
        }
    }
    team_sum2<1024>(q, more, slots[1]);
    const float rstd = norm_rstd(q, more, n, p.eps, &mean);
    if (threadIdx.x == 0 && p.mean) { p.mean[row] = mean; p.rstd[row] = rstd; }
    // whole groups of lanes go on together, for keep8
    for (int c0 = 0; c0 < p.dim; c0 += step) {
        const int c = c0 + threadIdx.x * 8, left = p.dim - c;
        load8(x + c, left, v);
        if (p.x8) keep8(p.x8, p.x8_scale, row, c, left, p.dim, v);
        load_param<T>(p.gamma, p.p32, c, left, 1.0f, g);
        load_param<T>(p.beta, p.p32, c, left, 0.0f, b);
        #pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (v[j] - mean) * rstd * g[j] + b[j];
        if (left > 0) store8((T*)p.y + row * p.ld_y + c, left, v);
        if (p.y8) {
            #pragma unroll
            for (int j = 0; j < 8; ++j)
                v[j] = j < left ? (float)(T)v[j] : 0.0f;
            keep8(p.y8, p.y8_scale, row, c, left, p.dim, v);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(1024) void norm_dx_wide_kernel(NormGradArgs p) {
    __shared__ float slots[32];
    const int row = blockIdx.x, step = 1024 * 8;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s1 = 0.0f, s2 = 0.0f, h[8], d[8], g[8], a[8];
    for (int c = threadIdx.x * 8; c < p.dim; c += step) {
        load_kept<T>(p, row, c, p.dim - c, mean, h);
        load8((const T*)p.dy + row * p.ld_dy + c, p.dim - c, d);
        load_param<T>(p.gamma, p.p32, c, p.dim - c, 1.0f, g);
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            s1 += d[j] * g[j];
            s2 += d[j] * g[j] * h[j] * rstd;
        }
    }
    team_sum2<1024>(s1, s2, slots);
    s1 /= p.dim;
    s2 /= p.dim;
    for (int c = threadIdx.x * 8; c < p.dim; c += step) {
        const int left = p.dim - c;
        load_kept<T>(p, row, c, left, mean, h);
        load8((const T*)p.dy + row * p.ld_dy + c, left, d);
        load_param<T>(p.gamma, p.p32, c, left, 1.0f, g);
        if (p.add) load8((const T*)p.add + row * p.ld_add + c, left, a);
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float v = rstd * (d[j] * g[j] - s1 - h[j] * rstd * s2);
            d[j] = p.add ? v + a[j] : v;
        }
        store8((T*)p.dx + (long long)row * p.dim + c, left, d);
    }
}

// ---- sums over rows -------------------------------------------------------------
// part[blockIdx.y][c] = sum over the slab's rows; 8 columns a thread.  NORM:
// dy xh and dy of the layer norm's gradients, else the rows of p.dy alone.
template <typename T, bool NORM>
__global__ __launch_bounds__(256) void row_sum_kernel(NormGradArgs p,
                                                      int per) {
    __shared__ float all[8 * 256];
    const int t = threadIdx.x & 31, r0 = threadIdx.x >> 5;
    const int c = (blockIdx.x * 32 + t) * 8, left = p.dim - c;
    const int first = blockIdx.y * per;
    const int last = p.rows - first < per ? p.rows : first + per;
    float sg[8] = {0, 0, 0, 0, 0, 0, 0, 0}, sb[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (left > 0) {
        const bool whole = (blockIdx.x + 1) * 256 <= p.dim;
        #pragma unroll 4
        for (int row = first + r0; row < last; row += 8) {
            float d[8], h[8];
            unpack8(fetch8((const T*)p.dy + row * p.ld_dy, c, p.dim), c, p.dim,
                    whole, d);
            if (NORM) {
                load_kept<T>(p, row, c, left, p.mean[row], h);
                #pragma unroll
                for (int j = 0; j < 8; ++j)
                    sg[j] += d[j] * h[j] * p.rstd[row];
            }
            #pragma unroll
            for (int j = 0; j < 8; ++j) sb[j] += d[j];
        }
    }
    for (int half = 0; half < (NORM ? 2 : 1); ++half) {
        #pragma unroll
        for (int j = 0; j < 8; ++j)
            all[r0 * 256 + t * 8 + j] = NORM && !half ? sg[j] : sb[j];
        __syncthreads();
        const int col = blockIdx.x * 256 + threadIdx.x;
        float s = 0.0f;
        for (int r = 0; r < 8; ++r) s += all[r * 256 + threadIdx.x];
        if (col < p.dim)
            p.part[((long long)blockIdx.y * (NORM ? 2 : 1) + half) * p.dim +
                   col] = s;
        __syncthreads();
    }
}

// out[c] = sum over `n` rows of part, width values each, in a fixed order; the
// first `first` columns go to `a`, the others to `b` (either may be null)
template <typename O>
__global__ __launch_bounds__(1024) void column_sum_kernel(
        const float* part, int n, int width, int first, O* a, O* b) {
    __shared__ float all[64][17];
    const int t = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const int c = blockIdx.x * 16 + t;
    float s = 0.0f;
    if (c < width) {
        #pragma unroll 4
        for (int r = r0; r < n; r += 64) s += part[(long long)r * width + c];
    }
    all[r0][t] = s;
    __syncthreads();
    if (threadIdx.x < 16 && c < width) {
        float v = 0.0f;
        #pragma unroll 8
        for (int r = 0; r < 64; ++r) v += all[r][t];
        if (c < first) { if (a) a[c] = (O)v; }
        else if (b) b[c - first] = (O)v;
    }
}

// ---- the 8-bit form by itself ------------------------------------------------------
// A group of 128 values for each 16 lanes, GROUPS of them at a time; I is the
// type that counts them.  17920 x 6000 in bf16, us: one group 66, two 64, four
// 66, and 74 with a quarter of the blocks; in a step, from memory, 77 (4.2 TB/s).
template <typename T, typename I>
__global__ __launch_bounds__(256) void act8_pack_kernel(
        const T* x, long long ld, I rows, int dim, signed char* codes,
        float* scales) {
    constexpr int GROUPS = 2;
    const I ng = groups_of(dim), groups = rows * ng;
    const int t = threadIdx.x >> 4, o = (threadIdx.x & 15) * 8;
    // all lanes of a wave go round as often, for max16
    for (I g0 = (I)blockIdx.x * 16 * GROUPS; g0 < groups;
         g0 += (I)gridDim.x * 16 * GROUPS) {
        typename Chunk<T>::V raw[GROUPS];
        I row[GROUPS];
        int c[GROUPS];
        #pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const I at = g0 + i * 16 + t, g = at < groups ? at : groups - 1;
            row[i] = g / ng;
            c[i] = (int)(g - row[i] * ng) * ACT8_GROUP + o;
            raw[i] = fetch8(x + (long long)row[i] * ld, c[i], dim);
            if (at >= groups) c[i] = dim;
        }
        #pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            float v[8];
            unpack8(raw[i], c[i], dim, dim % ACT8_GROUP == 0, v);
            keep8(codes, scales, row[i], c[i], dim - c[i], dim, v);
        }
    }
}

// Values of 8 bits to 16 or 32, rows ld apart, a chunk of 8 a thread: 17920 x 6000
// to fp32 93 us, with two to eight chunks a thread 115 to 137; in a step, from
// memory, 105 (5.1 TB/s).
template <typename O, typename I>
__global__ __launch_bounds__(256) void act8_unpack_kernel(
        const signed char* codes, const float* scales, I rows, int dim, O* out,
        long long ld) {
    const I nc = (dim + 7) / 8;
    // once, but for more chunks than a launch may have threads
    for (I i = (I)blockIdx.x * 256 + threadIdx.x; i < rows * nc;
         i += (I)gridDim.x * 256) {
        const I row = i / nc;
        const int c = (int)(i - row * nc) * 8;
        const signed char* p = codes + (long long)row * dim;
        i8x8 raw;
        if (dim >= 8) {
            raw = *reinterpret_cast<const i8x8*>(p + (c < dim - 8 ? c : dim - 8));
        } else {
            #pragma unroll
            for (int j = 0; j < 8; ++j) raw[j] = j < dim ? p[j] : (signed char)0;
        }
        const float scale =
            scales[(long long)row * groups_of(dim) + c / ACT8_GROUP];
        float v[8];
        unpack8(raw, c, dim, dim % 8 == 0, v);
        #pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= scale;
        store8(out + (long long)row * ld + c, dim - c, v);
    }
}
