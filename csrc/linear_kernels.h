// Kernels of linear layers: products with their epilogues, and the
// joining of products that were split over k.
#pragma once
#include <hip/hip_runtime.h>
#include "gemm.h"

enum Epilogue { EPI_FORWARD = 0, EPI_GRAD = 1, EPI_PLAIN = 2 };
// how the value before the activation is kept for the backward pass
enum Keep { KEEP_NONE = 0, KEEP_FULL = 1, KEEP_BITS = 2, KEEP_8BIT = 3 };

struct EpiArgs {
    void* out;             // [M, N] of T (EPI_PLAIN: of float where out_f32)
    long long ld_out;
    void* out_lo;          // EPI_GRAD: what rounding to `out` left, or null
    const void* bias;      // [N] of T (of float where bias_f32) or null
    const void* res;       // [M, N] of T or null
    long long ld_res;
    void* kept;            // [M, N] of T, [M, N / 8] bytes, or [M, N] codes
    float* kept_scale;     // [M, N / 128]
    signed char* out8;     // 8-bit form of `out`, or null
    float* out8_scale;
    float* colsum;         // EPI_GRAD: [row blocks, N] sums of `out`, or null
    int act, keep, bias_f32, out_f32;
};

template <typename T> struct IsHalf { static constexpr bool value = true; };
template <> struct IsHalf<float> { static constexpr bool value = false; };

// 8 neighbouring results of row m from column n on; `left` of them are there
// (0 or less: none).  All 16 lanes of a group of 128 columns come together.
template <typename T, int EPI>
__device__ __forceinline__ void finish8(float* v, long long m, int n, int left,
                                        int N, const EpiArgs& e, float* sums) {
    constexpr bool FAST = IsHalf<T>::value;
    const bool on = left > 0;
    if (EPI == EPI_PLAIN) {
        if (!on) return;
        if (e.out_f32) store8((float*)e.out + m * e.ld_out + n, left, v);
        else store8((T*)e.out + m * e.ld_out + n, left, v);
        return;
    }
    if (EPI == EPI_GRAD) {
        if (!on) return;
        // what comes from the layer above is of type T: rounded as such
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)(T)v[i];
        if (e.keep == KEEP_BITS) {
            const unsigned bits = ((const unsigned char*)e.kept)
                [m * ((N + 7) >> 3) + (n >> 3)];
            #pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!(bits >> i & 1)) v[i] = 0.0f;
        } else if (e.keep != KEEP_NONE) {
            float u[8];
            if (e.keep == KEEP_8BIT)
                load8_codes((const signed char*)e.kept + m * N + n, left,
                            e.kept_scale[m * ((N + ACT8_GROUP - 1) /
                                              ACT8_GROUP) + n / ACT8_GROUP],
                            u);
            else
                load8((const T*)e.kept + m * N + n, left, u);
            #pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= act_slope<FAST>(u[i], e.act);
        }
        #pragma unroll
        for (int i = 0; i < 8; ++i) sums[i] += i < left ? v[i] : 0.0f;
        store8((T*)e.out + m * e.ld_out + n, left, v);
        if (e.out_lo) {
            #pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float hi = (float)(T)v[i];
                v[i] = fabsf(hi) < __builtin_inff() ? v[i] - hi : 0.0f;
            }
            store8((T*)e.out_lo + m * e.ld_out + n, left, v);
        }
        return;
    }
    if (on && e.bias) {
        float b[8];
        if (e.bias_f32) load8((const float*)e.bias + n, left, b);
        else load8((const T*)e.bias + n, left, b);
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += b[i];
    }
    #pragma unroll
    for (int i = 0; i < 8; ++i) if (i >= left) v[i] = 0.0f;
    if (e.keep == KEEP_BITS) {
        unsigned bits = 0;
        #pragma unroll
        for (int i = 0; i < 8; ++i) bits |= (v[i] <= 0.0f ? 0u : 1u) << i;
        if (on)
            ((unsigned char*)e.kept)[m * ((N + 7) >> 3) + (n >> 3)] =
                (unsigned char)bits;
    } else if (e.keep == KEEP_FULL) {
        if (on) store8((T*)e.kept + m * N + n, left, v);
    } else if (e.keep == KEEP_8BIT) {
        const float a = max16(max8(v));
        const Act8Scale s = act8_scale(a, a < __builtin_inff());
        if (on) {
            store8_codes((signed char*)e.kept + m * N + n, left, v, s.by);
            if (n % ACT8_GROUP == 0)
                e.kept_scale[m * ((N + ACT8_GROUP - 1) / ACT8_GROUP) +
                             n / ACT8_GROUP] = s.scale;
        }
    }
    if (e.act != ACT_NONE) {
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = act_value<FAST>(v[i], e.act);
    }
    if (on && e.res) {
        float r[8];
        load8((const T*)e.res + m * e.ld_res + n, left, r);
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += r[i];
    }
    if (on) store8((T*)e.out + m * e.ld_out + n, left, v);
    if (e.out8) {
        #pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = i < left ? (float)(T)v[i] : 0.0f;
        const float a = max16(max8(v));
        const Act8Scale s = act8_scale(a, a < __builtin_inff());
        if (on) {
            store8_codes(e.out8 + m * N + n, left, v, s.by);
            if (n % ACT8_GROUP == 0)
                e.out8_scale[m * ((N + ACT8_GROUP - 1) / ACT8_GROUP) +
                             n / ACT8_GROUP] = s.scale;
        }
    }
}

// One block, one tile of C; blockIdx.y is the part of k.  With `part` the
// tile's fp32 sums go to part[blockIdx.y][m][n] (rows of ld_part values), and
// finish_kernel joins them; otherwise the epilogue follows at once.
template <typename T, int BM, int BN, int WM, int WN, bool AA, bool BA,
          int EPI>
__global__ __launch_bounds__(WM * WN * 64) void gemm_kernel(
        Operand a, Operand b, int M, int N, int K, int kper, float* part,
        long long ld_part, EpiArgs e) {
    typedef Gemm<T, BM, BN, WM, WN, AA, BA> G;
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const int tm = (M + BM - 1) / BM, tn = (N + BN - 1) / BN;
    int bm, bn;
    tile_of(blockIdx.x, tm, tn, &bm, &bn);
    const int m0 = bm * BM, n0 = bn * BN;
    const int k0 = blockIdx.y * kper;
    const int k1 = K - k0 < kper ? K : k0 + kper;

    G g(lds, a, b, M, N, K, m0, n0);
    g.run(k0, k1);
    if (a.lo) {
        g.a.p = a.lo;
        stage_wait<0>();
        g.run(k0, k1);
    }

    constexpr int CH = BN / 8;             // chunks of 8 columns
    constexpr int RS = G::THREADS / CH;    // rows a round
    const int c = threadIdx.x % CH, r0 = threadIdx.x / CH;
    const int n = n0 + 8 * c, left = N - n;
    float sums[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    #pragma unroll
    for (int i = 0; i < G::TM; ++i) {
        __syncthreads();
        g.stage_out(lds, i);
        __syncthreads();
        for (int r = r0; r < WM * 32; r += RS) {
            const float* s = reinterpret_cast<const float*>(lds) +
                             r * G::OUT_LD + 8 * c;
            float v[8];
            #pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = s[j];
            const int m = m0 + ((r >> 5) * G::TM + i) * 32 + (r & 31);
            const int here = m < M ? left : 0;
            if (part) {
                if (here > 0)
                    store8(part + ((long long)blockIdx.y * M + m) * ld_part +
                           n, here, v);
            } else {
                finish8<T, EPI>(v, m, n, here, N, e, sums);
            }
        }
    }
    if (EPI == EPI_GRAD && e.colsum && !part) {
        float* all = reinterpret_cast<float*>(lds);
        __syncthreads();
        #pragma unroll
        for (int j = 0; j < 8; ++j) all[r0 * BN + 8 * c + j] = sums[j];
        __syncthreads();
        for (int j = threadIdx.x; j < BN; j += G::THREADS) {
            float t = 0.0f;
            for (int r = 0; r < RS; ++r) t += all[r * BN + j];
            if (n0 + j < N) e.colsum[(long long)bm * N + n0 + j] = t;
        }
    }
}

// Few rows: 32 x 32 results a block, k shared out among its 8 waves.  The
// fragments come straight from memory, 16 bytes a lane along k: there is nothing
// to share, and no barrier before the end.  What bounds it is the weight's way
// from memory.  BA false (32 bits only): a lane's 4 values of B lie across k.
#define THIN_WAVES 8
template <typename T, bool BA, int EPI>
__global__ __launch_bounds__(THIN_WAVES * 64) void thin_kernel(
        Operand a, Operand b, int M, int N, int K, EpiArgs e) {
    static_assert(BA || sizeof(T) == 4, "across k needs 32 bits");
    constexpr int E = 16 / sizeof(T), U = 2 * E, LD = 36;
    typedef T V __attribute__((ext_vector_type(E), aligned(sizeof(T))));
    __shared__ float part[THIN_WAVES][32][LD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = lane & 31, off = E * (lane >> 5);
    const int m0 = blockIdx.y * 32, n0 = blockIdx.x * 32;
    // rows that are not there: the last one's values, for results not written
    const long long ma = m0 + row < M ? m0 + row : M - 1;
    const long long nb = n0 + row < N ? n0 + row : N - 1;
    const T* pa = (const T*)a.p + ma * a.ld + off;
    const T* pb = (const T*)b.p + (BA ? nb * b.ld + off : off * b.ld + nb);
    const int steps = (K + U - 1) / U;
    const int per = (steps + THIN_WAVES - 1) / THIN_WAVES;
    const int s0 = wave * per, s1 = s0 + per < steps ? s0 + per : steps;
    const int whole = K / U < s1 ? K / U : s1;
    f32x16 acc;
    #pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
    auto step = [&](int s, bool all) {
        typename Mfma<T>::V x, y;
        const int k = s * U;
        if (all) {
            x = *reinterpret_cast<const V*>(pa + k);
        } else {
            #pragma unroll
            for (int i = 0; i < E; ++i)
                x[i] = k + off + i < K ? pa[k + i] : (T)0.0f;
        }
        if (BA && all) {
            y = *reinterpret_cast<const V*>(pb + k);
        } else {
            #pragma unroll
            for (int i = 0; i < E; ++i)
                y[i] = all || k + off + i < K
                    ? pb[BA ? k + i : (long long)(k + i) * b.ld] : (T)0.0f;
        }
        acc = Mfma<T>::go(y, x, acc);
    };
    #pragma unroll 6
    for (int s = s0; s < whole; ++s) step(s, true);
    if (s0 < s1 && whole < s1) step(whole, false);
    #pragma unroll
    for (int g = 0; g < 4; ++g) {
        f32x4 v;
        #pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = acc[4 * g + i];
        *reinterpret_cast<f32x4*>(&part[wave][row][8 * g + 4 * (lane >> 5)]) = v;
    }
    __syncthreads();
    const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 8;
    float sums[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (threadIdx.x < 128) {
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        #pragma unroll
        for (int w = 0; w < THIN_WAVES; ++w)
            #pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += part[w][r][c + i];
        finish8<T, EPI>(v, m0 + r, n0 + c, m0 + r < M ? N - n0 - c : 0, N, e,
                        sums);
    }
    if (EPI == EPI_GRAD && e.colsum) {
        __syncthreads();
        if (threadIdx.x < 128) {
            #pragma unroll
            for (int i = 0; i < 8; ++i) part[0][r][c + i] = sums[i];
        }
        __syncthreads();
        if (threadIdx.x < 32 && n0 + threadIdx.x < N) {
            float t = 0.0f;
            for (int i = 0; i < 32; ++i) t += part[0][i][threadIdx.x];
            e.colsum[(long long)blockIdx.y * N + n0 + threadIdx.x] = t;
        }
    }
}

// Joins `splits` partial products, `rows` (a multiple of 16) x 128 columns a
// block, in the order of k, and finishes them as the product's own epilogue
// would.  With one "product" of type S it takes a gradient back through an
// activation.
template <typename T, int EPI, typename S>
__global__ __launch_bounds__(256) void finish_kernel(
        const S* part, long long ld_part, int splits, int rows, int M, int N,
        EpiArgs e) {
    __shared__ float all[16 * 128];
    const int c = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const int n = blockIdx.y * 128 + 8 * c, left = N - n;
    float sums[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int r = r0; r < rows; r += 16) {
        const long long m = (long long)blockIdx.x * rows + r;
        const int here = m < M ? left : 0;
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (here > 0) {
            #pragma unroll 4
            for (int s = 0; s < splits; ++s) {
                float w[8];
                load8(part + ((long long)s * M + m) * ld_part + n, here, w);
                #pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += w[j];
            }
        }
        finish8<T, EPI>(v, m, n, here, N, e, sums);
    }
    if (EPI == EPI_GRAD && e.colsum) {
        #pragma unroll
        for (int j = 0; j < 8; ++j) all[r0 * 128 + 8 * c + j] = sums[j];
        __syncthreads();
        if (threadIdx.x < 128) {
            float t = 0.0f;
            for (int r = 0; r < 16; ++r) t += all[r * 128 + threadIdx.x];
            const int col = blockIdx.y * 128 + threadIdx.x;
            if (col < N) e.colsum[(long long)blockIdx.x * N + col] = t;
        }
    }
}
