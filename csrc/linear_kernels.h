// Kernels of linear layers: products with their epilogues, and the
// joining of products that were split over k.
#pragma once
#include <hip/hip_runtime.h>
#include "gemm.h"

enum Epilogue { EPI_FORWARD = 0, EPI_GRAD = 1, EPI_PLAIN = 2 };
// how the value before the activation, u, is kept for the backward pass
enum Keep { KEEP_NONE = 0, KEEP_FULL = 1, KEEP_BITS = 2, KEEP_8BIT = 3 };

// What a u in full is kept as, where the results are T: with more bits than they.
// Its rounding goes into the slope and from there into each p, and the sums that
// follow a rounding of their own, the norm's gradients in the block, show it: kept
// in T, the norm bias's gradient was off by 1.8 times what its rounding makes, so by
// 1.1.  bf16: fp16 has 3 bits more in the same place, and where it ends, at 65504
// and 2^-24, a slope is 0, 1 or 1/2 already; a linear layer of 17920 x 1500 to 6000
// with gelu, forward and backward, takes 1265 us for 1267.  fp16: twice the bytes,
// there 215 MB more and 1359 us for 1291, at 700 rows 119 for 116.
template <typename T> struct KeptType { typedef float V; };
template <> struct KeptType<bf16_t> { typedef f16_t V; };

struct EpiArgs {
    void* out;             // [M, N] of T
    long long ld_out;
    void* out_lo;          // EPI_GRAD: what rounding to `out` left, or null
    const void* bias;      // [N] of T (of float where bias_f32) or null
    const void* res;       // [M, N] of T or null
    long long ld_res;
    void* kept;            // [M, N] of KeptType, [M, N / 8] bytes, or codes
    float* kept_scale;     // [M, N / 128]
    signed char* out8;     // 8-bit form of `out`, or null
    float* out8_scale;
    // EPI_GRAD: sums of `out` over the rows, or null: [row blocks, N] of float,
    // or, where all rows are one block's, [N] of float or of T.  EPI_PLAIN: sums
    // of A over k, [M] of float or of T, or null.
    void* colsum;
    int act, keep, bias_f32, colsum_out;
};
enum ColsumOut { COLSUM_FLOAT = 0, COLSUM_T = 1 };

template <typename T> struct IsHalf { static constexpr bool value = true; };
template <> struct IsHalf<float> { static constexpr bool value = false; };

// What a chunk of 8 results needs from memory besides: the residual, or what is
// kept of the value before the activation.  It is fetched long before its use.
template <typename T> struct Extra {
    typename Chunk<T>::V v;
    typename Chunk<typename KeptType<T>::V>::V u;
    u32x2 codes;
    float scale;
    unsigned bits;
};

__device__ __forceinline__ const float* scale_at(const float* scales,
                                                 long long m, int n, int N) {
    const int groups = (N + ACT8_GROUP - 1) / ACT8_GROUP;
    return scales + m * groups + (n < N ? n / ACT8_GROUP : groups - 1);
}

// for row m, which is there, and columns from n on, which may not be
template <typename T, int EPI>
__device__ __forceinline__ void fetch_extra(Extra<T>& x, const EpiArgs& e,
                                            long long m, int n, int N) {
    if (EPI == EPI_FORWARD) {
        if (e.res) x.v = fetch8((const T*)e.res + m * e.ld_res, n, N);
    } else if (EPI == EPI_GRAD) {
        if (e.keep == KEEP_FULL) {
            x.u = fetch8((const typename KeptType<T>::V*)e.kept + m * N, n, N);
        } else if (e.keep == KEEP_8BIT) {
            const signed char* p = (const signed char*)e.kept + m * N;
            if (N >= 8) {
                x.codes = __builtin_bit_cast(u32x2,
                    *reinterpret_cast<const i8x8*>(
                        p + (n < N - 8 ? n : N - 8)));
            } else {
                i8x8 c;
                #pragma unroll
                for (int i = 0; i < 8; ++i)
                    c[i] = i < N ? p[i] : (signed char)0;
                x.codes = __builtin_bit_cast(u32x2, c);
            }
            x.scale = *scale_at(e.kept_scale, m, n, N);
        } else if (e.keep == KEEP_BITS) {
            const int bytes = (N + 7) >> 3, at = n >> 3;
            x.bits = ((const unsigned char*)e.kept)
                [m * bytes + (at < bytes ? at : bytes - 1)];
        }
    }
}

template <typename T>
__device__ __forceinline__ void load_bias(const EpiArgs& e, int n, int N,
                                          float* b) {
    if (!e.bias) {
        #pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = 0.0f;
    } else if (e.bias_f32) {
        load8((const float*)e.bias + n, N - n, b);
    } else {
        load8((const T*)e.bias + n, N - n, b);
    }
}

// 8 neighbouring results of row m from column n on; `left` of them are there
// (0 or less: none), all 8 where it is `whole` (the same for all lanes).  All
// 16 lanes of a group of 128 columns come together.
template <typename T, int EPI>
__device__ __forceinline__ void finish8(float* v, long long m, int n, int left,
                                        int N, bool whole, const EpiArgs& e,
                                        const float* bias, const Extra<T>& x,
                                        float* sums) {
    constexpr bool FAST = IsHalf<T>::value;
    const bool on = left > 0;
    if (EPI == EPI_PLAIN) {
        if (on) store8((T*)e.out + m * e.ld_out + n, left, v);
        return;
    }
    if (EPI == EPI_GRAD) {
        // what comes from the layer above is of type T: rounded as such
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)(T)v[i];
        if (e.keep == KEEP_BITS) {
            #pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!(x.bits >> i & 1)) v[i] = 0.0f;
        } else if (e.keep != KEEP_NONE) {
            float u[8];
            if (e.keep == KEEP_8BIT) {
                unpack8(__builtin_bit_cast(i8x8, x.codes), n, N, whole, u);
                #pragma unroll
                for (int i = 0; i < 8; ++i) u[i] *= x.scale;
            } else {
                unpack8(x.u, n, N, whole, u);
            }
            #pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= act_slope<FAST>(u[i], e.act);
        }
        if (!on) return;
        #pragma unroll
        for (int i = 0; i < 8; ++i)
            sums[i] += whole || i < left ? v[i] : 0.0f;
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
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] += bias[i];
        if (!whole && i >= left) v[i] = 0.0f;
    }
    if (e.keep == KEEP_BITS) {
        unsigned bits = 0;
        #pragma unroll
        for (int i = 0; i < 8; ++i) bits |= (v[i] <= 0.0f ? 0u : 1u) << i;
        if (on)
            ((unsigned char*)e.kept)[m * ((N + 7) >> 3) + (n >> 3)] =
                (unsigned char)bits;
    } else if (e.keep == KEEP_FULL) {
        if (on)
            store8((typename KeptType<T>::V*)e.kept + m * N + n, left, v);
    } else if (e.keep == KEEP_8BIT) {
        const Act8Scale s = act8_scale(max16(max8(v)));
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
    if (e.res) {
        float r[8];
        unpack8(x.v, n, N, whole, r);
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += r[i];
    }
    if (on) store8((T*)e.out + m * e.ld_out + n, left, v);
    if (e.out8) {
        #pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = whole || i < left ? (float)(T)v[i] : 0.0f;
        const Act8Scale s = act8_scale(max16(max8(v)));
        if (on) {
            store8_codes(e.out8 + m * N + n, left, v, s.by);
            if (n % ACT8_GROUP == 0)
                e.out8_scale[m * ((N + ACT8_GROUP - 1) / ACT8_GROUP) +
                             n / ACT8_GROUP] = s.scale;
        }
    }
}

// column sums of a block of rows: one of several, to be joined, or the result
template <typename T>
__device__ __forceinline__ void put_colsum(const EpiArgs& e, long long block,
                                           int n, int N, float t) {
    if (e.colsum_out == COLSUM_T) ((T*)e.colsum)[n] = (T)t;
    else ((float*)e.colsum)[block * N + n] = t;
}

// the sum of A over k, which is column N of the product: `left` columns on
template <typename T>
__device__ __forceinline__ void put_sum(const EpiArgs& e, long long m, int left,
                                        const float* v) {
    #pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i == left) put_colsum<T>(e, 0, (int)m, 0, v[i]);
}

// One block, one tile of C; blockIdx.y is the part of k.  With `part` the
// tile's fp32 sums go to part[blockIdx.y][m][n] (rows of ld_part values), and
// finish_kernel joins them; otherwise the epilogue follows at once.
//
// What the epilogues cost, 17920 x 10000 results in bf16, operands on lines, us of
// the whole kernel at k = 64 and 1500: no bias 147 and 560 (the results alone take
// 69 at a copy's rate), bias 151 and 565, with gelu too 253 and 657, and its input
// kept 262 and 714, or kept in 8 bits 293 and 704; a residual 242 and 637; a
// gradient through gelu from the kept input 355 and 770, from its 8 bits 328 and
// 755.  Gelu and its slope are bound by the vector unit, the others by memory.
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

    const int ones = EPI == EPI_PLAIN && e.colsum ? 1 : 0;
    G g(lds, a, b, M, N, K, m0, n0, ones);
    g.run(k0, k1);
    if (a.lo) {
        g.a.p = a.lo;
        stage_wait();
        g.run(k0, k1);
    }

    constexpr int CH = BN / 8;             // chunks of 8 columns
    constexpr int RS = G::THREADS / CH;    // rows a round
    constexpr int ROUNDS = WM * 32 / RS;
    const int c = threadIdx.x % CH, r0 = threadIdx.x / CH;
    const int n = n0 + 8 * c, left = N - n;
    const bool whole = n0 + BN <= N;
    float sums[8] = {0, 0, 0, 0, 0, 0, 0, 0}, bias[8];
    if (EPI == EPI_FORWARD && !part) load_bias<T>(e, n, N, bias);
    auto row_of = [&](int i, int round) {
        const int r = r0 + round * RS;
        return m0 + ((r >> 5) * G::TM + i) * 32 + (r & 31);
    };
    // Each pass's extras are on their way while the pass before is written, or a
    // pass would wait for memory four times.  The passes share their code: what
    // they do is long, and instructions come through a cache too.
    Extra<T> x[ROUNDS];
    auto fetch = [&](int i, int q) {
        const int m = row_of(i, q);
        fetch_extra<T, EPI>(x[q], e, m < M ? m : M - 1, n, N);
    };
    if (!part) {
        #pragma unroll
        for (int q = 0; q < ROUNDS; ++q) fetch(0, q);
    }
    #pragma unroll 1
    for (int i = 0; i < G::TM; ++i) {
        __syncthreads();
        #pragma unroll
        for (int j = 0; j < G::TM; ++j)
            if (i == j) g.stage_out(lds, j);
        __syncthreads();
        #pragma unroll
        for (int q = 0; q < ROUNDS; ++q) {
            const float* s = reinterpret_cast<const float*>(lds) +
                             (r0 + q * RS) * G::OUT_LD + 8 * c;
            float v[8];
            #pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = s[j];
            const int m = row_of(i, q);
            const int here = m < M ? left : 0;
            if (part) {
                if (m < M && left + ones > 0)
                    store8(part + ((long long)blockIdx.y * M + m) * ld_part +
                           n, left + ones, v);
            } else {
                if (ones && m < M) put_sum<T>(e, m, left, v);
                finish8<T, EPI>(v, m, n, here, N, whole, e, bias, x[q], sums);
                if (i + 1 < G::TM) fetch(i + 1, q);
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
            if (n0 + j < N) put_colsum<T>(e, bm, n0 + j, N, t);
        }
    }
}

// Few rows: 32 x 32 results a block, k shared out among its 8 waves, which wait
// for nobody before the end.  What bounds it is the weight's way from memory, so
// each wave has two steps of 128 bytes of k on their way at once, in registers:
// copies into LDS would need 16 KB of it a wave.  From there they go through LDS
// (one stage a wave, no barrier: a wave's accesses keep their order) to get from
// rows of memory to fragments.  20 x 1500 by 10000 in bf16, us: fragments
// straight from memory 17 (16 bytes of each of 32 rows are 64 requests to the
// cache, 128 bytes of 8 rows 16 at most), copies into two stages a wave 13, this
// 10.6; three steps leave registers for one block a unit only, 12.8.
#define THIN_WAVES 8
#define THIN_AHEAD 2
template <typename T, bool BA, int EPI>
__global__ __launch_bounds__(THIN_WAVES * 64, 4) void thin_kernel(
        Operand a, Operand b, int M, int N, int K, EpiArgs e) {
    typedef Gemm<T, 32, 32, 1, 1, true, BA> G;
    typedef typename G::TA TA;
    typedef typename G::TB TB;
    constexpr int E = TA::E, STAGE = G::STAGE > 32 * 36 * 4 ? G::STAGE
                                                           : 32 * 36 * 4;
    typedef T V __attribute__((ext_vector_type(E), aligned(sizeof(T))));
    typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
    __shared__ __attribute__((aligned(1024)))
        unsigned char lds[THIN_WAVES][STAGE];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int m0 = blockIdx.y * 32, n0 = blockIdx.x * 32;
    lds_byte* own = (lds_byte*)lds[wave];
    const int steps = (K + G::BK - 1) / G::BK;
    const int per = (steps + THIN_WAVES - 1) / THIN_WAVES;
    const int s0 = wave * per, s1 = s0 + per < steps ? s0 + per : steps;
    f32x16 acc;
    #pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
    V x[THIN_AHEAD][4], y[THIN_AHEAD][4];
    // this lane's chunk i: stored row and first value in it
    auto row_a = [&](int i) { return i * TA::RPC + lane / TA::CH; };
    auto row_b = [&](int i) { return i * TB::RPC + lane / TB::CH; };
    auto col_a = [&](int i) {
        return ((lane % TA::CH) ^ TA::swizzle(row_a(i))) * E;
    };
    auto col_b = [&](int i) {
        return ((lane % TB::CH) ^ TB::swizzle(row_b(i))) * E;
    };
    auto load = [&](int s, V* to_x, V* to_y) {
        if (s >= s1) return;
        const int k = s * G::BK;
        // rows that are not there: the last one's values, for results that are
        // not written
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = m0 + row_a(i);
            to_x[i] = fetch<V, E>(
                (const T*)a.p + (long long)(m < M ? m : M - 1) * a.ld,
                k + col_a(i), K);
            const int r = (BA ? n0 : k) + row_b(i), end = BA ? N : K;
            to_y[i] = fetch<V, E>(
                (const T*)b.p + (long long)(r < end ? r : end - 1) * b.ld,
                (BA ? k : n0) + col_b(i), BA ? K : N);
        }
    };
    const int at_a = TA::lane_at(lane, 0), at_b = TB::lane_at(lane, 0);
    auto use = [&](int s, const V* from_x, const V* from_y) {
        if (s >= s1) return;
        const int k = s * G::BK;
        const bool last = k + G::BK > K;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            V p = from_x[i], q = from_y[i];
            if (last) {
                p = settle<E>(p, k + col_a(i), K);
                if constexpr (BA) {
                    q = settle<E>(q, k + col_b(i), K);
                } else if (k + row_b(i) >= K) {
                    #pragma unroll
                    for (int j = 0; j < E; ++j) q[j] = (T)0.0f;
                }
            }
            if constexpr (!BA)
                if (n0 + 32 > N) q = settle<E>(q, n0 + col_b(i), N);
            *(lds_u32x4*)(own + i * 1024 + lane * 16) =
                __builtin_bit_cast(u32x4, p);
            *(lds_u32x4*)(own + TA::BYTES + i * 1024 + lane * 16) =
                __builtin_bit_cast(u32x4, q);
        }
        #pragma unroll
        for (int j = 0; j < 4; ++j)
            acc = Mfma<T>::go(TB::frag(own + TA::BYTES, at_b, j),
                              TA::frag(own, at_a, j), acc);
    };
    #pragma unroll
    for (int d = 0; d < THIN_AHEAD; ++d) load(s0 + d, x[d], y[d]);
    for (int s = s0; s < s1; s += THIN_AHEAD) {
        #pragma unroll
        for (int d = 0; d < THIN_AHEAD; ++d) {
            use(s + d, x[d], y[d]);
            load(s + d + THIN_AHEAD, x[d], y[d]);
        }
    }
    const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 8;
    const bool whole = n0 + 32 <= N;
    Extra<T> extra;
    float bias[8], sums[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (threadIdx.x < 128) {
        fetch_extra<T, EPI>(extra, e, m0 + r < M ? m0 + r : M - 1, n0 + c, N);
        if (EPI == EPI_FORWARD) load_bias<T>(e, n0 + c, N, bias);
    }
    constexpr int LD = 36;
    float* out = reinterpret_cast<float*>(lds[wave]) + (lane & 31) * LD +
                 4 * (lane >> 5);
    #pragma unroll
    for (int g = 0; g < 4; ++g) {
        f32x4 v;
        #pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = acc[4 * g + i];
        *reinterpret_cast<f32x4*>(out + 8 * g) = v;
    }
    __syncthreads();
    if (threadIdx.x < 128) {
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        #pragma unroll
        for (int w = 0; w < THIN_WAVES; ++w) {
            const float* p = reinterpret_cast<const float*>(lds[w]) + r * LD +
                             c;
            #pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += p[i];
        }
        finish8<T, EPI>(v, m0 + r, n0 + c, m0 + r < M ? N - n0 - c : 0, N,
                        whole, e, bias, extra, sums);
    }
    if (EPI == EPI_GRAD && e.colsum) {
        float* all = reinterpret_cast<float*>(lds[0]);
        __syncthreads();
        if (threadIdx.x < 128) {
            #pragma unroll
            for (int i = 0; i < 8; ++i) all[r * 32 + c + i] = sums[i];
        }
        __syncthreads();
        if (threadIdx.x < 32 && n0 + threadIdx.x < N) {
            float t = 0.0f;
            for (int i = 0; i < 32; ++i) t += all[i * 32 + threadIdx.x];
            put_colsum<T>(e, blockIdx.y, n0 + threadIdx.x, N, t);
        }
    }
}

// Joins `splits` partial products, `rows` (a multiple of 16) x 128 columns a
// block, in the order of k, and finishes them as the product's own epilogue
// would.  With one "product" of type S it takes a gradient back through an
// activation.  Bound by the partial sums' way from memory: 7 parts of 6000 x
// 1500 in 37 us, 6.8 TB/s of them from the last cache.
template <typename T, int EPI, typename S>
__global__ __launch_bounds__(256) void finish_kernel(
        const S* part, long long ld_part, int splits, int rows, int M, int N,
        EpiArgs e) {
    __shared__ float all[16 * 128];
    const int c = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const int n = blockIdx.y * 128 + 8 * c, left = N - n;
    const bool whole = (int)(blockIdx.y + 1) * 128 <= N;
    float sums[8] = {0, 0, 0, 0, 0, 0, 0, 0}, bias[8];
    if (EPI == EPI_FORWARD) load_bias<T>(e, n, N, bias);
    const int ones = EPI == EPI_PLAIN && e.colsum ? 1 : 0;
    for (int r = r0; r < rows; r += 16) {
        const long long m = (long long)blockIdx.x * rows + r;
        const long long there = m < M ? m : M - 1;
        const int here = m < M ? left : 0;
        Extra<T> x;
        fetch_extra<T, EPI>(x, e, there, n, N);
        float v[8];
        #pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
        #pragma unroll 4
        for (int s = 0; s < splits; ++s) {
            float w[8];
            unpack8(fetch8(part + ((long long)s * M + there) * ld_part, n,
                           N + ones), n, N + ones, whole, w);
            #pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += w[j];
        }
        if (ones && m < M) put_sum<T>(e, m, left, v);
        finish8<T, EPI>(v, m, n, here, N, whole, e, bias, x, sums);
    }
    if (EPI == EPI_GRAD && e.colsum) {
        #pragma unroll
        for (int j = 0; j < 8; ++j) all[r0 * 128 + 8 * c + j] = sums[j];
        __syncthreads();
        if (threadIdx.x < 128) {
            float t = 0.0f;
            for (int r = 0; r < 16; ++r) t += all[r * 128 + threadIdx.x];
            const int col = blockIdx.y * 128 + threadIdx.x;
            if (col < N) put_colsum<T>(e, blockIdx.x, col, N, t);
        }
    }
}
