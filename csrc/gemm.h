// Matrix products on the matrix cores, C[M, N] = A B with fp32 sums, for the
// three orders that a linear layer's step needs:
//
//   forward          y  = x W^T   A = x  along k, B = W  along k
//   input's gradient dx = p W     A = p  along k, B = W  across k
//   weight's         dW = p^T x   A = p  across k, B = x  across k
//
// "along k": each row of the operand is one output row, k contiguous.
// "across k": stored [k][rows], the output's rows contiguous.
#pragma once
#include "ffn_common.h"

template <typename T> struct Mfma;
template <> struct Mfma<bf16_t> {
    typedef bf16_t V __attribute__((ext_vector_type(8)));
    __device__ static __forceinline__ f32x16 go(V a, V b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <> struct Mfma<f16_t> {
    typedef f16_t V __attribute__((ext_vector_type(8)));
    __device__ static __forceinline__ f32x16 go(V a, V b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

// fp32: four products of depth 2.  The lower half of the lanes holds k = 0..3
// of a step of 8, the upper half k = 4..7, and product j takes j and 4 + j.
template <> struct Mfma<float> {
    typedef f32x4 V;
    __device__ static __forceinline__ f32x16 go(V a, V b, f32x16 c) {
        #pragma unroll
        for (int j = 0; j < 4; ++j)
            c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};

typedef __attribute__((address_space(3))) unsigned char lds_byte;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// 64 lanes x 16 bytes from memory straight into LDS at `lds` + 16 * lane.
// Offsets at or past the descriptor's size read as zeros.  Nothing here tells
// the compiler that the bytes are on their way: stage_wait() does, for all.
__device__ __forceinline__ void dma16(u32x4 desc, unsigned lds, int voff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\t"
                 "buffer_load_dwordx4 %1, %2, 0 offen lds"
                 :: "s"(lds), "v"(voff), "s"(desc) : "m0");
}

// every copy into LDS and every read of LDS by this wave is done, and the
// whole block has come here
__device__ __forceinline__ void stage_wait() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

__device__ __forceinline__ u32x4 buffer_desc(const void* p, long long bytes) {
    const unsigned long long a = (unsigned long long)p;
    const unsigned n = bytes <= 0 ? 0u
        : bytes > 0x7fffffffLL ? 0x7fffffffu : (unsigned)bytes;
    u32x4 d;
    d[0] = (unsigned)a;
    d[1] = (unsigned)(a >> 32) & 0xffffu;
    d[2] = n;
    d[3] = 0x00020000u;
    return d;
}

// One operand's tile of ROWS output rows x BK k in LDS, in chunks of 16 bytes
// (E values); BK is 128 bytes of k, taken in 4 steps of two chunks.
// along k:  row r is 128 bytes; its chunk c lies at c ^ (r & 7), so that the
//           8 lanes that read one chunk of 8 neighbouring rows hit all banks.
// across k: k-row of ROWS values; 16 bits: chunk c lies at c ^ 2 (k & 3), as
//           the transposing read takes 32 bytes of 4 neighbouring k at a
//           time; 32 bits: at c ^ 8 (k / 4 % 2), as the two halves of the
//           lanes read 128 bytes each, 4 k apart.
template <typename T, int ROWS, bool ALONG, int NWAVES>
struct Tile {
    static constexpr int SZ = sizeof(T), E = 16 / SZ, BK = 128 / SZ;
    static constexpr int BYTES = ROWS * 128;
    static constexpr int COPIES = BYTES / 1024 / NWAVES;  // of this wave
    static constexpr int ROWB = ALONG ? 128 : ROWS * SZ;
    static constexpr int CH = ROWB / 16;       // chunks in a stored row
    static constexpr int RPC = 1024 / ROWB;    // stored rows in one copy
    typedef typename Mfma<T>::V Frag;
    static_assert(BYTES % (1024 * NWAVES) == 0 && CH >= 8, "tile");

    __device__ static __forceinline__ int swizzle(int r) {
        return ALONG ? r & 7 : SZ == 2 ? (r & 3) << 1
                     : CH >= 16 ? (r & 4) << 1 : 0;
    }

    // byte offset, from the tile's first value, of what this lane copies
    __device__ static __forceinline__ int source(int wave, int lane, int i,
                                                 int ld) {
        const int r = (wave * COPIES + i) * RPC + lane / CH;
        const int p = lane % CH;
        return r * ld * SZ + (p ^ swizzle(r)) * 16;
    }
    __device__ static __forceinline__ unsigned target(int wave, int i) {
        return (wave * COPIES + i) * 1024;
    }
    // lane part of the address of 32 rows' fragments; `row` a multiple of 32
    __device__ static __forceinline__ int lane_at(int lane, int row) {
        if (ALONG) {
            return (row + (lane & 31)) * 128 +
                   (((lane >> 5) ^ (lane & 7)) << 4);
        } else if (SZ == 2) {
            const int q = lane >> 4, j = lane & 15;
            const int k = 8 * (q >> 1) + (j >> 2);
            const int c = (row >> 3) + (2 * (q & 1) + ((j & 3) >> 1));
            return k * ROWB + ((c ^ swizzle(k)) << 4) + (j & 1) * 8;
        } else {
            const int k = 4 * (lane >> 5), n = row + (lane & 31);
            return k * ROWB + (((n >> 2) ^ swizzle(k)) << 4) + (n & 3) * 4;
        }
    }
    // step s: this lane's row, k = E (2 s + lane / 32) + 0..E-1
    __device__ static __forceinline__ Frag frag(lds_byte* tile, int at,
                                                int s) {
        if constexpr (ALONG) {
            return *reinterpret_cast<
                __attribute__((address_space(3))) Frag*>(
                    tile + (at ^ (s << 5)));
        } else if constexpr (SZ == 4) {
            lds_byte* p = tile + at + s * 8 * ROWB;
            Frag f;
            #pragma unroll
            for (int j = 0; j < 4; ++j)
                f[j] = *(__attribute__((address_space(3))) float*)
                    (p + j * ROWB);
            return f;
        } else {
            lds_byte* p = tile + at + s * 16 * ROWB;
            union { Frag f; s16x4 h[2]; } u;
            u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
            u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4*)(p + 4 * ROWB));
            return u.f;
        }
    }
    // Mends the last tile of k, of which kv (1..BK) are there.  Rows along k
    // go on with the next row's values: cleared, since garbage times 0 may be
    // NaN.  A copy takes dwords, and one that ends past the operand reads as
    // 0: the operand's very last value, if its row is of odd length, comes
    // from `p`.  rows, len: output rows and, across k, their number here;
    // `p` is the tile's first value in memory.
    __device__ static __forceinline__ bool needs_mending(int kv, int rows,
                                                         bool odd) {
        return (ALONG && kv < BK) || (odd && rows <= ROWS);
    }
    __device__ static __forceinline__ void mend(lds_byte* tile, int tid,
                                                int nthreads, int kv, int rows,
                                                bool odd, const T* p, int ld) {
        typedef __attribute__((address_space(3))) T* lds_T;
        if (ALONG) {
            for (int i = tid; i < ROWS * 8; i += nthreads) {
                const int r = i >> 3, c = i & 7;
                lds_T q = (lds_T)(tile + r * 128 + ((c ^ (r & 7)) << 4));
                #pragma unroll
                for (int j = 0; j < E; ++j) {
                    if (E * c + j >= kv) q[j] = (T)0.0f;
                    else if (odd && r == rows - 1 && E * c + j == kv - 1)
                        q[j] = p[(long long)r * ld + kv - 1];
                }
            }
        } else if (odd && rows <= ROWS && tid == 0) {
            const int r = kv - 1, n = rows - 1;
            lds_T q = (lds_T)(tile + r * ROWB +
                              (((n / E) ^ swizzle(r)) << 4));
            q[n % E] = p[(long long)r * ld + n];
        }
    }
};

// what an operand is in memory: stored rows lie ld values apart.  A value may be
// the sum of two of the type, `lo` what rounding to `p` left: the products of
// both with the other operand are summed.
struct Operand {
    const void* p;
    long long ld;
    const void* lo;
};

// ---- block index -> output tile ---------------------------------------------
// Blocks go round the 8 dies in turn; each die gets neighbouring tiles, 8 tile
// rows by all columns at a time, so that its L2 holds what they share.
__device__ __forceinline__ void tile_of(int bid, int tm, int tn, int* m,
                                        int* n) {
    const int nb = tm * tn, x = bid & 7;
    const int per = nb >> 3, more = nb & 7;
    const int id = (x < more ? x * (per + 1) : x * per + more) + (bid >> 3);
    const int G = 8;
    const int group = id / (G * tn), first = group * G;
    const int h = tm - first < G ? tm - first : G;
    const int in = id - group * G * tn;
    *m = first + in % h;
    *n = in / h;
}

// ---- main loop ---------------------------------------------------------------
template <typename T, int BM, int BN, int WM, int WN, bool AA, bool BA>
struct Gemm {
    static constexpr int SZ = sizeof(T), BK = 128 / SZ;
    static constexpr int NW = WM * WN, THREADS = NW * 64;
    static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
    typedef Tile<T, BM, AA, NW> TA;
    typedef Tile<T, BN, BA, NW> TB;
    static constexpr int STAGE = TA::BYTES + TB::BYTES;
    // fp32 results on their way to the epilogue: WM * 32 rows at a time
    static constexpr int OUT_LD = BN + 4;
    static constexpr int OUT_BYTES = WM * 32 * OUT_LD * 4;
    static constexpr int LDS =
        2 * STAGE > OUT_BYTES ? 2 * STAGE : OUT_BYTES;

    // acc[i][j]: tile rows m = (wm TM + i) 32 + lane % 32,
    //            columns n = (wn TN + j) 32 + 4 (lane / 32) + e % 4 + 8 (e / 4)
    // acc += a b over k0..k1; the block's LDS is free
    __device__ static __forceinline__ void loop(
            unsigned char* lds, Operand a, Operand b, int m0, int n0, int M,
            int N, int K, int k0, int k1, f32x16 acc[TM][TN]) {
        const int tid = threadIdx.x, lane = tid & 63;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int wm = wave / WN, wn = wave % WN;
        lds_byte* base = (lds_byte*)lds;
        const unsigned base_at = (unsigned)(unsigned long long)base;

        int va[TA::COPIES], vb[TB::COPIES], fa[TM], fb[TN];
        #pragma unroll
        for (int i = 0; i < TA::COPIES; ++i)
            va[i] = TA::source(wave, lane, i, (int)a.ld);
        #pragma unroll
        for (int i = 0; i < TB::COPIES; ++i)
            vb[i] = TB::source(wave, lane, i, (int)b.ld);
        #pragma unroll
        for (int i = 0; i < TM; ++i)
            fa[i] = TA::lane_at(lane, (wm * TM + i) * 32);
        #pragma unroll
        for (int j = 0; j < TN; ++j)
            fb[j] = TB::lane_at(lane, (wn * TN + j) * 32);

        // first value of the operand's tile at k, and the bytes from there to
        // the end of the operand
        auto at_a = [&](int k) {
            return (const T*)a.p + (AA ? (long long)m0 * a.ld + k
                                       : (long long)k * a.ld + m0);
        };
        auto at_b = [&](int k) {
            return (const T*)b.p + (BA ? (long long)n0 * b.ld + k
                                       : (long long)k * b.ld + n0);
        };
        auto desc_a = [&](int k) {
            return buffer_desc(at_a(k), SZ * (AA
                ? (M - m0 - 1) * a.ld + K - k : (K - k - 1) * a.ld + M - m0));
        };
        auto desc_b = [&](int k) {
            return buffer_desc(at_b(k), SZ * (BA
                ? (N - n0 - 1) * b.ld + K - k : (K - k - 1) * b.ld + N - n0));
        };
        auto copy = [&](int k, int buf) {
            const u32x4 da = desc_a(k), db = desc_b(k);
            const unsigned at = base_at + buf * STAGE;
            #pragma unroll
            for (int i = 0; i < TA::COPIES; ++i)
                dma16(da, at + TA::target(wave, i), va[i]);
            #pragma unroll
            for (int i = 0; i < TB::COPIES; ++i)
                dma16(db, at + TA::BYTES + TB::target(wave, i), vb[i]);
        };

        auto multiply = [&](int buf) {
            lds_byte* ta = base + buf * STAGE;
            lds_byte* tb = ta + TA::BYTES;
            #pragma unroll
            for (int s = 0; s < 4; ++s) {
                typename Mfma<T>::V xa[TM], xb[TN];
                #pragma unroll
                for (int i = 0; i < TM; ++i) xa[i] = TA::frag(ta, fa[i], s);
                #pragma unroll
                for (int j = 0; j < TN; ++j) xb[j] = TB::frag(tb, fb[j], s);
                #pragma unroll
                for (int i = 0; i < TM; ++i)
                    #pragma unroll
                    for (int j = 0; j < TN; ++j)
                        acc[i][j] = Mfma<T>::go(xb[j], xa[i], acc[i][j]);
            }
        };

        copy(k0, 0);
        int buf = 0, k = k0;
        for (; k + BK < k1; k += BK, buf ^= 1) {
            stage_wait();
            copy(k + BK, buf ^ 1);
            multiply(buf);
        }
        stage_wait();
        if (k1 == K) {
            const bool oa = SZ == 2 && ((AA ? K : M) & 1);
            const bool ob = SZ == 2 && ((BA ? K : N) & 1);
            const bool ma = TA::needs_mending(K - k, M - m0, oa);
            const bool mb = TB::needs_mending(K - k, N - n0, ob);
            if (ma)
                TA::mend(base + buf * STAGE, tid, THREADS, K - k, M - m0, oa,
                         at_a(k), (int)a.ld);
            if (mb)
                TB::mend(base + buf * STAGE + TA::BYTES, tid, THREADS, K - k,
                         N - n0, ob, at_b(k), (int)b.ld);
            if (ma || mb) stage_wait();
        }
        multiply(buf);
    }

    // rows (w 32 + 0..31 for each of the WM wave rows) of pass i, in fp32
    __device__ static __forceinline__ void stage_out(
            unsigned char* lds, int i, const f32x16* acc) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int wm = wave / WN, wn = wave % WN;
        float* out = reinterpret_cast<float*>(lds) +
                     (wm * 32 + (lane & 31)) * OUT_LD +
                     wn * TN * 32 + 4 * (lane >> 5);
        #pragma unroll
        for (int j = 0; j < TN; ++j)
            #pragma unroll
            for (int g = 0; g < 4; ++g) {
                f32x4 v;
                #pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[j][4 * g + e];
                *reinterpret_cast<f32x4*>(out + j * 32 + 8 * g) = v;
            }
    }
};
