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

// 64 lanes x 16 bytes from memory straight into LDS at `lds` + PLUS + 16 * lane.
// Offsets (both parts of it) at or past the descriptor's size read as zeros.
// Nothing here tells the compiler that the bytes are on their way: stage_wait()
// does, for all.  m0 is set anew by each copy; it is reserved, cannot be named as
// clobbered, and the compiler's own code for these kernels does not touch it.
template <int PLUS>
__device__ __forceinline__ void dma16(u32x4 desc, unsigned lds, int voff,
                                      unsigned soff) {
    asm volatile("s_add_u32 m0, %0, %4\n\ts_nop 0\n\t"
                 "buffer_load_dwordx4 %1, %2, %3 offen lds"
                 :: "s"(lds), "v"(voff), "s"(desc), "s"(soff), "n"(PLUS)
                 : "scc");
}

// every copy into LDS and every read of LDS by this wave is done, and the whole
// block has come here
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
// LDS gives 256 bytes a cycle where the 16-byte chunks of a group of lanes fall
// on different 16 bytes of 256, so the chunks of a stored row are permuted:
// along k:  row r is 128 bytes, its chunk c lies at c ^ (r / 2 % 8).  A read of
//           16 bytes a lane goes in four groups of 16 lanes, the first of them
//           lanes 0-3, 12-15, 20-23 and 24-27: there r / 2 takes each value
//           mod 8 once for odd and once for even r.
// across k: a stored row is one k.  16 bits: chunk c lies at c ^ 4 (k % 4), as
//           the transposing read takes 32 bytes of 4 neighbouring k for each
//           of 2 neighbouring blocks of 16 columns (rows of 128 bytes: c ^ 4
//           (k / 2 % 2), of 64 bytes: c); 32 bits: at c ^ 8 (k / 4 % 2), as the two halves of
//           the lanes read 128 bytes each, 4 k apart.
// Counters: conflicts fell from 97 to 1 of 100 read cycles at 8192^3; with the
// epilogue's passes through LDS they are 2 to 15 of 100, the most where k is short.
template <typename T, int ROWS, bool ALONG, int NWAVES>
struct Tile {
    static constexpr int SZ = sizeof(T), E = 16 / SZ, BK = 128 / SZ;
    static constexpr int BYTES = ROWS * 128;
    static constexpr int COPIES = BYTES / 1024 / NWAVES;  // of this wave
    static constexpr int ROWB = ALONG ? 128 : ROWS * SZ;
    static constexpr int CH = ROWB / 16;       // chunks in a stored row
    static constexpr int RPC = 1024 / ROWB;    // stored rows in one copy
    typedef typename Mfma<T>::V Frag;
    static_assert(BYTES % (1024 * NWAVES) == 0 && CH >= 4, "tile");

    __device__ static __forceinline__ int swizzle(int r) {
        return ALONG ? (r >> 1) & 7
             : SZ == 2 ? (CH >= 16 ? (r & 3) << 2 : CH == 8 ? (r & 2) << 1 : 0)
                       : CH >= 16 ? (r & 4) << 1 : 0;
    }

    // byte offset, from the tile's first value, of what this lane copies
    __device__ static __forceinline__ int source(int wave, int lane, int i,
                                                 int ld) {
        const int r = (wave * COPIES + i) * RPC + lane / CH;
        const int p = lane % CH;
        return r * ld * SZ + (p ^ swizzle(r)) * 16;
    }
    // lane part of the address of 32 rows' fragments; `row` a multiple of 32
    __device__ static __forceinline__ int lane_at(int lane, int row) {
        if (ALONG) {
            return (row + (lane & 31)) * 128 +
                   (((lane >> 5) ^ ((lane >> 1) & 7)) << 4);
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
                lds_T q = (lds_T)(tile + r * 128 + ((c ^ swizzle(r)) << 4));
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
// rows by all columns at a time, so that its L2 holds what they share (4 or 16
// rows: 1 % slower over a block's training step of 17920 rows).
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

// ---- the product ----------------------------------------------------------------
// Sums of one tile BM x BN in registers, WM x WN waves.  Two stages of LDS: while
// one is multiplied, the next tile of k comes into the other.
//
// What bounds it: copies into LDS come at 8 to 12 TB/s over all units, the more
// the fewer lines of 128 bytes they touch.  256 x 256 tiles multiply a byte 128
// times and need 12 at 1.5 PFLOP/s, 64 x 64 tiles 32 times: small products are
// better split over k than over tiles, and more stages (4 and 6, tried) gain
// nothing.  One barrier a tile of k; a wave loads its fragments a step ahead,
// among the products of the step before, so that neither the barrier nor LDS's
// latency shows.  Measured, bf16 along/along, us at 8192^3: each step's
// fragments loaded just before its products 890; a step ahead 817 (1345
// TFLOP/s); two groups of waves that take turns at loading and multiplying 840;
// 4 waves of 128 x 128 instead of 8 of 128 x 64 980.  fp32 at 4096^3: 994 and
// 943 (146 TFLOP/s).  A block that went on to a next tile, its first copies
// under way while this one is written, gained nothing.
template <typename T, int BM, int BN, int WM, int WN, bool AA, bool BA>
struct Gemm {
    static constexpr int SZ = sizeof(T), BK = 128 / SZ;
    static constexpr int NW = WM * WN, THREADS = NW * 64;
    static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
    typedef Tile<T, BM, AA, NW> TA;
    typedef Tile<T, BN, BA, NW> TB;
    static constexpr int STAGE = TA::BYTES + TB::BYTES;
    static constexpr int COPIES = TA::COPIES + TB::COPIES, LOADS = TM + TN;
    // fp32 results on their way to the epilogue: WM * 32 rows at a time
    static constexpr int OUT_LD = BN + 4;
    static constexpr int OUT_BYTES = WM * 32 * OUT_LD * 4;
    static constexpr int LDS =
        2 * STAGE > OUT_BYTES ? 2 * STAGE : OUT_BYTES;

    Operand a, b;
    int M, N, K, m0, n0;
    int tid, lane, wave, wm, wn;
    lds_byte* base;
    unsigned base_at;
    int va[TA::COPIES], vb[TB::COPIES], fa[TM], fb[TN];
    u32x4 da, db;
    unsigned sa, sb, step_a, step_b, to;
    int ka, kb;
    typename Mfma<T>::V xa[2][TM], xb[2][TN];
    f32x16 acc[TM][TN];
    // Both operands across k: B may go on with a column of ones behind its N,
    // where the last tile has room, so that C's column N is the sum of A over k.
    static constexpr bool ONES = !AA && !BA;
    bool one[TN], any_one;     // this lane's column of B is the one of ones

    __device__ __forceinline__ Gemm(unsigned char* lds, const Operand& a_,
                                    const Operand& b_, int M_, int N_, int K_,
                                    int m0_, int n0_, bool ones)
        : a(a_), b(b_), M(M_), N(N_), K(K_), m0(m0_), n0(n0_) {
        tid = threadIdx.x;
        lane = tid & 63;
        wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        wm = wave / WN;
        wn = wave % WN;
        base = (lds_byte*)lds;
        base_at = (unsigned)(unsigned long long)base;
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
        #pragma unroll
        for (int j = 0; j < TN; ++j)
            one[j] = ONES && ones &&
                     n0 + (wn * TN + j) * 32 + (lane & 31) == N;
        any_one = ONES && ones && N >= n0 + wn * TN * 32 &&
                  N < n0 + (wn + 1) * TN * 32;
        #pragma unroll
        for (int i = 0; i < TM; ++i)
            #pragma unroll
            for (int j = 0; j < TN; ++j)
                #pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    }

    // first value of the operand's tile at k
    __device__ __forceinline__ const T* at_a(int k) const {
        return (const T*)a.p + (AA ? (long long)m0 * a.ld + k
                                   : (long long)k * a.ld + m0);
    }
    __device__ __forceinline__ const T* at_b(int k) const {
        return (const T*)b.p + (BA ? (long long)n0 * b.ld + k
                                   : (long long)k * b.ld + n0);
    }
    // Copies come from a descriptor that starts at a tile of k and ends with its
    // operand, by offsets that grow with k; across k, where 32 bits would not
    // hold them, it starts again after each 2^30 bytes.
    __device__ __forceinline__ void aim_a(int k) {
        da = buffer_desc(at_a(k), SZ * (AA
            ? (M - m0 - 1) * a.ld + K - k : (K - k - 1) * a.ld + M - m0));
        sa = 0;
        ka = k;
    }
    __device__ __forceinline__ void aim_b(int k) {
        db = buffer_desc(at_b(k), SZ * (BA
            ? (N - n0 - 1) * b.ld + K - k : (K - k - 1) * b.ld + N - n0));
        sb = 0;
        kb = k;
    }
    // the copies that follow are of the next tile of k, into stage buf
    __device__ __forceinline__ void advance(int buf) {
        sa += step_a;
        sb += step_b;
        if (!AA && sa >= (1u << 30)) aim_a(ka + sa / (unsigned)(a.ld * SZ));
        if (!BA && sb >= (1u << 30)) aim_b(kb + sb / (unsigned)(b.ld * SZ));
        to = base_at + buf * STAGE;
    }
    template <int I>
    __device__ __forceinline__ void copy_one() {
        if constexpr (I < TA::COPIES)
            dma16<I * 1024>(da, to + wave * TA::COPIES * 1024, va[I], sa);
        else
            dma16<TA::BYTES + (I - TA::COPIES) * 1024>(
                db, to + wave * TB::COPIES * 1024, vb[I - TA::COPIES], sb);
    }
    template <int FROM, int TO>
    __device__ __forceinline__ void copy() {
        if constexpr (FROM < TO) {
            copy_one<FROM>();
            copy<FROM + 1, TO>();
        }
    }
    __device__ __forceinline__ void load_one(lds_byte* tile, int s, int set,
                                             int i) {
        if (i < TN) xb[set][i] = TB::frag(tile + TA::BYTES, fb[i], s);
        else xa[set][i - TN] = TA::frag(tile, fa[i - TN], s);
    }
    template <int I, int CUR, bool LOAD, int FROM, int COUNT>
    __device__ __forceinline__ void step_rows(lds_byte* next, int ns) {
        if constexpr (I < TM) {
            if (ONES && I == 0 && any_one) {
                // by waves that have the column only: its 4 instructions for
                // each fragment cost a tenth of the product
                #pragma unroll
                for (int j = 0; j < TN; ++j)
                    #pragma unroll
                    for (int e = 0; e < 16 / SZ; ++e)
                        xb[CUR][j][e] = one[j] ? (T)1.0f : xb[CUR][j][e];
            }
            if (LOAD) {
                #pragma unroll
                for (int l = I * LOADS / TM; l < (I + 1) * LOADS / TM; ++l)
                    load_one(next, ns, CUR ^ 1, l);
            }
            copy<FROM + I * COUNT / TM, FROM + (I + 1) * COUNT / TM>();
            #pragma unroll
            for (int j = 0; j < TN; ++j)
                acc[I][j] = Mfma<T>::go(xb[CUR][j], xa[CUR][I], acc[I][j]);
            __builtin_amdgcn_sched_barrier(0);
            step_rows<I + 1, CUR, LOAD, FROM, COUNT>(next, ns);
        }
    }
    // products of fragment set CUR; among them the loads of step ns from
    // `next` into the other set, and COUNT copies from number FROM on
    template <int CUR, bool LOAD, int FROM, int COUNT>
    __device__ __forceinline__ void step(lds_byte* next, int ns) {
        step_rows<0, CUR, LOAD, FROM, COUNT>(next, ns);
    }
    // the last tile of k has come
    __device__ __forceinline__ void mend(int k, int k1, int buf) {
        if (k1 != K) return;
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

    // acc += a b over k0..k1; nobody uses the block's LDS
    __device__ __forceinline__ void run(int k0, int k1) {
        step_a = (unsigned)(SZ * BK * (AA ? 1 : a.ld));
        step_b = (unsigned)(SZ * BK * (BA ? 1 : b.ld));
        aim_a(k0);
        aim_b(k0);
        to = base_at;
        copy<0, COPIES>();
        // Fragments a step ahead.  A stage is read until the barrier before
        // its last step; from there on the tile after the next may come into
        // it, half of it at once and half in the next tile's first step.
        constexpr int HALF = COPIES / 2, REST = COPIES - HALF;
        int buf = 0, k = k0;
        const bool one = k0 + BK >= k1;
        stage_wait();
        if (one) {
            mend(k, k1, 0);
        } else {
            advance(1);
            copy<0, HALF>();
        }
        #pragma unroll
        for (int l = 0; l < LOADS; ++l) load_one(base, 0, 0, l);
        for (; k + 2 * BK < k1; k += BK, buf ^= 1) {
            lds_byte* p = base + buf * STAGE;
            step<0, true, HALF, REST>(p, 1);
            step<1, true, 0, 0>(p, 2);
            step<0, true, 0, 0>(p, 3);
            stage_wait();
            advance(buf);
            step<1, true, 0, HALF>(base + (buf ^ 1) * STAGE, 0);
        }
        if (!one) {
            lds_byte* p = base + buf * STAGE;
            step<0, true, HALF, REST>(p, 1);
            step<1, true, 0, 0>(p, 2);
            step<0, true, 0, 0>(p, 3);
            stage_wait();
            buf ^= 1;
            mend(k + BK, k1, buf);
            step<1, true, 0, 0>(base + buf * STAGE, 0);
        }
        lds_byte* p = base + buf * STAGE;
        step<0, true, 0, 0>(p, 1);
        step<1, true, 0, 0>(p, 2);
        step<0, true, 0, 0>(p, 3);
        step<1, false, 0, 0>(p, 0);
    }

    // acc[i][j]: tile rows m = (wm TM + i) 32 + lane % 32,
    //            columns n = (wn TN + j) 32 + 4 (lane / 32) + e % 4 + 8 (e / 4)
    // Pass i: rows 0..31 of (w TM + i) 32 for each of the WM wave rows, fp32.
    __device__ __forceinline__ void stage_out(unsigned char* lds, int i) {
        float* out = reinterpret_cast<float*>(lds) +
                     (wm * 32 + (lane & 31)) * OUT_LD +
                     wn * TN * 32 + 4 * (lane >> 5);
        #pragma unroll
        for (int j = 0; j < TN; ++j)
            #pragma unroll
            for (int g = 0; g < 4; ++g) {
                f32x4 v;
                #pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * g + e];
                *reinterpret_cast<f32x4*>(out + j * 32 + 8 * g) = v;
            }
    }
};
