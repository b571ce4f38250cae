// Products of linear layers: choice of tile and of the split over k, launches.
#include <hip/hip_runtime.h>
#include "ffn_launch.h"
#include "linear_kernels.h"

namespace ffn {

// up to this many rows of an operand along k go to thin_kernel
#define THIN_ROWS 64

struct Plan { int tile, splits; };

// Estimated us of the product with each tile and number of parts of k; the
// least one wins.  A tile's step over 128 bytes of k takes `step` us, `more`
// longer for each further block (up to `at_once`) that shares its compute unit,
// and a block spends `over` us outside its loop; parts cost `join` us and their
// way to memory and back at `rate` bytes a us.  The numbers fit 74 products of
// 1 to 17920 rows, each timed with all tiles and up to 16 parts: the choice is
// 1.5 % slower than the best one in the mean, and 19 % at worst.
static Plan plan_product(long long M, long long N, long long K, int size,
                         bool quantises) {
    struct Shape { int tile, at_once; float over, step, more; };
    static const Shape half[] = {{256, 1, 10.3f, 1.16f, 0.0f},
                                 {128, 2, 4.5f, 0.65f, 0.24f},
                                 {64, 5, 3.05f, 0.284f, 0.177f}};
    static const Shape full[] = {{128, 2, 5.6f, 1.8f, 0.58f},
                                 {64, 5, 3.05f, 0.49f, 0.33f}};
    const Shape* shapes = size == 2 ? half : full;
    const int n = size == 2 ? 3 : 2;
    const float join = size == 2 ? 5.3f : 3.2f;
    const float rate = size == 2 ? 5.44e6f : 3.3e6f;
    const long long units = 256;
    const long long steps = (K * size + 127) / 128;
    Plan best{shapes[0].tile, 1};
    float least = 1e30f;
    for (int i = 0; i < n; ++i) {
        const Shape& s = shapes[i];
        if (quantises && s.tile < ACT8_GROUP) continue;
        const long long tiles = ((M + s.tile - 1) / s.tile) *
                                ((N + s.tile - 1) / s.tile);
        for (int parts = 1; parts <= 16 && parts <= steps; ++parts) {
            const long long per = (steps + parts - 1) / parts;
            if ((steps + per - 1) / per != parts) continue;
            const long long all = tiles * parts, slots = units * s.at_once;
            const long long rest = all % slots;
            float t = all / slots *
                (per * (s.step + s.more * (s.at_once - 1)) + s.over);
            if (rest)
                t += per * (s.step + s.more * ((rest - 1) / units)) + s.over;
            if (parts > 1) t += join + 8.0f * M * N * parts / rate;
            if (t < least) { least = t; best = {s.tile, parts}; }
        }
    }
    return best;
}

// rows a block of finish_kernel: as many as leave it 512 blocks, up to 64
static int finish_rows(long long M, long long N) {
    int rows = 64;
    while (rows > 16 && (M + rows - 1) / rows * ((N + 127) / 128) < 512)
        rows /= 2;
    return rows;
}

template <typename T, int BM, int BN, int WM, int WN, bool AA, bool BA,
          int EPI>
static void launch(const Operand& a, const Operand& b, int M, int N, int K,
                   int splits, EpiArgs e, const at::Tensor& like,
                   long long* blocks) {
    typedef Gemm<T, BM, BN, WM, WN, AA, BA> G;
    const auto s = stream_now();
    const long long tm = (M + BM - 1) / BM, tn = (N + BN - 1) / BN;
    TORCH_CHECK(tm * tn < (1LL << 32) / G::THREADS, "product of ", M, " x ", N,
                " is too large");
    const int steps = (K + G::BK - 1) / G::BK;
    const int per = (steps + splits - 1) / splits;
    const int parts = (steps + per - 1) / per;
    // the column of ones has to find room in the last tile
    if (EPI == EPI_PLAIN && N % BN == 0) e.colsum = nullptr;
    const int wide = EPI == EPI_PLAIN && e.colsum ? N + 1 : N;
    const long long ld_part = (wide + 3) / 4 * 4;
    at::Tensor part;
    if (parts > 1)
        part = at::empty({parts, M, ld_part},
                         like.options().dtype(at::kFloat));
    float* pp = parts > 1 ? part.data_ptr<float>() : nullptr;
    const dim3 grid((unsigned)(tm * tn), (unsigned)parts);
    auto k = gemm_kernel<T, BM, BN, WM, WN, AA, BA, EPI>;
    hipLaunchKernelGGL(k, grid, G::THREADS, G::LDS, s, a, b, M, N, K, per * G::BK, pp,
                                       ld_part, e);
    FFN_OK();
    *blocks = tm;
    if (parts > 1) {
        const int rows = finish_rows(M, N);
        const dim3 fgrid((unsigned)((M + rows - 1) / rows),
                         (unsigned)((wide + 127) / 128));
        auto f = finish_kernel<T, EPI, float>;
        hipLaunchKernelGGL(f, fgrid, 256, 0, s, pp, ld_part, parts, rows, M, N,
                           e);
        FFN_OK();
        *blocks = fgrid.x;
    }
    if (EPI == EPI_PLAIN) *blocks = e.colsum ? 1 : 0;
}

// C = A B with the epilogue; `blocks`: rows of e.colsum that were written (none
// where EPI_PLAIN's sums found no room)
template <bool AA, bool BA, int EPI>
static void product(at::ScalarType type, const Operand& a, const Operand& b,
                    long long M, long long N, long long K, EpiArgs e,
                    const at::Tensor& like, long long* blocks) {
    const bool quantises = EPI == EPI_FORWARD &&
                           (e.out8 || e.keep == KEEP_8BIT);
    if constexpr (AA) {
        if (M <= THIN_ROWS && !quantises && !a.lo) {
            const dim3 grid((unsigned)((N + 31) / 32),
                            (unsigned)((M + 31) / 32));
            FFN_TYPES(type,
                auto k = thin_kernel<T, BA, EPI>;
                hipLaunchKernelGGL(k, grid, THIN_WAVES * 64, 0, stream_now(),
                                   a, b, (int)M, (int)N, (int)K, e));
            FFN_OK();
            *blocks = grid.y;
            return;
        }
    }
    const Plan p = plan_product(M, N, a.lo ? 2 * K : K,
                                type == at::kFloat ? 4 : 2, quantises);
    FFN_TYPES(type,
        if (p.tile == 256) {
            if constexpr (sizeof(T) == 2)
                launch<T, 256, 256, 2, 4, AA, BA, EPI>(
                    a, b, (int)M, (int)N, (int)K, p.splits, e, like, blocks);
        } else if (p.tile == 128) {
            launch<T, 128, 128, 2, 2, AA, BA, EPI>(
                a, b, (int)M, (int)N, (int)K, p.splits, e, like, blocks);
        } else {
            launch<T, 64, 64, 2, 2, AA, BA, EPI>(
                a, b, (int)M, (int)N, (int)K, p.splits, e, like, blocks);
        });
}

static Operand operand(const Mat& m) {
    return {m.t.data_ptr(), m.ld, m.lo.defined() ? m.lo.data_ptr() : nullptr};
}

static Kept empty_kept(int act, bool act8, long long rows, long long dim,
                       const at::Tensor& like) {
    Kept u;
    if (act == ACT_RELU) {
        u.how = KEEP_BITS;
        u.data = at::empty({rows, (dim + 7) / 8},
                           like.options().dtype(at::kByte));
    } else if (act != ACT_NONE && act8) {
        Packed p = empty_packed(rows, dim, like);
        u.how = KEEP_8BIT;
        u.data = p.codes;
        u.scales = p.scales;
    } else if (act != ACT_NONE) {
        u.how = KEEP_FULL;
        // KeptType
        const auto t = like.scalar_type() == at::kBFloat16 ? at::kHalf
                                                           : at::kFloat;
        u.data = at::empty({rows, dim}, like.options().dtype(t));
    }
    return u;
}

static void set_kept(EpiArgs& e, const Kept& u) {
    e.keep = u.how;
    e.kept = u.data.defined() ? u.data.data_ptr() : nullptr;
    e.kept_scale = u.scales.defined() ? u.scales.data_ptr<float>() : nullptr;
}

LinearOut linear_forward(const Mat& x, const Mat& w, const at::Tensor& bias,
                         const Mat* res, int act, bool keep, bool act8,
                         bool keep_y8, at::IntArrayRef sizes) {
    LinearOut o;
    const long long M = x.rows, N = w.rows;
    o.y = sizes.empty() ? empty_rows(M, N, x.t, x.t.scalar_type())
                        : empty_result(sizes, x.t, x.t.scalar_type());
    if (keep) o.u = empty_kept(act, act8, M, N, x.t);
    if (keep_y8) o.y8 = empty_packed(M, N, x.t);
    if (!M) return o;
    EpiArgs e{};
    e.out = o.y.t.data_ptr();
    e.ld_out = o.y.ld;
    if (bias.defined()) {
        e.bias = bias.data_ptr();
        e.bias_f32 = bias.scalar_type() == at::kFloat;
    }
    if (res) {
        e.res = res->t.data_ptr();
        e.ld_res = res->ld;
    }
    set_kept(e, o.u);
    if (keep_y8) {
        e.out8 = (signed char*)o.y8.codes.data_ptr();
        e.out8_scale = o.y8.scales.data_ptr<float>();
    }
    e.act = act;
    long long blocks;
    product<true, true, EPI_FORWARD>(x.t.scalar_type(), operand(x), operand(w),
                                     M, N, x.dim, e, x.t, &blocks);
    return o;
}

// Sums over the rows on their way: partial ones, one row of them for each block
// of rows, or where one block has all rows (`one`) the result itself.
struct Colsum {
    at::Tensor out, part;
    void aim(EpiArgs& e, long long rows, long long dim, const at::Tensor& bias,
             bool one) {
        out = at::empty({dim}, bias.options());
        if (one) {
            e.colsum = out.data_ptr();
            e.colsum_out = bias.scalar_type() == at::kFloat ? COLSUM_FLOAT
                                                            : COLSUM_T;
            return;
        }
        // of 64 rows or more, or finish_kernel's
        const int least = rows <= THIN_ROWS ? 16 : finish_rows(rows, dim);
        part = at::empty({(rows + least - 1) / least, dim},
                         bias.options().dtype(at::kFloat));
        e.colsum = part.data_ptr();
    }
    at::Tensor join(long long blocks) {
        if (part.defined()) sum_partials(part, blocks, out);
        return out;
    }
};

static Mat empty_grad(long long rows, long long dim, const at::Tensor& like,
                      bool split, const Kept& u) {
    Mat p = empty_rows(rows, dim, like, like.scalar_type());
    // through relu a value passes whole; fp32 rounds as the sums themselves do
    if (split && (u.how == KEEP_FULL || u.how == KEEP_8BIT) &&
        like.scalar_type() != at::kFloat)
        p.lo = empty_rows(rows, dim, like, like.scalar_type()).t;
    return p;
}

Mat through_act(const Mat& dy, int act, const Kept& u, const at::Tensor& bias,
                at::Tensor* dbias, bool split) {
    if (act == ACT_NONE) return dy;
    Mat p = empty_grad(dy.rows, dy.dim, dy.t, split, u);
    if (!p.rows) {
        if (bias.defined()) *dbias = at::zeros_like(bias);
        return p;
    }
    EpiArgs e{};
    e.out = p.t.data_ptr();
    e.out_lo = p.lo.defined() ? p.lo.data_ptr() : nullptr;
    e.ld_out = p.ld;
    e.act = act;
    set_kept(e, u);
    // all of a few rows in one block a column: their sums are the gradient of the
    // bias at once, where a second launch costs 4 us and blocks of 16 rows win 1
    const int rows = bias.defined() && p.rows <= 64 ? 64
                                                    : finish_rows(p.rows, p.dim);
    Colsum sum;
    if (bias.defined()) sum.aim(e, p.rows, p.dim, bias, p.rows <= rows);
    const dim3 grid((unsigned)((p.rows + rows - 1) / rows),
                    (unsigned)((p.dim + 127) / 128));
    FFN_TYPES(dy.t.scalar_type(),
        auto f = finish_kernel<T, EPI_GRAD, T>;
        hipLaunchKernelGGL(f, grid, 256, 0, stream_now(), (const T*)dy.t.data_ptr(), dy.ld, 1, rows,
                                          (int)p.rows, (int)p.dim, e));
    FFN_OK();
    if (bias.defined()) *dbias = sum.join(grid.x);
    return p;
}

Mat input_grad(const Mat& p, const Mat& w, int act, const Kept& u,
               const at::Tensor& bias, at::Tensor* dbias, bool split,
               at::IntArrayRef sizes) {
    const long long M = p.rows, N = w.dim;
    const auto type = p.t.scalar_type();
    const int64_t plain[] = {M, N};
    const Mat out =
        act != ACT_NONE ? empty_grad(M, N, p.t, split, u) // goes into products
                        : empty_result(sizes.empty() ? plain : sizes, p.t, type);
    if (!M) {
        if (bias.defined()) *dbias = at::zeros_like(bias);
        return out;
    }
    EpiArgs e{};
    e.out = out.t.data_ptr();
    e.out_lo = out.lo.defined() ? out.lo.data_ptr() : nullptr;
    e.ld_out = out.ld;
    e.act = act;
    set_kept(e, u);
    Colsum sum;
    if (bias.defined()) sum.aim(e, M, N, bias, M <= 16);
    long long blocks;
    product<true, false, EPI_GRAD>(type, operand(p), operand(w), M, N, p.dim,
                                   e, p.t, &blocks);
    if (bias.defined()) *dbias = sum.join(blocks);
    return out;
}

// The sum of p's rows is a column of ones on x, where the last tile has room for
// it: by itself it reads p once more, at 17920 x 10000 in bf16 97 us beside 450.
at::Tensor weight_grad(const Mat& p, const Mat& x, const at::Tensor& bias,
                       at::Tensor* dbias) {
    auto out = at::empty({p.dim, x.dim}, p.t.options());
    if (bias.defined()) *dbias = at::empty({p.dim}, bias.options());
    if (!p.rows) {
        if (bias.defined()) dbias->zero_();
        return out.zero_();
    }
    EpiArgs e{};
    e.out = out.data_ptr();
    e.ld_out = x.dim;
    if (bias.defined()) {
        e.colsum = dbias->data_ptr();
        e.colsum_out = bias.scalar_type() == at::kFloat ? COLSUM_FLOAT
                                                        : COLSUM_T;
    }
    long long blocks;
    product<false, false, EPI_PLAIN>(p.t.scalar_type(), operand(p), operand(x),
                                     p.dim, x.dim, p.rows, e, p.t, &blocks);
    if (bias.defined() && !blocks) *dbias = row_sums(p, bias.scalar_type());
    return out;
}

}  // namespace ffn
