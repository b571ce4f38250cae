// Layer norm forward and backward, the 8-bit form of activations, and sums
// over rows: launches.
#include <hip/hip_runtime.h>
#include "ffn_launch.h"
#include "layernorm_kernels.h"

namespace ffn {

Mat as_rows(const at::Tensor& x) {
    Mat m;
    m.dim = x.size(-1);
    m.rows = 1;
    for (int64_t i = 0; i + 1 < x.dim(); ++i) m.rows *= x.size(i);
    m.t = x.dim() == 2 ? x : x.reshape({m.rows, m.dim});
    if (m.dim > 1 && m.t.stride(1) != 1) m.t = m.t.contiguous();
    if (m.rows > 1 && m.t.stride(0) < m.dim) m.t = m.t.contiguous();
    // the products address 256 rows by 32-bit byte offsets
    if (m.rows > 1 && m.t.stride(0) > 4000000 && m.t.stride(0) != m.dim)
        m.t = m.t.contiguous();
    m.ld = m.rows > 1 ? m.t.stride(0) : m.dim;
    return m;
}

void check_params(const at::Tensor& x, const at::Tensor& p, long long n,
                  const char* name) {
    if (!p.defined()) return;
    TORCH_CHECK(p.dim() == 1 && p.size(0) == n, name, " must have shape [", n,
                "], got ", p.sizes());
    TORCH_CHECK(p.device() == x.device(), name, " is on ", p.device(),
                ", x on ", x.device());
    TORCH_CHECK(p.scalar_type() == x.scalar_type() ||
                p.scalar_type() == at::kFloat, name, " must be ",
                x.scalar_type(), " or Float, got ", p.scalar_type());
}

static long long groups_in(long long dim) {
    return (dim + ACT8_GROUP - 1) / ACT8_GROUP;
}

Packed empty_packed(long long rows, long long dim, const at::Tensor& like) {
    return {at::empty({rows, dim}, like.options().dtype(at::kChar)),
            at::empty({rows, groups_in(dim)}, like.options().dtype(at::kFloat))};
}

// 64-bit divisions take long: runs the statement with I as the type that counts
// n pieces, and some blocks more
#define FFN_COUNT(n, ...) do { \
    if ((n) < (1LL << 30)) { typedef int I; __VA_ARGS__; } \
    else { typedef long long I; __VA_ARGS__; } \
} while (0)

Packed pack(const Mat& x) {
    Packed p = empty_packed(x.rows, x.dim, x.t);
    pack_to(x, p);
    return p;
}

void pack_to(const Mat& x, const Packed& p) {
    const long long groups = x.rows * groups_in(x.dim);
    if (!groups) return;
    const int grid = (int)std::min<long long>((groups + 31) / 32, 256 * 64);
    FFN_TYPES(x.t.scalar_type(), FFN_COUNT(groups,
        auto k = act8_pack_kernel<T, I>;
        hipLaunchKernelGGL(k, grid, 256, 0, stream_now(),
                           (const T*)x.t.data_ptr(), x.ld, (I)x.rows,
                           (int)x.dim, (signed char*)p.codes.data_ptr(),
                           p.scales.data_ptr<float>())));
    FFN_OK();
}

Mat empty_result(at::IntArrayRef sizes, const at::Tensor& like,
                 at::ScalarType type) {
    Mat m;
    m.t = at::empty(sizes, like.options().dtype(type));
    m.dim = m.ld = sizes.back();
    m.rows = 1;
    for (size_t i = 0; i + 1 < sizes.size(); ++i) m.rows *= sizes[i];
    return m;
}

Mat empty_rows(long long rows, long long dim, const at::Tensor& like,
               at::ScalarType type) {
    const long long line = 128 / c10::elementSize(type);
    Mat m;
    m.rows = rows;
    m.dim = dim;
    m.ld = dim < 4 * line ? dim : (dim + line - 1) / line * line;
    m.t = at::empty({rows, m.ld}, like.options().dtype(type));
    if (m.ld != dim) m.t = m.t.narrow(1, 0, dim);
    return m;
}

// A product of two 16-bit operands with a wide other side gains 1.2e-10 us for
// each value of this one and each line of the other, when its rows start on lines
// (about 6 %; 17920 x 1500 to 10000, us: forward 630, one operand on lines 585,
// both 563; dx with the weight on lines 605 to 581, dW with x 474 to 450), and a
// copy takes 8e-7 us a value and a launch (10000 x 1500: 13).
Mat on_lines(const Mat& m, long long other) {
    const long long line = 64;
    if (m.t.scalar_type() == at::kFloat || m.dim < 4 * line ||
        (m.ld % line == 0 && (uintptr_t)m.t.data_ptr() % 128 == 0) ||
        (double)m.rows * m.dim * (1.2e-10 * other - 8e-7) < 4.0)
        return m;
    Mat out = empty_rows(m.rows, m.dim, m.t, m.t.scalar_type());
    out.t.copy_(m.t);
    return out;
}

Mat unpack(const at::Tensor& codes, const at::Tensor& scales,
           at::ScalarType type, at::IntArrayRef sizes) {
    const long long rows = codes.size(0), dim = codes.size(1);
    const Mat out = sizes.empty() ? empty_rows(rows, dim, codes, type)
                                  : empty_result(sizes, codes, type);
    const long long n = rows * ((dim + 7) / 8);
    if (!n) return out;
    const int grid = (int)std::min<long long>((n + 255) / 256, 1 << 22);
    FFN_TYPES(type, FFN_COUNT(n,
        auto k = act8_unpack_kernel<T, I>;
        hipLaunchKernelGGL(k, grid, 256, 0, stream_now(),
                           (const signed char*)codes.data_ptr(),
                           scales.data_ptr<float>(), (I)rows, (int)dim,
                           (T*)out.t.data_ptr(), out.ld)));
    FFN_OK();
    return out;
}

// team of threads a row, chunks of 8 a thread.  Forward: as few threads as hold
// the row in 4 chunks each, so that a row of up to 2048 values needs no barrier.
// Backward: about as many threads as there are chunks, up to 1024, since a chunk
// takes 32 registers and both kernels are bound by instructions: 17920 x 1500 in
// bf16, x in 8 bits, us: 64 threads with 3 chunks (194 registers, two waves a
// unit) 68 where 256 with one took 42; 192 with one, fewer instructions a value,
// 30, at 4.5 TB/s.
#define NORM_BACKWARD_SHAPES(dim, WIDE, GO) do { \
    const long long chunks = ((dim) + 7) / 8; \
    if (chunks <= 64) GO(64, 1); \
    else if (chunks <= 128) GO(128, 1); \
    else if (chunks <= 192) GO(192, 1); \
    else if (chunks <= 256) GO(256, 1); \
    else if (chunks <= 384) GO(384, 1); \
    else if (chunks <= 512) GO(512, 1); \
    else if (chunks <= 768) GO(768, 1); \
    else if (chunks <= 1024) GO(1024, 1); \
    else if (chunks <= 2048) GO(1024, 2); \
    else if (chunks <= 4096) GO(1024, 4); \
    else WIDE; \
} while (0)
#define NORM_SHAPES(dim, WIDE, GO) do { \
    const long long chunks = ((dim) + 7) / 8; \
    if (chunks <= 64) GO(64, 1); \
    else if (chunks <= 128) GO(64, 2); \
    else if (chunks <= 192) GO(64, 3); \
    else if (chunks <= 256) GO(64, 4); \
    else if (chunks <= 512) GO(256, 2); \
    else if (chunks <= 1024) GO(256, 4); \
    else if (chunks <= 2048) GO(1024, 2); \
    else if (chunks <= 4096) GO(1024, 4); \
    else WIDE; \
} while (0)

NormOut norm_forward(const Mat& x, const at::Tensor& gamma,
                     const at::Tensor& beta, double eps, bool stats,
                     bool keep_x8, bool keep_y8, at::IntArrayRef sizes) {
    NormOut o;
    const auto type = x.t.scalar_type();
    o.y = sizes.empty() ? empty_rows(x.rows, x.dim, x.t, type)
                        : empty_result(sizes, x.t, type);
    if (stats)
        o.stats = at::empty({2, x.rows}, x.t.options().dtype(at::kFloat));
    if (keep_x8) o.x8 = empty_packed(x.rows, x.dim, x.t);
    if (keep_y8) o.y8 = empty_packed(x.rows, x.dim, x.t);
    if (!x.rows) return o;
    NormArgs a{};
    a.x = x.t.data_ptr();
    a.ld = x.ld;
    a.gamma = gamma.defined() ? gamma.data_ptr() : nullptr;
    a.beta = beta.defined() ? beta.data_ptr() : nullptr;
    a.p32 = gamma.defined() ? gamma.scalar_type() == at::kFloat
          : beta.defined() && beta.scalar_type() == at::kFloat;
    a.y = o.y.t.data_ptr();
    a.ld_y = o.y.ld;
    if (stats) {
        a.mean = o.stats.data_ptr<float>();
        a.rstd = a.mean + x.rows;
    }
    if (keep_x8) {
        a.x8 = (signed char*)o.x8.codes.data_ptr();
        a.x8_scale = o.x8.scales.data_ptr<float>();
    }
    if (keep_y8) {
        a.y8 = (signed char*)o.y8.codes.data_ptr();
        a.y8_scale = o.y8.scales.data_ptr<float>();
    }
    a.rows = (int)x.rows;
    a.dim = (int)x.dim;
    a.eps = (float)eps;
    const auto s = stream_now();
    #define GO(NT, R) do { \
        const int teams = NT == 64 ? 4 : 1, threads = NT == 64 ? 256 : NT; \
        const int grid = (int)std::min<long long>( \
            (x.rows + teams - 1) / teams, 256 * 8); \
        auto k = norm_forward_kernel<T, NT, R>; \
        hipLaunchKernelGGL(k, grid, threads, 0, s, a); \
    } while (0)
    #define WIDE do { \
        auto k = norm_forward_wide_kernel<T>; \
        hipLaunchKernelGGL(k, (int)x.rows, 1024, 0, s, a); \
    } while (0)
    FFN_TYPES(type, NORM_SHAPES(x.dim, WIDE, GO));
    #undef GO
    #undef WIDE
    FFN_OK();
    return o;
}

static void sum_columns(const at::Tensor& part, long long n, long long width,
                        long long first, at::Tensor a, at::Tensor b) {
    const auto type = a.defined() ? a.scalar_type() : b.scalar_type();
    const int grid = (int)((width + 15) / 16);
    FFN_TYPES(type,
        auto k = column_sum_kernel<T>;
        hipLaunchKernelGGL(k, grid, 1024, 0, stream_now(), part.data_ptr<float>(), (int)n, (int)width, (int)first,
            a.defined() ? (T*)a.data_ptr() : nullptr,
            b.defined() ? (T*)b.data_ptr() : nullptr));
    FFN_OK();
}

NormGrads norm_backward(const Mat& x, const Packed& x8, const Mat& dy,
                        const Mat* add, const at::Tensor& gamma,
                        const at::Tensor& beta, const at::Tensor& stats,
                        bool need_dx, bool need_params,
                        at::IntArrayRef sizes) {
    const long long rows = dy.rows, dim = dy.dim;
    NormGrads g;
    if (need_dx) g.dx = at::empty(sizes, dy.t.options());
    if (need_params && gamma.defined()) g.dgamma = at::empty_like(gamma);
    if (need_params && beta.defined()) g.dbeta = at::empty_like(beta);
    const bool params = g.dgamma.defined() || g.dbeta.defined();
    if (!rows) {
        if (g.dgamma.defined()) g.dgamma.zero_();
        if (g.dbeta.defined()) g.dbeta.zero_();
        return g;
    }
    NormGradArgs a{};
    if (x8.codes.defined()) {
        a.x8 = (const signed char*)x8.codes.data_ptr();
        a.x8_scale = x8.scales.data_ptr<float>();
    } else {
        a.x = x.t.data_ptr();
        a.ld = x.ld;
    }
    a.dy = dy.t.data_ptr();
    a.ld_dy = dy.ld;
    if (add) {
        a.add = add->t.data_ptr();
        a.ld_add = add->ld;
    }
    a.gamma = gamma.defined() ? gamma.data_ptr() : nullptr;
    a.p32 = gamma.defined() && gamma.scalar_type() == at::kFloat;
    a.mean = stats.data_ptr<float>();
    a.rstd = a.mean + rows;
    a.dx = need_dx ? g.dx.data_ptr() : nullptr;
    a.rows = (int)rows;
    a.dim = (int)dim;
    const auto s = stream_now();
    const auto f32 = dy.t.options().dtype(at::kFloat);
    at::Tensor part;
    long long blocks = 0;
    #define GO(NT, R) do { \
        const int teams = NT == 64 ? 4 : 1, threads = NT == 64 ? 256 : NT; \
        blocks = std::min<long long>((rows + teams - 1) / teams, \
                                     NT <= 256 ? 1024 : NT <= 512 ? 512 : 256); \
        if (params) { \
            part = at::empty({blocks, 2, dim}, f32); \
            a.part = part.data_ptr<float>(); \
        } \
        auto k = a.x8 ? norm_backward_kernel<T, NT, R, true> \
                      : norm_backward_kernel<T, NT, R, false>; \
        hipLaunchKernelGGL(k, (int)blocks, threads, 0, s, a); \
    } while (0)
    #define WIDE do { \
        if (need_dx) { \
            auto k = norm_dx_wide_kernel<T>; \
            hipLaunchKernelGGL(k, (int)rows, 1024, 0, s, a); \
        } \
        if (params) { \
            const int per = (int)std::max<long long>(64, (rows + 63) / 64); \
            blocks = (rows + per - 1) / per; \
            part = at::empty({blocks, 2, dim}, f32); \
            a.part = part.data_ptr<float>(); \
            const dim3 grid((unsigned)((dim + 255) / 256), (unsigned)blocks); \
            auto k = row_sum_kernel<T, true>; \
            hipLaunchKernelGGL(k, grid, 256, 0, s, a, per); \
        } \
    } while (0)
    FFN_TYPES(dy.t.scalar_type(), NORM_BACKWARD_SHAPES(dim, WIDE, GO));
    #undef GO
    #undef WIDE
    FFN_OK();
    if (params) sum_columns(part, blocks, 2 * dim, dim, g.dgamma, g.dbeta);
    return g;
}

at::Tensor row_sums(const Mat& p, at::ScalarType type) {
    auto out = at::empty({p.dim}, p.t.options().dtype(type));
    if (!p.rows) return out.zero_();
    // about 2048 blocks, of 32 rows at least
    const long long cols = (p.dim + 255) / 256;
    const long long slabs = std::max<long long>(1, 2048 / cols);
    const int per = (int)std::max<long long>(32, (p.rows + slabs - 1) / slabs);
    const long long blocks = (p.rows + per - 1) / per;
    auto part = at::empty({blocks, p.dim}, p.t.options().dtype(at::kFloat));
    NormGradArgs a{};
    a.dy = p.t.data_ptr();
    a.ld_dy = p.ld;
    a.part = part.data_ptr<float>();
    a.rows = (int)p.rows;
    a.dim = (int)p.dim;
    const dim3 grid((unsigned)cols, (unsigned)blocks);
    FFN_TYPES(p.t.scalar_type(),
        auto k = row_sum_kernel<T, false>;
        hipLaunchKernelGGL(k, grid, 256, 0, stream_now(), a, per));
    FFN_OK();
    sum_columns(part, blocks, p.dim, p.dim, out, at::Tensor());
    return out;
}

void sum_partials(const at::Tensor& part, long long n, at::Tensor& out) {
    sum_columns(part, n, out.numel(), out.numel(), out, at::Tensor());
}

}  // namespace ffn
