// Launchers of the feed-forward operators, over checked tensors.
#pragma once
#include <torch/extension.h>

namespace ffn {

// [rows, dim] with neighbouring columns; rows lie ld values apart
struct Mat {
    at::Tensor t;     // keeps the memory
    at::Tensor lo;    // what rounding to t left, laid out the same, or none
    long long rows = 0, dim = 0, ld = 0;
};
Mat as_rows(const at::Tensor& x);
// the result of a call, allocated as it is returned: of a view of its rows torch
// would refuse to modify it in place
Mat empty_result(at::IntArrayRef sizes, const at::Tensor& like,
                 at::ScalarType type);

// the 8-bit form of [rows, dim]
struct Packed { at::Tensor codes, scales; };
Packed empty_packed(long long rows, long long dim, const at::Tensor& like);
Packed pack(const Mat& x);
void pack_to(const Mat& x, const Packed& p);
// `sizes` here and below: those of the result; where they are empty, it goes to
// another operator, in rows on lines
Mat unpack(const at::Tensor& codes, const at::Tensor& scales,
           at::ScalarType type, at::IntArrayRef sizes);
// rows that start on lines of 128 bytes, unless they are short: what a product
// reads in lines, it reads with up to 16 % fewer requests
Mat empty_rows(long long rows, long long dim, const at::Tensor& like,
               at::ScalarType type);

// m, or a copy whose rows start on lines where a product with `other` rows or
// columns gains more by them than the copy takes
Mat on_lines(const Mat& m, long long other);

// what the backward pass sees of a value: itself, its 8-bit form, or for relu
// the sign in bits
struct Kept {
    at::Tensor data, scales;
    int how = 0;      // Keep of linear_kernels.h
};

void check_params(const at::Tensor& x, const at::Tensor& p, long long n,
                  const char* name);

// stats: [2, rows], the means and the 1 / deviations
struct NormOut { Mat y; at::Tensor stats; Packed x8, y8; };
NormOut norm_forward(const Mat& x, const at::Tensor& gamma,
                     const at::Tensor& beta, double eps, bool stats,
                     bool keep_x8, bool keep_y8, at::IntArrayRef sizes);
struct NormGrads { at::Tensor dx, dgamma, dbeta; };
// x or, where it is defined, x8; `add` (or nothing) goes onto dx, of `sizes`
NormGrads norm_backward(const Mat& x, const Packed& x8, const Mat& dy,
                        const Mat* add, const at::Tensor& gamma,
                        const at::Tensor& beta, const at::Tensor& stats,
                        bool need_dx, bool need_params,
                        at::IntArrayRef sizes);

struct LinearOut { Mat y; Kept u; Packed y8; };
LinearOut linear_forward(const Mat& x, const Mat& w, const at::Tensor& bias,
                         const Mat* res, int act, bool keep, bool act8,
                         bool keep_y8, at::IntArrayRef sizes);
// p = dy act'(u), and the sum of its rows in bias's type where bias is defined
// (without an activation: dy, and no sum).  `split`: p keeps what rounding
// leaves, where the activation makes it round.
Mat through_act(const Mat& dy, int act, const Kept& u, const at::Tensor& bias,
                at::Tensor* dbias, bool split);
// dx = p W, rounded, then through the activation below as through_act does;
// without one of `sizes`, or where they are empty [rows, dim]
Mat input_grad(const Mat& p, const Mat& w, int act, const Kept& u,
               const at::Tensor& bias, at::Tensor* dbias, bool split,
               at::IntArrayRef sizes);
// dW = p^T x, and the sum of p's rows in bias's type where bias is defined
at::Tensor weight_grad(const Mat& p, const Mat& x, const at::Tensor& bias,
                       at::Tensor* dbias);
at::Tensor row_sums(const Mat& p, at::ScalarType type);
// out = sum of the first n rows of partial sums
void sum_partials(const at::Tensor& part, long long n, at::Tensor& out);

// autograd entry points, bound in gtopk_ext.hip
at::Tensor layer_norm(at::Tensor x, c10::optional<at::Tensor> weight,
                      c10::optional<at::Tensor> bias, double eps, bool act8);
at::Tensor linear_act(at::Tensor x, at::Tensor weight,
                      c10::optional<at::Tensor> bias,
                      c10::optional<at::Tensor> residual, int64_t act,
                      bool act8);
at::Tensor ffn_block(at::Tensor x, c10::optional<at::Tensor> norm_weight,
                     c10::optional<at::Tensor> norm_bias, at::Tensor w1,
                     c10::optional<at::Tensor> b1, at::Tensor w2,
                     c10::optional<at::Tensor> b2, int64_t act, double eps,
                     bool act8);
void check_cast_leaves(const std::vector<at::Tensor>& all);
std::vector<at::Tensor> act8_pack(at::Tensor x);
at::Tensor act8_unpack(at::Tensor codes, at::Tensor scales, int64_t type);

}  // namespace ffn
