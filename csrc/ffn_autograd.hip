// The feed-forward operators as autograd functions: checks of arguments, what
// is kept for the backward pass, and the backward pass itself.
#include "ffn_ops.h"
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>

namespace ffn {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

static Tensor or_none(const c10::optional<Tensor>& t) {
    return t.has_value() ? *t : Tensor();
}

static void check_values(const Tensor& x, const char* name) {
    TORCH_CHECK(x.is_cuda(), name, " must be on the GPU, got ", x.device());
    TORCH_CHECK(x.scalar_type() == at::kBFloat16 ||
                x.scalar_type() == at::kHalf || x.scalar_type() == at::kFloat,
                name, " must be BFloat16, Half or Float, got ",
                x.scalar_type());
    TORCH_CHECK(x.dim() >= 1, name, " must have at least one dimension");
    TORCH_CHECK(x.size(-1) > 0, name, "'s last dimension must not be empty");
    // a launch has less than 2^32 threads, and a thread at least four rows
    TORCH_CHECK(x.size(-1) < (1LL << 30) &&
                x.numel() / x.size(-1) <= 1000000000, name, " of shape ",
                x.sizes(), " is too large");
}

static void check_same(const Tensor& x, const Tensor& t, const char* name) {
    TORCH_CHECK(t.device() == x.device(), name, " is on ", t.device(),
                ", x on ", x.device());
    TORCH_CHECK(t.scalar_type() == x.scalar_type(), name, " must be ",
                x.scalar_type(), " as x is, got ", t.scalar_type());
}

static void check_weight(const Tensor& x, const Tensor& w, long long in,
                         const char* name) {
    TORCH_CHECK(w.dim() == 2 && w.size(1) == in && w.size(0) > 0, name,
                " must have shape [out, ", in, "], got ", w.sizes());
    check_same(x, w, name);
    // 256 rows of an operand are addressed by 32-bit byte offsets
    TORCH_CHECK(w.size(0) <= 4000000 && in <= 4000000, name, " of shape ",
                w.sizes(), " is too large");
}

static void check_norm_params(const Tensor& x, const Tensor& gamma,
                              const Tensor& beta, const char* weight_name,
                              const char* bias_name) {
    check_params(x, gamma, x.size(-1), weight_name);
    check_params(x, beta, x.size(-1), bias_name);
    TORCH_CHECK(!gamma.defined() || !beta.defined() ||
                gamma.scalar_type() == beta.scalar_type(), weight_name, " is ",
                gamma.scalar_type(), ", ", bias_name, " ",
                beta.scalar_type());
}

static void check_act(int64_t act) {
    TORCH_CHECK(act >= 0 && act <= 3, "no activation ", act);
}

// The kernels are launched past torch's dispatcher.  What follows a call there
// would see no more of it than the allocation of its result: a derivative of
// zero in forward mode, a graph without the kernel.
static void check_seen(const char* name, std::initializer_list<Tensor> all) {
    using Modes = c10::impl::TorchDispatchModeTLS;
    using Mode = c10::impl::TorchDispatchModeKey;
    TORCH_CHECK(!torch::jit::tracer::isTracing() &&
                !Modes::get_mode(Mode::PROXY) && !Modes::get_mode(Mode::FAKE) &&
                !Modes::get_mode(Mode::FUNCTIONAL),
                name, " cannot be traced: its kernels are no operators of torch");
    for (const Tensor& t : all) {
        if (!t.defined()) continue;
        TORCH_CHECK(t.has_storage() &&
                    !t.unsafeGetTensorImpl()->key_set().has_any(
                        c10::DispatchKeySet({c10::DispatchKey::FuncTorchBatched,
                            c10::DispatchKey::FuncTorchGradWrapper,
                            c10::DispatchKey::Functionalize})),
                    name, " has no form for the transforms of torch.func");
        TORCH_CHECK(!t._fw_grad(0).defined(), name,
                    " has no derivative in forward mode");
    }
}

static bool wants_grad(const Tensor& t) {
    return t.defined() && t.requires_grad();
}

static bool recording(std::initializer_list<Tensor> all) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor& t : all) if (wants_grad(t)) return true;
    return false;
}

// A leaf's gradient goes to it on the stream on which its first graph that still
// lives was recorded.  Captured, that would be work on a stream that is not part
// of the capture, which the autograd engine's thread does not survive.
static void check_capture(at::ArrayRef<Tensor> all) {
    const auto stream = c10::hip::getCurrentHIPStream();
    hipStreamCaptureStatus status;
    if (hipStreamIsCapturing(stream, &status) == hipSuccess &&
        status == hipStreamCaptureStatusNone)
        return;
    for (const Tensor& t : all) {
        if (!wants_grad(t) || !t.is_leaf()) continue;
        const auto sink = torch::autograd::impl::try_get_grad_accumulator(t);
        if (!sink) continue;
        const auto theirs = sink->stream();
        TORCH_CHECK(!theirs.has_value() || theirs->id() == stream.id(),
                    "a graph recorded on another stream keeps a parameter or "
                    "input of this captured call: free that graph (its outputs)"
                    " before the capture begins");
    }
}

// the same for leaves that the caller casts before it passes them on
void check_cast_leaves(const std::vector<Tensor>& all) {
    if (!at::GradMode::is_enabled() || all.empty() || !all[0].is_cuda()) return;
    const at::DeviceGuard guard(all[0].device());
    check_capture(all);
}

static void check_once(const char* name) {
    TORCH_CHECK(!at::GradMode::is_enabled(), name, " has no second derivative "
                "(backward with create_graph=True)");
}

// Absent inputs are passed on as nothing and have no edge: bit i of the mask
// says that input i is there, and an input's edge is found by counting.
static int64_t present(std::initializer_list<Tensor> all) {
    int64_t mask = 0, bit = 1;
    for (const Tensor& t : all) {
        if (t.defined()) mask |= bit;
        bit <<= 1;
    }
    return mask;
}

static bool needs(AutogradContext* ctx, int i) {
    const int64_t mask = ctx->saved_data["inputs"].toInt();
    if (!(mask >> i & 1)) return false;
    return ctx->needs_input_grad(
        __builtin_popcountll(mask & ((1LL << i) - 1)));
}

using Maybe = c10::optional<Tensor>;
static Maybe maybe(const Tensor& t) {
    return t.defined() ? Maybe(t) : Maybe();
}

// a view costs the host as much as an allocation: none where the shape is right
static Tensor shaped(const Tensor& t, at::IntArrayRef sizes) {
    return t.sizes() == sizes ? t : t.view(sizes);
}

static Tensor contiguous_or_none(const Tensor& t) {
    return t.defined() ? t.contiguous() : t;
}

// ---- layer norm -----------------------------------------------------------------
struct NormFn : public torch::autograd::Function<NormFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x,
                          const Maybe& weight, const Maybe& bias, double eps,
                          bool act8) {
        const Tensor gamma = or_none(weight), beta = or_none(bias);
        const Mat m = as_rows(x);
        NormOut o = norm_forward(m, contiguous_or_none(gamma),
                                 contiguous_or_none(beta), eps, true, act8,
                                 false, x.sizes());
        ctx->save_for_backward({act8 ? Tensor() : x, gamma, beta, o.stats,
                                o.x8.codes, o.x8.scales});
        ctx->saved_data["inputs"] = present({x, gamma, beta});
        return o.y.t;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_once("layer_norm");
        const auto s = ctx->get_saved_variables();
        const Tensor& dy = grads[0];
        const at::DeviceGuard guard(dy.device());
        const Mat d = as_rows(dy);
        const Mat x = s[0].defined() ? as_rows(s[0]) : Mat();
        NormGrads g = norm_backward(
            x, {s[4], s[5]}, d, nullptr, contiguous_or_none(s[1]),
            contiguous_or_none(s[2]), s[3], needs(ctx, 0),
            needs(ctx, 1) || needs(ctx, 2), dy.sizes());
        return {g.dx, g.dgamma, g.dbeta, Tensor(), Tensor()};
    }
};

Tensor layer_norm(Tensor x, c10::optional<Tensor> weight,
                  c10::optional<Tensor> bias, double eps, bool act8) {
    const Tensor gamma = or_none(weight), beta = or_none(bias);
    check_seen("layer_norm", {x, gamma, beta});
    check_values(x, "x");
    check_norm_params(x, gamma, beta, "weight", "bias");
    TORCH_CHECK(x.size(-1) < (1LL << 25), "rows of ", x.size(-1),
                " are too long");
    const at::DeviceGuard guard(x.device());
    if (recording({x, gamma, beta})) {
        check_capture({x, gamma, beta});
        return NormFn::apply(x, maybe(gamma), maybe(beta), eps, act8);
    }
    return norm_forward(as_rows(x), contiguous_or_none(gamma),
                        contiguous_or_none(beta), eps, false, false, false,
                        x.sizes()).y.t;
}

// ---- linear layer ----------------------------------------------------------------
static std::vector<int64_t> out_sizes(const Tensor& x, int64_t n) {
    std::vector<int64_t> s = x.sizes().vec();
    s.back() = n;
    return s;
}

struct LinearFn : public torch::autograd::Function<LinearFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x,
                          const Tensor& w, const Maybe& maybe_bias,
                          const Maybe& maybe_res, int64_t act, bool act8) {
        const Tensor bias = or_none(maybe_bias), res = or_none(maybe_res);
        const Mat mx = as_rows(x), mw = as_rows(w);
        const Mat m = on_lines(mx, mw.rows), wm = on_lines(mw, mx.rows);
        Mat r;
        if (res.defined()) r = as_rows(res);
        const bool through = wants_grad(x) || wants_grad(w) ||
                             wants_grad(bias);
        LinearOut o = linear_forward(m, wm, contiguous_or_none(bias),
                                     res.defined() ? &r : nullptr, (int)act,
                                     through, act8, false,
                                     out_sizes(x, w.size(0)));
        Packed x8;
        if (wants_grad(w) && act8) x8 = pack(m);
        // a copy that was made serves the backward pass too
        const Tensor& kept_x = m.t.is_same(mx.t) ? x : m.t;
        const Tensor& kept_w = wm.t.is_same(mw.t) ? w : wm.t;
        ctx->save_for_backward({wants_grad(w) && !act8 ? kept_x : Tensor(),
                                wants_grad(x) ? kept_w : Tensor(), x8.codes,
                                x8.scales, o.u.data, o.u.scales, bias});
        ctx->saved_data["inputs"] = present({x, w, bias, res});
        ctx->saved_data["act"] = act;
        ctx->saved_data["how"] = (int64_t)o.u.how;
        return o.y.t;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_once("linear_act");
        const auto s = ctx->get_saved_variables();
        const Tensor& dy = grads[0];
        const at::DeviceGuard guard(dy.device());
        const bool need_x = needs(ctx, 0), need_w = needs(ctx, 1);
        const bool need_b = needs(ctx, 2);
        Tensor dx, dw, db;
        if (need_x || need_w || need_b) {
            const Kept u{s[4], s[5], (int)ctx->saved_data["how"].toInt()};
            const int act = (int)ctx->saved_data["act"].toInt();
            // The matrix cores take 16 bits: p is rounded to its type for dx and
            // dW, in the place of the gradient that an activation by itself
            // would hand on.  With the result's own rounding that makes 1.4
            // times its error: through gelu in bf16 0.0024 of the norm, 0.0017
            // with p in two parts, which takes a product of twice the length:
            // 17920 x 1500 to 6000, forward and backward, 1315 and 1915 us, 700
            // rows 121 and 154.  Two parts are kept where a third rounding would
            // follow: for dW beside an x unpacked from 8 bits, which rounds to
            // 16.  (That is off by 2^-8 of a value at most in bf16, 2^-11 in
            // fp16, and the 8-bit form by 2^-8 of its group's largest: dW from a
            // second part of x would be 0.0017 for 0.0024 of its norm, or 0.0002
            // for 0.0003 in fp16, beside 0.0065 that the form itself is off by.)
            const bool act8 = need_w && s[2].defined();
            // without an activation the bias's gradient comes with dW, or alone
            const bool plain = need_b && act == 0;
            Mat p = through_act(as_rows(dy), act, u,
                                need_b && !plain ? s[6] : Tensor(), &db, act8);
            if (need_w)
                dw = weight_grad(p, act8
                    ? unpack(s[2], s[3], dy.scalar_type(), {})
                    : as_rows(s[0]), plain ? s[6] : Tensor(), &db);
            else if (plain)
                db = row_sums(p, s[6].scalar_type());
            p.lo = Tensor();
            if (need_x)
                dx = input_grad(p, as_rows(s[1]), 0, Kept(), Tensor(), nullptr,
                                false, out_sizes(dy, s[1].size(1))).t;
        }
        return {dx, dw, db, needs(ctx, 3) ? dy : Tensor(),
                Tensor(), Tensor()};
    }
};

Tensor linear_act(Tensor x, Tensor weight, c10::optional<Tensor> bias,
                  c10::optional<Tensor> residual, int64_t act, bool act8) {
    const Tensor b = or_none(bias), r = or_none(residual);
    check_seen("linear_act", {x, weight, b, r});
    check_values(x, "x");
    check_weight(x, weight, x.size(-1), "weight");
    check_params(x, b, weight.size(0), "bias");
    check_act(act);
    if (r.defined()) {
        check_same(x, r, "residual");
        TORCH_CHECK(r.sizes() == at::IntArrayRef(out_sizes(x, weight.size(0))),
                    "residual must have the output's shape ",
                    at::IntArrayRef(out_sizes(x, weight.size(0))), ", got ",
                    r.sizes());
    }
    const at::DeviceGuard guard(x.device());
    if (recording({x, weight, b, r})) {
        check_capture({x, weight, b, r});
        return LinearFn::apply(x, weight, maybe(b), maybe(r), act, act8);
    }
    Mat rm;
    const Mat m = as_rows(x);
    if (r.defined()) rm = as_rows(r);
    return linear_forward(on_lines(m, weight.size(0)),
                          on_lines(as_rows(weight), m.rows),
                          contiguous_or_none(b), r.defined() ? &rm : nullptr,
                          (int)act, false, false, false,
                          out_sizes(x, weight.size(0))).y.t;
}

// ---- the block ---------------------------------------------------------------------
struct BlockFn : public torch::autograd::Function<BlockFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x,
                          const Maybe& norm_weight, const Maybe& norm_bias,
                          const Tensor& w1, const Maybe& bias1,
                          const Tensor& w2, const Maybe& bias2, int64_t act,
                          double eps, bool act8) {
        const Tensor gamma = or_none(norm_weight), beta = or_none(norm_bias);
        const Tensor b1 = or_none(bias1), b2 = or_none(bias2);
        const Mat m = as_rows(x);
        NormOut n = norm_forward(m, contiguous_or_none(gamma),
                                 contiguous_or_none(beta), eps, true, act8,
                                 act8, {});
        const Mat r1 = as_rows(w1), r2 = as_rows(w2);
        const Mat m1 = on_lines(r1, m.rows), m2 = on_lines(r2, m.rows);
        LinearOut a = linear_forward(n.y, m1, contiguous_or_none(b1), nullptr,
                                     (int)act, true, act8, act8, {});
        LinearOut o = linear_forward(a.y, m2, contiguous_or_none(b2), &m, 0,
                                     false, false, false, x.sizes());
        const Tensor& kept1 = m1.t.is_same(r1.t) ? w1 : m1.t;
        const Tensor& kept2 = m2.t.is_same(r2.t) ? w2 : m2.t;
        const Tensor none;
        ctx->save_for_backward(
            {act8 ? none : x, act8 ? none : n.y.t, act8 ? none : a.y.t, n.x8.codes,
             n.x8.scales, n.y8.codes, n.y8.scales, a.y8.codes, a.y8.scales,
             a.u.data, a.u.scales, n.stats, gamma, beta, kept1, b1, kept2,
             b2});
        ctx->saved_data["inputs"] = present({x, gamma, beta, w1, b1, w2, b2});
        ctx->saved_data["act"] = act;
        ctx->saved_data["how"] = (int64_t)a.u.how;
        return o.y.t;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_once("ffn_block");
        const auto s = ctx->get_saved_variables();
        const Tensor& dy = grads[0];
        const at::DeviceGuard guard(dy.device());
        const auto type = dy.scalar_type();
        const Mat d = as_rows(dy);
        const Tensor &w1 = s[14], &b1 = s[15], &w2 = s[16], &b2 = s[17];
        auto need = [&](int i) { return needs(ctx, i); };
        auto kept = [&](int plain, int packed) {
            return s[plain].defined()
                ? as_rows(s[plain])
                : unpack(s[packed], s[packed + 1], type, {});
        };
        Tensor dw1, db1, dw2, db2;
        NormGrads g;
        if (need(5))
            dw2 = weight_grad(d, kept(2, 7), need(6) ? b2 : Tensor(), &db2);
        else if (need(6))
            db2 = row_sums(d, b2.scalar_type());
        const bool norm = need(0) || need(1) || need(2);
        const bool bias = need(4);
        if (norm || need(3) || bias) {
            const Kept u{s[9], s[10], (int)ctx->saved_data["how"].toInt()};
            // The norm's gradients are sums over dh, which is rounded as it
            // comes from the product: were p rounded before, dh would round
            // to other values.  Both parts go into dW1, too: 268 us for 254 at
            // 700 x 1500, hidden 6000, where LinearFn's two products would take
            // half as long again; dW1 is off by what its own rounding makes,
            // not 1.4 times that.
            Mat p = input_grad(d, as_rows(w2),
                               (int)ctx->saved_data["act"].toInt(), u,
                               bias ? b1 : Tensor(), &db1, norm || need(3),
                               {});
            if (norm) {
                const Mat dh = input_grad(p, as_rows(w1), 0, Kept(), Tensor(),
                                          nullptr, false, {});
                g = norm_backward(
                    s[0].defined() ? as_rows(s[0]) : Mat(), {s[3], s[4]},
                    dh, &d, contiguous_or_none(s[12]),
                    contiguous_or_none(s[13]), s[11], need(0),
                    need(1) || need(2), dy.sizes());
            }
            if (need(3))
                dw1 = weight_grad(p, kept(1, 5), Tensor(), nullptr);
        }
        return {g.dx, g.dgamma, g.dbeta, dw1, db1, dw2, db2, Tensor(), Tensor(),
                Tensor()};
    }
};

Tensor ffn_block(Tensor x, c10::optional<Tensor> norm_weight,
                 c10::optional<Tensor> norm_bias, Tensor w1,
                 c10::optional<Tensor> b1, Tensor w2,
                 c10::optional<Tensor> b2, int64_t act, double eps,
                 bool act8) {
    const Tensor gamma = or_none(norm_weight), beta = or_none(norm_bias);
    const Tensor c1 = or_none(b1), c2 = or_none(b2);
    check_seen("ffn_block", {x, gamma, beta, w1, c1, w2, c2});
    check_values(x, "x");
    check_norm_params(x, gamma, beta, "norm_weight", "norm_bias");
    check_weight(x, w1, x.size(-1), "w1");
    check_weight(x, w2, w1.size(0), "w2");
    TORCH_CHECK(w2.size(0) == x.size(-1), "w2 must have shape [", x.size(-1),
                ", ", w1.size(0), "], got ", w2.sizes());
    check_params(x, c1, w1.size(0), "b1");
    check_params(x, c2, x.size(-1), "b2");
    check_act(act);
    const at::DeviceGuard guard(x.device());
    if (recording({x, gamma, beta, w1, c1, w2, c2})) {
        check_capture({x, gamma, beta, w1, c1, w2, c2});
        return BlockFn::apply(x, maybe(gamma), maybe(beta), w1, maybe(c1), w2,
                              maybe(c2), act, eps, act8);
    }
    const Mat m = as_rows(x);
    const NormOut n = norm_forward(m, contiguous_or_none(gamma),
                                   contiguous_or_none(beta), eps, false, false,
                                   false, {});
    const LinearOut a = linear_forward(n.y, on_lines(as_rows(w1), m.rows),
                                       contiguous_or_none(c1), nullptr,
                                       (int)act, false, false, false, {});
    return linear_forward(a.y, on_lines(as_rows(w2), m.rows),
                          contiguous_or_none(c2), &m, 0, false, false, false,
                          x.sizes()).y.t;
}

// ---- the 8-bit form ------------------------------------------------------------------
std::vector<Tensor> act8_pack(Tensor x) {
    check_seen("act8_pack", {x});
    check_values(x, "x");
    const at::DeviceGuard guard(x.device());
    const Packed p{at::empty(x.sizes(), x.options().dtype(at::kChar)),
                   at::empty(out_sizes(x, (x.size(-1) + 127) / 128),
                             x.options().dtype(at::kFloat))};
    pack_to(as_rows(x), p);
    return {p.codes, p.scales};
}

Tensor act8_unpack(Tensor codes, Tensor scales, int64_t type) {
    check_seen("act8_unpack", {codes, scales});
    TORCH_CHECK(!recording({scales}), "act8_unpack has no gradient: scales must "
                "not require one");
    TORCH_CHECK(codes.is_cuda() && scales.device() == codes.device(),
                "codes and scales must be on one GPU, got ", codes.device(),
                " and ", scales.device());
    TORCH_CHECK(codes.scalar_type() == at::kChar &&
                scales.scalar_type() == at::kFloat,
                "codes must be Char and scales Float, got ",
                codes.scalar_type(), " and ", scales.scalar_type());
    TORCH_CHECK(codes.dim() >= 1 && codes.size(-1) > 0 &&
                codes.size(-1) < (1LL << 30),
                "codes of shape ", codes.sizes());
    std::vector<int64_t> s = codes.sizes().vec();
    const int64_t dim = s.back();
    s.back() = (dim + 127) / 128;
    TORCH_CHECK(scales.sizes() == at::IntArrayRef(s), "scales must have shape ",
                at::IntArrayRef(s), ", got ", scales.sizes());
    const at::DeviceGuard guard(codes.device());
    const auto t = type == 0 ? at::kFloat : type == 1 ? at::kBFloat16
                                                      : at::kHalf;
    const int64_t rows = codes.numel() / dim;
    return unpack(shaped(codes.contiguous(), {rows, dim}),
                  shaped(scales.contiguous(), {rows, s.back()}), t,
                  codes.sizes()).t;
}

}  // namespace ffn
