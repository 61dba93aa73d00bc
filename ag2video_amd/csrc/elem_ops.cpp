// Host side of the fp32 / bf16 / fp16 operators: argument checks, views, workspaces and autograd nodes over the C entry points of
// include/ag2v.h.  The nodes are C++ because the tape's backward runs on a thread of its own: a node written in Python costs 40 to 100 us
// there (the interpreter and its objects move between cores), more than the kernels of a small map.  Every refusal of a value is a
// RuntimeError.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <limits>
#include <string>
#include <tuple>

#include "../../include/ag2v.h"

namespace {
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t INT_LIMIT = int64_t(1) << 31;

// The entry points of the library that ag2video_amd._lib has loaded.
struct Entries {
    decltype(&ag2v_embed_fwd) embed_fwd = nullptr;
    decltype(&ag2v_embed_bwd_workspace_floats) embed_bwd_ws = nullptr;
    decltype(&ag2v_embed_bwd) embed_bwd = nullptr;
    decltype(&ag2v_group_norm_workspace_floats) norm_ws = nullptr;
    decltype(&ag2v_group_norm_fwd) norm_fwd = nullptr;
    decltype(&ag2v_group_norm_bwd) norm_bwd = nullptr;
} lib;

void bind(uintptr_t embed_fwd, uintptr_t embed_bwd_ws, uintptr_t embed_bwd, uintptr_t norm_ws, uintptr_t norm_fwd, uintptr_t norm_bwd) {
    lib.embed_fwd = reinterpret_cast<decltype(lib.embed_fwd)>(embed_fwd);
    lib.embed_bwd_ws = reinterpret_cast<decltype(lib.embed_bwd_ws)>(embed_bwd_ws);
    lib.embed_bwd = reinterpret_cast<decltype(lib.embed_bwd)>(embed_bwd);
    lib.norm_ws = reinterpret_cast<decltype(lib.norm_ws)>(norm_ws);
    lib.norm_fwd = reinterpret_cast<decltype(lib.norm_fwd)>(norm_fwd);
    lib.norm_bwd = reinterpret_cast<decltype(lib.norm_bwd)>(norm_bwd);
}

int elem_of(at::ScalarType t) {
    return t == at::kFloat ? AG2V_F32 : t == at::kBFloat16 ? AG2V_BF16 : t == at::kHalf ? AG2V_F16 : -1;
}
void elem_check(const char* name, const Tensor& t) {
    TORCH_CHECK(t.is_cuda(), name, ": expected a HIP device tensor, got ", t.device(), " (no CPU fallback)");
    TORCH_CHECK(elem_of(t.scalar_type()) >= 0, name, ": expected float32, bfloat16 or float16, got ", t.scalar_type());
}
void checked(const char* name, int rc) {
    TORCH_CHECK(rc == AG2V_OK, name, " failed: ", rc == AG2V_EINVAL ? "AG2V_EINVAL (rejected argument)" : "AG2V_EHIP (HIP launch error)");
}
// The tensors' device for the duration of a launch, and its current stream.
struct OnDevice {
    c10::DeviceGuard guard;
    void* stream;
    explicit OnDevice(const Tensor& t)
        : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};
Tensor workspace_of(const Tensor& like, size_t floats) {
    return floats ? at::empty({int64_t(floats)}, like.options().dtype(at::kFloat)) : Tensor();
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// The tokens in row-major order, `stride` elements apart; a copy only if no one stride walks them.
std::pair<Tensor, int64_t> token_rows(const Tensor& idx) {
    if (idx.is_contiguous()) return {idx, 1};
    int64_t stride = -1, run = 1;
    for (int64_t d = idx.dim() - 1; d >= 0; --d) {
        if (idx.size(d) == 1) continue;
        if (stride < 0) stride = idx.stride(d);
        else if (idx.stride(d) != stride * run) return {idx.contiguous(), 1};
        run *= idx.size(d);
    }
    return {idx, stride < 0 ? 1 : stride};
}
// x [N, ..., C] as (tensor, sample stride, row stride): positions a row stride apart, channels adjacent.  Channel slices, channels-last
// views of NCHW tensors and broadcast gradients keep their memory; other orders are copied.
std::tuple<Tensor, int64_t, int64_t> channel_rows(const Tensor& x) {
    const int64_t C = x.size(-1), last = x.dim() - 1;
    const auto dense = [&](const Tensor& t) {
        return std::make_tuple(t, t.size(0) ? t.numel() / t.size(0) : int64_t(0), C);
    };
    if (x.is_contiguous()) return dense(x);
    if (C > 1 && x.stride(last) != 1) return dense(x.contiguous());
    int64_t row = -1, run = 1;
    for (int64_t d = last - 1; d >= 1; --d) {
        if (x.size(d) == 1) continue;
        if (row < 0) row = x.stride(d);
        else if (x.stride(d) != row * run) return dense(x.contiguous());
        run *= x.size(d);
    }
    return std::make_tuple(x, x.stride(0), row < 0 ? C : row);
}

// A node without a second derivative: with create_graph=True its gradients would count as constants.
void first_derivative_only(const char* name) {
    TORCH_CHECK(!at::GradMode::is_enabled(), name, " has no second derivative: its backward pass is refused with create_graph=True");
}

// ---------------------------------------------------------------- embedding
Tensor embed_forward(const Tensor& idx, const Tensor& table, double scale) {
    const int64_t n = idx.numel(), V = table.size(0), D = table.size(1);
    auto shape = idx.sizes().vec();
    shape.push_back(D);
    Tensor out = at::empty(shape, table.options().requires_grad(false));
    if (n == 0 || D == 0) return out;
    const auto [tok, st] = token_rows(idx);
    OnDevice on(table);
    checked("ag2v_embed_fwd", lib.embed_fwd(elem_of(table.scalar_type()), tok.data_ptr(), int(tok.element_size()), st, table.data_ptr(),
                                            V > 1 ? table.stride(0) : D, out.data_ptr(), n, V, int(D), float(scale), on.stream));
    return out;
}

struct EmbeddingScaled : torch::autograd::Function<EmbeddingScaled> {
    static Tensor forward(AutogradContext* ctx, const Tensor& idx, const Tensor& table, double scale, int64_t pad) {
        ctx->save_for_backward({idx});
        ctx->saved_data["V"] = table.size(0);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["pad"] = pad;
        return embed_forward(idx, table, scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_derivative_only("embedding_scaled");
        const Tensor idx = ctx->get_saved_variables()[0];
        const int64_t V = ctx->saved_data["V"].toInt(), pad = ctx->saved_data["pad"].toInt();
        const double scale = ctx->saved_data["scale"].toDouble();
        const int64_t n = idx.numel(), D = grads[0].size(-1);
        if (n == 0 || D == 0) return {Tensor(), at::zeros({V, D}, grads[0].options()), Tensor(), Tensor()};
        const auto [dout, sample, ds] = channel_rows(grads[0].unsqueeze(0));
        const auto [tok, st] = token_rows(idx);
        Tensor dtable = at::empty({V, D}, dout.options());
        OnDevice on(dout);
        const int type = elem_of(dout.scalar_type());
        const size_t floats = lib.embed_bwd_ws(type, n, V, int(D));
        Tensor ws = workspace_of(dout, floats);
        checked("ag2v_embed_bwd", lib.embed_bwd(type, tok.data_ptr(), int(tok.element_size()), st, dout.data_ptr(), ds, dtable.data_ptr(), n, V, int(D),
                                                float(scale), pad, static_cast<float*>(ptr(ws)), floats, on.stream));
        return {Tensor(), dtable, Tensor(), Tensor()};
    }
};

Tensor embedding_scaled(const Tensor& idx, Tensor table, double scale, std::optional<int64_t> padding_idx) {
    elem_check("embedding_scaled", table);
    TORCH_CHECK(table.dim() == 2 && table.size(0) > 0, "embedding_scaled: expected a table [V > 0, D], got ", table.sizes());
    TORCH_CHECK(idx.scalar_type() == at::kInt || idx.scalar_type() == at::kLong, "embedding_scaled: expected int32 or int64 tokens, got ",
                idx.scalar_type());
    TORCH_CHECK(idx.device() == table.device(), "embedding_scaled: tokens on ", idx.device(), ", table on ", table.device());
    TORCH_CHECK(idx.numel() < INT_LIMIT && table.size(0) < INT_LIMIT - 1 && table.size(1) < INT_LIMIT / 2, "embedding_scaled: ", idx.numel(),
                " tokens, table ", table.sizes(), ": fewer than 2^31 tokens and rows, 2^30 columns");
    TORCH_CHECK(!padding_idx || (*padding_idx >= 0 && *padding_idx < table.size(0)), "embedding_scaled: padding_idx ", padding_idx.value_or(0),
                " outside [0, ", table.size(0), ")");
    if ((table.size(1) > 1 && table.stride(1) != 1) || table.stride(0) < table.size(1)) table = table.contiguous();
    if (at::GradMode::is_enabled() && table.requires_grad()) return EmbeddingScaled::apply(idx, table, scale, padding_idx.value_or(-1));
    return embed_forward(idx, table, scale);
}

// ---------------------------------------------------------------- group norm
int param_type(const Tensor& weight, const Tensor& bias) {
    return weight.defined() ? elem_of(weight.scalar_type()) : bias.defined() ? elem_of(bias.scalar_type()) : AG2V_F32;
}
int64_t positions(const Tensor& x) { return x.numel() ? x.numel() / x.size(0) / x.size(-1) : 0; }

std::pair<Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t groups, double eps, int64_t act,
                                       double slope) {
    const int64_t N = x.size(0), C = x.size(-1), S = positions(x);
    Tensor y = at::empty(x.sizes(), x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
    Tensor stats = at::empty({2, N, groups}, x.options().requires_grad(false).dtype(at::kFloat));
    if (x.numel() == 0) return {y, stats};
    const auto [rows, xs, xr] = channel_rows(x);
    OnDevice on(x);
    const int type = elem_of(x.scalar_type());
    const size_t floats = lib.norm_ws(type, int(N), int(S), int(C), int(groups), 0);
    Tensor ws = workspace_of(x, floats);
    float* mean = stats.data_ptr<float>();
    checked("ag2v_group_norm_fwd", lib.norm_fwd(type, rows.data_ptr(), xs, xr, ptr(weight), ptr(bias), param_type(weight, bias), y.data_ptr(), mean,
                                                mean + N * groups, int(N), int(S), int(C), int(groups), float(eps), int(act), float(slope),
                                                static_cast<float*>(ptr(ws)), floats, on.stream));
    return {y, stats};
}

struct GroupNormAct : torch::autograd::Function<GroupNormAct> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight_, const std::optional<Tensor>& bias_,
                          int64_t groups, double eps, int64_t act, double slope) {
        const Tensor weight = weight_ ? *weight_ : Tensor(), bias = bias_ ? *bias_ : Tensor();
        auto [y, stats] = norm_forward(x, weight, bias, groups, eps, act, slope);
        ctx->save_for_backward({x, weight, bias, stats});
        ctx->saved_data["act"] = act;
        ctx->saved_data["slope"] = slope;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_derivative_only("group_norm_act");
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3];
        const bool some = x.numel() > 0;
        const auto made = [&](const Tensor& like) {
            return some ? at::empty(like.sizes(), like.options().memory_format(at::MemoryFormat::Contiguous)) : at::zeros(like.sizes(), like.options());
        };
        Tensor dx, dw, db;
        if (ctx->needs_input_grad(0)) dx = made(x);
        // (the edges are those of the tensors that are there)
        if (weight.defined() && ctx->needs_input_grad(1)) dw = made(weight);
        if (bias.defined() && ctx->needs_input_grad(weight.defined() ? 2 : 1)) db = made(bias);
        if (some) {
            const int64_t N = x.size(0), C = x.size(-1), S = positions(x), groups = stats.size(2);
            const auto [xrows, xs, xr] = channel_rows(x);
            const auto [drows, ds, dr] = channel_rows(grads[0]);
            OnDevice on(x);
            const int type = elem_of(x.scalar_type());
            const size_t floats = lib.norm_ws(type, int(N), int(S), int(C), int(groups), 1);
            Tensor ws = workspace_of(x, floats);
            const float* mean = stats.data_ptr<float>();
            checked("ag2v_group_norm_bwd", lib.norm_bwd(type, drows.data_ptr(), ds, dr, xrows.data_ptr(), xs, xr, ptr(weight), ptr(bias),
                                                        param_type(weight, bias), mean, mean + N * groups, ptr(dx), ptr(dw), ptr(db), int(N), int(S), int(C),
                                                        int(groups), int(ctx->saved_data["act"].toInt()), float(ctx->saved_data["slope"].toDouble()),
                                                        static_cast<float*>(ptr(ws)), floats, on.stream));
        }
        return {dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor group_norm_act(const Tensor& x, int64_t groups, const std::optional<Tensor>& weight_, const std::optional<Tensor>& bias_, double eps,
                      const std::string& act, double slope) {
    const char* name = "group_norm_act";
    elem_check(name, x);
    TORCH_CHECK(x.dim() >= 2 && x.size(-1) > 0, name, ": expected x [N, ..., C > 0], got ", x.sizes());
    const int64_t N = x.size(0), C = x.size(-1);
    TORCH_CHECK(groups > 0 && C % groups == 0, name, ": ", C, " channels do not divide into ", groups, " groups");
    const int64_t code = act == "silu" ? 1 : act == "lrelu" ? 2 : act == "none" ? 0 : -1;
    TORCH_CHECK(code >= 0, name, ": unknown activation '", act, "' (silu, lrelu, none)");
    TORCH_CHECK(eps >= 0 && eps < std::numeric_limits<double>::infinity() && !std::isnan(slope), name, ": eps ", eps, ", slope ", slope);
    TORCH_CHECK(N * groups < (int64_t(1) << 24) && positions(x) < INT_LIMIT / 2 && C < INT_LIMIT / 2, name, ": ", x.sizes(), " in ", groups,
                " groups: fewer than 2^24 (sample, group) pairs, 2^30 positions and channels");
    const auto given = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
    Tensor p[2] = {weight_ ? *weight_ : Tensor(), bias_ ? *bias_ : Tensor()};
    for (int k = 0; k < 2; ++k) {
        if (!p[k].defined()) continue;
        TORCH_CHECK(p[k].dim() == 1 && p[k].size(0) == C && p[k].device() == x.device() &&
                        (p[k].scalar_type() == x.scalar_type() || p[k].scalar_type() == at::kFloat),
                    name, ": ", k ? "bias" : "weight", " must be [", C, "] on ", x.device(), " in ", x.scalar_type(), " or float32, got ", p[k].sizes(), " ",
                    p[k].scalar_type(), " on ", p[k].device());
        p[k] = p[k].contiguous();
    }
    if (p[0].defined() && p[1].defined())
        TORCH_CHECK(p[0].scalar_type() == p[1].scalar_type(), name, ": weight is ", p[0].scalar_type(), ", bias ", p[1].scalar_type());
    const auto wants = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
    if (at::GradMode::is_enabled() && (wants(x) || wants(p[0]) || wants(p[1])))
        return GroupNormAct::apply(x, given(p[0]), given(p[1]), groups, eps, code, slope);
    return norm_forward(x, p[0], p[1], groups, eps, code, slope).first;
}
}  // namespace

PYBIND11_MODULE(_elem_ops, m) {
    m.def("bind", &bind);
    m.def("embedding_scaled", &embedding_scaled, py::call_guard<py::gil_scoped_release>());
    m.def("group_norm_act", &group_norm_act, py::call_guard<py::gil_scoped_release>());
    m.def("token_rows", &token_rows);
    m.def("channel_rows", &channel_rows);
}
