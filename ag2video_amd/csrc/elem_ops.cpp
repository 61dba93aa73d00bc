// Host side of the fp32 / bf16 / fp16 operators: argument checks, views, workspaces and autograd nodes over the C entry points of
// include/ag2v.h.  They are operators of torch's dispatcher (torch.ops.ag2v), each with a device kernel, an autograd kernel and one that gives
// the results' shapes: what watches a program at the dispatcher -- traces, dispatch modes, fake tensors, forward-mode duals -- sees a call of an
// operator, and not the empty result that the library writes behind its back.
// The nodes are C++ because the tape's backward runs on a thread of its own: a node written in Python costs 40 to 100 us there (the
// interpreter and its objects move between cores), more than the kernels of a small map.  Every refusal of a value is a RuntimeError.
#include <torch/extension.h>
#include <torch/library.h>

#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <array>
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
} entries;

void bind(uintptr_t embed_fwd, uintptr_t embed_bwd_ws, uintptr_t embed_bwd, uintptr_t norm_ws, uintptr_t norm_fwd, uintptr_t norm_bwd) {
    entries.embed_fwd = reinterpret_cast<decltype(entries.embed_fwd)>(embed_fwd);
    entries.embed_bwd_ws = reinterpret_cast<decltype(entries.embed_bwd_ws)>(embed_bwd_ws);
    entries.embed_bwd = reinterpret_cast<decltype(entries.embed_bwd)>(embed_bwd);
    entries.norm_ws = reinterpret_cast<decltype(entries.norm_ws)>(norm_ws);
    entries.norm_fwd = reinterpret_cast<decltype(entries.norm_fwd)>(norm_fwd);
    entries.norm_bwd = reinterpret_cast<decltype(entries.norm_bwd)>(norm_bwd);
}

const Entries& library() {
    TORCH_CHECK(entries.embed_fwd, "ag2video_amd: its library is not loaded yet (ag2video_amd._lib.elem_ops())");
    return entries;
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
// Nor a tangent: without a check its result would count as a constant.
void reverse_mode_only(const char* name, std::initializer_list<const Tensor*> inputs) {
    for (const Tensor* t : inputs) TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), name, " has no forward-mode derivative");
}
const Tensor& given(const std::optional<Tensor>& t) {
    static const Tensor none;
    return t ? *t : none;
}
std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
bool wants_grad(std::initializer_list<const Tensor*> inputs) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : inputs)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}
// An operator of this library, as the dispatcher calls it.
template <class F>
c10::TypedOperatorHandle<F> op_of(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

// ---------------------------------------------------------------- embedding
// padding_idx is -1 for none in all of these
void embedding_check(const Tensor& idx, const Tensor& table, int64_t pad) {
    TORCH_CHECK(elem_of(table.scalar_type()) >= 0, "embedding_scaled: expected float32, bfloat16 or float16, got ", table.scalar_type());
    TORCH_CHECK(table.dim() == 2 && table.size(0) > 0, "embedding_scaled: expected a table [V > 0, D], got ", table.sizes());
    TORCH_CHECK(idx.scalar_type() == at::kInt || idx.scalar_type() == at::kLong, "embedding_scaled: expected int32 or int64 tokens, got ",
                idx.scalar_type());
    TORCH_CHECK(idx.device() == table.device(), "embedding_scaled: tokens on ", idx.device(), ", table on ", table.device());
    TORCH_CHECK(idx.numel() < INT_LIMIT && table.size(0) < INT_LIMIT - 1 && table.size(1) < INT_LIMIT / 2, "embedding_scaled: ", idx.numel(),
                " tokens, table ", table.sizes(), ": fewer than 2^31 tokens and rows, 2^30 columns");
    TORCH_CHECK(pad >= -1 && pad < table.size(0), "embedding_scaled: padding_idx ", pad, " outside [0, ", table.size(0), ")");
}
Tensor embedding_result(const Tensor& idx, const Tensor& table) {
    auto shape = idx.sizes().vec();
    shape.push_back(table.size(1));
    return at::empty(shape, table.options().requires_grad(false));
}
Tensor embedding_meta(const Tensor& idx, const Tensor& table, double, int64_t pad) {
    embedding_check(idx, table, pad);
    return embedding_result(idx, table);
}
Tensor embedding_device(const Tensor& idx, const Tensor& table_, double scale, int64_t pad) {
    embedding_check(idx, table_, pad);
    Tensor out = embedding_result(idx, table_);
    const int64_t n = idx.numel(), V = table_.size(0), D = table_.size(1);
    if (n == 0 || D == 0) return out;
    const bool rows = (D == 1 || table_.stride(1) == 1) && table_.stride(0) >= D;
    const Tensor table = rows ? table_ : table_.contiguous();
    const auto [tok, st] = token_rows(idx);
    OnDevice on(table);
    checked("ag2v_embed_fwd", library().embed_fwd(elem_of(table.scalar_type()), tok.data_ptr(), int(tok.element_size()), st, table.data_ptr(),
                                            V > 1 ? table.stride(0) : D, out.data_ptr(), n, V, int(D), float(scale), on.stream));
    return out;
}
void embedding_backward_check(const Tensor& dout, const Tensor& idx, int64_t V, int64_t pad) {
    TORCH_CHECK(elem_of(dout.scalar_type()) >= 0 && dout.device() == idx.device() && dout.dim() == idx.dim() + 1 &&
                    dout.sizes().slice(0, idx.dim()) == idx.sizes() && (idx.scalar_type() == at::kInt || idx.scalar_type() == at::kLong),
                "embedding_scaled_backward: gradient ", dout.sizes(), " ", dout.scalar_type(), " on ", dout.device(), " of tokens ", idx.sizes(), " ",
                idx.scalar_type(), " on ", idx.device());
    TORCH_CHECK(V > 0 && V < INT_LIMIT - 1 && pad >= -1 && pad < V && idx.numel() < INT_LIMIT && dout.size(-1) < INT_LIMIT / 2,
                "embedding_scaled_backward: ", V, " rows, padding_idx ", pad, ", gradient ", dout.sizes());
}
Tensor embedding_backward_meta(const Tensor& dout, const Tensor& idx, int64_t V, double, int64_t pad) {
    embedding_backward_check(dout, idx, V, pad);
    return at::empty({V, dout.size(-1)}, dout.options());
}
Tensor embedding_backward_device(const Tensor& grad, const Tensor& idx, int64_t V, double scale, int64_t pad) {
    embedding_backward_check(grad, idx, V, pad);
    const int64_t n = idx.numel(), D = grad.size(-1);
    if (n == 0 || D == 0) return at::zeros({V, D}, grad.options());
    const auto [dout, sample, ds] = channel_rows(grad.unsqueeze(0));
    const auto [tok, st] = token_rows(idx);
    Tensor dtable = at::empty({V, D}, dout.options());
    OnDevice on(dout);
    const int type = elem_of(dout.scalar_type());
    const size_t floats = library().embed_bwd_ws(type, n, V, int(D));
    Tensor ws = workspace_of(dout, floats);
    checked("ag2v_embed_bwd", library().embed_bwd(type, tok.data_ptr(), int(tok.element_size()), st, dout.data_ptr(), ds, dtable.data_ptr(), n, V, int(D),
                                            float(scale), pad, static_cast<float*>(ptr(ws)), floats, on.stream));
    return dtable;
}
Tensor embedding_call(const Tensor& idx, const Tensor& table, double scale, int64_t pad) {
    static const auto op = op_of<decltype(embedding_device)>("ag2v::embedding_scaled");
    return op.call(idx, table, scale, pad);
}
Tensor embedding_backward_call(const Tensor& dout, const Tensor& idx, int64_t V, double scale, int64_t pad) {
    static const auto op = op_of<decltype(embedding_backward_device)>("ag2v::embedding_scaled_backward");
    return op.call(dout, idx, V, scale, pad);
}

struct EmbeddingScaled : torch::autograd::Function<EmbeddingScaled> {
    static Tensor forward(AutogradContext* ctx, const Tensor& idx, const Tensor& table, double scale, int64_t pad) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({idx});
        ctx->saved_data["V"] = table.size(0);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["pad"] = pad;
        return embedding_call(idx, table, scale, pad);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_derivative_only("embedding_scaled");
        const Tensor idx = ctx->get_saved_variables()[0];      // (above the guard: a checkpoint runs its forward pass again in here)
        at::AutoDispatchBelowADInplaceOrView below;
        Tensor dtable = embedding_backward_call(grads[0], idx, ctx->saved_data["V"].toInt(), ctx->saved_data["scale"].toDouble(),
                                                ctx->saved_data["pad"].toInt());
        return {Tensor(), dtable, Tensor(), Tensor()};
    }
};
Tensor embedding_autograd(const Tensor& idx, const Tensor& table, double scale, int64_t pad) {
    reverse_mode_only("embedding_scaled", {&table});
    if (wants_grad({&table})) return EmbeddingScaled::apply(idx, table, scale, pad);
    at::AutoDispatchBelowADInplaceOrView below;
    return embedding_call(idx, table, scale, pad);
}

Tensor embedding_scaled(const Tensor& idx, const Tensor& table, double scale, std::optional<int64_t> padding_idx) {
    elem_check("embedding_scaled", table);
    TORCH_CHECK(!padding_idx || *padding_idx >= 0, "embedding_scaled: padding_idx ", padding_idx.value_or(0), " is negative");
    return embedding_call(idx, table, scale, padding_idx.value_or(-1));
}

// ---------------------------------------------------------------- group norm
int param_type(const Tensor& weight, const Tensor& bias) {
    return weight.defined() ? elem_of(weight.scalar_type()) : bias.defined() ? elem_of(bias.scalar_type()) : AG2V_F32;
}
int64_t positions(const Tensor& x) { return x.numel() ? x.numel() / x.size(0) / x.size(-1) : 0; }
Tensor dense_like(const Tensor& t) { return at::empty(t.sizes(), t.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous)); }

Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

void norm_check(const Tensor& x, int64_t groups, const Tensor& weight, const Tensor& bias, double eps, int64_t act, double slope) {
    const char* name = "group_norm_act";
    TORCH_CHECK(elem_of(x.scalar_type()) >= 0, name, ": expected float32, bfloat16 or float16, got ", x.scalar_type());
    TORCH_CHECK(x.dim() >= 2 && x.size(-1) > 0, name, ": expected x [N, ..., C > 0], got ", x.sizes());
    const int64_t N = x.size(0), C = x.size(-1);
    TORCH_CHECK(groups > 0 && C % groups == 0, name, ": ", C, " channels do not divide into ", groups, " groups");
    TORCH_CHECK(act >= 0 && act <= 2, name, ": unknown activation code ", act);
    TORCH_CHECK(eps >= 0 && eps < std::numeric_limits<double>::infinity() && !std::isnan(slope), name, ": eps ", eps, ", slope ", slope);
    TORCH_CHECK(N * groups < (int64_t(1) << 24) && positions(x) < INT_LIMIT / 2 && C < INT_LIMIT / 2, name, ": ", x.sizes(), " in ", groups,
                " groups: fewer than 2^24 (sample, group) pairs, 2^30 positions and channels");
    for (const Tensor* p : {&weight, &bias}) {
        if (!p->defined()) continue;
        TORCH_CHECK(p->dim() == 1 && p->size(0) == C && p->device() == x.device() &&
                        (p->scalar_type() == x.scalar_type() || p->scalar_type() == at::kFloat),
                    name, ": ", p == &bias ? "bias" : "weight", " must be [", C, "] on ", x.device(), " in ", x.scalar_type(), " or float32, got ", p->sizes(),
                    " ", p->scalar_type(), " on ", p->device());
    }
    if (weight.defined() && bias.defined())
        TORCH_CHECK(weight.scalar_type() == bias.scalar_type(), name, ": weight is ", weight.scalar_type(), ", bias ", bias.scalar_type());
}
typedef std::optional<Tensor> Param;
std::tuple<Tensor, Tensor> norm_results(const Tensor& x, int64_t groups) {
    return {dense_like(x), at::empty({2, x.size(0), groups}, x.options().requires_grad(false).dtype(at::kFloat))};
}
std::tuple<Tensor, Tensor> norm_stats_meta(const Tensor& x, int64_t groups, const Param& weight, const Param& bias, double eps, int64_t act, double slope) {
    norm_check(x, groups, given(weight), given(bias), eps, act, slope);
    return norm_results(x, groups);
}
// y, and mean and 1 / std of every (sample, group)
std::tuple<Tensor, Tensor> norm_stats_device(const Tensor& x, int64_t groups, const Param& weight_, const Param& bias_, double eps, int64_t act, double slope) {
    norm_check(x, groups, given(weight_), given(bias_), eps, act, slope);
    auto [y, stats] = norm_results(x, groups);
    if (x.numel() == 0) return {y, stats};
    const Tensor weight = dense(given(weight_)), bias = dense(given(bias_));
    const int64_t N = x.size(0), C = x.size(-1), S = positions(x);
    const auto [rows, xs, xr] = channel_rows(x);
    OnDevice on(x);
    const int type = elem_of(x.scalar_type());
    const size_t floats = library().norm_ws(type, int(N), int(S), int(C), int(groups), 0);
    Tensor ws = workspace_of(x, floats);
    float* mean = stats.data_ptr<float>();
    checked("ag2v_group_norm_fwd", library().norm_fwd(type, rows.data_ptr(), xs, xr, ptr(weight), ptr(bias), param_type(weight, bias), y.data_ptr(), mean,
                                                mean + N * groups, int(N), int(S), int(C), int(groups), float(eps), int(act), float(slope),
                                                static_cast<float*>(ptr(ws)), floats, on.stream));
    return {y, stats};
}
Tensor norm_meta(const Tensor& x, int64_t groups, const Param& weight, const Param& bias, double eps, int64_t act, double slope) {
    return std::get<0>(norm_stats_meta(x, groups, weight, bias, eps, act, slope));
}
Tensor norm_device(const Tensor& x, int64_t groups, const Param& weight, const Param& bias, double eps, int64_t act, double slope) {
    return std::get<0>(norm_stats_device(x, groups, weight, bias, eps, act, slope));
}
void norm_backward_check(const Tensor& dy, const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& stats, int64_t act, double slope) {
    const char* name = "group_norm_act_backward";
    TORCH_CHECK(x.dim() >= 2 && stats.dim() == 3 && stats.size(0) == 2 && stats.size(1) == x.size(0) && stats.scalar_type() == at::kFloat &&
                    stats.is_contiguous() && stats.device() == x.device(), name, ": statistics ", stats.sizes(), " of x ", x.sizes());
    TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() && dy.device() == x.device(), name, ": gradient ", dy.sizes(), " ",
                dy.scalar_type(), " on ", dy.device(), " of x ", x.sizes(), " ", x.scalar_type(), " on ", x.device());
    norm_check(x, stats.size(2), weight, bias, 0.0, act, slope);
}
typedef std::tuple<Tensor, Tensor, Tensor> Grads;      // of x, weight and bias; undefined where not wanted
Grads norm_backward_meta(const Tensor& dy, const Tensor& x, const Param& weight_, const Param& bias_, const Tensor& stats, int64_t act, double slope,
                         std::array<bool, 3> wanted) {
    const Tensor &weight = given(weight_), &bias = given(bias_);
    norm_backward_check(dy, x, weight, bias, stats, act, slope);
    return {wanted[0] ? dense_like(x) : Tensor(), wanted[1] && weight.defined() ? dense_like(weight) : Tensor(),
            wanted[2] && bias.defined() ? dense_like(bias) : Tensor()};
}
Grads norm_backward_device(const Tensor& dy, const Tensor& x, const Param& weight_, const Param& bias_, const Tensor& stats, int64_t act, double slope,
                           std::array<bool, 3> wanted) {
    auto [dx, dw, db] = norm_backward_meta(dy, x, weight_, bias_, stats, act, slope, wanted);
    if (x.numel() == 0) {
        for (Tensor* t : {&dw, &db})
            if (t->defined()) t->zero_();
        return {dx, dw, db};
    }
    const Tensor weight = dense(given(weight_)), bias = dense(given(bias_));
    const int64_t N = x.size(0), C = x.size(-1), S = positions(x), groups = stats.size(2);
    const auto [xrows, xs, xr] = channel_rows(x);
    const auto [drows, ds, dr] = channel_rows(dy);
    OnDevice on(x);
    const int type = elem_of(x.scalar_type());
    const size_t floats = library().norm_ws(type, int(N), int(S), int(C), int(groups), 1);
    Tensor ws = workspace_of(x, floats);
    const float* mean = stats.data_ptr<float>();
    checked("ag2v_group_norm_bwd", library().norm_bwd(type, drows.data_ptr(), ds, dr, xrows.data_ptr(), xs, xr, ptr(weight), ptr(bias),
                                                param_type(weight, bias), mean, mean + N * groups, ptr(dx), ptr(dw), ptr(db), int(N), int(S), int(C),
                                                int(groups), int(act), float(slope), static_cast<float*>(ptr(ws)), floats, on.stream));
    return {dx, dw, db};
}
Tensor norm_call(const Tensor& x, int64_t groups, const Param& weight, const Param& bias, double eps, int64_t act, double slope) {
    static const auto op = op_of<decltype(norm_device)>("ag2v::group_norm_act");
    return op.call(x, groups, weight, bias, eps, act, slope);
}
std::tuple<Tensor, Tensor> norm_stats_call(const Tensor& x, int64_t groups, const Param& weight, const Param& bias, double eps, int64_t act,
                                           double slope) {
    static const auto op = op_of<decltype(norm_stats_device)>("ag2v::group_norm_act_stats");
    return op.call(x, groups, weight, bias, eps, act, slope);
}
Grads norm_backward_call(const Tensor& dy, const Tensor& x, const Param& weight, const Param& bias, const Tensor& stats, int64_t act, double slope,
                         std::array<bool, 3> wanted) {
    static const auto op = op_of<decltype(norm_backward_device)>("ag2v::group_norm_act_backward");
    return op.call(dy, x, weight, bias, stats, act, slope, wanted);
}

struct GroupNormAct : torch::autograd::Function<GroupNormAct> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Param& weight, const Param& bias, int64_t groups, double eps, int64_t act,
                          double slope) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [y, stats] = norm_stats_call(x, groups, weight, bias, eps, act, slope);
        ctx->save_for_backward({x, given(weight), given(bias), stats});
        ctx->saved_data["act"] = act;
        ctx->saved_data["slope"] = slope;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_derivative_only("group_norm_act");
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3];
        at::AutoDispatchBelowADInplaceOrView below;
        // (the edges are those of the tensors that are there)
        const auto [dx, dw, db] = norm_backward_call(grads[0], x, maybe(weight), maybe(bias), stats, ctx->saved_data["act"].toInt(),
                                                     ctx->saved_data["slope"].toDouble(),
                                                     {ctx->needs_input_grad(0), weight.defined() && ctx->needs_input_grad(1),
                                                      bias.defined() && ctx->needs_input_grad(weight.defined() ? 2 : 1)});
        return {dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};
Tensor norm_autograd(const Tensor& x, int64_t groups, const Param& weight, const Param& bias, double eps, int64_t act, double slope) {
    reverse_mode_only("group_norm_act", {&x, &given(weight), &given(bias)});
    if (wants_grad({&x, &given(weight), &given(bias)})) return GroupNormAct::apply(x, weight, bias, groups, eps, act, slope);
    at::AutoDispatchBelowADInplaceOrView below;
    return norm_call(x, groups, weight, bias, eps, act, slope);
}

Tensor group_norm_act(const Tensor& x, int64_t groups, const Param& weight, const Param& bias, double eps, const std::string& act, double slope) {
    elem_check("group_norm_act", x);
    const int64_t code = act == "silu" ? 1 : act == "lrelu" ? 2 : act == "none" ? 0 : -1;
    TORCH_CHECK(code >= 0, "group_norm_act: unknown activation '", act, "' (silu, lrelu, none)");
    return norm_call(x, groups, weight, bias, eps, code, slope);
}
}  // namespace

TORCH_LIBRARY(ag2v, m) {
    m.def("embedding_scaled(Tensor idx, Tensor table, float scale, int padding_idx) -> Tensor");
    m.def("embedding_scaled_backward(Tensor dout, Tensor idx, int rows, float scale, int padding_idx) -> Tensor");
    m.def("group_norm_act(Tensor x, int groups, Tensor? weight, Tensor? bias, float eps, int act, float slope) -> Tensor");
    // with the statistics, for the tape: no derivative of its own
    m.def("group_norm_act_stats(Tensor x, int groups, Tensor? weight, Tensor? bias, float eps, int act, float slope) -> (Tensor, Tensor)");
    m.def("group_norm_act_backward(Tensor dy, Tensor x, Tensor? weight, Tensor? bias, Tensor stats, int act, float slope, bool[3] wanted)"
          " -> (Tensor, Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(ag2v, CUDA, m) {         // (the key of HIP devices)
    m.impl("embedding_scaled", &embedding_device);
    m.impl("embedding_scaled_backward", &embedding_backward_device);
    m.impl("group_norm_act", &norm_device);
    m.impl("group_norm_act_stats", &norm_stats_device);
    m.impl("group_norm_act_backward", &norm_backward_device);
}
TORCH_LIBRARY_IMPL(ag2v, Meta, m) {
    m.impl("embedding_scaled", &embedding_meta);
    m.impl("embedding_scaled_backward", &embedding_backward_meta);
    m.impl("group_norm_act", &norm_meta);
    m.impl("group_norm_act_stats", &norm_stats_meta);
    m.impl("group_norm_act_backward", &norm_backward_meta);
}
TORCH_LIBRARY_IMPL(ag2v, Autograd, m) {
    m.impl("embedding_scaled", &embedding_autograd);
    m.impl("group_norm_act", &norm_autograd);
}

PYBIND11_MODULE(_elem_ops, m) {
    m.def("bind", &bind);
    m.def("embedding_scaled", &embedding_scaled, py::call_guard<py::gil_scoped_release>());
    m.def("group_norm_act", &group_norm_act, py::call_guard<py::gil_scoped_release>());
    m.def("token_rows", &token_rows);
    m.def("channel_rows", &channel_rows);
}
