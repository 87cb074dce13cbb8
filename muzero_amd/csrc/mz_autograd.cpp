// torch's side of group norm, the categorical loss and clipping: argument checks, strides, outputs and autograd nodes around the C
// entries of libmzhip.so.  Built as muzero_amd/_autograd.so.  In C++ because a node in Python costs more than these
// operators do: its backward pass runs on the autograd thread, has to take the interpreter from the thread that waits for
// it, and moves Python's objects between the cores of both (120 to 130 us a forward and backward pass of a small state,
// of which an empty node takes 22 to 46).
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <cstring>
#include <string>
#include <unordered_set>
#include <vector>

#include "../../include/mzhip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Refused : std::runtime_error {            // MuZeroError
    using std::runtime_error::runtime_error;
};
struct Failed : std::runtime_error {             // MuZeroHipError
    int status;
    Failed(int s, const char* m) : std::runtime_error(m), status(s) {}
};

template <typename... A>
[[noreturn]] void refuse(const A&... a) {
    throw Refused(c10::str(a...));
}
int64_t done(int64_t status) {
    if (status < 0) throw Failed((int)status, mz_last_error());
    return status;
}

int dtype_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return MZ_F32;
        case at::kHalf: return MZ_F16;
        case at::kBFloat16: return MZ_BF16;
        default: return -1;
    }
}
void require_type(const char* name, const Tensor& t, bool fits, const char* expected) {
    if (!fits) refuse(name, ": expected ", expected, ", got ", t.scalar_type());
}
void require_device(const char* name, const Tensor& t, const c10::Device& d) {
    if (t.device() != d) refuse(name, " is on ", t.device(), ", expected ", d);
}
void require_hip(const c10::Device& d) {
    if (!d.is_cuda()) refuse("the tensors must be on a HIP device, not ", d, "; muzero_amd has no CPU fallback");
}

// What the kernels cannot take from t's memory, or nullptr.  Derivatives that travel with a tensor instead of a graph would be
// lost without a word.
const char* unreadable(const Tensor& t) {
    if (t.layout() != at::kStrided) return "is not a strided tensor";
    // a null pointer would pass for an input that is not given
    if (!t.has_storage() || (t.numel() && !t._is_zerotensor() && !t.const_data_ptr()))
        return "has no memory of its own (a tensor inside a transform of torch.func, or one that wraps others)";
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
        return "carries a forward-mode derivative: muzero_amd's training operators are differentiable in reverse mode alone";
    return nullptr;
}
void require_readable(const char* name, const Tensor& t) {
    if (const char* why = unreadable(t)) refuse(name, " ", why);
}
void require_readable(const char* name, const OptTensor& t) {
    if (t) require_readable(name, *t);
}

// t with what torch does lazily carried out, which t's memory does not hold: its sign, and zeros without any
Tensor written_out(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t._is_zerotensor() ? t.clone() : t; }

// A recording of torch's operations would hold the outputs' allocation and not the kernel that fills them.
void refuse_while_recording() {
    using c10::impl::TorchDispatchModeKey;
    using c10::impl::TorchDispatchModeTLS;
    if (torch::jit::tracer::isTracing()) refuse("muzero_amd's operators cannot be recorded by torch.jit.trace");
    if (TorchDispatchModeTLS::any_modes_set() &&
        (TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY) || TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FAKE) ||
         TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FUNCTIONAL)))
        refuse("muzero_amd's operators cannot be recorded by torch.fx or torch.export, nor run on fake tensors");
}

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool wants_grad(const OptTensor& t) { return t && t->requires_grad(); }

// The device of the call made current, and its current stream
struct On {
    c10::DeviceGuard guard;
    void* stream;
    explicit On(const c10::Device& d) : guard(d), stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(d.index()).stream()) {}
};

// A backward pass runs every node of the graph on the stream the node was made on; a leaf's accumulation node lives as long
// as any graph that holds it.  A backward pass captured while the captured graph reaches a node of a stream outside the
// capture -- through a leaf that an eager graph holds, or an eager graph in front -- would leave the capture, which ends the
// process: refused when the forward pass is captured, before anything is launched.
void refuse_nodes_outside_capture(const c10::Device& d, std::initializer_list<const Tensor*> inputs) {
    const auto here = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(d.index());
    if (!done(mz_stream_is_capturing(here.stream()))) return;
    std::vector<std::shared_ptr<torch::autograd::Node>> todo;
    std::unordered_set<torch::autograd::Node*> seen;
    const auto visit = [&](std::shared_ptr<torch::autograd::Node> node) {
        if (node && seen.insert(node.get()).second) todo.push_back(std::move(node));
    };
    for (const Tensor* t : inputs)
        if (t->defined() && t->requires_grad()) visit(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
    while (!todo.empty()) {
        const auto node = std::move(todo.back());
        todo.pop_back();
        const auto made_on = node->stream();
        if (made_on && *made_on != here.unwrap() &&
            !done(mz_stream_is_capturing(c10::hip::HIPStreamMasqueradingAsCUDA(*made_on).stream())))
            refuse("this forward pass is being captured, and its backward pass would reach a node (", node->name(), ") of a stream outside "
                   "the capture: an eager autograd graph of the same leaf tensors is alive, or lies in front of this call; delete its "
                   "outputs (the loss among them), or detach the input, before capturing");
        for (const auto& edge : node->next_edges()) visit(edge.function);
    }
}

// Differentiable once: under create_graph the gradients pass through a node that depends on all they were computed from and
// refuses to be differentiated.
struct Once : torch::autograd::Function<Once> {
    static Tensor forward(AutogradContext*, const Tensor& gradient, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                          const OptTensor&) {
        return gradient.view_as(gradient);
    }
    static variable_list backward(AutogradContext*, variable_list) {
        throw std::runtime_error("muzero_amd's training operators are differentiable once");
    }
};
variable_list once(variable_list gradients, const std::array<Tensor, 5>& from) {
    if (at::GradMode::is_enabled()) {
        const auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
        for (Tensor& g : gradients)
            if (g.defined()) g = Once::apply(g, opt(from[0]), opt(from[1]), opt(from[2]), opt(from[3]), opt(from[4]));
    }
    return gradients;
}

// ---- group norm -------------------------------------------------------------------------------------------------------

// t or a dense copy of it, as [batch][positions][C] with adjacent channels and one stride each for batch and positions
Tensor states(const Tensor& t, int64_t (&strides)[2]) {
    const auto shape = t.sizes();
    const int64_t n = t.dim();
    if (!t.is_contiguous() && (t.stride(n - 1) == 1 || shape[n - 1] == 1)) {
        const auto st = t.strides();
        int64_t step = 0, span = 1;
        bool even = true;
        for (int64_t i = n - 2; i > 0; --i) {
            if (shape[i] == 1) continue;
            if (span == 1) step = st[i];
            even = even && st[i] == step * span;
            span *= shape[i];
        }
        if (even) {
            strides[0] = st[0];
            strides[1] = step;
            return t;
        }
    }
    const Tensor c = t.contiguous();
    strides[0] = c.stride(0);
    strides[1] = shape[n - 1];
    return c;
}

struct NormCall {
    mz_group_norm_t config;
    Tensor x, residual, weight, bias;            // as the kernels read them
};

Tensor norm_forward(NormCall& c, Tensor* stats) {
    const Tensor y = at::empty(c.x.sizes(), c.x.options().memory_format(at::MemoryFormat::Contiguous));
    float *mean = nullptr, *rstd = nullptr;
    if (stats) {
        *stats = at::empty({2, c.config.batch, c.config.groups}, c.x.options().dtype(at::kFloat));
        mean = stats->data_ptr<float>();
        rstd = mean + c.config.batch * c.config.groups;
    }
    const int64_t bytes = done(mz_group_norm_workspace(&c.config, 0));
    const Tensor ws = bytes ? at::empty({bytes}, c.x.options().dtype(at::kByte)) : Tensor();
    const On on(c.x.device());
    done(mz_group_norm_forward(on.stream, &c.config, data(c.x), data(c.residual), data(c.weight), data(c.bias), data(y), mean, rstd,
                               data(ws), bytes));
    return y;
}

struct GroupNorm : torch::autograd::Function<GroupNorm> {
    // the differentiable tensors once as they came, for the graph, and in `call` as the kernels read them
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, const OptTensor& residual,
                          NormCall* call) {
        Tensor stats;
        const Tensor y = norm_forward(*call, &stats);
        // the residual enters the gradients through the activation's argument alone
        ctx->save_for_backward({call->x, call->weight, call->bias, call->config.activation ? call->residual : Tensor(), stats});
        ctx->saved_data["config"] = std::string(reinterpret_cast<const char*>(&call->config), sizeof(call->config));
        ctx->saved_data["residual"] = call->residual.defined();
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list dys) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &residual = saved[3], &stats = saved[4];
        mz_group_norm_t config;
        memcpy(&config, ctx->saved_data["config"].toStringRef().data(), sizeof(config));
        require_readable("the gradient", dys[0]);
        const Tensor dy = states(written_out(dys[0]), config.dy_strides);
        const auto like = [&](int input, const Tensor& t) {
            return ctx->needs_input_grad(input) ? at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous)) : Tensor();
        };
        const bool has_weight = weight.defined(), has_bias = bias.defined();
        // inputs that are absent have no edge, and the others move up
        int edge = 0;
        const Tensor dx = like(edge++, x), dweight = has_weight ? like(edge++, weight) : Tensor(), dbias = has_bias ? like(edge++, bias) : Tensor();
        const Tensor dresidual = ctx->saved_data["residual"].toBool() ? like(edge, x) : Tensor();
        const int64_t bytes = done(mz_group_norm_workspace(&config, 1));
        const Tensor ws = bytes ? at::empty({bytes}, x.options().dtype(at::kByte)) : Tensor();
        {
            const On on(x.device());
            const float* mean = stats.data_ptr<float>();
            done(mz_group_norm_backward(on.stream, &config, data(x), data(residual), data(weight), data(bias), mean,
                                        mean + config.batch * config.groups, data(dy), data(dx), data(dresidual), data(dweight),
                                        data(dbias), data(ws), bytes));
        }
        return once({dx, dweight, dbias, dresidual, Tensor()}, {x, weight, bias, residual, dys[0]});
    }
};

int activation_of(const std::optional<std::string>& name) {
    if (!name) return MZ_ACT_NONE;
    if (*name == "relu") return MZ_ACT_RELU;
    if (*name == "silu") return MZ_ACT_SILU;
    if (*name == "gelu") return MZ_ACT_GELU;
    if (*name == "tanh") return MZ_ACT_TANH;
    refuse("activation '", *name, "' is not one of None, 'relu', 'silu', 'gelu', 'tanh'");
}

Tensor group_norm(const Tensor& x, int64_t groups, const OptTensor& weight, const OptTensor& bias, double eps,
                  const std::optional<std::string>& activation, const OptTensor& residual) {
    refuse_while_recording();
    require_readable("x", x);
    require_readable("weight", weight);
    require_readable("bias", bias);
    require_readable("residual", residual);
    require_type("x", x, dtype_of(x) >= 0, "float32, float16 or bfloat16");
    if (x.dim() < 2) refuse("x must be [B, ..., C], got shape ", x.sizes());
    const int64_t channels = x.size(-1);
    if (channels > MZ_GROUP_NORM_MAX_CHANNELS) refuse("at most ", MZ_GROUP_NORM_MAX_CHANNELS, " channels, got ", channels);
    if (groups < 1 || channels < 1 || channels % groups) refuse(channels, " channels cannot be split into ", groups, " groups");
    const int act = activation_of(activation);
    if (!(eps >= 0) || !std::isfinite(eps)) refuse("eps must be finite and >= 0, got ", eps);
    for (const auto& [name, p] : {std::pair<const char*, const OptTensor&>("weight", weight), {"bias", bias}}) {
        if (!p) continue;
        require_type(name, *p, p->scalar_type() == at::kFloat || p->scalar_type() == x.scalar_type(), "float32 or the type of x");
        require_device(name, *p, x.device());
        if (p->dim() != 1 || p->size(0) != channels) refuse(name, " must have shape [", channels, "], got ", p->sizes());
    }
    if (weight && bias && weight->scalar_type() != bias->scalar_type())
        refuse("weight is ", weight->scalar_type(), ", bias ", bias->scalar_type(), ": both must be of one type");
    if (residual) {
        require_type("residual", *residual, residual->scalar_type() == x.scalar_type(), "the type of x");
        require_device("residual", *residual, x.device());
        if (residual->sizes() != x.sizes()) refuse("residual has shape ", residual->sizes(), ", x ", x.sizes());
    }
    require_hip(x.device());
    NormCall c = {};
    c.config.batch = x.size(0);
    c.config.positions = 1;
    for (int64_t i = 1; i + 1 < x.dim(); ++i) c.config.positions *= x.size(i);
    c.config.channels = (int32_t)channels;
    c.config.groups = (int32_t)groups;
    c.config.dtype = dtype_of(x);
    c.config.param_dtype = weight ? dtype_of(*weight) : bias ? dtype_of(*bias) : (int)MZ_F32;
    c.config.activation = act;
    c.config.eps = eps;
    const bool differentiable = at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(weight) || wants_grad(bias) || wants_grad(residual));
    if (differentiable)
        refuse_nodes_outside_capture(x.device(), {&x, weight ? &*weight : &x, bias ? &*bias : &x, residual ? &*residual : &x});
    {
        const at::NoGradGuard off;
        c.x = states(written_out(x), c.config.x_strides);
        if (residual) c.residual = states(written_out(*residual), c.config.residual_strides);
        if (weight) c.weight = written_out(*weight).contiguous();
        if (bias) c.bias = written_out(*bias).contiguous();
        if (!differentiable) return norm_forward(c, nullptr);
    }
    return GroupNorm::apply(x, weight, bias, residual, &c);
}

// ---- categorical loss -------------------------------------------------------------------------------------------------

struct LossCall {
    mz_categorical_t config;
    Tensor logits, targets, game, position, weights;      // as the kernel reads them
};

// a tensor of the rows' shape or a dense copy of it, with its (unroll, batch) strides
Tensor rows_of(const Tensor& t, int64_t (&strides)[2]) {
    if (t.dim() == 2) {
        strides[0] = t.stride(0);
        strides[1] = t.stride(1);
        return t;
    }
    strides[0] = 0;
    strides[1] = 1;
    return t.contiguous();
}

LossCall describe(const Tensor& logits, const Tensor& targets, const OptTensor& game, const OptTensor& position, const OptTensor& weights) {
    refuse_while_recording();
    require_readable("logits", logits);
    require_readable("targets", targets);
    require_readable("game", game);
    require_readable("position", position);
    require_readable("weights", weights);
    require_type("logits", logits, dtype_of(logits) >= 0, "float32, float16 or bfloat16");
    const c10::Device device = logits.device();
    const auto shape = logits.sizes();
    if (shape.size() < 2 || shape.back() < 1 || shape.back() > 4096)
        refuse("logits must be [..., classes] with 1 to 4096 classes, got ", shape);
    const int64_t classes = shape.back();
    const auto rows = shape.slice(0, shape.size() - 1);
    require_type("targets", targets, targets.scalar_type() == at::kFloat, "float32");
    require_device("targets", targets, device);
    if (targets.requires_grad()) refuse("the loss is not differentiable with respect to targets");
    LossCall c = {};
    c.config.classes = (int32_t)classes;
    c.config.dtype = dtype_of(logits);
    c.config.index_bytes = 4;
    if (game || position) {
        if (shape.size() != 3) refuse("with game and position, logits must be [unroll, batch, classes], got ", shape);
        if (!game || !position) refuse("game and position: both or neither");
        if (targets.dim() != 3 || targets.size(2) != classes) refuse("targets must be [positions, games, ", classes, "], got ", targets.sizes());
        for (const auto& [name, t] : {std::pair<const char*, const OptTensor&>("game", game), {"position", position}}) {
            require_type(name, *t, t->scalar_type() == at::kInt || t->scalar_type() == at::kLong, "int32 or int64");
            require_device(name, *t, device);
            if (t->dim() != 1 || t->size(0) != rows[1]) refuse(name, " must have shape [", rows[1], "], got ", t->sizes());
        }
        if (game->scalar_type() != position->scalar_type())
            refuse("game is ", game->scalar_type(), ", position ", position->scalar_type(), ": both must be of one type");
        c.config.index_bytes = (int32_t)game->element_size();
        c.config.target_positions = targets.size(0);
        c.config.target_games = targets.size(1);
    } else if (targets.sizes() != shape) {
        refuse("targets have shape ", targets.sizes(), ", logits ", shape);
    }
    Tensor w;
    if (weights) {
        require_type("weights", *weights, weights->scalar_type() == at::kFloat, "float32");
        require_device("weights", *weights, device);
        if (weights->requires_grad()) refuse("the loss is not differentiable with respect to weights");
        bool fits = weights->dim() <= (int64_t)rows.size();
        for (int64_t i = 1; fits && i <= weights->dim(); ++i) fits = weights->size(-i) == 1 || weights->size(-i) == rows[rows.size() - i];
        if (!fits) refuse("weights of shape ", weights->sizes(), " do not broadcast to ", rows);
        w = weights->sizes() == rows ? *weights : weights->expand(rows);
    }
    require_hip(device);
    const at::NoGradGuard off;
    c.logits = written_out(logits);
    if (rows.size() == 2) {
        if (c.logits.stride(2) != 1 && classes > 1) c.logits = c.logits.contiguous();
        c.config.unroll = rows[0];
        c.config.batch = rows[1];
        c.config.logits_strides[0] = c.logits.stride(0);
        c.config.logits_strides[1] = c.logits.stride(1);
    } else {
        c.logits = c.logits.contiguous();
        c.config.unroll = 1;
        c.config.batch = c10::multiply_integers(rows);
        c.config.logits_strides[1] = classes;
    }
    if (game) {
        c.game = written_out(*game).contiguous();
        c.position = written_out(*position).contiguous();
    } else {
        c.config.target_positions = c.config.unroll;
        c.config.target_games = c.config.batch;
    }
    if (w.defined()) c.weights = rows_of(written_out(w), c.config.weight_strides);
    c.targets = written_out(targets).contiguous();
    return c;
}

std::pair<Tensor, Tensor> loss_run(LossCall& c, bool with_loss, bool with_grad, const Tensor& dloss) {
    Tensor loss, grad, up;
    if (with_loss) loss = at::empty(c.logits.sizes().slice(0, c.logits.dim() - 1), c.logits.options().dtype(at::kFloat));
    if (with_grad) grad = at::empty(c.logits.sizes(), c.logits.options().memory_format(at::MemoryFormat::Contiguous));
    if (dloss.defined()) up = rows_of(written_out(dloss), c.config.dloss_strides);
    const On on(c.logits.device());
    done(mz_categorical_loss(on.stream, &c.config, data(c.logits), static_cast<const float*>(data(c.targets)), data(c.game), data(c.position),
                             static_cast<const float*>(data(c.weights)), static_cast<const float*>(data(up)),
                             static_cast<float*>(data(loss)), data(grad)));
    return {loss, grad};
}

struct CategoricalLoss : torch::autograd::Function<CategoricalLoss> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, LossCall* call) {
        const Tensor loss = loss_run(*call, true, false, Tensor()).first;
        ctx->save_for_backward({call->logits, call->targets, call->game, call->position, call->weights});
        ctx->saved_data["config"] = std::string(reinterpret_cast<const char*>(&call->config), sizeof(call->config));
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list dloss) {
        const variable_list saved = ctx->get_saved_variables();
        LossCall c;
        memcpy(&c.config, ctx->saved_data["config"].toStringRef().data(), sizeof(c.config));
        c.logits = saved[0];
        c.targets = saved[1];
        c.game = saved[2];
        c.position = saved[3];
        c.weights = saved[4];
        require_readable("the gradient", dloss[0]);
        const Tensor grad = loss_run(c, false, true, dloss[0]).second;
        return once({grad, Tensor()}, {c.logits, dloss[0]});
    }
};

Tensor categorical_loss(const Tensor& logits, const Tensor& targets, const OptTensor& game, const OptTensor& position, const OptTensor& weights) {
    LossCall c = describe(logits, targets, game, position, weights);
    if (!at::GradMode::is_enabled() || !logits.requires_grad()) return loss_run(c, true, false, Tensor()).first;
    refuse_nodes_outside_capture(logits.device(), {&logits});
    return CategoricalLoss::apply(logits, &c);
}

std::pair<Tensor, Tensor> categorical_loss_and_grad(const Tensor& logits, const Tensor& targets, const OptTensor& game, const OptTensor& position,
                                                    const OptTensor& weights) {
    LossCall c = describe(logits, targets, game, position, weights);
    return loss_run(c, true, true, Tensor());
}

// ---- global norm and clipping -----------------------------------------------------------------------------------------

// every element of t's memory span once: contiguous in some order of its dimensions
bool dense(const Tensor& t) {
    if (t.is_contiguous()) return true;
    std::vector<std::pair<int64_t, int64_t>> dims;
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) != 1) dims.emplace_back(t.stride(i), t.size(i));
    std::sort(dims.begin(), dims.end());
    int64_t span = 1;
    for (const auto& [stride, size] : dims) {
        if (stride != span) return false;
        span *= size;
    }
    return true;
}

// one element's place in both is the same
bool alike(const Tensor& t, const Tensor& u) {
    return t.sizes() == u.sizes() && ((t.is_contiguous() && u.is_contiguous()) || t.strides() == u.strides());
}

struct TensorList {
    std::vector<Tensor> tensors, out;
    std::vector<mz_tensor_t> described;
    std::vector<void*> outputs;
    c10::Device device = at::kCPU;

    TensorList(std::vector<Tensor> t, std::optional<std::vector<Tensor>> o) : tensors(std::move(t)) {
        refuse_while_recording();
        const size_t n = tensors.size();
        if (n < 1 || n > MZ_GLOBAL_NORM_MAX_TENSORS) refuse("1 to ", MZ_GLOBAL_NORM_MAX_TENSORS, " tensors, got ", n);
        device = tensors[0].device();
        described.reserve(n);
        for (size_t i = 0; i < n; ++i) {
            const Tensor& t = tensors[i];
            if (const char* why = unreadable(t)) refuse("tensor ", i, " ", why);
            if (dtype_of(t) < 0) refuse("tensor ", i, ": expected float32, float16 or bfloat16, got ", t.scalar_type());
            if (t.is_neg() || t._is_zerotensor()) refuse("tensor ", i, " is the lazy negative of its memory, or zeros without any");
            if (t.device() != device) refuse("tensor ", i, " is on ", t.device(), ", expected ", device);
            if (!dense(t)) refuse("tensor ", i, " is not dense: shape ", t.sizes(), ", strides ", t.strides());
            described.push_back({t.data_ptr(), t.numel(), dtype_of(t), 0});
        }
        if (o) {
            out = std::move(*o);
            if (out.size() != n) refuse(n, " tensors, ", out.size(), " outputs");
            for (size_t i = 0; i < n; ++i) {
                const Tensor &t = tensors[i], &u = out[i];
                if (const char* why = unreadable(u)) refuse("output ", i, " ", why);
                if (u.is_neg() || u._is_zerotensor()) refuse("output ", i, " is the lazy negative of its memory, or zeros without any");
                if (u.scalar_type() != t.scalar_type() || u.device() != device || !alike(u, t))
                    refuse("output ", i, " must be like its tensor: ", t.scalar_type(), " ", t.sizes(), ", strides ", t.strides(), ", on ", device);
                outputs.push_back(u.data_ptr());
            }
        }
        require_hip(device);
    }
    // every tensor is where it was, of the size and type it had, and dense
    void check_unchanged() const {
        const auto same = [&](const Tensor& t, const mz_tensor_t& was, void* data) {
            return t.data_ptr() == data && t.numel() == was.elements && dtype_of(t) == was.dtype && dense(t);
        };
        for (size_t i = 0; i < tensors.size(); ++i) {
            if (!same(tensors[i], described[i], described[i].data) || (!outputs.empty() && !same(out[i], described[i], outputs[i])))
                refuse("tensor ", i, " or its output has other memory, or another shape or type, than when the set was made");
            if (!outputs.empty() && !alike(out[i], tensors[i])) refuse("tensor ", i, " and its output are laid out unlike each other");
        }
    }
    const std::vector<Tensor>& written() const { return outputs.empty() ? tensors : out; }
    void* const* output_table() const { return outputs.empty() ? nullptr : outputs.data(); }
    void check_clip(double max_norm) const {
        if (!(max_norm >= 0)) refuse("max_norm must be >= 0, got ", max_norm);
        for (const Tensor& t : written())
            if (t.requires_grad()) refuse("a tensor that requires grad cannot be written by clipping");
    }
    void changed() const {
        for (const Tensor& t : written())
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
    // call(stream, workspace, its size, norm) -> status
    template <typename F>
    Tensor run(F call) const {
        refuse_while_recording();
        const auto options = at::TensorOptions().device(device);
        const Tensor ws = at::empty({MZ_GLOBAL_NORM_WORKSPACE}, options.dtype(at::kByte)), norm = at::empty({}, options.dtype(at::kFloat));
        const On on(device);
        done(call(on.stream, ws.data_ptr(), MZ_GLOBAL_NORM_WORKSPACE, norm.data_ptr<float>()));
        return norm;
    }
};

Tensor global_norm(std::vector<Tensor> tensors) {
    const TensorList l(std::move(tensors), std::nullopt);
    return l.run([&](void* stream, void* ws, int64_t bytes, float* norm) {
        return mz_global_norm(stream, (int32_t)l.described.size(), l.described.data(), ws, bytes, norm);
    });
}

Tensor clip_by_global_norm(std::vector<Tensor> tensors, double max_norm, std::optional<std::vector<Tensor>> out) {
    const TensorList l(std::move(tensors), std::move(out));
    l.check_clip(max_norm);
    const Tensor norm = l.run([&](void* stream, void* ws, int64_t bytes, float* norm) {
        return mz_clip_by_global_norm(stream, (int32_t)l.described.size(), l.described.data(), l.output_table(), max_norm, ws, bytes, norm);
    });
    l.changed();
    return norm;
}

class GradientSet {
    TensorList list_;
    mz_tensor_table_t table_;
    Tensor memory_;                              // the table on the device
    c10::Stream made_on_;
    std::string overlap_;

    c10::Stream current() const { return c10::impl::VirtualGuardImpl(list_.device.type()).getStream(list_.device); }
    void* table() const {
        const c10::Stream stream = current();
        if (stream != made_on_ && !done(mz_stream_is_capturing(On(list_.device).stream))) memory_.record_stream(stream);
        return memory_.data_ptr();
    }

  public:
    GradientSet(std::vector<Tensor> tensors, std::optional<std::vector<Tensor>> out)
        : list_(std::move(tensors), std::move(out)), made_on_(current()) {
        if (done(mz_stream_is_capturing(On(list_.device).stream))) refuse("a GradientSet uploads its table: make it before the capture");
        const int32_t n = (int32_t)list_.described.size();
        Tensor host = at::empty({(int64_t)n * MZ_TENSOR_TABLE_ENTRY}, at::kByte);
        done(mz_tensor_table_build(n, list_.described.data(), list_.output_table(), host.data_ptr(), &table_));
        if (!table_.writable) overlap_ = mz_last_error();
        memory_ = host.to(list_.device);
    }
    Tensor global_norm() const {
        list_.check_unchanged();
        void* const table = this->table();
        return list_.run([&](void* stream, void* ws, int64_t bytes, float* norm) {
            return mz_tensor_table_global_norm(stream, &table_, table, ws, bytes, norm);
        });
    }
    Tensor clip_by_global_norm(double max_norm) const {
        list_.check_clip(max_norm);
        if (!overlap_.empty()) refuse("cannot clip: ", overlap_);
        list_.check_unchanged();
        void* const table = this->table();
        const Tensor norm = list_.run([&](void* stream, void* ws, int64_t bytes, float* norm) {
            return mz_tensor_table_clip(stream, &table_, table, max_norm, ws, bytes, norm);
        });
        list_.changed();
        return norm;
    }
};

}  // namespace

PYBIND11_MODULE(_autograd, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        const char* module = "muzero_amd.exceptions";
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Refused& e) {
            py::object type = py::module_::import(module).attr("MuZeroError");
            PyErr_SetObject(type.ptr(), type(std::string(e.what())).ptr());
        } catch (const Failed& e) {
            py::object type = py::module_::import(module).attr("MuZeroHipError");
            PyErr_SetObject(type.ptr(), type(e.status, std::string(e.what())).ptr());
        }
    });
    m.def("group_norm", &group_norm, py::call_guard<py::gil_scoped_release>());
    m.def("categorical_loss", &categorical_loss, py::call_guard<py::gil_scoped_release>());
    m.def("categorical_loss_and_grad", &categorical_loss_and_grad, py::call_guard<py::gil_scoped_release>());
    m.def("global_norm", &global_norm, py::call_guard<py::gil_scoped_release>());
    m.def("clip_by_global_norm", &clip_by_global_norm, py::call_guard<py::gil_scoped_release>());
    py::class_<GradientSet>(m, "GradientSet")
        .def(py::init<std::vector<Tensor>, std::optional<std::vector<Tensor>>>(), py::call_guard<py::gil_scoped_release>())
        .def("global_norm", &GradientSet::global_norm, py::call_guard<py::gil_scoped_release>())
        .def("clip_by_global_norm", &GradientSet::clip_by_global_norm, py::call_guard<py::gil_scoped_release>());
}
