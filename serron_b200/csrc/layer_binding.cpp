// The layer operators as torch sees them: torch.ops.serron.*, with outputs and workspaces from torch's caching allocator,
// work on torch's current stream, and backward nodes that call the C ABI (include/serron_b200.h) without passing
// through Python.
//
// A pass of these operators over a small tensor takes a few microseconds on the GPU, and a custom function written in
// Python about forty on the host, forward and backward; from here the two passes cost a few each.  Arguments are
// checked by the Python functions (serron_b200/functional.py) before they come here; what would let a kernel leave its
// tensors is checked once more, since torch.ops is open to all.
//
// They are operators of the dispatcher, and not mere functions, so that whatever stands between a call and its kernel
// in torch sees them: tracers record them, fake tensors take their shapes from the Meta kernels, function transforms
// unwrap their tensors.  `layer_norm`, `dropout` and `dropout_add_layer_norm` record the backward nodes; the ones that
// begin with an underscore are what those and the nodes call below autograd.
#include "serron_b200.h"

#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/library.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <array>
#include <numeric>
#include <optional>
#include <stdexcept>
#include <tuple>
#include <utility>
#include <vector>

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

void raise_for(int rc) {
    if (rc != SERRON_OK) throw std::runtime_error(serron_last_error());
}

int32_t dtype_code(at::ScalarType t) {
    switch (t) {
    case at::kFloat: return SERRON_F32;
    case at::kDouble: return SERRON_F64;
    case at::kHalf: return SERRON_F16;
    case at::kBFloat16: return SERRON_BF16;
    default: throw std::runtime_error("serron: unsupported dtype");
    }
}

void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor given(const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); }
Tensor plain(const MaybeTensor& t) { return t.has_value() && t->defined() ? t->contiguous() : Tensor(); }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
int32_t ordinal_of(const Tensor& t) { return t.device().index(); }

// How the memory of a dense tensor holds the rows along `dim`.
struct Layout {
    int64_t outer = 1, len = 1, inner = 1;
};
using Order = c10::SmallVector<int64_t, 8>;

// The dimensions of x from the outermost in memory inwards; x becomes a contiguous copy where they do not lie densely in
// some order.
Order order_of(Tensor& x) {
    const int64_t n = x.dim();
    Order order(n);
    std::iota(order.begin(), order.end(), 0);
    if (x.is_contiguous()) return order;
    std::stable_sort(order.begin(), order.end(), [&](int64_t a, int64_t b) { return x.stride(a) > x.stride(b); });
    int64_t expected = 1;
    bool dense = true;
    for (int64_t k = n - 1; k >= 0; --k) {
        if (x.size(order[k]) == 1) continue;
        dense = dense && x.stride(order[k]) == expected;
        expected *= x.size(order[k]);
    }
    if (!dense) {
        x = x.contiguous();
        std::iota(order.begin(), order.end(), 0);
    }
    return order;
}

Layout layout_of(Tensor& x, int64_t dim) {
    Layout l;
    const Order order = order_of(x);
    l.len = x.size(dim);
    bool behind = false;
    for (const int64_t d : order) {
        if (d == dim)
            behind = true;
        else
            (behind ? l.inner : l.outer) *= x.size(d);
    }
    return l;
}

// t in the dense memory order of x
Tensor like(const Tensor& t, const Tensor& x) {
    return t.strides() == x.strides() ? t : at::empty_like(x).copy_(t);
}

// ------------------------------------------------------------------------------------------------
// what the kernels rely on
// ------------------------------------------------------------------------------------------------
void check_beside(const char* name, const Tensor& t, const Tensor& x) {
    TORCH_CHECK(t.device() == x.device(), "serron::", name, ": all tensors must be on one device");
    TORCH_CHECK(t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type(), "serron::", name,
                ": tensors of the input's shape and dtype are needed, got ", t.sizes(), " of ", t.scalar_type(),
                " beside ", x.sizes(), " of ", x.scalar_type());
}

int64_t check_dim(const char* name, const Tensor& x, int64_t dim) {
    TORCH_CHECK(x.dim() > 0 && dim >= -x.dim() && dim < x.dim(), "serron::", name, ": dim ", dim,
                " is out of range for a ", x.dim(), "-D input");
    return dim < 0 ? dim + x.dim() : dim;
}

void check_params(const char* name, const Tensor& x, int64_t dim, const Tensor& weight, const Tensor& bias) {
    for (const Tensor* t : {&weight, &bias}) {
        if (!t->defined()) continue;
        TORCH_CHECK(t->device() == x.device(), "serron::", name, ": all tensors must be on one device");
        TORCH_CHECK(t->dim() == 1 && t->size(0) == x.size(dim), "serron::", name, ": weight and bias must have the shape (",
                    x.size(dim), ",) of the normalised dimension, got ", t->sizes());
    }
    TORCH_CHECK(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(), "serron::", name,
                ": weight and bias must share a dtype");
}

void check_param_type(const char* name, const Tensor& weight, at::ScalarType params) {
    TORCH_CHECK(!weight.defined() || weight.scalar_type() == params, "serron::", name, ": a weight of ", params,
                " is needed, got ", weight.scalar_type());
}

void check_seed(const char* name, const Tensor& x, const Tensor& seed) {
    if (!seed.defined()) return;
    TORCH_CHECK(seed.device() == x.device(), "serron::", name, ": all tensors must be on one device");
    TORCH_CHECK(seed.scalar_type() == at::kLong && seed.numel() == 1, "serron::", name,
                ": a seed in a tensor is one int64, got ", seed.numel(), " of ", seed.scalar_type());
}

at::ScalarType stats_type(const Tensor& x) { return x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat; }

// mean in the first row, 1 / sqrt(var + eps) in the second
Tensor empty_stats(const Tensor& x, const Layout& l) {
    return at::empty({2, l.outer * l.inner}, x.options().dtype(stats_type(x)));
}
void* second(const Tensor& stats) {
    return stats.defined() ? static_cast<char*>(stats.data_ptr()) + stats.size(1) * stats.element_size() : nullptr;
}
Tensor checked_stats(const char* name, const Tensor& stats, const Tensor& x, const Layout& l) {
    TORCH_CHECK(stats.device() == x.device(), "serron::", name, ": all tensors must be on one device");
    TORCH_CHECK(stats.dim() == 2 && stats.size(0) == 2 && stats.size(1) == l.outer * l.inner &&
                    stats.scalar_type() == stats_type(x),
                "serron::", name, ": statistics of another input");
    return stats.contiguous();
}

struct Workspace {
    Tensor buffer;
    int64_t bytes;
    Workspace(const Tensor& x, const Layout& l, bool backward)
        : bytes(serron_layer_norm_workspace_bytes(l.outer, l.len, l.inner, dtype_code(x.scalar_type()), backward)) {
        if (bytes < 0) raise_for(SERRON_ERR_INVALID);
        if (bytes > 0) buffer = at::empty({bytes}, x.options().dtype(at::kByte));
    }
};

at::ScalarType param_type(const Tensor& x, const Tensor& weight, const Tensor& bias) {
    return weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : x.scalar_type();
}

// ------------------------------------------------------------------------------------------------
// CUDA and Meta kernels: a tensor that is not on a GPU has shapes and strides alone, and nothing is launched for it
// ------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> norm_kernel(const Tensor& input, const MaybeTensor& weight, const MaybeTensor& bias,
                                       int64_t dim, double eps, bool stats) {
    const char* name = "layer_norm";
    Tensor x = input, s;
    dim = check_dim(name, x, dim);
    const Layout l = layout_of(x, dim);
    const Tensor w = plain(weight), b = plain(bias);
    check_params(name, x, dim, w, b);
    const Tensor y = at::empty_like(x);
    if (stats) s = empty_stats(x, l);
    if (x.is_cuda()) {
        const Workspace ws(x, l, false);
        raise_for(serron_layer_norm(address(x), l.outer, l.len, l.inner, dtype_code(x.scalar_type()), address(w),
                                    address(b), dtype_code(param_type(x, w, b)), eps, address(y), address(s), second(s),
                                    address(ws.buffer), ws.bytes, ordinal_of(x), stream_of(x)));
    }
    return {y, s};
}

std::tuple<Tensor, Tensor, Tensor> norm_backward_kernel(const Tensor& grad_output, const Tensor& input,
                                                        const Tensor& stats, const MaybeTensor& weight, int64_t dim,
                                                        at::ScalarType params, std::array<bool, 3> wanted) {
    const char* name = "layer_norm_backward";
    Tensor x = input;
    dim = check_dim(name, x, dim);
    check_beside(name, grad_output, x);
    const Layout l = layout_of(x, dim);
    const Tensor gy = like(grad_output, x), w = plain(weight), s = checked_stats(name, stats, x, l);
    check_params(name, x, dim, w, Tensor());
    check_param_type(name, w, params);
    std::array<Tensor, 3> out;
    if (wanted[0]) out[0] = at::empty_like(x);
    for (const int i : {1, 2})
        if (wanted[i]) out[i] = at::empty({l.len}, x.options().dtype(params));
    if (x.is_cuda()) {
        const Workspace ws(x, l, true);
        raise_for(serron_layer_norm_backward(address(gy), address(x), address(s), second(s), l.outer, l.len, l.inner,
                                             dtype_code(x.scalar_type()), address(w), dtype_code(params),
                                             address(out[0]), address(out[1]), address(out[2]), address(ws.buffer),
                                             ws.bytes, ordinal_of(x), stream_of(x)));
    }
    return {out[0], out[1], out[2]};
}

// Decisions are counted in the row-major order of the elements.
Tensor dropout_kernel(const Tensor& input, const MaybeTensor& residual, int64_t span, double p, int64_t seed,
                      const MaybeTensor& seed_tensor, int64_t sequence) {
    const char* name = "dropout";
    const Tensor x = input.contiguous(), r = plain(residual), key = given(seed_tensor);
    if (r.defined()) check_beside(name, r, x);
    check_seed(name, x, key);
    const Tensor y = at::empty_like(x);
    if (x.is_cuda())
        raise_for(serron_dropout(address(x), address(r), x.numel(), span, dtype_code(x.scalar_type()), p,
                                 static_cast<uint64_t>(seed), address(key), static_cast<uint64_t>(sequence), address(y),
                                 ordinal_of(x), stream_of(x)));
    return y;
}

std::tuple<Tensor, Tensor, Tensor> join_kernel(const Tensor& input, const Tensor& residual, const MaybeTensor& weight,
                                               const MaybeTensor& bias, double p, int64_t seed,
                                               const MaybeTensor& seed_tensor, int64_t sequence, int64_t dim, double eps,
                                               bool stats) {
    const char* name = "dropout_add_layer_norm";
    dim = check_dim(name, input, dim);
    Tensor x = input.contiguous(), s;
    const Tensor r = residual.contiguous(), w = plain(weight), b = plain(bias), key = given(seed_tensor);
    const Layout l = layout_of(x, dim);
    check_beside(name, r, x);
    check_params(name, x, dim, w, b);
    check_seed(name, x, key);
    const Tensor y = at::empty_like(x), h = at::empty_like(x);
    if (stats) s = empty_stats(x, l);
    if (x.is_cuda()) {
        const Workspace ws(x, l, false);
        raise_for(serron_dropout_add_layer_norm(
            address(x), address(r), l.outer, l.len, l.inner, dtype_code(x.scalar_type()), address(w), address(b),
            dtype_code(param_type(x, w, b)), p, static_cast<uint64_t>(seed), address(key),
            static_cast<uint64_t>(sequence), eps, address(h), address(y), address(s), second(s), address(ws.buffer),
            ws.bytes, ordinal_of(x), stream_of(x)));
    }
    return {y, h, s};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> join_backward_kernel(
    const Tensor& grad_output, const MaybeTensor& grad_sum, const Tensor& sum, const Tensor& stats,
    const MaybeTensor& weight, int64_t dim, at::ScalarType params, double p, int64_t seed, const MaybeTensor& seed_tensor,
    int64_t sequence, std::array<bool, 4> wanted) {
    const char* name = "dropout_add_layer_norm_backward";
    dim = check_dim(name, sum, dim);
    Tensor h = sum.contiguous();
    const Layout l = layout_of(h, dim);
    const Tensor gy = grad_output.contiguous(), gh = plain(grad_sum), w = plain(weight), key = given(seed_tensor),
                 s = checked_stats(name, stats, h, l);
    check_beside(name, gy, h);
    if (gh.defined()) check_beside(name, gh, h);
    check_params(name, h, dim, w, Tensor());
    check_param_type(name, w, params);
    check_seed(name, h, key);
    std::array<Tensor, 4> out;
    for (const int i : {0, 1})
        if (wanted[i]) out[i] = at::empty_like(h);
    for (const int i : {2, 3})
        if (wanted[i]) out[i] = at::empty({l.len}, h.options().dtype(params));
    if (h.is_cuda()) {
        const Workspace ws(h, l, true);
        raise_for(serron_dropout_add_layer_norm_backward(
            address(gy), address(gh), address(h), address(s), second(s), l.outer, l.len, l.inner,
            dtype_code(h.scalar_type()), address(w), dtype_code(params), p, static_cast<uint64_t>(seed), address(key),
            static_cast<uint64_t>(sequence), address(out[0]), address(out[1]), address(out[2]), address(out[3]),
            address(ws.buffer), ws.bytes, ordinal_of(h), stream_of(h)));
    }
    return {out[0], out[1], out[2], out[3]};
}

// ------------------------------------------------------------------------------------------------
// calls through the dispatcher
// ------------------------------------------------------------------------------------------------
template <typename F>
c10::TypedOperatorHandle<F> operator_of(const char* name, F*) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
#define SERRON_OPERATOR(name, kernel)                                                 \
    const auto& name() {                                                              \
        static const auto op = operator_of("serron::" #name, static_cast<decltype(&kernel)>(nullptr)); \
        return op;                                                                    \
    }
SERRON_OPERATOR(_layer_norm, norm_kernel)
SERRON_OPERATOR(_layer_norm_backward, norm_backward_kernel)
SERRON_OPERATOR(dropout, dropout_kernel)
SERRON_OPERATOR(_dropout_add_layer_norm, join_kernel)
SERRON_OPERATOR(_dropout_add_layer_norm_backward, join_backward_kernel)

// There are no forward-mode derivatives; an output without a tangent would stand for one of zero.
template <typename... T>
void refuse_tangents(const char* name, const T&... inputs) {
    const auto has = [](const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); };
    TORCH_CHECK_NOT_IMPLEMENTED(!(has(inputs) || ...), "serron::", name,
                                ": an input carries a tangent, and there is no forward-mode derivative");
}

// Gradients of a backward pass cannot be differentiated again: what asks for it, along whichever of `edges`, is an error.
template <typename Tensors>
void once(Tensors& grads, torch::autograd::edge_list&& edges) {
    const auto error = std::make_shared<torch::autograd::Error>(
        "serron: a gradient of layer_norm or dropout_add_layer_norm is once_differentiable", std::move(edges));
    for (const Tensor& g : grads)
        if (g.defined()) torch::autograd::set_history(g, error);
}

// The same for what a node computed while a graph of its gradients is recorded: they depend on its own inputs and on those
// that came to it.
void once_from(const Node& node, const variable_list& came, variable_list& grads) {
    if (!at::GradMode::is_enabled()) return;
    torch::autograd::edge_list edges = node.next_edges();
    for (const Tensor& g : came)
        if (g.defined()) edges.push_back(torch::autograd::impl::gradient_edge(g));
    once(grads, std::move(edges));
}

// ------------------------------------------------------------------------------------------------
// layer norm
// ------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor, Tensor> norm_backward_autograd(const Tensor& grad_output, const Tensor& input,
                                                          const Tensor& stats, const MaybeTensor& weight, int64_t dim,
                                                          at::ScalarType params, std::array<bool, 3> wanted) {
    refuse_tangents("layer_norm_backward", grad_output, input, given(weight));
    std::array<Tensor, 3> out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        std::tie(out[0], out[1], out[2]) =
            _layer_norm_backward().call(grad_output, input, stats, weight, dim, params, wanted);
    }
    const Tensor w = given(weight);
    if (torch::autograd::compute_requires_grad(grad_output, input, w))
        once(out, torch::autograd::collect_next_edges(grad_output, input, w));
    return {out[0], out[1], out[2]};
}

struct LayerNormBackward : public Node {
    SavedVariable x, weight, stats;
    c10::SmallVector<int64_t, 8> strides;  // of x: the statistics lie in the order of its memory
    int64_t dim = 0;
    at::ScalarType params = at::kFloat;

    std::string name() const override { return "SerronLayerNormBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        x.reset_data();
        weight.reset_data();
        stats.reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(3);
        if (!grads[0].defined()) return out;
        Tensor input = x.unpack();
        const Tensor w = weight.unpack();
        // hooks on saved tensors (as to keep them on the host) may bring x back in another order
        if (input.strides() != at::IntArrayRef(strides))
            input = at::empty_strided(input.sizes(), strides, input.options()).copy_(input);
        std::tie(out[0], out[1], out[2]) = _layer_norm_backward().call(
            grads[0], input, stats.unpack(), w.defined() ? MaybeTensor(w) : MaybeTensor(), dim, params,
            {task_should_compute_output(0), task_should_compute_output(1), task_should_compute_output(2)});
        once_from(*this, grads, out);
        return out;
    }
};

Tensor norm_autograd(const Tensor& input, const MaybeTensor& weight, const MaybeTensor& bias, int64_t dim, double eps) {
    const Tensor given_w = given(weight), given_b = given(bias);
    refuse_tangents("layer_norm", input, given_w, given_b);
    const bool records = torch::autograd::compute_requires_grad(input, given_w, given_b);
    Tensor x = input, y, stats;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        if (records) order_of(x);  // the copy of an input that does not lie densely is kept for the backward pass
        std::tie(y, stats) = _layer_norm().call(x, weight, bias, dim, eps, records);
    }
    if (records) {
        auto node = std::make_shared<LayerNormBackward>();
        node->set_next_edges(torch::autograd::collect_next_edges(input, given_w, given_b));
        node->x = SavedVariable(x, false);
        node->weight = SavedVariable(given_w, false);
        node->stats = SavedVariable(stats, false);
        node->strides = c10::SmallVector<int64_t, 8>(x.strides().begin(), x.strides().end());
        node->dim = dim;
        node->params = param_type(x, given_w, given_b);
        torch::autograd::set_history(y, node);
    }
    return y;
}

// below autograd
Tensor norm_alone(const Tensor& input, const MaybeTensor& weight, const MaybeTensor& bias, int64_t dim, double eps) {
    return std::get<0>(_layer_norm().call(input, weight, bias, dim, eps, false));
}

// ------------------------------------------------------------------------------------------------
// dropout
// ------------------------------------------------------------------------------------------------
struct Rule {
    double p = 0.0;
    int64_t seed = 0, sequence = 0;
};

struct DropoutBackward : public Node {
    SavedVariable seed;
    Rule rule;
    int64_t span = 1;

    std::string name() const override { return "SerronDropoutBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        seed.reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(2);
        if (!grads[0].defined()) return out;
        if (task_should_compute_output(0)) {
            const Tensor key = seed.unpack();
            out[0] = dropout().call(grads[0], std::nullopt, span, rule.p, rule.seed,
                                    key.defined() ? MaybeTensor(key) : MaybeTensor(), rule.sequence);
        }
        if (task_should_compute_output(1)) out[1] = grads[0];
        return out;
    }
};

Tensor dropout_autograd(const Tensor& input, const MaybeTensor& residual, int64_t span, double p, int64_t seed,
                        const MaybeTensor& seed_tensor, int64_t sequence) {
    const Tensor given_r = given(residual);
    refuse_tangents("dropout", input, given_r);
    const bool records = torch::autograd::compute_requires_grad(input, given_r);
    Tensor y;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        y = dropout().call(input, residual, span, p, seed, seed_tensor, sequence);
    }
    if (records) {
        auto node = std::make_shared<DropoutBackward>();
        node->set_next_edges(torch::autograd::collect_next_edges(input, given_r));
        node->seed = SavedVariable(given(seed_tensor), false);
        node->rule = {p, seed, sequence};
        node->span = span;
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ------------------------------------------------------------------------------------------------
// the join
// ------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor, Tensor, Tensor> join_backward_autograd(
    const Tensor& grad_output, const MaybeTensor& grad_sum, const Tensor& sum, const Tensor& stats,
    const MaybeTensor& weight, int64_t dim, at::ScalarType params, double p, int64_t seed, const MaybeTensor& seed_tensor,
    int64_t sequence, std::array<bool, 4> wanted) {
    refuse_tangents("dropout_add_layer_norm_backward", grad_output, given(grad_sum), sum, given(weight));
    std::array<Tensor, 4> out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        std::tie(out[0], out[1], out[2], out[3]) = _dropout_add_layer_norm_backward().call(
            grad_output, grad_sum, sum, stats, weight, dim, params, p, seed, seed_tensor, sequence, wanted);
    }
    const Tensor gh = given(grad_sum), w = given(weight);
    if (torch::autograd::compute_requires_grad(grad_output, gh, sum, w))
        once(out, torch::autograd::collect_next_edges(grad_output, gh, sum, w));
    return {out[0], out[1], out[2], out[3]};
}

struct DropoutAddLayerNormBackward : public Node {
    SavedVariable sum, weight, stats, seed;
    int64_t dim = 0;
    Rule rule;
    at::ScalarType params = at::kFloat;

    std::string name() const override { return "SerronDropoutAddLayerNormBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        sum.reset_data();
        weight.reset_data();
        stats.reset_data();
        seed.reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(4);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        const Tensor key = seed.unpack();
        const MaybeTensor seed_tensor = key.defined() ? MaybeTensor(key) : MaybeTensor();
        if (!grads[0].defined()) {
            // the norm's output was not used: what it would be at this input, finite or not, is in no gradient
            if (task_should_compute_output(0))
                out[0] = dropout().call(grads[1], std::nullopt, 1, rule.p, rule.seed, seed_tensor, rule.sequence);
            if (task_should_compute_output(1)) out[1] = grads[1];
            for (const int i : {2, 3})
                if (task_should_compute_output(i))
                    out[i] = at::zeros({grads[1].size(dim)}, grads[1].options().dtype(params));
            return out;
        }
        const Tensor h = sum.unpack(shared_from_this()), w = weight.unpack();
        std::tie(out[0], out[1], out[2], out[3]) = _dropout_add_layer_norm_backward().call(
            grads[0], grads[1].defined() ? MaybeTensor(grads[1]) : MaybeTensor(), h, stats.unpack(),
            w.defined() ? MaybeTensor(w) : MaybeTensor(), dim, params, rule.p, rule.seed, seed_tensor, rule.sequence,
            {task_should_compute_output(0), task_should_compute_output(1), task_should_compute_output(2),
             task_should_compute_output(3)});
        once_from(*this, grads, out);
        return out;
    }
};

std::tuple<Tensor, Tensor> join_autograd(const Tensor& input, const Tensor& residual, const MaybeTensor& weight,
                                         const MaybeTensor& bias, double p, int64_t seed, const MaybeTensor& seed_tensor,
                                         int64_t sequence, int64_t dim, double eps) {
    const Tensor given_w = given(weight), given_b = given(bias);
    refuse_tangents("dropout_add_layer_norm", input, residual, given_w, given_b);
    const bool records = torch::autograd::compute_requires_grad(input, residual, given_w, given_b);
    Tensor y, h, stats;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        std::tie(y, h, stats) = _dropout_add_layer_norm().call(input, residual, weight, bias, p, seed, seed_tensor,
                                                               sequence, dim, eps, records);
    }
    if (records) {
        auto node = std::make_shared<DropoutAddLayerNormBackward>();
        node->set_next_edges(torch::autograd::collect_next_edges(input, residual, given_w, given_b));
        torch::autograd::set_history(y, node);
        torch::autograd::set_history(h, node);
        node->sum = SavedVariable(h, true);
        node->weight = SavedVariable(given_w, false);
        node->stats = SavedVariable(stats, false);
        node->seed = SavedVariable(given(seed_tensor), false);
        node->dim = dim;
        node->rule = {p, seed, sequence};
        node->params = param_type(input, given_w, given_b);
    }
    return {y, h};
}

// below autograd
std::tuple<Tensor, Tensor> join_alone(const Tensor& input, const Tensor& residual, const MaybeTensor& weight,
                                      const MaybeTensor& bias, double p, int64_t seed, const MaybeTensor& seed_tensor,
                                      int64_t sequence, int64_t dim, double eps) {
    const auto out = _dropout_add_layer_norm().call(input, residual, weight, bias, p, seed, seed_tensor, sequence, dim,
                                                    eps, false);
    return {std::get<0>(out), std::get<1>(out)};
}

SERRON_OPERATOR(layer_norm, norm_alone)
SERRON_OPERATOR(dropout_add_layer_norm, join_alone)

}  // namespace

// Seeds and sequence numbers are 64 bits without a sign; an operator's integer holds the same bits with one.
TORCH_LIBRARY_FRAGMENT(serron, m) {
    m.def("layer_norm(Tensor input, Tensor? weight, Tensor? bias, int dim, float eps) -> Tensor");
    m.def("_layer_norm(Tensor input, Tensor? weight, Tensor? bias, int dim, float eps, bool stats) -> (Tensor, Tensor)");
    m.def("_layer_norm_backward(Tensor grad_output, Tensor input, Tensor stats, Tensor? weight, int dim, "
          "ScalarType params, bool[3] wanted) -> (Tensor, Tensor, Tensor)");
    m.def("dropout(Tensor input, Tensor? residual, int span, float p, int seed, Tensor? seed_tensor, int sequence) "
          "-> Tensor");
    m.def("dropout_add_layer_norm(Tensor input, Tensor residual, Tensor? weight, Tensor? bias, float p, int seed, "
          "Tensor? seed_tensor, int sequence, int dim, float eps) -> (Tensor, Tensor)");
    m.def("_dropout_add_layer_norm(Tensor input, Tensor residual, Tensor? weight, Tensor? bias, float p, int seed, "
          "Tensor? seed_tensor, int sequence, int dim, float eps, bool stats) -> (Tensor, Tensor, Tensor)");
    m.def("_dropout_add_layer_norm_backward(Tensor grad_output, Tensor? grad_sum, Tensor sum, Tensor stats, "
          "Tensor? weight, int dim, ScalarType params, float p, int seed, Tensor? seed_tensor, int sequence, "
          "bool[4] wanted) -> (Tensor, Tensor, Tensor, Tensor)");
}

#define SERRON_KERNELS(m)                                              \
    m.impl("_layer_norm", &norm_kernel);                               \
    m.impl("_layer_norm_backward", &norm_backward_kernel);             \
    m.impl("dropout", &dropout_kernel);                                \
    m.impl("_dropout_add_layer_norm", &join_kernel);                   \
    m.impl("_dropout_add_layer_norm_backward", &join_backward_kernel);
TORCH_LIBRARY_IMPL(serron, CUDA, m) { SERRON_KERNELS(m) }
TORCH_LIBRARY_IMPL(serron, Meta, m) { SERRON_KERNELS(m) }

TORCH_LIBRARY_IMPL(serron, CompositeExplicitAutograd, m) {
    m.impl("layer_norm", &norm_alone);
    m.impl("dropout_add_layer_norm", &join_alone);
}

TORCH_LIBRARY_IMPL(serron, Autograd, m) {
    m.impl("layer_norm", &norm_autograd);
    m.impl("dropout", &dropout_autograd);
    m.impl("dropout_add_layer_norm", &join_autograd);
    m.impl("_layer_norm_backward", &norm_backward_autograd);
    m.impl("_dropout_add_layer_norm_backward", &join_backward_autograd);
    m.impl("_layer_norm", torch::autograd::autogradNotImplementedFallback());
    m.impl("_dropout_add_layer_norm", torch::autograd::autogradNotImplementedFallback());
}

PYBIND11_MODULE(_layers, m) {
    m.doc() = "Layer norm, dropout and their join: the operators torch.ops.serron.*, called without their Python layer.";
    m.def("layer_norm", [](const Tensor& input, const MaybeTensor& weight, const MaybeTensor& bias, int64_t dim,
                           double eps) { return layer_norm().call(input, weight, bias, dim, eps); });
    m.def("dropout", [](const Tensor& input, const MaybeTensor& residual, int64_t span, double p, uint64_t seed,
                        const MaybeTensor& seed_tensor, uint64_t sequence) {
        return dropout().call(input, residual, span, p, static_cast<int64_t>(seed), seed_tensor,
                              static_cast<int64_t>(sequence));
    });
    m.def("dropout_add_layer_norm",
          [](const Tensor& input, const Tensor& residual, const MaybeTensor& weight, const MaybeTensor& bias, double p,
             uint64_t seed, const MaybeTensor& seed_tensor, uint64_t sequence, int64_t dim, double eps) {
              return dropout_add_layer_norm().call(input, residual, weight, bias, p, static_cast<int64_t>(seed),
                                                   seed_tensor, static_cast<int64_t>(sequence), dim, eps);
          });
}
